"""Packed batches and single tokens of the Mamba mixer: conv1d + SiLU and selective scan over sequences that lie back to
back, their caches and gradients, against a sequence-by-sequence, step-by-step evaluation in float64.

Tolerances.  Inputs are the same numbers on both sides and the kernels work in float32, so a result differs by float32
rounding and, in bfloat16, by one rounding at the end: at most half a step, 2^-8 of the value.  Float32: a state is a sum
of terms that each step scales by its decay; the decay's argument, its exponential and the update round by about 6 half
steps (2^-24) of the state, and a decay of at most exp(-dt) with dt around 0.05 remembers some 20 to 50 steps, so that
300 * 2^-24 = 1.8e-5 of the largest value bounds a result.  Sums over rows (parameters' gradients) add a random walk of
less than that.
"""
import pytest
import torch
import torch.nn.functional as F

from _parity_report import record

pytestmark = pytest.mark.gpu
EPS32 = 300 * 2.0 ** -24
BF16 = torch.bfloat16
F32 = torch.float32


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    from ossm_b200 import _lib

    torch.cuda.synchronize()
    assert _lib.device_status() == 0


def close(got, want, what="", steps=1.0):
    """Within float32 rounding of the whole and ``steps`` final roundings of the element."""
    want = want.double().cpu()
    g = got.detach().double().cpu()
    assert g.shape == want.shape, (what, g.shape, want.shape)
    if not want.numel():
        return
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != F32 else 0.0
    limit = steps * half * want.abs() + EPS32 * want.abs().max().clamp_min(1e-30)
    worst = float(((g - want).abs() / limit).max())
    assert worst <= 1.0, f"{what}: {worst:.3g} times the limit"


def offsets_of(lengths, first=0):
    at = [first]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32)


# ---- float64 reference -------------------------------------------------------------------------------
def ref_scan(u, dt, A, B, C, z, D, bias, softplus, offsets, start, end_too=True):
    """Differentiable; returns (out, states behind the sequences)."""
    step = dt + bias if bias is not None else dt
    step = F.softplus(step) if softplus else step
    out, ends = [], []
    at = offsets.tolist()
    out.append(0 * u[:at[0]])
    for i in range(len(at) - 1):
        h = start[i]
        for t in range(at[i], at[i + 1]):
            h = torch.exp(step[t][:, None] * A) * h + (step[t] * u[t])[:, None] * B[t][None, :]
            y = h @ C[t]
            if D is not None:
                y = y + D * u[t]
            if z is not None:
                y = y * F.silu(z[t])
            out.append(y[None])
        ends.append(h)
    out.append(0 * u[at[-1]:])
    return torch.cat(out), torch.stack(ends) if ends else start


def ref_conv(x, w, bias, offsets, start):
    K = w.size(-1)
    at = offsets.tolist()
    out, ends = [0 * x[:at[0]]], []
    for i in range(len(at) - 1):
        seq = torch.cat([start[i], x[at[i]:at[i + 1]]])
        n = at[i + 1] - at[i]
        pre = sum(w[:, k] * seq[k:k + n] for k in range(K))
        out.append(F.silu(pre + bias if bias is not None else pre))
        ends.append(seq[n:])
    out.append(0 * x[at[-1]:])
    return torch.cat(out), torch.stack(ends) if ends else start


def scan_case(lengths, D, N, io=F32, dt_type=None, seed=0, first=0, pad=0, pitched=True):
    gen = torch.Generator().manual_seed(seed + 31 * D + N + len(lengths))
    off = offsets_of(lengths, first)
    T = int(off[-1]) + pad
    r = lambda *s: torch.randn(*s, generator=gen)
    proj = r(T, 3 + 2 * N).to(io)
    xz = r(T, 2 * D).to(io)
    c = {"u": xz[:, :D], "z": xz[:, D:], "B": proj[:, 3:3 + N], "C": proj[:, 3 + N:]}
    if not pitched:
        c = {k: v.contiguous() for k, v in c.items()}
    c["dt"] = (r(T, D) * 0.5).to(dt_type or io)
    c["A"] = -torch.exp(r(D, N) * 0.5) * 2
    c["bias"] = r(D) * 0.5 - 3.0
    c["D"] = r(D)
    c["start"] = r(len(lengths), D, N)
    return c, off


def spoil(c, off):
    """NaN and infinities in the rows of no sequence: they must not reach a result."""
    for name in ("u", "z", "B", "C", "dt"):
        c[name][: int(off[0])] = float("nan")
        c[name][int(off[-1]):] = float("inf")


SHAPES = [([1], 32, 16), ([5, 0, 0, 1, 37], 33, 16), ([0, 0], 8, 4), ([3, 700, 1, 0, 260], 40, 16), ([513], 128, 16),
          ([64, 128, 65], 31, 8), ([100, 30], 20, 1), ([17, 90], 64, 3), ([300, 200], 48, 17), ([150, 2, 31], 36, 32),
          ([129], 32, 48), ([200, 77], 32, 64), ([90, 60, 1], 40, 100), ([70, 140], 24, 128), ([40, 150], 128, 256),
          ([33], 5, 250), ([1] * 70, 129, 16), ([2, 0, 1] * 30, 64, 5)]


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (BF16, F32)], ids=["f32", "bf16", "bf16_dt32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{len(s[0])}x{sum(s[0])}_D{s[1]}_N{s[2]}")
def test_scan_training(shape, types):
    from ossm_b200.selective_scan import selective_scan_packed

    lengths, D, N = shape
    c, off = scan_case(lengths, D, N, *types, first=2, pad=3)
    names = ["u", "dt", "A", "B", "C", "z", "D", "bias", "start"]
    gen = torch.Generator().manual_seed(9)
    g_out, g_end = torch.randn(c["u"].shape, generator=gen).to(types[0]), torch.randn(c["start"].shape, generator=gen)
    r = {k: c[k].double().detach().requires_grad_(True) for k in names}
    want, want_end = ref_scan(r["u"], r["dt"], r["A"], r["B"], r["C"], r["z"], r["D"], r["bias"], True, off, r["start"])
    w_grads = torch.autograd.grad((want, want_end), [r[k] for k in names], (g_out.double(), g_end.double()), allow_unused=True)
    spoil(c, off)
    d = {k: c[k].cuda().detach().requires_grad_(True) for k in names}
    # column slices of wider tensors, as the projections give them
    wide = torch.cat([c["B"], c["C"], c["z"]], 1).cuda()
    d["B"], d["C"], d["z"] = (v.detach().requires_grad_(True) for v in (wide[:, :N], wide[:, N:2 * N], wide[:, 2 * N:]))
    got, got_end = selective_scan_packed(d["u"], d["dt"], d["A"], d["B"], d["C"], off.cuda(), d["z"], d["D"],
                                         delta_bias=d["bias"], delta_softplus=True, initial_state=d["start"], return_state=True)
    grads = torch.autograd.grad((got, got_end), [d[k] for k in names], (g_out.cuda(), g_end.cuda()))
    close(got, want.detach(), "out")
    close(got_end, want_end.detach(), "end")
    for k, a, b in zip(names, grads, w_grads):
        assert a.dtype == d[k].dtype
        close(a, torch.zeros_like(r[k]) if b is None else b, "grad_" + k)


@pytest.mark.parametrize("drop", ["z", "D", "bias", "softplus", "start", "end_only", "out_only"])
def test_scan_options(drop):
    from ossm_b200.selective_scan import selective_scan_packed

    lengths, D, N = [150, 0, 45], 40, 16
    c, off = scan_case(lengths, D, N, seed=4)
    if drop == "softplus":
        c["dt"] = c["dt"].abs() * 0.2
        c["bias"] = c["bias"].abs() * 0.01
    use = {k: None if k == drop else c[k] for k in ("z", "D", "bias")}
    softplus = drop not in ("softplus",)
    if drop == "bias":
        c["dt"] = c["dt"] - 3
    gen = torch.Generator().manual_seed(9)
    g_out, g_end = torch.randn(c["u"].shape, generator=gen), torch.randn(c["start"].shape, generator=gen)
    names = [k for k in ("u", "dt", "A", "B", "C", "z", "D", "bias", "start") if k != drop]
    r = {k: c[k].double().detach().requires_grad_(True) for k in names}
    d = {k: c[k].cuda().detach().requires_grad_(True) for k in names}
    zero = torch.zeros_like(c["start"])
    want = ref_scan(r["u"], r["dt"], r["A"], r["B"], r["C"], r.get("z"), r.get("D"), r.get("bias"), softplus, off,
                    r.get("start", zero.double()))
    got = selective_scan_packed(d["u"], d["dt"], d["A"], d["B"], d["C"], off.cuda(), d.get("z"), d.get("D"),
                                delta_bias=d.get("bias"), delta_softplus=softplus, initial_state=d.get("start"),
                                return_state=True)
    pick = {"end_only": [1], "out_only": [0]}.get(drop, [0, 1])
    gs = [g_out, g_end]
    w_grads = torch.autograd.grad([want[i] for i in pick], [r[k] for k in names], [gs[i].double() for i in pick], allow_unused=True)
    grads = torch.autograd.grad([got[i] for i in pick], [d[k] for k in names], [gs[i].cuda() for i in pick])
    for i in (0, 1):
        close(got[i], want[i].detach(), f"result {i}")
    for k, a, b in zip(names, grads, w_grads):
        close(a, torch.zeros_like(r[k]) if b is None else b, "grad_" + k)
    assert use is not None


def test_scan_gradient_against_differences():
    """Along a random direction of all operands: the central difference of the float64 definition."""
    from ossm_b200.selective_scan import selective_scan_packed

    c, off = scan_case([40, 25], 33, 16, seed=2)
    names = ["u", "dt", "A", "B", "C", "z", "D", "bias", "start"]
    gen = torch.Generator().manual_seed(1)
    way = {k: torch.randn(c[k].shape, generator=gen).double() for k in names}
    w = torch.randn(c["u"].shape, generator=gen).double()
    w_end = torch.randn(c["start"].shape, generator=gen).double()

    def loss(e):
        v = {k: c[k].double() + e * way[k] for k in names}
        y, end = ref_scan(v["u"], v["dt"], v["A"], v["B"], v["C"], v["z"], v["D"], v["bias"], True, off, v["start"])
        return float((y * w).sum() + (end * w_end).sum())

    e = 1e-5
    want = (loss(e) - loss(-e)) / (2 * e)
    d = {k: c[k].cuda().detach().requires_grad_(True) for k in names}
    got = selective_scan_packed(d["u"], d["dt"], d["A"], d["B"], d["C"], off.cuda(), d["z"], d["D"], delta_bias=d["bias"],
                                delta_softplus=True, initial_state=d["start"], return_state=True)
    grads = torch.autograd.grad(got, [d[k] for k in names], (w.float().cuda(), w_end.float().cuda()))
    terms = [float((g.double().cpu() * way[k]).sum()) for k, g in zip(names, grads)]
    size = sum(float((g.double().cpu() * way[k]).abs().sum()) for k, g in zip(names, grads))
    assert abs(sum(terms) - want) <= 1e-6 * size


@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [([5, 0, 0, 1, 37], 33, 16), ([3, 700, 1, 0, 260], 40, 16), ([90, 60, 1], 40, 100),
                                   ([40, 0, 150], 128, 256), ([1] * 40, 64, 3)], ids=lambda s: f"{len(s[0])}_D{s[1]}_N{s[2]}")
def test_scan_prompts_into_a_cache(shape, io):
    """Slots in any order, resumed and fresh sequences, one without a slot; other entries and rows stay as they were."""
    from ossm_b200.selective_scan import selective_scan_packed

    lengths, D, N = shape
    S = len(lengths)
    c, off = scan_case(lengths, D, N, io, seed=3, first=1, pad=5)
    gen = torch.Generator().manual_seed(5)
    slots = torch.randperm(S + 4, generator=gen)[:S].int()
    slots[min(1, S - 1)] = -1
    resume = torch.rand(S, generator=gen) < 0.5
    cache = torch.randn(S + 4, D, N, generator=gen)
    start = torch.zeros(S, D, N, dtype=torch.float64)
    for i in range(S):
        if resume[i] and slots[i] >= 0:
            start[i] = cache[slots[i]].double()
    args = [c[k].double() for k in ("u", "dt", "A", "B", "C", "z", "D", "bias")]
    want, want_end = ref_scan(*args, True, off, start)
    want_cache = cache.double().clone()
    for i in range(S):
        if slots[i] >= 0:
            want_cache[slots[i]] = want_end[i]
    spoil(c, off)
    d = {k: v.cuda() for k, v in c.items()}
    call = lambda cached, out=None: selective_scan_packed(
        d["u"], d["dt"], d["A"], d["B"], d["C"], off.cuda(), d["z"], d["D"], delta_bias=d["bias"], delta_softplus=True,
        cache=cached, slots=slots.cuda(), resume=resume.cuda(), out=out)
    cached = cache.cuda()
    got = call(cached)
    close(got, want, "out")
    close(cached, want_cache, "cache")
    touched = set(int(v) for v in slots if v >= 0)
    for e in range(S + 4):
        if e not in touched:
            assert torch.equal(cached[e].cpu(), cache[e])
    again = cache.cuda()
    wide = torch.full((got.size(0), D + 7), 3.0, dtype=io, device="cuda")
    mine = wide[:, 4:4 + D]
    assert call(again, mine).data_ptr() == mine.data_ptr()
    lo, hi = int(off[0]), int(off[-1])
    assert torch.equal(mine[lo:hi], got[lo:hi]) and torch.equal(again, cached)      # run to run the same
    assert bool((wide[:lo] == 3).all()) and bool((wide[hi:] == 3).all()) and bool((wide[:, :4] == 3).all())


def test_no_rows_at_all():
    """A batch of sequences without rows: states and windows go through unchanged, fresh ones become zeros, gradients too."""
    from ossm_b200.mixer import causal_conv1d_silu_packed
    from ossm_b200.selective_scan import selective_scan_packed

    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    resume = torch.tensor([True, False], device="cuda")
    for N in (16, 256):
        none = lambda w: torch.empty(0, w, device="cuda")
        A = -torch.rand(33, N, device="cuda")
        cache = torch.randn(2, 33, N, device="cuda")
        before = cache.clone()
        assert selective_scan_packed(none(33), none(33), A, none(N), none(N), off, cache=cache, resume=resume).shape == (0, 33)
        assert torch.equal(cache[0], before[0]) and not cache[1].any()
        start = before.clone().requires_grad_(True)
        u = none(33).requires_grad_(True)
        out, end = selective_scan_packed(u, none(33), A, none(N), none(N), off, initial_state=start, return_state=True)
        assert torch.equal(end, before)
        gu, gs = torch.autograd.grad((end * 2).sum() + out.sum(), (u, start))
        assert gu.shape == (0, 33) and bool((gs == 2).all())
    w, window = torch.randn(33, 4, device="cuda"), torch.randn(2, 3, 33, device="cuda")
    before = window.clone()
    assert causal_conv1d_silu_packed(torch.empty(0, 33, device="cuda"), w, None, off, cache=window, resume=resume).shape == (0, 33)
    assert torch.equal(window[0], before[0]) and not window[1].any()
    start, x = before.clone().requires_grad_(True), torch.empty(0, 33, device="cuda").requires_grad_(True)
    out, end = causal_conv1d_silu_packed(x, w, None, off, initial_window=start, return_window=True)
    assert torch.equal(end, before)
    gs, = torch.autograd.grad(end.sum(), start)
    assert bool((gs == 1).all())


@pytest.mark.parametrize("N", [1, 3, 4, 8, 16, 20, 64, 100, 256])
@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
def test_scan_step(N, io):
    from ossm_b200.selective_scan import selective_scan_step

    for S, D in ((1, 33), (37, 64), (300, 5)):
        c, _ = scan_case([1] * S, D, N, io, seed=6)
        gen = torch.Generator().manual_seed(5)
        cache = torch.randn(S + 3, D, N, generator=gen)
        slots = torch.randperm(S + 3, generator=gen)[:S].int()
        if S > 1:
            slots[1] = -1
        start = torch.stack([cache[s].double() if s >= 0 else torch.zeros(D, N).double() for s in slots.tolist()])
        args = [c[k].double() for k in ("u", "dt", "A", "B", "C", "z", "D", "bias")]
        want, end = ref_scan(*args, True, offsets_of([1] * S), start)
        want_cache = cache.double().clone()
        for i, s in enumerate(slots.tolist()):
            if s >= 0:
                want_cache[s] = end[i]
        d = {k: v.cuda() for k, v in c.items()}
        cached = cache.cuda()
        got = selective_scan_step(d["u"], d["dt"], d["A"], d["B"], d["C"], cached, d["z"], d["D"], delta_bias=d["bias"],
                                  delta_softplus=True, slots=slots.cuda())
        close(got, want, f"out {S} {D}")
        close(cached, want_cache, f"cache {S} {D}")


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (BF16, F32)], ids=["f32", "bf16", "bf16_w32"])
@pytest.mark.parametrize("K", [1, 2, 3, 4])
@pytest.mark.parametrize("shape", [([1], 8), ([5, 0, 0, 1, 37], 33), ([2, 1, 0, 3, 1, 700, 2], 40), ([0], 3), ([300, 259], 129),
                                   ([1] * 50, 64)], ids=lambda s: f"{len(s[0])}x{sum(s[0])}_D{s[1]}")
def test_conv_training(shape, K, types):
    from ossm_b200.mixer import causal_conv1d_silu_packed

    lengths, D = shape
    io, wt = types
    gen = torch.Generator().manual_seed(sum(lengths) + K)
    off = offsets_of(lengths, 2)
    T, S = int(off[-1]) + 3, len(lengths)
    xz = torch.randn(T, 2 * D + 1, generator=gen).to(io)
    c = {"x": xz[:, :D], "w": (torch.randn(D, K, generator=gen) * 0.5).to(wt), "b": (torch.randn(D, generator=gen) * 0.3).to(wt),
         "start": torch.randn(S, K - 1, D, generator=gen).to(io)}
    g_out, g_end = torch.randn(T, D, generator=gen).to(io), torch.randn(S, K - 1, D, generator=gen).to(io)
    r = {k: v.double().detach().requires_grad_(True) for k, v in c.items()}
    want = ref_conv(r["x"], r["w"], r["b"], off, r["start"])
    w_grads = torch.autograd.grad(want, list(r.values()), (g_out.double(), g_end.double()), allow_unused=True)
    xd = xz.cuda()
    xd[: int(off[0])] = float("nan")
    xd[int(off[-1]):] = float("inf")
    d = {k: v.cuda().detach().requires_grad_(True) for k, v in c.items()}
    d["x"] = xd[:, :D].detach().requires_grad_(True)
    got = causal_conv1d_silu_packed(d["x"], d["w"].view(D, 1, K), d["b"], off.cuda(), initial_window=d["start"], return_window=True)
    g_bad = g_out.clone()
    g_bad[int(off[-1]):] = float("nan")            # the gradient of rows of no sequence is not read either
    grads = torch.autograd.grad(got, [d["x"], d["w"], d["b"], d["start"]], (g_bad.cuda(), g_end.cuda()))
    close(got[0], want[0].detach(), "out")
    assert torch.equal(got[1].cpu().double(), want[1].detach())
    for k, a, b in zip(r, grads, w_grads):
        close(a, torch.zeros_like(r[k]) if b is None else b, "grad_" + k)


@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("D", [40, 33])
def test_conv_prompts_then_steps(D, io):
    """A prompt in two pieces and single tokens give what the whole sequence gives, bit for bit in the windows."""
    from ossm_b200.mixer import causal_conv1d_silu_packed, causal_conv1d_silu_step

    gen = torch.Generator().manual_seed(D)
    K, lengths = 4, [9, 2, 30, 1]
    w, b = (torch.randn(D, K, generator=gen) * 0.5).to(io).cuda(), torch.randn(D, generator=gen).to(io).cuda()
    x = torch.randn(sum(lengths), D, generator=gen).to(io).cuda()
    off = offsets_of(lengths)
    whole = causal_conv1d_silu_packed(x, w, b, off.cuda())
    slots = torch.tensor([3, 0, 5, 1], dtype=torch.int32).cuda()
    cache = torch.full((6, K - 1, D), 7.0, dtype=io, device="cuda")
    first = [4, 2, 17, 0]
    rows = [torch.arange(off[i], off[i] + n) for i, n in enumerate(first)]
    got = causal_conv1d_silu_packed(x[torch.cat(rows)], w, b, offsets_of(first).cuda(), cache=cache, slots=slots, resume=False)
    assert torch.equal(got, whole[torch.cat(rows)])
    second = [3, 0, 12, 0]
    rows = [torch.arange(off[i] + first[i], off[i] + first[i] + n) for i, n in enumerate(second)]
    got = causal_conv1d_silu_packed(x[torch.cat(rows)], w, b, offsets_of(second).cuda(), cache=cache, slots=slots, resume=True)
    assert torch.equal(got, whole[torch.cat(rows)])
    done = [a + b for a, b in zip(first, second)]
    while any(n < m for n, m in zip(done, lengths)):
        at = [int(off[i]) + min(done[i], lengths[i] - 1) for i in range(4)]
        use = torch.tensor([int(slots[i]) if done[i] < lengths[i] else -1 for i in range(4)], dtype=torch.int32).cuda()
        got = causal_conv1d_silu_step(x[at], w, b, cache, slots=use)
        for i in range(4):
            if done[i] < lengths[i]:
                assert torch.equal(got[i], whole[at[i]])
                done[i] += 1
    for i, n in enumerate(lengths):
        last = x[int(off[i + 1]) - min(n, K - 1): int(off[i + 1])]
        want = torch.cat([torch.zeros(K - 1 - last.size(0), D, dtype=io, device="cuda"), last])
        assert torch.equal(cache[slots[i].item()], want)
    assert bool((cache[[2, 4]] == 7).all())


class Mixer(torch.nn.Module):
    """A mixer with the attributes of ossm's ``_MambaMixer`` (``mambarec.py:64-135``)."""

    def __init__(self, d_model, d_state, d_conv=4, expand=2):
        super().__init__()
        self.d_inner, self.d_state, self.d_conv = expand * d_model, d_state, d_conv
        self.dt_rank = -(-d_model // 16)
        self.in_proj = torch.nn.Linear(d_model, 2 * self.d_inner, bias=False)
        self.conv1d = torch.nn.Conv1d(self.d_inner, self.d_inner, d_conv, groups=self.d_inner)
        self.x_proj = torch.nn.Linear(self.d_inner, self.dt_rank + 2 * d_state, bias=False)
        self.dt_proj = torch.nn.Linear(self.dt_rank, self.d_inner)
        self.A_log = torch.nn.Parameter(torch.log(torch.arange(1.0, d_state + 1)).repeat(self.d_inner, 1))
        self.out_proj = torch.nn.Linear(self.d_inner, d_model, bias=False)


def ref_mixer(m, x):
    """One sequence ``[L, d_model]`` in the mixer's dtype."""
    xz = m.in_proj(x)
    u, z = xz[:, :m.d_inner], xz[:, m.d_inner:]
    u = F.silu(F.conv1d(F.pad(u.t()[None], (m.d_conv - 1, 0)), m.conv1d.weight, m.conv1d.bias, groups=m.d_inner))[0].t()
    dt, B, C = torch.split(m.x_proj(u), [m.dt_rank, m.d_state, m.d_state], dim=-1)
    start = torch.zeros(1, m.d_inner, m.d_state, dtype=x.dtype)
    y, _ = ref_scan(u, m.dt_proj(dt), -torch.exp(m.A_log), B, C, z, None, None, True, offsets_of([x.size(0)]), start)
    return m.out_proj(y)


@pytest.mark.parametrize("d_state", [16, 256])
def test_mixer_packed_and_stepwise(d_state):
    """The whole mixer: packed training with gradients, then prompts in pieces and single tokens through a cache, then the
    step captured into a graph -- all against one sequence at a time in float64."""
    import copy

    from ossm_b200.mixer import MambaCache, mamba_mixer_packed, mamba_mixer_step

    torch.manual_seed(1)
    m = Mixer(32, d_state)
    m64 = copy.deepcopy(m).double()
    m = m.cuda()
    lengths = [12, 1, 0, 30]
    off = offsets_of(lengths)
    x = torch.randn(sum(lengths), 32)
    w = torch.randn(sum(lengths), 32)
    x64 = x.double().requires_grad_(True)
    want = torch.cat([ref_mixer(m64, x64[off[i]:off[i + 1]]) for i in range(4) if lengths[i]])
    (want * w.double()).sum().backward()
    xd = x.cuda().requires_grad_(True)
    got = mamba_mixer_packed(m, xd, off.cuda())
    (got * w.cuda()).sum().backward()
    rel = lambda a, b: float((a.double().cpu() - b).abs().max() / b.abs().max().clamp_min(1e-30))
    # the projections are float32 GEMMs of the library: the bound of the fused mixer's own test
    assert record("packed mixer", "output", rel(got.detach(), want.detach()), 2e-4) <= 2e-4
    assert rel(xd.grad, x64.grad) <= 2e-4
    for (n, p), (_, q) in zip(m.named_parameters(), m64.named_parameters()):
        assert rel(p.grad, q.grad) <= 2e-4, n
    # prompts, a second piece of them, then steps
    cache = MambaCache(m, 6)
    slots = torch.tensor([4, 1, 3, 0], dtype=torch.int32).cuda()
    done = [0, 0, 0, 0]
    for piece, resume in (([5, 1, 0, 11], False), ([2, 0, 0, 9], True)):
        rows = torch.cat([torch.arange(off[i] + done[i], off[i] + done[i] + n) for i, n in enumerate(piece)])
        y = mamba_mixer_packed(m, x[rows].cuda(), offsets_of(piece).cuda(), cache, slots=slots, resume=resume)
        assert rel(y, want.detach()[rows]) <= 2e-4
        done = [a + b for a, b in zip(done, piece)]
    token = torch.zeros(4, 32, device="cuda")
    use = torch.full((4,), -1, dtype=torch.int32, device="cuda")
    mamba_mixer_step(m, token, cache, slots=use)      # warm-up: rows of padding only, the cache stays as it is
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mamba_mixer_step(m, token, cache, slots=use)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mamba_mixer_step(m, token, cache, slots=use)
    count = 0
    while any(d < n for d, n in zip(done, lengths)):
        at = [int(off[i]) + done[i] if done[i] < lengths[i] else 0 for i in range(4)]
        token.copy_(x[at])
        use.copy_(torch.tensor([int(slots[i]) if done[i] < lengths[i] else -1 for i in range(4)], dtype=torch.int32))
        if count % 2:
            y = mamba_mixer_step(m, token, cache, slots=use)
        else:
            graph.replay()
            y = out
        for i in range(4):
            if done[i] < lengths[i]:
                assert rel(y[i], want.detach()[at[i]]) <= 4e-4
                done[i] += 1
        count += 1


def test_other_stream_and_graphs():
    """A call on a side stream; forward and backward captured into two graphs that replay in turn on new inputs."""
    from ossm_b200.selective_scan import selective_scan_packed

    c, off = scan_case([300, 20, 500], 64, 16, seed=8)
    names = ["u", "dt", "A", "B", "C", "z", "D", "bias", "start"]
    d = {k: v.cuda() for k, v in c.items()}
    offd = off.cuda()
    g = torch.randn(d["u"].shape, device="cuda")

    def run():
        leaves = [d[k].detach().requires_grad_(True) for k in names]
        u, dt, A, B, C, z, D, bias, start = leaves
        y, end = selective_scan_packed(u, dt, A, B, C, offd, z, D, delta_bias=bias, delta_softplus=True, initial_state=start,
                                       return_state=True)
        return (y.detach(), end.detach()) + torch.autograd.grad((y, end), leaves, (g, torch.ones_like(end)))

    want = [t.clone() for t in run()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(on_side, want):
        assert torch.equal(a, b)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = run()
        graphs.append((graph, res))
    with torch.no_grad():
        d["u"].mul_(0.5)
    fresh = [t.clone() for t in run()]
    for graph, res in graphs + graphs:
        graph.replay()
        for a, b in zip(res, fresh):
            assert torch.equal(a, b)


@pytest.mark.parametrize("N", [16, 64, 256])
def test_long_sequences_cross_seams(N):
    """Rows enough for many time segments, summaries in several pieces: sequences that span segments, begin and end inside
    them, and a cache updated in place -- against the same sequences one by one, each its own call, in float64 where the
    whole would take too long here: the float64 recurrence runs vectorised over channels, row by row."""
    from ossm_b200.selective_scan import selective_scan_packed

    lengths, D = [1300, 0, 40, 2600, 1, 700], 33
    c, off = scan_case(lengths, D, N, seed=12, first=3, pad=9)
    S = len(lengths)
    slots = torch.tensor([5, 1, 6, 0, 2, 3], dtype=torch.int32)
    cache = torch.randn(7, D, N, generator=torch.Generator().manual_seed(2))
    start = torch.stack([cache[i] for i in slots.tolist()]).double()
    f = {k: v.double().cuda() for k, v in c.items()}
    step = F.softplus(f["dt"] + f["bias"])
    want, h_all = torch.zeros(c["u"].shape, dtype=torch.float64, device="cuda"), start.cuda().clone()
    for i in range(S):
        h = h_all[i]
        for t in range(int(off[i]), int(off[i + 1])):
            h = torch.exp(step[t][:, None] * f["A"]) * h + (step[t] * f["u"][t])[:, None] * f["B"][t]
            want[t] = (h @ f["C"][t] + f["D"] * f["u"][t]) * F.silu(f["z"][t])
        h_all[i] = h
    d = {k: v.cuda() for k, v in c.items()}
    cached = cache.cuda()
    got = selective_scan_packed(d["u"], d["dt"], d["A"], d["B"], d["C"], off.cuda(), d["z"], d["D"], delta_bias=d["bias"],
                                delta_softplus=True, cache=cached, slots=slots.cuda(), resume=True)
    close(got, want, "out")
    close(cached[slots.long().cuda()], h_all, "cache")
    # the gradients of the same rows, by the adjoint recurrence from right to left
    g_out, g_end = torch.randn(c["u"].shape), torch.randn(S, D, N)
    names = ["u", "dt", "A", "B", "C", "z", "D", "bias"]
    leaves = [d[k].detach().requires_grad_(True) for k in names] + [start.float().cuda().requires_grad_(True)]
    u, dt, A, B, C, z, Dv, bias, st = leaves
    y, end = selective_scan_packed(u, dt, A, B, C, off.cuda(), z, Dv, delta_bias=bias, delta_softplus=True, initial_state=st,
                                   return_state=True)
    grads = torch.autograd.grad((y, end), leaves, (g_out.cuda(), g_end.cuda()))
    gate = F.silu(f["z"])
    dy = g_out.cuda().double() * gate
    r = {k: torch.zeros_like(f[k]) for k in names}
    r_start = torch.zeros(S, D, N, dtype=torch.float64, device="cuda")
    for i in range(S):
        lo, hi = int(off[i]), int(off[i + 1])
        states = [start[i].cuda()]
        for t in range(lo, hi):
            states.append(torch.exp(step[t][:, None] * f["A"]) * states[-1] + (step[t] * f["u"][t])[:, None] * f["B"][t])
        g = g_end[i].double().cuda()
        for t in range(hi - 1, lo - 1, -1):
            h, before = states[t - lo + 1], states[t - lo]
            a = torch.exp(step[t][:, None] * f["A"])
            g = g + dy[t][:, None] * f["C"][t]
            r["C"][t] = dy[t] @ h
            r["B"][t] = (step[t] * f["u"][t]) @ g
            force = g @ f["B"][t]
            through = g * before * a
            r["A"] += through * step[t][:, None]
            r["dt"][t] = ((through * f["A"]).sum(1) + force * f["u"][t]) * -torch.expm1(-step[t])
            r["u"][t] = force * step[t] + dy[t] * f["D"]
            ungated = h @ f["C"][t] + f["D"] * f["u"][t]
            sig = torch.sigmoid(f["z"][t])
            r["z"][t] = g_out[t].cuda().double() * ungated * sig * (1 + f["z"][t] * (1 - sig))
            g = g * a
        r_start[i] = g
    real = slice(int(off[0]), int(off[-1]))
    r["D"], r["bias"] = (dy * f["u"])[real].sum(0), r["dt"].sum(0)
    for k, a in zip(names, grads):
        close(a, r[k], "grad_" + k)
    close(grads[-1], r_start, "grad_start")


def test_offsets_and_slots_out_of_range_are_held():
    """Nothing is accessed out of range: the kernels hold offsets and slots inside the tensors and say so."""
    from ossm_b200 import _lib
    from ossm_b200.mixer import causal_conv1d_silu_packed, causal_conv1d_silu_step
    from ossm_b200.selective_scan import selective_scan_packed, selective_scan_step

    c, _ = scan_case([40], 32, 16)
    d = {k: v.cuda() for k, v in c.items()}
    w = torch.randn(32, 4, device="cuda")
    scan = lambda off, **k: selective_scan_packed(d["u"], d["dt"], d["A"], d["B"], d["C"],
                                                  torch.tensor(off, dtype=torch.int32, device="cuda"), d["z"], **k)
    conv = lambda off, **k: causal_conv1d_silu_packed(d["u"], w, None, torch.tensor(off, dtype=torch.int32, device="cuda"), **k)
    for off in ([0, 30, 10, 41], [-5, 20, 1000], [0, 1 << 30, 40]):
        for call in (scan, conv):
            call(off)
            torch.cuda.synchronize()
            assert _lib.device_status() == 3, off
    state, window = torch.zeros(2, 32, 16, device="cuda"), torch.zeros(2, 3, 32, device="cuda")
    past = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    for call in (lambda: scan([0, 20, 40], cache=state, slots=past), lambda: conv([0, 20, 40], cache=window, slots=past),
                 lambda: selective_scan_step(d["u"][:2], d["dt"][:2], d["A"], d["B"][:2], d["C"][:2], state, slots=past),
                 lambda: causal_conv1d_silu_step(d["u"][:2], w, None, window, slots=past)):
        call()
        torch.cuda.synchronize()
        assert _lib.device_status() == 4


def test_refusals_on_the_device():
    from ossm_b200.mixer import causal_conv1d_silu_step
    from ossm_b200.selective_scan import selective_scan_packed, selective_scan_step

    c, off = scan_case([10], 32, 16)
    d = {k: v.cuda() for k, v in c.items()}
    args = (d["u"], d["dt"], d["A"], d["B"], d["C"])
    cache = torch.zeros(2, 32, 16, device="cuda")
    good = dict(offsets=off.cuda(), gate=d["z"])
    for change, words in (({"offsets": off}, "device"), ({"offsets": off.cuda().float()}, "int32"),
                          ({"cache": cache.double()}, "cache"), ({"cache": cache[:, :, :8]}, "cache"),
                          ({"slots": off.cuda()[:1]}, "cache"), ({"cache": cache, "slots": off.cuda()}, "one entry"),
                          ({"cache": cache, "return_state": True}, "exclude"), ({"out": torch.empty_like(d["dt"])}, "out"),
                          ({"cache": cache, "out": d["u"]}, "share"), ({"cache": cache, "out": d["u"].bfloat16()}, "out"),
                          ({"cache": cache, "resume": off.cuda()}, "resume"), ({"gate": d["z"].bfloat16()}, "gate"),
                          ({"initial_state": cache}, "initial_state"), ({"D": d["D"][:3]}, "D must")):
        with pytest.raises(RuntimeError, match=words):
            selective_scan_packed(*args, **{**good, **change})
    with pytest.raises(RuntimeError, match="not differentiable"):
        selective_scan_packed(d["u"].detach().requires_grad_(True), *args[1:], off.cuda(), cache=cache)
    with pytest.raises(RuntimeError, match="not differentiable"):
        selective_scan_step(*args[:2], d["A"].detach().requires_grad_(True), *args[3:], cache)
    with pytest.raises(RuntimeError, match="cache"):
        causal_conv1d_silu_step(d["u"], torch.zeros(32, 4, device="cuda"), None, torch.zeros(10, 4, 32, device="cuda"))
    u = d["u"].detach().requires_grad_(True)
    first, = torch.autograd.grad(selective_scan_packed(u, *args[1:], off.cuda()).square().sum(), u, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        first.sum().backward()
    big = torch.zeros(32, 257, device="cuda")
    with pytest.raises(RuntimeError, match="state size"):
        selective_scan_step(d["u"], d["dt"], big, big[:10], big[:10], torch.zeros(10, 32, 257, device="cuda"))
