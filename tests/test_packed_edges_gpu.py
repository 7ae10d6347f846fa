"""Packed and single-token operators at their edges: what they allocate, refuse, leave alone and tell autograd, and the
regimes that only larger calls reach -- against the float64 definitions of ``test_packed_gpu``, whose derivation of the
tolerances holds here too."""
import ctypes

import pytest
import torch
import torch.nn.functional as F

from test_packed_gpu import BF16, F32, Mixer, close, offsets_of, ref_conv, ref_mixer, ref_scan, scan_case

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    from ossm_b200 import _lib

    torch.cuda.synchronize()
    assert _lib.device_status() == 0


def on_gpu(lengths, D, N, *types, **more):
    c, off = scan_case(lengths, D, N, *types, **more)
    return {k: v.cuda() for k, v in c.items()}, off.cuda()


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_no_states_are_kept_where_no_gradient_can_follow(mode):
    """Operands that require gradients (a mixer's own parameters) cost no memory while gradients are off."""
    from ossm_b200.selective_scan import selective_scan_packed

    d, off = on_gpu([900, 600, 548], 64, 256)

    def peak(require):
        leaves = {k: v.detach().requires_grad_(require) for k, v in d.items()}
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        with mode():
            out, end = selective_scan_packed(leaves["u"], leaves["dt"], leaves["A"], leaves["B"], leaves["C"], off, leaves["z"],
                                             leaves["D"], delta_bias=leaves["bias"], delta_softplus=True,
                                             initial_state=leaves["start"], return_state=True)
        return torch.cuda.max_memory_allocated() - base, out, end

    plain, out, end = peak(False)
    with_parameters, out2, end2 = peak(True)
    assert with_parameters == plain
    assert torch.equal(out, out2) and torch.equal(end, end2)


def test_cache_with_fewer_entries_than_sequences():
    """Without slots row i is entry i: a cache without one refuses the call and stays as it is."""
    from ossm_b200.mixer import (MambaCache, causal_conv1d_silu_packed, causal_conv1d_silu_step, mamba_mixer_packed,
                                 mamba_mixer_step)
    from ossm_b200.selective_scan import selective_scan_packed, selective_scan_step

    d, off = on_gpu([2, 0, 3], 8, 16)
    state, window = torch.ones(2, 8, 16, device="cuda"), torch.ones(2, 3, 8, device="cuda")
    w = torch.randn(8, 4, device="cuda")
    args = (d["u"], d["dt"], d["A"], d["B"], d["C"])
    three = tuple(t if t is d["A"] else t[:3] for t in args)
    m = Mixer(8, 16).cuda()
    cache = MambaCache(m, 2)
    x = torch.randn(5, 8, device="cuda")
    for call in (lambda: selective_scan_packed(*args, off, cache=state), lambda: selective_scan_step(*three, state),
                 lambda: causal_conv1d_silu_packed(d["u"], w, None, off, cache=window),
                 lambda: causal_conv1d_silu_step(d["u"][:3], w, None, window),
                 lambda: mamba_mixer_packed(m, x, off, cache), lambda: mamba_mixer_step(m, x[:3], cache)):
        with pytest.raises(RuntimeError, match="2 entries"):
            call()
    assert bool((state == 1).all()) and bool((window == 1).all()) and not cache.conv.any() and not cache.ssm.any()
    slots = torch.tensor([1, -1, 0], dtype=torch.int32, device="cuda")
    selective_scan_packed(*args, off, cache=state, slots=slots)
    causal_conv1d_silu_step(d["u"][:3], w, None, window, slots=slots)


def test_mixer_cache_under_autocast():
    """float32 parameters under bfloat16 autocast: prompts in pieces and single tokens, the cache made inside or outside of
    the region.  Some twelve roundings to bfloat16 (2^-8 each) lie between the input and the output."""
    import copy

    from ossm_b200.mixer import MambaCache, mamba_mixer_packed, mamba_mixer_step

    torch.manual_seed(3)
    m = Mixer(32, 16)
    m64 = copy.deepcopy(m).double()
    m = m.cuda()
    lengths = [9, 4]
    off = offsets_of(lengths)
    x = torch.randn(13, 32)
    want = torch.cat([ref_mixer(m64, x.double()[off[i]:off[i + 1]]) for i in range(2)]).detach()
    near = lambda got, rows: float((got.double().cpu() - want[rows]).abs().max() / want.abs().max()) <= 12 * 2.0 ** -8
    outside = MambaCache(m, 2)
    assert outside.conv.dtype == F32
    for inside in (True, False):
        with torch.autocast("cuda", BF16):
            cache = MambaCache(m, 2) if inside else outside
            assert cache.conv.dtype == (BF16 if inside else F32) and cache.ssm.dtype == F32
            assert near(mamba_mixer_packed(m, x.cuda(), off.cuda()).detach(), slice(0, 13))
            rows = torch.tensor([0, 1, 2, 9])
            assert near(mamba_mixer_packed(m, x[rows].cuda(), offsets_of([3, 1]).cuda(), cache), rows)
            rows = torch.tensor([3, 4, 5, 6, 7, 10])
            assert near(mamba_mixer_packed(m, x[rows].cuda(), offsets_of([5, 1]).cuda(), cache, resume=True), rows)
            rows = torch.tensor([8, 11])
            assert near(mamba_mixer_step(m, x[rows].cuda(), cache), rows)


@pytest.mark.parametrize("D, N", [(24, 16), (24, 200), (72, 16), (72, 20)])
@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (BF16, F32)], ids=["f32", "bf16", "bf16_dt32"])
def test_backward_outputs_off_the_vector_boundary(D, N, types):
    """The C entry writes its gradients wherever their types allow: dense, one element behind a 16-byte boundary."""
    from ossm_b200 import _lib

    io, step = types
    d, off = on_gpu([40, 0, 27], D, N, *types, pad=3, pitched=False)
    rows, S = d["u"].size(0), 3
    lib = _lib.load()
    codes = (int(io == BF16), int(step == BF16))
    kept = torch.empty(-(-rows // lib.ossm_b200_selective_scan_packed_tile(N)), D, N, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    p = lambda t: ctypes.c_void_p(t.data_ptr())
    operands = (p(d["u"]), D, p(d["dt"]), D, p(d["A"]), p(d["B"]), N, p(d["C"]), N, p(d["z"]), D, p(d["D"]), p(d["bias"]), 1)
    out = torch.empty_like(d["u"])
    ws = torch.empty(max(lib.ossm_b200_selective_scan_packed_workspace_bytes(rows, D, N, *codes), 16), dtype=torch.uint8, device="cuda")
    _lib.check(lib.ossm_b200_selective_scan_packed_forward(
        *operands, p(off), None, None, 1, p(d["start"]), None, S, p(out), D, 1, p(kept), p(ws), ws.numel(), rows, S, D, N, *codes,
        stream), "forward")
    grad = torch.randn(rows, D, generator=torch.Generator().manual_seed(1)).to(io).cuda()
    ws = torch.empty(lib.ossm_b200_selective_scan_packed_backward_workspace_bytes(rows, D, N, *codes), dtype=torch.uint8, device="cuda")

    def backward(shift):
        shapes = [((rows, D), io), ((rows, D), step), ((D, N), F32), ((rows, N), io), ((rows, N), io), ((rows, D), io), ((D,), F32),
                  ((D,), F32), ((S, D, N), F32)]
        outs = []
        for shape, dtype in shapes:
            count = torch.Size(shape).numel()
            flat = torch.full((count + shift + 1,), 5.0, dtype=dtype, device="cuda")
            outs.append((flat, flat[shift:shift + count].view(shape)))
        _lib.check(lib.ossm_b200_selective_scan_packed_backward(
            p(grad), D, *operands, p(off), p(d["start"]), None, p(kept), *(p(v) for _, v in outs), p(ws), ws.numel(), rows, S, D, N,
            *codes, stream), "backward")
        assert all(bool((flat[:shift] == 5).all()) and float(flat[-1]) == 5 for flat, _ in outs)
        return [v for _, v in outs]

    for a, b in zip(backward(0), backward(1)):
        assert torch.equal(a, b)


def test_wide_integers_are_not_wrapped():
    """int64 slots and offsets past 32 bits are wrong slots and offsets, not others that lie in range."""
    from ossm_b200 import _lib
    from ossm_b200.selective_scan import selective_scan_packed, selective_scan_step

    d, off = on_gpu([2], 8, 16)
    state = torch.ones(2, 8, 16, device="cuda")
    args = (d["u"], d["dt"], d["A"], d["B"], d["C"])
    slots = torch.tensor([1 << 32, 1], device="cuda")
    selective_scan_step(*args, state, slots=slots)
    torch.cuda.synchronize()
    assert _lib.device_status() == 4
    assert bool((state[0] == 1).all()) and not bool((state[1] == 1).all())
    before = state.clone()
    selective_scan_step(*args, state, slots=torch.tensor([-(1 << 32), -(1 << 40)], device="cuda"))
    assert torch.equal(state, before)
    selective_scan_packed(*args, torch.tensor([0, (1 << 32) + 2], device="cuda"))
    torch.cuda.synchronize()
    assert _lib.device_status() == 3
    want = selective_scan_packed(*args, off)
    assert torch.equal(selective_scan_packed(*args, off.long()), want)


def test_autograd_sees_what_is_written_in_place():
    """A cache that a graph still needs is not changed behind its back, and a cache or a result that requires a gradient
    is refused."""
    from ossm_b200.mixer import causal_conv1d_silu_packed, causal_conv1d_silu_step
    from ossm_b200.selective_scan import selective_scan_packed, selective_scan_step

    d, off = on_gpu([2, 3], 8, 16)
    args = (d["u"], d["dt"], d["A"], d["B"], d["C"])
    two = tuple(t if t is d["A"] else t[:2] for t in args)
    w = torch.randn(8, 4, device="cuda")
    state, window = torch.ones(2, 8, 16, device="cuda"), torch.ones(2, 3, 8, device="cuda")
    calls = [(state, lambda c, **k: selective_scan_packed(*args, off, cache=c, **k), d["u"]),
             (state, lambda c, **k: selective_scan_step(*two, c, **k), d["u"][:2]),
             (window, lambda c, **k: causal_conv1d_silu_packed(d["u"], w, None, off, cache=c, **k), d["u"]),
             (window, lambda c, **k: causal_conv1d_silu_step(d["u"][:2], w, None, c, **k), d["u"][:2])]
    for cache, call, like in calls:
        scale = torch.ones_like(cache, requires_grad=True)
        loss = (cache * scale).sum()              # keeps the cache for its backward pass
        call(cache)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        out, scale = torch.ones_like(like), torch.ones_like(like, requires_grad=True)
        loss = (out * scale).sum()
        call(cache, out=out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        with pytest.raises(RuntimeError, match="not differentiable"):
            call(cache.clone().requires_grad_(True))
        with pytest.raises(RuntimeError, match="not differentiable"):
            call(cache, out=torch.empty_like(like).requires_grad_(True))
        with torch.inference_mode():
            call(cache.clone())
    # the state that preceded a training call, stepped on before its backward pass
    u = d["u"].detach().requires_grad_(True)
    out = selective_scan_packed(u, *args[1:], off, initial_state=state)
    selective_scan_step(*two, state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@pytest.mark.parametrize("N", [16, 20, 256])
@pytest.mark.parametrize("D", [24, 72])
def test_rows_of_no_sequence_have_zero_gradients_beside_infinities(D, N):
    """NaN in the first sequence's gradient and in the last one's state stay with those sequences."""
    from ossm_b200.selective_scan import selective_scan_packed

    d, off = on_gpu([5, 6, 5], D, N, first=5, pad=6)
    d["u"][19] = float("nan")
    g = torch.randn_like(d["u"])
    g[5] = float("inf")
    names = ["u", "dt", "A", "B", "C", "z"]
    leaves = {k: d[k].detach().requires_grad_(True) for k in names}
    out = selective_scan_packed(*(leaves[k] for k in names[:5]), off, leaves["z"], delta_bias=d["bias"], delta_softplus=True)
    grads = torch.autograd.grad(out, list(leaves.values()), g)
    for k, a in zip(names, grads):
        if k != "A":
            assert not a[:5].any() and not a[21:].any(), k
            assert bool(a[10:16].isfinite().all()), k


def test_growing_states_that_are_zero_at_a_seam():
    """States may grow (A dt > 0).  Where a state, or its adjoint, is still zero, the growth over a whole segment, which is no
    float32 number, must not make it anything else."""
    from ossm_b200.selective_scan import selective_scan_packed

    T, D, N = 2000, 33, 16
    d, off = on_gpu([T], D, N)
    d["A"] = 2.5 + torch.rand(D, N, device="cuda")
    d["dt"] = torch.full((T, D), 1.0, device="cuda")
    d["u"] = d["u"].clone()
    d["u"][: T - 8] = 0
    g = torch.randn(T, D, device="cuda")
    g[8:] = 0
    names = ["u", "dt", "A", "B", "C"]
    leaves = {k: d[k].detach().requires_grad_(True) for k in names}
    got = selective_scan_packed(*leaves.values(), off)
    grads = torch.autograd.grad(got, list(leaves.values()), g)
    r = {k: d[k].double().cpu().requires_grad_(True) for k in names}
    want, _ = ref_scan(*r.values(), None, None, None, False, off.cpu(), torch.zeros(1, D, N, dtype=torch.float64))
    w_grads = torch.autograd.grad(want, list(r.values()), g.double().cpu())
    close(got, want.detach(), "out")
    for k, a, b in zip(names, grads, w_grads):
        close(a, b, "grad_" + k)


def cut_of(bytes_of, D, N, extra=0):
    """``(segments, pieces)`` that a workspace of ``bytes_of`` stands for: the only pair whose parts add up to it."""
    up = lambda v: (v + 255) // 256 * 256
    found = []
    for pieces in (1, 2, 4):
        for g in range(1, 4096):
            if up(g * pieces * D * N * 4) + up(g * D * N * 4) + up(g * pieces * D * 4) + up(g * pieces * 4) \
                    + (up(g * 2 * D * 4) + extra if extra else 0) == bytes_of:
                found.append((g, pieces))
    assert len(found) == 1, found
    return found[0]


def walk(f, off, start, dy_of, g_end, softplus_slope):
    """The recurrence and its adjoint in float64, place by place over all sequences at once: ``(y, ends, gradients)``."""
    at = torch.tensor(off)
    lengths = at[1:] - at[:-1]
    order = lengths.argsort(descending=True, stable=True)
    begin, order_d = at[:-1][order].cuda(), order.cuda()
    counts = [int((lengths > t).sum()) for t in range(int(lengths.max()))]
    step, A = f["step"], f["A"]
    h = start[order_d].clone()
    y = torch.zeros_like(f["u"])
    kept = torch.zeros(*f["u"].shape, A.size(1), dtype=torch.float64, device="cuda")
    for t, n in enumerate(counts):
        r = begin[:n] + t
        kept[r] = h[:n]
        h[:n] = torch.exp(step[r][:, :, None] * A) * h[:n] + (step[r] * f["u"][r])[:, :, None] * f["B"][r][:, None, :]
        y[r] = (h[:n] * f["C"][r][:, None, :]).sum(-1) + f["D"] * f["u"][r]
    ends = torch.empty_like(h)
    ends[order_d] = h
    dy = dy_of(y)
    g = g_end[order_d].clone()
    r_ = {k: torch.zeros_like(f[k]) for k in ("u", "B", "C", "A", "step")}
    for t in range(len(counts) - 1, -1, -1):
        n = counts[t]
        r = begin[:n] + t
        a = torch.exp(step[r][:, :, None] * A)
        now = a * kept[r] + (step[r] * f["u"][r])[:, :, None] * f["B"][r][:, None, :]
        g[:n] += dy[r][:, :, None] * f["C"][r][:, None, :]
        r_["C"][r] = (now * dy[r][:, :, None]).sum(1)
        r_["B"][r] = (g[:n] * (step[r] * f["u"][r])[:, :, None]).sum(1)
        force = (g[:n] * f["B"][r][:, None, :]).sum(-1)
        g[:n] *= a
        through = g[:n] * kept[r]
        r_["A"] += (through * step[r][:, :, None]).sum(0)
        r_["step"][r] = (through * A).sum(-1) + force * f["u"][r]
        r_["u"][r] = force * step[r] + dy[r] * f["D"]
    g_start = torch.empty_like(g)
    g_start[order_d] = g
    r_["D"] = (dy * f["u"]).sum(0)
    r_["dt"] = r_.pop("step") * softplus_slope
    r_["bias"] = r_["dt"].sum(0)
    return y, ends, {**r_, "start": g_start}


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16)], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows, D, N, pieces", [(6000, 2048, 16, (2, 4)), (3200, 2048, 16, (1, 2)), (12000, 2048, 16, (4, 4)),
                                                (6000, 1024, 32, (2, 4)), (12800, 128, 256, (4, 4)), (6001, 127, 250, (2, 2))])
def test_segments_in_several_pieces(rows, D, N, pieces, types):
    """Segments long enough to be summarised in 2 and 4 pieces, forward and backward: sequences that begin and end inside
    pieces, on their borders and on the segments' borders, some without rows, one over many segments."""
    from ossm_b200 import _lib
    from ossm_b200.selective_scan import selective_scan_packed

    io, step = types
    lib, codes = _lib.load(), (int(io == BF16), int(step == BF16))
    forward = cut_of(lib.ossm_b200_selective_scan_packed_workspace_bytes(rows, D, N, *codes), D, N)
    back_bytes = lib.ossm_b200_selective_scan_packed_backward_workspace_bytes(rows, D, N, *codes)
    backward = cut_of(back_bytes, D, N, extra=-(-D // 32) * rows * 2 * N * 4)
    assert (forward[1], backward[1]) == pieces, (forward, backward)
    cuts = {0, rows}
    for (g, k), multiple in ((forward, 16), (backward, lib.ossm_b200_selective_scan_packed_tile(N))):
        m = -(-rows // g)
        m = -(-m // multiple) * multiple           # rows of a segment
        part = m // k
        cuts |= {2 * m, 3 * m + part, 3 * m + part + 5, 4 * m + 2 * part - 1, 5 * m + 1, 7 * m - 1, 7 * m, 9 * m + m // 2,
                 g // 2 * m + 3, (g - 2) * m + part, (g - 1) * m + 1}
    cuts = sorted(c for c in cuts if 0 <= c <= rows)
    cuts = cuts[:4] + [cuts[3]] * 2 + cuts[4:] + [rows]     # sequences without rows, inside and at the end
    lengths = [b - a for a, b in zip(cuts[:-1], cuts[1:])]
    c, off = scan_case(lengths, D, N, *types, seed=21)
    d = {k: v.cuda() for k, v in c.items()}
    S = len(lengths)
    gen = torch.Generator(device="cuda").manual_seed(4)
    g_out = torch.randn(rows, D, generator=gen, device="cuda").to(io)
    g_end = torch.randn(S, D, N, generator=gen, device="cuda")
    f = {k: v.double() for k, v in d.items()}
    raw = f["dt"] + f["bias"]
    f["step"] = F.softplus(raw)
    sig = torch.sigmoid(f["z"])
    y, ends, want = walk(f, cuts, f["start"], lambda y: g_out.double() * f["z"] * sig, g_end.double(), torch.sigmoid(raw))
    want["z"] = g_out.double() * y * sig * (1 + f["z"] * (1 - sig))
    names = ["u", "dt", "A", "B", "C", "z", "D", "bias", "start"]
    leaves = {k: d[k].detach().requires_grad_(True) for k in names}
    out, end = selective_scan_packed(*(leaves[k] for k in names[:5]), off.cuda(), leaves["z"], leaves["D"],
                                     delta_bias=leaves["bias"], delta_softplus=True, initial_state=leaves["start"],
                                     return_state=True)
    close(out, y * f["z"] * sig, "out")
    close(end, ends, "end")
    for k, a in zip(names, torch.autograd.grad((out, end), list(leaves.values()), (g_out, g_end))):
        close(a, want[k], "grad_" + k)
    # the same through a cache, updated in place
    slots = torch.randperm(S + 3, generator=torch.Generator().manual_seed(1))[:S].int().cuda()
    cache = torch.full((S + 3, D, N), 7.0, device="cuda")
    cache[slots.long()] = d["start"]
    got = selective_scan_packed(*(d[k] for k in names[:5]), off.cuda(), d["z"], d["D"], delta_bias=d["bias"],
                                delta_softplus=True, cache=cache, slots=slots, resume=True)
    assert torch.equal(got, out) and torch.equal(cache[slots.long()], end)


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (BF16, F32)], ids=["f32", "bf16", "bf16_dt32"])
@pytest.mark.parametrize("S, D, N", [(512, 4096, 16), (130, 1024, 256), (200, 4097, 16), (700, 2050, 8), (300, 2049, 4),
                                     (150, 777, 128), (260, 1000, 64), (400, 4096, 20), (500, 3000, 3), (300, 1500, 100),
                                     (300, 1501, 50)])
def test_many_tokens_of_a_block(S, D, N, types):
    """Sequences enough that a block takes many entries one after the other (the ring of bulk copies turns several times),
    padding rows between them; entries of no row stay as they were, and a second run gives the same bits."""
    from ossm_b200.selective_scan import selective_scan_step

    io, step = types
    gen = torch.Generator(device="cuda").manual_seed(S + N)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    u, z, dt = r(S, D).to(io), r(S, 2 * D).to(io)[:, D:], (r(S, D) * 0.5).to(step)
    proj = r(S, 4 + 2 * N).to(io)
    B, C = proj[:, 4:4 + N], proj[:, 4 + N:]
    A, bias, skip = -torch.exp(r(D, N) * 0.5) * 2, r(D) * 0.5 - 3.0, r(D)
    slots = torch.randperm(S + 9, generator=torch.Generator().manual_seed(S))[:S].int()
    slots[::7] = -1
    slots[S // 2:S // 2 + 11] = -3                 # more in a row than the ring has places
    before = r(S + 9, D, N)
    runs = []
    for _ in range(2):
        cache = before.clone()
        runs.append((selective_scan_step(u, dt, A, B, C, cache, z, skip, delta_bias=bias, delta_softplus=True, slots=slots.cuda()),
                     cache))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    got, cache = runs[0]
    at, real = slots.long().cuda(), slots.cuda() >= 0
    x = F.softplus(dt.double() + bias.double())
    want_cache, want = before.double(), torch.empty(S, D, dtype=torch.float64, device="cuda")
    for lo in range(0, S, 64):                     # in parts: 64 bits of every state
        p = slice(lo, lo + 64)
        h = torch.where(real[p, None, None], want_cache[at[p].clamp(min=0)], 0.0)
        h = torch.exp(x[p, :, None] * A.double()) * h + (x[p] * u[p].double())[:, :, None] * B[p].double()[:, None, :]
        want[p] = ((h * C[p].double()[:, None, :]).sum(-1) + skip.double() * u[p].double()) * F.silu(z[p].double())
        want_cache[at[p][real[p]]] = h[real[p]]
    close(got, want, "out")
    close(cache, want_cache, "cache")
    rest = torch.ones(S + 9, dtype=torch.bool)
    rest[slots[slots >= 0].long()] = False
    assert torch.equal(cache[rest.cuda()], before[rest.cuda()])


def conv_against_64_bits(x, w, b, start, off, g_out, g_end):
    from ossm_b200.mixer import causal_conv1d_silu_packed

    leaves = [t.detach().requires_grad_(True) for t in (x, w, b, start)]
    got = causal_conv1d_silu_packed(*leaves[:3], off.cuda(), initial_window=leaves[3], return_window=True)
    grads = torch.autograd.grad(got, leaves, (g_out, g_end))
    r = [t.double().detach().requires_grad_(True) for t in (x, w, b, start)]
    want = ref_conv(*r[:3], off, r[3])
    w_grads = torch.autograd.grad(want, r, (g_out.double(), g_end.double()))
    close(got[0], want[0].detach(), "out")
    assert torch.equal(got[1].double(), want[1].detach())
    for k, a, b_ in zip(("x", "w", "b", "start"), grads, w_grads):
        close(a, b_, "grad_" + k)


def conv_operands(lengths, D, K, io, wt, pitch=None, w_shift=0, first=0, pad=0):
    gen = torch.Generator(device="cuda").manual_seed(D + K + sum(lengths))
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    off = offsets_of(lengths, first)
    rows, S = int(off[-1]) + pad, len(lengths)
    flat = (r(D * K + w_shift) * 0.5).to(wt)
    return (r(rows, pitch or 2 * D).to(io)[:, :D], flat[w_shift:].view(D, K), (r(D) * 0.3).to(wt), r(S, K - 1, D).to(io), off,
            r(rows, D).to(io), r(S, K - 1, D).to(io))


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (BF16, F32)], ids=["f32", "bf16", "bf16_w32"])
@pytest.mark.parametrize("K", [1, 2, 3, 4])
@pytest.mark.parametrize("D, w_shift", [(40, 0), (64, 1), (136, 0)])
def test_conv_of_sixteen_bytes_a_thread(D, w_shift, K, types):
    """Rows on 16 bytes: a thread takes 4 or 8 channels, their taps in vector loads or (weights off that boundary) one by one."""
    conv_against_64_bits(*conv_operands([5, 0, 0, 1, 37, 2, 1, 700, 3], D, K, *types, w_shift=w_shift, first=2, pad=3))


@pytest.mark.parametrize("rows, D, K, io", [(20000, 2048, 4, F32), (30000, 4096, 3, BF16), (20000, 2048, 2, F32),
                                            (9000, 1001, 4, F32)])
def test_conv_runs_of_many_rows(rows, D, K, io):
    """Rows enough that a thread walks a hundred of them, with sequences that begin and end anywhere in such a run."""
    gen = torch.Generator().manual_seed(rows)
    cuts = sorted(torch.randint(0, rows - 7, (40,), generator=gen).tolist() + [0, 1, 2, 5, 64, 66, 256, rows - 7])
    conv_against_64_bits(*conv_operands([b - a for a, b in zip(cuts[:-1], cuts[1:])], D, K, io, io, pad=7))


@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("S, D, K", [(512, 4096, 4), (37, 64, 3), (5, 33, 2), (64, 40, 1)])
def test_conv_tokens_against_64_bits(S, D, K, io):
    from ossm_b200.mixer import causal_conv1d_silu_step

    x, w, b, _, _, _, _ = conv_operands([S], D, K, io, io)
    gen = torch.Generator().manual_seed(S)
    slots = torch.randperm(S + 4, generator=gen)[:S].int()
    slots[3:5] = -1
    before = torch.randn(S + 4, K - 1, D, generator=gen).to(io).cuda()
    cache = before.clone()
    got = causal_conv1d_silu_step(x, w, b, cache, slots=slots.cuda())
    at, real = slots.long().cuda(), slots.cuda() >= 0
    window = torch.cat([torch.where(real[:, None, None], before[at.clamp(min=0)], torch.zeros((), dtype=io, device="cuda")),
                        x[:, None]], 1)
    close(got, F.silu((window.double() * w.double().t()).sum(1) + b.double()), "out")
    want = before.clone()
    want[at[real]] = window[real][:, 1:]
    assert torch.equal(cache, want)


def test_two_segments_where_there_is_no_room_for_more():
    """Channel blocks that fill more than a third of the GPU, a few sequences: the rows are cut in two, forward and backward."""
    from ossm_b200 import _lib
    from ossm_b200.selective_scan import selective_scan_packed

    rows, D, N = 400, 2048, 256
    lib = _lib.load()
    assert cut_of(lib.ossm_b200_selective_scan_packed_workspace_bytes(rows, D, N, 0, 0), D, N)[0] == 2
    assert lib.ossm_b200_selective_scan_packed_workspace_bytes(128, D, N, 0, 0) == 0
    for few in (rows, 64):
        back = lib.ossm_b200_selective_scan_packed_backward_workspace_bytes(few, D, N, 0, 0)
        assert cut_of(back, D, N, extra=D // 32 * few * 2 * N * 4)[0] == 2
    lengths = [130, 0, 69, 2, 199]                 # one over the middle
    cuts = [0, 130, 130, 199, 201, 400]
    c, off = scan_case(lengths, D, N, seed=33)
    d = {k: v.cuda() for k, v in c.items() if k != "z"}
    gen = torch.Generator(device="cuda").manual_seed(4)
    g_out, g_end = torch.randn(rows, D, generator=gen, device="cuda"), torch.randn(5, D, N, generator=gen, device="cuda")
    f = {k: v.double() for k, v in d.items()}
    raw = f["dt"] + f["bias"]
    f["step"] = F.softplus(raw)
    y, ends, want = walk(f, cuts, f["start"], lambda y: g_out.double(), g_end.double(), torch.sigmoid(raw))
    names = ["u", "dt", "A", "B", "C", "D", "bias", "start"]
    leaves = {k: d[k].detach().requires_grad_(True) for k in names}
    out, end = selective_scan_packed(*(leaves[k] for k in names[:5]), off.cuda(), None, leaves["D"], delta_bias=leaves["bias"],
                                     delta_softplus=True, initial_state=leaves["start"], return_state=True)
    close(out, y, "out")
    close(end, ends, "end")
    for k, a in zip(names, torch.autograd.grad((out, end), list(leaves.values()), (g_out, g_end))):
        close(a, want[k], "grad_" + k)
