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
