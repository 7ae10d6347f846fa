"""What the packed and single-token operators refuse, as far as that can be seen without a GPU."""
import ctypes

import pytest
import torch

from ossm_b200 import _lib, packed
from ossm_b200.mixer import causal_conv1d_silu_packed, causal_conv1d_silu_step, mamba_mixer_packed, mamba_mixer_step
from ossm_b200.selective_scan import selective_scan_packed, selective_scan_step


def operands(T=6, D=8, N=4):
    u = torch.randn(T, D)
    return u, torch.rand(T, D), -torch.rand(D, N), torch.randn(T, N), torch.randn(T, N)


OFF = torch.tensor([0, 6], dtype=torch.int32)


def test_cpu_tensors_are_refused():
    u, dt, A, B, C = operands()
    with pytest.raises(RuntimeError, match="CUDA"):
        selective_scan_packed(u, dt, A, B, C, OFF)
    with pytest.raises(RuntimeError, match="CUDA"):
        selective_scan_step(u, dt, A, B, C, torch.zeros(6, 8, 4))
    with pytest.raises(RuntimeError, match="CUDA"):
        causal_conv1d_silu_packed(u, torch.randn(8, 4), None, OFF)
    with pytest.raises(RuntimeError, match="CUDA"):
        causal_conv1d_silu_step(u, torch.randn(8, 4), None, torch.zeros(6, 3, 8))


@pytest.mark.parametrize("change, words", [
    ({0: torch.randn(2, 3, 8)}, "rows, channels"), ({1: torch.rand(6, 7)}, "dt"), ({2: -torch.rand(7, 4)}, "A must"),
    ({2: -torch.rand(8, 0)}, "state size"), ({3: torch.randn(6, 5)}, "B and C"), ({4: torch.randn(5, 4)}, "B and C")])
def test_scan_shapes(change, words):
    args = list(operands())
    for i, t in change.items():
        args[i] = t
    with pytest.raises(RuntimeError, match=words):
        selective_scan_packed(*args, OFF)
    with pytest.raises(RuntimeError, match=words):
        selective_scan_step(*args, torch.zeros(6, 8, 4))


def test_mixer_shapes():
    with pytest.raises(ValueError, match="rows, channels"):
        mamba_mixer_packed(None, torch.randn(1, 2, 3), OFF)
    with pytest.raises(ValueError, match="sequences, channels"):
        mamba_mixer_step(None, torch.randn(1, 2, 3), None)
    with pytest.raises(RuntimeError, match="cache"):
        mamba_mixer_packed(None, torch.randn(2, 3), OFF, slots=OFF)


def test_row_pitch():
    wide = torch.randn(6, 20)
    t, ld = packed._rows(wide[:, 3:11])
    assert ld == 20 and t.data_ptr() == wide[:, 3:11].data_ptr()
    for odd in (wide.t()[:, :5], wide[:, :1].expand(6, 8), wide[:, ::2], wide[:1].expand(6, 20)):
        t, ld = packed._rows(odd)
        assert t.is_contiguous() and ld == odd.size(1) and torch.equal(t, odd)
    assert packed._rows(wide[:1, 3:11])[1] == 8 and packed._rows(wide[:0, 3:11])[1] == 8


def test_library_refuses_without_a_gpu():
    lib = _lib.load()
    p = ctypes.c_void_p(256)

    def scan(rows=4, count=1, D=8, N=4, io=0, dt=0, u=p, ldu=8, ws=None, ws_bytes=0):
        return lib.ossm_b200_selective_scan_packed_forward(u, ldu, p, 8, p, p, 4, p, 4, None, 0, None, None, 0, p, None,
                                                           None, 0, None, None, 0, p, 8, 1, None, ws, ws_bytes, rows,
                                                           count, D, N, io, dt, None)

    def why(rc, words):
        assert rc < 0 and words in lib.ossm_b200_last_error().decode(), lib.ossm_b200_last_error()

    why(scan(rows=-1), "negative")
    why(scan(N=257), "state size")
    why(scan(N=0), "state size")
    why(scan(io=7), "element types")
    why(scan(io=0, dt=1), "element types")
    why(scan(u=None), "null pointer")
    why(scan(ldu=7), "pitch")
    why(scan(rows=1 << 31), "too many")
    assert lib.ossm_b200_selective_scan_packed_workspace_bytes(4096, 8, 4, 0, 0) > 0
    why(scan(rows=4096), "workspace")
    assert scan(rows=0, count=0) == 0
    conv = lambda taps, ld=8: lib.ossm_b200_conv1d_silu_packed_forward(p, ld, p, None, p, None, None, 0, None, None, 0, p, 8, 1,
                                                                       4, 1, 8, taps, 0, 0, None)
    why(conv(5), "kernel size")
    why(conv(0), "kernel size")
    why(conv(4, 7), "pitch")
    why(lib.ossm_b200_conv1d_silu_step(p, 8, p, None, None, None, 4, p, 8, 2, 8, 4, 0, 0, None), "null pointer")
    back = lambda rows: lib.ossm_b200_selective_scan_packed_backward(
        p, 8, p, 8, p, 8, p, p, 4, p, 4, None, 0, None, None, 0, p, None, None, p, p, p, p, p, p, None, None, None, None, None, 0,
        rows, 1, 8, 4, 0, 0, None)
    why(back(0), "no rows")
    why(back(4), "workspace")
