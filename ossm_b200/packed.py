"""Packed batches and single tokens of the Mamba mixer: checked calls into the C ABI.

Sequences of different lengths lie back to back in ``[rows, channels]`` tensors; ``offsets`` (int32 ``[S + 1]`` on the
device) says which rows are whose, so that no length has to be known on the host.  The differentiable and documented
entry points are :func:`ossm_b200.selective_scan.selective_scan_packed`, :func:`~ossm_b200.selective_scan.selective_scan_step`,
:func:`ossm_b200.mixer.causal_conv1d_silu_packed` and :func:`~ossm_b200.mixer.causal_conv1d_silu_step`.
"""
from __future__ import annotations

import contextlib
import functools
from typing import NamedTuple, Optional, Tuple, Union

import torch
from torch import Tensor

from . import _lib
from .kernels import _IO_DTYPES, _require_cuda

_SAME_DEVICE = contextlib.nullcontext()
MAX_STATE = 256


def _ptr(t: Optional[Tensor]):
    return None if t is None else t.data_ptr()


def _on(device):
    """The device of the operands around a call; nothing to do where it is the current one."""
    return _SAME_DEVICE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _stream(device) -> int:
    """The current stream's handle, without the Stream object around it (a step of one token is mostly host time)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


@functools.lru_cache(maxsize=256)
def _scan_workspace(backward: bool, rows: int, ch: int, n: int, io: int, dt: int, device: int) -> int:
    """Workspace bytes, asked for on the device of the operands; they depend on nothing but these sizes."""
    lib = _lib.load()
    ask = (lib.ossm_b200_selective_scan_packed_backward_workspace_bytes if backward
           else lib.ossm_b200_selective_scan_packed_workspace_bytes)
    return int(ask(rows, ch, n, io, dt))


def _rows(t: Tensor) -> Tuple[Tensor, int]:
    """``t [rows, C]`` with contiguous channels and a row pitch: as it is (a column slice of a wider tensor too), else copied."""
    (rows, width), (pitch, step) = t.shape, t.stride()
    if (step == 1 or width <= 1) and (pitch >= width or rows <= 1):
        return t, (pitch if rows > 1 else max(width, 1))
    return t.contiguous(), max(width, 1)


class Sequences(NamedTuple):
    """Where the sequences of a packed batch lie, and which entries of a cache are theirs."""
    offsets: Tensor
    slots: Optional[Tensor]
    resume: Optional[Tensor]
    resume_all: int
    count: int


def _index(name: str, t: Tensor, device, count: Optional[int] = None) -> Tensor:
    if not torch.is_tensor(t) or t.dim() != 1 or t.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"ossm_b200: {name} must be a 1-D int32 (or int64) tensor")
    if t.device != device:
        raise RuntimeError(f"ossm_b200: {name} must be on the device of the inputs")
    if count is not None and t.size(0) != count:
        raise RuntimeError(f"ossm_b200: {name} must have one entry for each sequence ({count})")
    if t.dtype == torch.int64:      # what does not fit 32 bits stays out of range
        t = t.clamp(-1, 2 ** 31 - 1).to(torch.int32)
    return t.contiguous()


def sequences(offsets: Tensor, device, slots: Optional[Tensor] = None,
              resume: Union[bool, Tensor, None] = None) -> Sequences:
    offsets = _index("offsets", offsets, device)
    count = offsets.size(0) - 1
    if count < 0:
        raise RuntimeError("ossm_b200: offsets must have one entry more than there are sequences")
    if slots is not None:
        slots = _index("slots", slots, device, count)
    flags, every = None, 0
    if torch.is_tensor(resume):
        if resume.shape != (count,) or resume.dtype not in (torch.bool, torch.uint8) or resume.device != device:
            raise RuntimeError("ossm_b200: resume must be a bool, or a bool tensor with one entry for each sequence on "
                               "the device of the inputs")
        flags = resume.contiguous()
    else:
        every = int(bool(resume))
    return Sequences(offsets, slots, flags, every, count)


def _check_out(out: Optional[Tensor], like: Tensor, *inputs: Optional[Tensor]) -> None:
    if out is None:
        return
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device:
        raise RuntimeError("ossm_b200: out must have the shape, dtype and device of the inputs")
    if out.numel() and ((out.size(1) > 1 and out.stride(1) != 1) or (out.size(0) > 1 and out.stride(0) < out.size(1))):
        raise RuntimeError("ossm_b200: out needs contiguous channels and rows that do not overlap")
    memory = out.untyped_storage().data_ptr()
    if out.numel() and any(t is not None and t.untyped_storage().data_ptr() == memory for t in inputs):
        raise RuntimeError("ossm_b200: out must not share memory with an input")


def _out_pitch(out: Tensor) -> int:
    return out.stride(0) if out.size(0) > 1 else max(out.size(1), 1)


def _check_cache(name: str, cache: Tensor, shape: Tuple[int, ...], dtype, device, count: int, slots: Optional[Tensor]) -> None:
    if (cache.dim() != 3 or cache.shape[1:] != shape or cache.dtype != dtype or cache.device != device
            or not cache.is_contiguous()):
        raise RuntimeError(f"ossm_b200: {name} must be a contiguous {dtype} tensor [entries, {shape[0]}, {shape[1]}] on the "
                           "device of the inputs")
    if slots is None and cache.size(0) < count and 0 not in shape:
        raise RuntimeError(f"ossm_b200: {name} has {cache.size(0)} entries for {count} sequences: without slots each needs its own")


def refuse_grad(what: str, *tensors: Optional[Tensor]) -> None:
    if not torch.is_grad_enabled():
        return
    for t in tensors:
        if t is not None and t.requires_grad:
            raise RuntimeError(f"ossm_b200: {what} is not differentiable: call it under torch.no_grad() or on detached tensors")


def written(*tensors: Optional[Tensor]) -> None:
    """Tells autograd that a kernel changed these: a graph that kept one for its backward pass must not use it any more."""
    for t in tensors:
        if t is not None and not t.is_inference():
            torch.autograd.graph.increment_version(t)


# ---- convolution -------------------------------------------------------------------------------------
def check_conv(x: Tensor, weight: Tensor, bias: Optional[Tensor]) -> Tuple[Tensor, Optional[Tensor], int]:
    """``(weight [D, K], bias, K)`` as handed to the library."""
    if x.dim() != 2 or x.dtype not in _IO_DTYPES:
        raise RuntimeError("ossm_b200: x must be a float32 or bfloat16 [rows, channels] tensor")
    _require_cuda("x", x)
    D = x.size(1)
    if (weight.dim() not in (2, 3) or weight.size(0) != D or (weight.dim() == 3 and weight.size(1) != 1)
            or not 1 <= weight.size(-1) <= 4):
        raise RuntimeError("ossm_b200: conv weight must be [D, 1, K] or [D, K] with K <= 4")
    if weight.dtype not in (x.dtype, torch.float32) or weight.device != x.device:
        raise RuntimeError("ossm_b200: conv weight must be float32 or of the dtype of x, on its device")
    if bias is not None and (bias.shape != (D,) or bias.dtype != weight.dtype or bias.device != x.device):
        raise RuntimeError("ossm_b200: conv bias must be [D] with the dtype and device of the weight")
    taps = weight.size(-1)
    if not weight.is_contiguous():
        weight = weight.contiguous()
    return (weight if weight.dim() == 2 else weight.view(D, taps)), (bias.contiguous() if bias is not None else None), taps


def conv_forward(x: Tensor, weight: Tensor, bias: Optional[Tensor], seq: Sequences, start: Optional[Tensor],
                 end: Optional[Tensor], out: Optional[Tensor]) -> Tensor:
    """``weight [D, K]``, ``start`` / ``end [entries, K - 1, D]`` as described for the C entry."""
    rows, D = x.shape
    taps = weight.size(1)
    state = end if end is not None else start
    xr, ldx = _rows(x)
    fresh = out is None
    if fresh:
        out = torch.empty((rows, D), dtype=x.dtype, device=x.device)
    with _on(x.device):
        rc = _lib.load().ossm_b200_conv1d_silu_packed_forward(
            xr.data_ptr(), ldx, weight.data_ptr(), _ptr(bias), seq.offsets.data_ptr(), _ptr(seq.slots), _ptr(seq.resume),
            seq.resume_all, _ptr(start), _ptr(end), state.size(0) if state is not None else 0, out.data_ptr(),
            _out_pitch(out), int(fresh), rows, seq.count, D, taps, _IO_DTYPES[x.dtype], _IO_DTYPES[weight.dtype],
            _stream(x.device))
    _lib.check(rc, "conv1d_silu_packed_forward")
    if end is not None and end is start:
        written(end, None if fresh else out)
    return out


def conv_step(x: Tensor, weight: Tensor, bias: Optional[Tensor], slots: Optional[Tensor], cache: Tensor,
              out: Optional[Tensor]) -> Tensor:
    count, D = x.shape
    xr, ldx = _rows(x)
    given = out
    if out is None:
        out = torch.empty((count, D), dtype=x.dtype, device=x.device)
    with _on(x.device):
        rc = _lib.load().ossm_b200_conv1d_silu_step(
            xr.data_ptr(), ldx, weight.data_ptr(), _ptr(bias), _ptr(slots), cache.data_ptr(), cache.size(0),
            out.data_ptr(), _out_pitch(out), count, D, weight.size(1), _IO_DTYPES[x.dtype], _IO_DTYPES[weight.dtype],
            _stream(x.device))
    _lib.check(rc, "conv1d_silu_step")
    written(cache, given)
    return out


def conv_backward(grad: Tensor, x: Tensor, weight: Tensor, bias: Optional[Tensor], seq: Sequences,
                  start: Optional[Tensor], grad_end: Optional[Tensor]):
    """``(grad_x, grad_weight [D, K], grad_bias, grad_start)``; ``start`` / ``grad_start [S, K - 1, D]``."""
    rows, D = x.shape
    taps = weight.size(1)
    dev = x.device
    grad_x = torch.empty((rows, D), dtype=x.dtype, device=dev)
    grad_w = torch.empty_like(weight)
    grad_b = torch.empty_like(bias) if bias is not None else None
    grad_start = torch.empty_like(start) if start is not None else None
    if rows == 0 or D == 0:
        if grad_start is not None:
            grad_start.zero_() if grad_end is None else grad_start.copy_(grad_end)
        return grad_x, grad_w.zero_(), grad_b.zero_() if grad_b is not None else None, grad_start
    lib = _lib.load()
    io = _IO_DTYPES[x.dtype]
    xr, ldx = _rows(x)
    gr, ldg = _rows(grad)
    with _on(dev):
        ws_bytes = lib.ossm_b200_conv1d_silu_packed_backward_workspace_bytes(rows, D, taps, io)
        workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        rc = lib.ossm_b200_conv1d_silu_packed_backward(
            gr.data_ptr(), ldg, xr.data_ptr(), ldx, weight.data_ptr(), _ptr(bias), seq.offsets.data_ptr(), _ptr(start),
            _ptr(grad_end), grad_x.data_ptr(), grad_w.data_ptr(), _ptr(grad_b), _ptr(grad_start), workspace.data_ptr(),
            ws_bytes, rows, seq.count, D, taps, io, _IO_DTYPES[weight.dtype], _stream(dev))
    _lib.check(rc, "conv1d_silu_packed_backward")
    return grad_x, grad_w, grad_b, grad_start


# ---- selective scan ------------------------------------------------------------------------------------
def check_scan(inputs: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, gate: Optional[Tensor], D: Optional[Tensor],
               delta_bias: Optional[Tensor]) -> None:
    if inputs.dim() != 2:
        raise RuntimeError("inputs must have shape (rows, channels)")
    if dt.shape != inputs.shape:
        raise RuntimeError("dt must match the shape of inputs")
    rows, ch = inputs.shape
    if A.dim() != 2 or A.size(0) != ch:
        raise RuntimeError("A must have shape (channels, state)")
    n = A.size(1)
    if not 1 <= n <= MAX_STATE:
        raise RuntimeError(f"ossm_b200: the state size must be 1..{MAX_STATE}")
    if B.shape != (rows, n) or C.shape != (rows, n):
        raise RuntimeError("B and C must have shape (rows, state)")
    if gate is not None and gate.shape != inputs.shape:
        raise RuntimeError("gate must match the shape of inputs")
    for name, t in (("D", D), ("delta_bias", delta_bias)):
        if t is not None and t.shape != (ch,):
            raise RuntimeError(f"{name} must have shape (channels,)")
    _require_cuda("inputs", inputs)
    if inputs.dtype not in _IO_DTYPES:
        raise RuntimeError("ossm_b200: selective scan supports float32 or bfloat16 inputs")
    io = inputs.dtype
    for name, t in (("B", B), ("C", C), ("gate", gate)):
        if t is not None and t.dtype != io:
            raise RuntimeError(f"ossm_b200: {name} must have the dtype of inputs ({io})")
    if dt.dtype != io and dt.dtype != torch.float32:
        raise RuntimeError(f"ossm_b200: dt must be float32 or have the dtype of inputs ({io})")
    dev = inputs.device
    for t in (dt, A, B, C, gate, D, delta_bias):
        if t is not None and t.device != dev:
            raise RuntimeError("ossm_b200: all selective-scan operands must be on one device")


def _f32(t: Optional[Tensor]) -> Optional[Tensor]:
    if t is None or (t.dtype == torch.float32 and t.is_contiguous()):
        return t
    return t.to(torch.float32).contiguous()


def scan_kept(rows: int, ch: int, n: int, device) -> Tensor:
    """Room for the states entering every tile of rows, which the backward reads."""
    tile = _lib.load().ossm_b200_selective_scan_packed_tile(n)
    return torch.empty(((rows + tile - 1) // tile, ch, n), dtype=torch.float32, device=device)


def scan_forward(inputs: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, gate: Optional[Tensor],
                 D: Optional[Tensor], delta_bias: Optional[Tensor], delta_softplus: bool, seq: Sequences,
                 start: Optional[Tensor], end: Optional[Tensor], out: Optional[Tensor],
                 kept: Optional[Tensor] = None) -> Tensor:
    """``A``, ``D``, ``delta_bias`` float32 and contiguous; ``start`` / ``end [entries, channels, state]``."""
    rows, ch = inputs.shape
    n = A.size(1)
    dev = inputs.device
    lib = _lib.load()
    io, step = _IO_DTYPES[inputs.dtype], _IO_DTYPES[dt.dtype]
    state = end if end is not None else start
    fresh = out is None
    if fresh:
        out = torch.empty((rows, ch), dtype=inputs.dtype, device=dev)
    (u, ldu), (d, lddt), (b, ldb), (c, ldc) = _rows(inputs), _rows(dt), _rows(B), _rows(C)
    z, ldz = _rows(gate) if gate is not None else (None, 0)
    with _on(dev):
        ws_bytes = _scan_workspace(False, rows, ch, n, io, step, dev.index)
        workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
        rc = lib.ossm_b200_selective_scan_packed_forward(
            u.data_ptr(), ldu, d.data_ptr(), lddt, A.data_ptr(), b.data_ptr(), ldb, c.data_ptr(), ldc, _ptr(z), ldz,
            _ptr(D), _ptr(delta_bias), int(delta_softplus), seq.offsets.data_ptr(), _ptr(seq.slots), _ptr(seq.resume),
            seq.resume_all, _ptr(start), _ptr(end), state.size(0) if state is not None else 0, out.data_ptr(),
            _out_pitch(out), int(fresh), _ptr(kept), _ptr(workspace), ws_bytes, rows, seq.count, ch, n, io, step, _stream(dev))
    _lib.check(rc, "selective_scan_packed_forward")
    if end is not None and end is start:
        written(end, None if fresh else out)
    return out


def scan_step(inputs: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, gate: Optional[Tensor], D: Optional[Tensor],
              delta_bias: Optional[Tensor], delta_softplus: bool, slots: Optional[Tensor], cache: Tensor,
              out: Optional[Tensor]) -> Tensor:
    count, ch = inputs.shape
    dev = inputs.device
    given = out
    if out is None:
        out = torch.empty((count, ch), dtype=inputs.dtype, device=dev)
    (u, ldu), (d, lddt), (b, ldb), (c, ldc) = _rows(inputs), _rows(dt), _rows(B), _rows(C)
    z, ldz = _rows(gate) if gate is not None else (None, 0)
    with _on(dev):
        rc = _lib.load().ossm_b200_selective_scan_step(
            u.data_ptr(), ldu, d.data_ptr(), lddt, A.data_ptr(), b.data_ptr(), ldb, c.data_ptr(), ldc, _ptr(z), ldz,
            _ptr(D), _ptr(delta_bias), int(delta_softplus), _ptr(slots), cache.data_ptr(), cache.size(0), out.data_ptr(),
            _out_pitch(out), count, ch, A.size(1), _IO_DTYPES[inputs.dtype], _IO_DTYPES[dt.dtype], _stream(dev))
    _lib.check(rc, "selective_scan_step")
    written(cache, given)
    return out


def scan_backward(grad: Tensor, inputs: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, gate: Optional[Tensor],
                  D: Optional[Tensor], delta_bias: Optional[Tensor], delta_softplus: bool, seq: Sequences,
                  start: Optional[Tensor], grad_end: Optional[Tensor], kept: Tensor):
    """``(du, ddt, dA, dB, dC, dgate, dD, dbias, dstart)``, ``None`` for what is absent."""
    rows, ch = inputs.shape
    n = A.size(1)
    dev = inputs.device

    def like(t, shape=None):
        return None if t is None else torch.empty(shape or t.shape, dtype=t.dtype, device=dev)

    du, ddt, dA, dB, dC = like(inputs), like(dt), like(A), like(B), like(C)
    dz, dD, dbias, dstart = like(gate), like(D), like(delta_bias), like(start)
    if rows == 0 or ch == 0:
        if dstart is not None:
            dstart.zero_() if grad_end is None else dstart.copy_(grad_end)
        for t in (dA, dD, dbias):
            if t is not None:
                t.zero_()
        return du, ddt, dA, dB, dC, dz, dD, dbias, dstart
    lib = _lib.load()
    io, step = _IO_DTYPES[inputs.dtype], _IO_DTYPES[dt.dtype]
    (g, ldg), (u, ldu), (d, lddt), (b, ldb), (c, ldc) = _rows(grad), _rows(inputs), _rows(dt), _rows(B), _rows(C)
    z, ldz = _rows(gate) if gate is not None else (None, 0)
    with _on(dev):
        ws_bytes = _scan_workspace(True, rows, ch, n, io, step, dev.index)
        workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        rc = lib.ossm_b200_selective_scan_packed_backward(
            g.data_ptr(), ldg, u.data_ptr(), ldu, d.data_ptr(), lddt, A.data_ptr(), b.data_ptr(), ldb, c.data_ptr(), ldc,
            _ptr(z), ldz, _ptr(D), _ptr(delta_bias), int(delta_softplus), seq.offsets.data_ptr(), _ptr(start),
            _ptr(grad_end), kept.data_ptr(), du.data_ptr(), ddt.data_ptr(), dA.data_ptr(), dB.data_ptr(), dC.data_ptr(),
            _ptr(dz), _ptr(dD), _ptr(dbias), _ptr(dstart), workspace.data_ptr(), ws_bytes, rows, seq.count, ch, n, io, step,
            _stream(dev))
    _lib.check(rc, "selective_scan_packed_backward")
    return du, ddt, dA, dB, dC, dz, dD, dbias, dstart
