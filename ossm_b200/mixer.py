"""Neighbours of the selective scan inside ossm's Mamba mixer, folded into kernels of this library.

``_MambaMixer.forward`` (``src/ossm/models/mambarec.py:136-184``) runs, around the scan,

* ``transpose -> F.pad -> conv1d(groups=D) -> SiLU -> transpose`` on ``x [B, L, D]``: here one kernel
  (:func:`causal_conv1d_silu`) that reads ``x`` once and writes the result both time-contiguous (the scan's
  operand) and channel-contiguous (the ``x_proj`` GEMM's operand);
* ``dt = softplus(dt_proj(dt_raw))`` as a separate pass over ``[B, D, L]``: here the scan takes the projection
  without its bias, the bias as ``delta_bias`` and ``delta_softplus=True``.

:func:`mamba_mixer_forward` is the mixer's forward written with those two; ``install_as_ossm_kernels(
fuse_mixer=True)`` puts it behind the unmodified ``_MambaMixer`` class (same parameters, same state dict).

:func:`mamba_mixer_packed` runs the same mixer over sequences of different lengths that lie back to back, without padding,
and :func:`mamba_mixer_step` over one token of each: with a :class:`MambaCache` the sequences' convolution windows and scan
states stay on the device between calls, so that a new item costs one step and not the whole history again.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
import torch.nn.functional as F
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib, packed
from .kernels import _p, _require_cuda, _stream

__all__ = ["causal_conv1d_silu", "causal_conv1d_silu_packed", "causal_conv1d_silu_step", "mamba_mixer_forward",
           "mamba_mixer_packed", "mamba_mixer_step", "MambaCache", "MAX_TAPS"]

MAX_TAPS = 4


def _row_pitch(x: Tensor) -> int:
    """``x [B, L, D]`` with contiguous channels and rows ``ldx`` floats apart (a dense tensor or the first /
    second half of a ``[B, L, 2D]`` one); raises otherwise."""
    B, L, D = x.shape
    if x.stride(2) != 1 or (L > 1 and x.stride(0) != L * x.stride(1)) or x.stride(1) < D:
        raise RuntimeError("ossm_b200: causal_conv1d_silu needs x [B, L, D] with contiguous channels and evenly spaced rows")
    return int(x.stride(1))


class _ConvSiluFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: Tensor, weight: Tensor, bias: Optional[Tensor]) -> Tuple[Tensor, Tensor]:
        B, L, D = x.shape
        taps = weight.size(-1)
        w2 = weight.reshape(D, taps).contiguous()
        b1 = bias.contiguous() if bias is not None else None
        ldx = _row_pitch(x)
        out_bdl = torch.empty((B, D, L), dtype=torch.float32, device=x.device)
        out_bld = torch.empty((B, L, D), dtype=torch.float32, device=x.device)
        with torch.cuda.device(x.device):
            rc = _lib.load().ossm_b200_conv1d_silu_forward(_p(x), ldx, _p(w2), _p(b1), _p(out_bdl), _p(out_bld), B, L, D,
                                                           taps, _stream(x.device))
        _lib.check(rc, "conv1d_silu_forward")
        ctx.save_for_backward(x, w2, b1 if b1 is not None else x.new_empty(0))
        ctx.has_bias = bias is not None
        ctx.weight_shape = tuple(weight.shape)
        return out_bdl, out_bld

    @staticmethod
    def backward(ctx, g_bdl: Optional[Tensor], g_bld: Optional[Tensor]):
        x, w2, b1 = ctx.saved_tensors
        bias = b1 if ctx.has_bias else None
        B, L, D = x.shape
        taps = w2.size(1)
        g1 = g_bdl.contiguous() if g_bdl is not None else None
        g2 = g_bld.contiguous() if g_bld is not None else None
        grad_x = torch.empty((B, L, D), dtype=torch.float32, device=x.device)
        grad_w = torch.empty_like(w2)
        grad_b = torch.empty(D, dtype=torch.float32, device=x.device) if bias is not None else None
        if g1 is None and g2 is None:
            return torch.zeros_like(grad_x), torch.zeros(ctx.weight_shape, device=x.device), (
                torch.zeros_like(grad_b) if grad_b is not None else None)
        with torch.cuda.device(x.device):
            rc = _lib.load().ossm_b200_conv1d_silu_backward(_p(x), _row_pitch(x), _p(w2), _p(bias), _p(g1), _p(g2),
                                                            _p(grad_x), _p(grad_w), _p(grad_b), B, L, D, taps,
                                                            _stream(x.device))
        _lib.check(rc, "conv1d_silu_backward")
        return grad_x, grad_w.view(ctx.weight_shape), grad_b


def causal_conv1d_silu(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """``silu(conv1d(left-padded x^T) + bias)`` for ``x [B, L, D]`` float32 (channels contiguous, rows evenly
    spaced), ``weight [D, 1, K]`` or ``[D, K]`` (``K <= 4``), ``bias [D]``.  Returns the result as ``[B, D, L]``
    and as ``[B, L, D]``."""
    _require_cuda("x", x)
    if x.dim() != 3 or x.dtype != torch.float32:
        raise RuntimeError("ossm_b200: causal_conv1d_silu needs a float32 [B, L, D] tensor")
    D = x.size(2)
    if weight.numel() % max(D, 1) or weight.size(0) != D or weight.size(-1) > MAX_TAPS or weight.dtype != torch.float32:
        raise RuntimeError(f"ossm_b200: conv weight must be float32 [D, 1, K] with K <= {MAX_TAPS}")
    if bias is not None and (bias.shape != (D,) or bias.dtype != torch.float32):
        raise RuntimeError("ossm_b200: conv bias must be float32 [D]")
    if x.numel() == 0:
        return x.new_zeros(x.size(0), D, x.size(1)), x.new_zeros(x.shape)
    return _ConvSiluFn.apply(x, weight, bias)


class _ConvSiluPackedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: Tensor, weight: Tensor, bias: Optional[Tensor], initial_window: Optional[Tensor], offsets: Tensor,
                want_window: bool):
        w, b, taps = packed.check_conv(x, weight, bias)
        seq = packed.sequences(offsets, x.device, resume=True)
        start = initial_window.contiguous() if initial_window is not None else None
        end = torch.empty((seq.count, taps - 1, x.size(1)), dtype=x.dtype, device=x.device) if want_window else None
        out = packed.conv_forward(x, w, b, seq, start, end, None)
        ctx.save_for_backward(x, w, b, start, seq.offsets)
        ctx.weight_shape = tuple(weight.shape)
        ctx.set_materialize_grads(False)
        return out, end

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out: Optional[Tensor], grad_end: Optional[Tensor]):
        x, w, b, start, offsets = ctx.saved_tensors
        seq = packed.sequences(offsets, x.device, resume=True)
        grad_out = torch.zeros_like(x) if grad_out is None else grad_out.to(x.dtype)
        grad_end = None if grad_end is None else grad_end.to(x.dtype).contiguous()
        gx, gw, gb, gs = packed.conv_backward(grad_out, x, w, b, seq, start, grad_end)
        return gx, gw.view(ctx.weight_shape), gb, gs, None, None


def causal_conv1d_silu_packed(x: Tensor, weight: Tensor, bias: Optional[Tensor], offsets: Tensor, *,
                              initial_window: Optional[Tensor] = None, return_window: bool = False,
                              cache: Optional[Tensor] = None, slots: Optional[Tensor] = None,
                              resume: Union[bool, Tensor, None] = None,
                              out: Optional[Tensor] = None) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """:func:`causal_conv1d_silu` over sequences that lie back to back: ``x [T, D]`` (float32 or bfloat16, contiguous
    channels, any row pitch), sequence ``i`` in the rows ``offsets[i] .. offsets[i + 1] - 1``; the result is ``[T, D]``.
    ``weight [D, 1, K]`` or ``[D, K]`` (``K <= 4``) and ``bias [D]`` have the dtype of ``x`` or float32.

    The ``K - 1`` inputs before a sequence are its window, oldest first (zeros by default).  *Training*:
    ``initial_window [S, K - 1, D]``, and ``return_window=True`` for ``(out, windows behind the sequences)``; everything is
    differentiable.  *Prompts*: ``cache [entries, K - 1, D]`` with ``slots``, ``resume`` and ``out`` as in
    :func:`ossm_b200.selective_scan.selective_scan_packed`; updated in place, not differentiable."""
    w, b, taps = packed.check_conv(x, weight, bias)
    shape = (taps - 1, x.size(1))
    if cache is None:
        if slots is not None or resume is not None:
            raise RuntimeError("ossm_b200: slots and resume go with a cache")
        if out is not None:
            raise RuntimeError("ossm_b200: out goes with a cache; the differentiable form allocates its result")
        offsets = packed._index("offsets", offsets, x.device)
        if initial_window is not None and (tuple(initial_window.shape) != (offsets.size(0) - 1, *shape)
                                           or initial_window.dtype != x.dtype or initial_window.device != x.device):
            raise RuntimeError(f"initial_window must have shape {(offsets.size(0) - 1, *shape)}, the dtype and the device of x")
        res, end = _ConvSiluPackedFn.apply(x, weight, bias, initial_window, offsets, bool(return_window))
        return (res, end) if return_window else res
    if initial_window is not None or return_window:
        raise RuntimeError("ossm_b200: initial_window / return_window and cache exclude each other")
    packed.refuse_grad("causal_conv1d_silu_packed with a cache", x, weight, bias, cache, out)
    seq = packed.sequences(offsets, x.device, slots, resume)
    packed._check_cache("cache", cache, shape, x.dtype, x.device, seq.count, slots)
    packed._check_out(out, x, x, weight, bias, cache)
    return packed.conv_forward(x, w, b, seq, cache, cache, out)


def causal_conv1d_silu_step(x: Tensor, weight: Tensor, bias: Optional[Tensor], cache: Tensor, *,
                            slots: Optional[Tensor] = None, out: Optional[Tensor] = None) -> Tensor:
    """One token of each sequence, ``x [S, D]``, against its window in ``cache [entries, K - 1, D]`` (updated in place): row
    ``i`` uses entry ``slots[i]`` (int32, default ``i``; negative: a row of padding with an empty window).  The slots must
    differ.  Types as in :func:`causal_conv1d_silu_packed`."""
    w, b, taps = packed.check_conv(x, weight, bias)
    packed.refuse_grad("causal_conv1d_silu_step", x, weight, bias, cache, out)
    packed._check_cache("cache", cache, (taps - 1, x.size(1)), x.dtype, x.device, x.size(0), slots)
    packed._check_out(out, x, x, weight, bias, cache)
    if slots is not None:
        slots = packed._index("slots", slots, x.device, x.size(0))
    return packed.conv_step(x, w, b, slots, cache, out)


def mamba_mixer_forward(mixer, inputs: Tensor) -> Tensor:
    """Forward of ossm's ``_MambaMixer`` (``mambarec.py:136-184``) on its own parameters with the conv + SiLU
    kernel and the step transform folded into the scan.  ``inputs [B, L, d_model]`` on a CUDA device."""
    from .selective_scan import selective_scan

    if inputs.ndim != 3:
        raise ValueError("Inputs to Mamba mixer must have shape (batch, length, channels)")
    batch, seqlen, _ = inputs.shape
    if seqlen == 0:
        return torch.zeros_like(inputs)
    xz = mixer.in_proj(inputs).float()
    d_inner = mixer.d_inner
    x, z = xz[..., :d_inner], xz[..., d_inner:]
    x_bdl, x_bld = causal_conv1d_silu(x, mixer.conv1d.weight.float(),
                                      mixer.conv1d.bias.float() if mixer.conv1d.bias is not None else None)
    proj = mixer.x_proj(x_bld.to(mixer.x_proj.weight.dtype)).float()
    dt_raw, B_gen, C_gen = torch.split(proj, [mixer.dt_rank, mixer.d_state, mixer.d_state], dim=-1)
    # dt_proj without its bias, produced time-contiguous [B, D, L]; bias and softplus happen inside the scan
    dt_bdl = torch.matmul(mixer.dt_proj.weight.float(), dt_raw.transpose(1, 2))
    A = -torch.exp(mixer.A_log.float())
    gated = selective_scan(x_bdl, dt_bdl, A, B_gen, C_gen, z.transpose(1, 2), None,
                           delta_bias=mixer.dt_proj.bias.float(), delta_softplus=True)
    return mixer.out_proj(gated.transpose(1, 2).to(mixer.out_proj.weight.dtype))


class MambaCache:
    """What a mixer has to remember of each sequence: the last ``d_conv - 1`` inputs of its convolution and the state of its
    scan.  ``conv [entries, d_conv - 1, d_inner]`` (dtype of ``in_proj``'s output: the autocast dtype where the cache is made
    inside such a region) and ``ssm [entries, d_inner, d_state]`` (float32), zeros to begin with; a sequence is an entry,
    whose number the caller hands out.  A float32 cache takes bfloat16 projections too (they are widened); a bfloat16 cache
    does not take float32 ones."""

    def __init__(self, mixer, entries: int):
        weight = mixer.in_proj.weight
        dtype = torch.get_autocast_dtype("cuda") if weight.is_cuda and torch.is_autocast_enabled("cuda") else weight.dtype
        self.conv = torch.zeros((entries, mixer.d_conv - 1, mixer.d_inner), dtype=_io_dtype(dtype), device=weight.device)
        self.ssm = torch.zeros((entries, mixer.d_inner, mixer.d_state), dtype=torch.float32, device=weight.device)


def _io_dtype(dtype: torch.dtype) -> torch.dtype:
    return dtype if dtype in (torch.float32, torch.bfloat16) else torch.float32


def _packed_mixer(mixer, inputs: Tensor, conv, scan, window: Optional[torch.dtype] = None) -> Tensor:
    """``window``: dtype of the cached windows, if there are any."""
    xz = mixer.in_proj(inputs)
    io = torch.float32 if window == torch.float32 else _io_dtype(xz.dtype)
    xz = xz.to(io)
    x, z = xz[..., :mixer.d_inner], xz[..., mixer.d_inner:]
    weight, bias = mixer.conv1d.weight, mixer.conv1d.bias
    if weight.dtype not in (io, torch.float32):
        weight, bias = weight.float(), bias.float() if bias is not None else None
    x = conv(x, weight, bias)
    proj = mixer.x_proj(x.to(mixer.x_proj.weight.dtype))
    dt_raw, B, C = torch.split(proj, [mixer.dt_rank, mixer.d_state, mixer.d_state], dim=-1)
    dt = F.linear(dt_raw, mixer.dt_proj.weight)   # its bias and the softplus happen inside the scan
    dt = dt if dt.dtype in (io, torch.float32) else dt.float()
    gated = scan(x, dt, -torch.exp(mixer.A_log.float()), B.to(io), C.to(io), z, mixer.dt_proj.bias.float())
    return mixer.out_proj(gated.to(mixer.out_proj.weight.dtype))


def mamba_mixer_packed(mixer, inputs: Tensor, offsets: Tensor, cache: Optional[MambaCache] = None, *,
                       slots: Optional[Tensor] = None, resume: Union[bool, Tensor, None] = None) -> Tensor:
    """:func:`mamba_mixer_forward` over ``inputs [T, d_model]``, sequence ``i`` in the rows ``offsets[i] .. offsets[i + 1] - 1``
    (int32 ``[S + 1]`` on the device).  Without a cache every sequence starts afresh and the call is differentiable.  With
    one, sequence ``i`` leaves its window and state in entry ``slots[i]`` (and continues from it where ``resume`` says so:
    a prompt in pieces), and the call runs under ``torch.no_grad()``."""
    from .selective_scan import selective_scan_packed

    if inputs.ndim != 2:
        raise ValueError("Packed inputs to the Mamba mixer must have shape (rows, channels)")
    if cache is None:
        if slots is not None or resume is not None:
            raise RuntimeError("ossm_b200: slots and resume go with a cache")
        return _packed_mixer(mixer, inputs, lambda x, w, b: causal_conv1d_silu_packed(x, w, b, offsets),
                             lambda x, dt, A, B, C, z, bias: selective_scan_packed(
                                 x, dt, A, B, C, offsets, z, delta_bias=bias, delta_softplus=True))
    packed.refuse_grad("mamba_mixer_packed with a cache", inputs)
    with torch.no_grad():
        return _packed_mixer(
            mixer, inputs,
            lambda x, w, b: causal_conv1d_silu_packed(x, w, b, offsets, cache=cache.conv, slots=slots, resume=resume),
            lambda x, dt, A, B, C, z, bias: selective_scan_packed(
                x, dt, A, B, C, offsets, z, delta_bias=bias, delta_softplus=True, cache=cache.ssm, slots=slots, resume=resume),
            cache.conv.dtype)


def mamba_mixer_step(mixer, inputs: Tensor, cache: MambaCache, *, slots: Optional[Tensor] = None) -> Tensor:
    """One token of each sequence, ``inputs [S, d_model]``: the output the mixer gives at that token after everything that
    entry ``slots[i]`` has seen (int32, default ``i``; negative: a row of padding).  Runs under ``torch.no_grad()``; all its
    work is on the device, so that a step can be captured into a CUDA graph."""
    from .selective_scan import selective_scan_step

    if inputs.ndim != 2:
        raise ValueError("Inputs to a step of the Mamba mixer must have shape (sequences, channels)")
    packed.refuse_grad("mamba_mixer_step", inputs)
    with torch.no_grad():
        return _packed_mixer(
            mixer, inputs, lambda x, w, b: causal_conv1d_silu_step(x, w, b, cache.conv, slots=slots),
            lambda x, dt, A, B, C, z, bias: selective_scan_step(x, dt, A, B, C, cache.ssm, z, delta_bias=bias,
                                                                delta_softplus=True, slots=slots), cache.conv.dtype)
