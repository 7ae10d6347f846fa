"""Mamba selective scan with ossm's signature:
``try_selective_scan(inputs, dt, A, B, C, gate)`` (``src/ossm/models/_selective_scan.py:127-196``)
and the autograd bridge ``_SelectiveScanFn`` (:199-297).

Differences from the reference, on purpose: bfloat16 ``inputs/B/C/gate`` are
accepted (state arithmetic stays float32) where the reference returns ``None``
for anything but float32; an optional skip vector ``D`` is supported; the
backward recomputes the ungated output instead of saving it; errors raise
instead of returning ``None``.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import kernels, packed

__all__ = ["try_selective_scan", "selective_scan", "selective_scan_packed", "selective_scan_step", "SelectiveScanFn",
           "SelectiveScanPackedFn", "has_kernels"]


def has_kernels() -> bool:
    try:
        from . import _lib

        _lib.load()
        return True
    except (RuntimeError, OSError):
        return False


class SelectiveScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, inputs: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, gate: Optional[Tensor],
                D: Optional[Tensor], delta_bias: Optional[Tensor] = None, delta_softplus: bool = False) -> Tensor:
        needs_grad = any(ctx.needs_input_grad)
        out, states = kernels.selective_scan_fwd(inputs, dt, A, B, C, gate, D, save_states=needs_grad,
                                                 delta_bias=delta_bias, delta_softplus=delta_softplus)
        ctx.has_gate = gate is not None
        ctx.has_skip = D is not None
        ctx.has_bias = delta_bias is not None
        ctx.delta_softplus = bool(delta_softplus)
        if needs_grad:
            none = inputs.new_empty(0)
            ctx.save_for_backward(inputs, dt, A, B, C, gate if gate is not None else none,
                                  D if D is not None else none, delta_bias if delta_bias is not None else none,
                                  states)
        return out

    @staticmethod
    def backward(ctx, grad_output: Tensor):
        inputs, dt, A, B, C, gate, D, bias, states = ctx.saved_tensors
        res = kernels.selective_scan_bwd(
            grad_output, inputs, dt, A, B, C, gate if ctx.has_gate else None, states, D if ctx.has_skip else None,
            delta_bias=bias if ctx.has_bias else None, delta_softplus=ctx.delta_softplus)
        du, ddt, dA, dB, dC, dz, dD = res[:7]
        dbias = res[7] if len(res) > 7 else None
        return du, ddt, dA, dB, dC, dz, dD, dbias, None


def selective_scan(inputs: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, gate: Optional[Tensor] = None,
                   D: Optional[Tensor] = None, delta_bias: Optional[Tensor] = None,
                   delta_softplus: bool = False) -> Tensor:
    """``out[b,d,t] = (sum_n C[b,t,n] h[b,d,t,n] + D[d] u) * silu(gate)`` with
    ``h_t = exp(dt A) h_{t-1} + dt B u``.  Shapes: ``inputs, dt, gate [B,D,L]``, ``A [D,N]``,
    ``B, C [B,L,N]``, ``D [D]``.  ``delta_bias [D]`` / ``delta_softplus`` fold the mixer's
    ``softplus(dt_proj(.))`` (``mambarec.py:155``) into the scan: pass the projection without its bias
    as ``dt`` and the bias here, and the separate softplus pass over ``[B,D,L]`` disappears."""
    if inputs.numel() == 0:
        return inputs
    return SelectiveScanFn.apply(inputs, dt, A, B, C, gate, D, delta_bias, delta_softplus)


def try_selective_scan(inputs: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor,
                       gate: Optional[Tensor]) -> Optional[Tensor]:
    """Drop-in for ``ossm.models._selective_scan.try_selective_scan``."""
    return selective_scan(inputs, dt, A, B, C, gate)


class SelectiveScanPackedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, inputs: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, gate: Optional[Tensor],
                D: Optional[Tensor], delta_bias: Optional[Tensor], initial_state: Optional[Tensor], offsets: Tensor,
                delta_softplus: bool, want_state: bool, grad_enabled: bool = True):
        seq = packed.sequences(offsets, inputs.device, resume=True)
        Af, Df, bf = packed._f32(A), packed._f32(D), packed._f32(delta_bias)
        start = packed._f32(initial_state)
        rows, ch = inputs.shape
        n = A.size(1)
        end = torch.empty((seq.count, ch, n), dtype=torch.float32, device=inputs.device) if want_state else None
        # an operand that requires a gradient looks the same in here whether gradients are on or off: the caller says which
        kept = packed.scan_kept(rows, ch, n, inputs.device) if grad_enabled and any(ctx.needs_input_grad) else None
        out = packed.scan_forward(inputs, dt, Af, B, C, gate, Df, bf, delta_softplus, seq, start, end, None, kept)
        if kept is not None:
            ctx.save_for_backward(inputs, dt, Af, B, C, gate, Df, bf, start, seq.offsets, kept)
            ctx.delta_softplus = delta_softplus
            ctx.dtypes = tuple(None if t is None else t.dtype for t in (A, D, delta_bias, initial_state))
        ctx.set_materialize_grads(False)
        return out, end

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out: Optional[Tensor], grad_end: Optional[Tensor]):
        inputs, dt, A, B, C, gate, D, bias, start, offsets, kept = ctx.saved_tensors
        seq = packed.sequences(offsets, inputs.device, resume=True)
        grad_out = torch.zeros_like(inputs) if grad_out is None else grad_out.to(inputs.dtype)
        grad_end = None if grad_end is None else grad_end.float().contiguous()
        du, ddt, dA, dB, dC, dz, dD, dbias, dstart = packed.scan_backward(
            grad_out, inputs, dt, A, B, C, gate, D, bias, ctx.delta_softplus, seq, start, grad_end, kept)
        cast = [None if t is None else t.to(to) for t, to in zip((dA, dD, dbias, dstart), ctx.dtypes)]
        return du, ddt, cast[0], dB, dC, dz, cast[1], cast[2], cast[3], None, None, None, None


def selective_scan_packed(inputs: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, offsets: Tensor,
                          gate: Optional[Tensor] = None, D: Optional[Tensor] = None, *,
                          delta_bias: Optional[Tensor] = None, delta_softplus: bool = False,
                          initial_state: Optional[Tensor] = None, return_state: bool = False,
                          cache: Optional[Tensor] = None, slots: Optional[Tensor] = None,
                          resume: Union[bool, Tensor, None] = None,
                          out: Optional[Tensor] = None) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """:func:`selective_scan` over sequences of different lengths that lie back to back.

    ``inputs, dt, gate [T, channels]`` and ``B, C [T, state]`` hold the rows of all sequences, channels contiguous, any
    row pitch (the column slices of the mixer's projections are read where they lie); sequence ``i`` has the rows
    ``offsets[i] .. offsets[i + 1] - 1`` (int32 ``[S + 1]`` on the device; it may have none).  ``A [channels, state]``,
    ``D`` and ``delta_bias [channels]`` as there.  float32 or bfloat16; ``dt`` of the inputs' dtype or float32; states are
    float32.  Rows outside every sequence are not read, and the output is zero there (left alone in ``out``).

    *Training*: every operand is differentiable.  ``initial_state [S, channels, state]`` (default: zeros) precedes the
    sequences; with ``return_state=True`` the result is ``(out, states behind the sequences)``.

    *Prompts*: ``cache [entries, channels, state]`` holds the states instead and is updated in place: sequence ``i`` uses
    entry ``slots[i]`` (default ``i``, and then ``entries >= S``; negative: starts from zeros and keeps nothing).  ``resume``
    (bool, or bool ``[S]`` on the device; default False) says which sequences continue from their entry; the others start
    from zeros.  The slots must differ.  This form is not differentiable.  ``out [T, channels]`` takes the result, if given.

    Offsets and slots are on the device and cannot be checked here: wrong ones are held inside the tensors and reported
    by ``ossm_b200._lib.device_status()``.
    """
    packed.check_scan(inputs, dt, A, B, C, gate, D, delta_bias)
    if cache is None:
        if slots is not None or resume is not None:
            raise RuntimeError("ossm_b200: slots and resume go with a cache")
        if out is not None:
            raise RuntimeError("ossm_b200: out goes with a cache; the differentiable form allocates its result")
        offsets = packed._index("offsets", offsets, inputs.device)
        if initial_state is not None:
            shape = (offsets.size(0) - 1, inputs.size(1), A.size(1))
            if tuple(initial_state.shape) != shape or initial_state.device != inputs.device:
                raise RuntimeError(f"initial_state must have shape {shape} on the device of inputs")
        res, end = SelectiveScanPackedFn.apply(inputs, dt, A, B, C, gate, D, delta_bias, initial_state, offsets,
                                               bool(delta_softplus), bool(return_state), torch.is_grad_enabled())
        return (res, end) if return_state else res
    if initial_state is not None or return_state:
        raise RuntimeError("ossm_b200: initial_state / return_state and cache exclude each other")
    packed.refuse_grad("selective_scan_packed with a cache", inputs, dt, A, B, C, gate, D, delta_bias, cache, out)
    seq = packed.sequences(offsets, inputs.device, slots, resume)
    packed._check_cache("cache", cache, (inputs.size(1), A.size(1)), torch.float32, inputs.device, seq.count, slots)
    packed._check_out(out, inputs, inputs, dt, A, B, C, gate, D, delta_bias, cache)
    return packed.scan_forward(inputs, dt, packed._f32(A), B, C, gate, packed._f32(D), packed._f32(delta_bias),
                               bool(delta_softplus), seq, cache, cache, out)


def selective_scan_step(inputs: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, cache: Tensor,
                        gate: Optional[Tensor] = None, D: Optional[Tensor] = None, *,
                        delta_bias: Optional[Tensor] = None, delta_softplus: bool = False,
                        slots: Optional[Tensor] = None, out: Optional[Tensor] = None) -> Tensor:
    """One token of each sequence: ``h = exp(dt A) h + dt u B`` in ``cache [entries, channels, state]`` (float32, updated in
    place) and ``out = (C . h + D u) silu(gate)``.  Row ``i`` of ``inputs, dt, gate [S, channels]`` and ``B, C [S, state]``
    uses entry ``slots[i]`` (int32, default ``i``; negative: a row of padding, which starts from zeros and keeps nothing).
    The slots must differ.  Types, strides and the step transform as in :func:`selective_scan_packed`."""
    packed.check_scan(inputs, dt, A, B, C, gate, D, delta_bias)
    packed.refuse_grad("selective_scan_step", inputs, dt, A, B, C, gate, D, delta_bias, cache, out)
    packed._check_cache("cache", cache, (inputs.size(1), A.size(1)), torch.float32, inputs.device, inputs.size(0), slots)
    packed._check_out(out, inputs, inputs, dt, A, B, C, gate, D, delta_bias, cache)
    if slots is not None:
        slots = packed._index("slots", slots, inputs.device, inputs.size(0))
    return packed.scan_step(inputs, dt, packed._f32(A), B, C, gate, packed._f32(D), packed._f32(delta_bias),
                            bool(delta_softplus), slots, cache, out)
