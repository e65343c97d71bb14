"""A gated linear recurrence along packed sequences.

Per channel, ``h_t = (1 - a_t) h_{t-1} + a_t x_t`` with ``a_t =
sigmoid(gate_t)``: the "over" recurrence of alpha compositing with a learned
opacity, walked along a refiner's tokens. It carries context over the whole
sequence at a cost linear in its length.

:func:`gated_scan` runs whole sequences (differentiable), :func:`gated_scan_step`
one new token of each of a batch of streams.
"""

from __future__ import annotations

import ctypes

import torch

from . import native
from .sequences import (PackedSequences, address, call, changed_in_place, check_cuda,
                        check_packed, check_tokens, element_type, tile_arguments)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` itself where its channels are contiguous, else a copy."""
    return t if t.stride(-1) == 1 and t.stride(0) >= 0 else t.contiguous()


def _check_pair(what, x, gate, rows_name):
    if x.dim() != 2 or x.shape != gate.shape or x.shape[1] < 1:
        raise ValueError(f"{what}: expected x and gate [{rows_name}, channels], got "
                         f"{tuple(x.shape)} and {tuple(gate.shape)}")
    if x.dtype != gate.dtype:
        raise ValueError(f"{what}: x is {x.dtype}, gate is {gate.dtype}")
    return element_type(x.dtype, what)


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, initial, packed, dtype):
        x, gate = _rows(x), _rows(gate)
        if initial is not None:
            initial = initial.contiguous()
        tokens, channels = x.shape
        device = x.device
        layout = tile_arguments(packed, tokens)
        y = x.new_empty((tokens, channels))
        last = x.new_empty((layout["sequences"], channels), dtype=torch.float32)
        entering = x.new_empty((layout["num_tiles"], channels), dtype=torch.float32)
        args = native.GatedScanArgs(
            tokens=tokens, **layout, channels=channels, dtype=dtype, x=address(x),
            gate=address(gate), x_stride=x.stride(0), gate_stride=gate.stride(0), initial=address(initial),
            y=address(y), last=address(last), entering=address(entering))
        lib = native.lib()
        size = lib.gs_gated_scan_workspace_size(ctypes.byref(args))
        workspace = x.new_empty((size,), dtype=torch.uint8)
        args.workspace, args.workspace_size = address(workspace), size
        call("gs_gated_scan", device, ctypes.byref(args))
        ctx.save_for_backward(x, gate, entering)
        ctx.packed, ctx.args, ctx.size = packed, args, size
        ctx.has_initial = initial is not None
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y, grad_last):
        x, gate, entering = ctx.saved_tensors
        # A saved-tensor hook may have brought back tensors that lie differently.
        x, gate, entering = _rows(x), _rows(gate), entering.contiguous()
        device = x.device
        grad_y = x.new_zeros(x.shape) if grad_y is None \
            else grad_y.contiguous()
        grad_last = None if grad_last is None else grad_last.contiguous()
        grad_x, grad_gate = x.new_empty(x.shape), x.new_empty(x.shape)
        args = native.GatedScanArgs.from_buffer_copy(ctx.args)
        args.x, args.gate, args.entering = address(x), address(gate), address(entering)
        args.x_stride, args.gate_stride = x.stride(0), gate.stride(0)
        args.initial = args.y = args.last = None
        grad_initial = None
        if ctx.has_initial and ctx.needs_input_grad[2]:
            grad_initial = x.new_empty((args.sequences, args.channels), dtype=torch.float32)
        workspace = x.new_empty((ctx.size,), dtype=torch.uint8)
        args.grad_y, args.grad_last = address(grad_y), address(grad_last)
        args.grad_x, args.grad_gate = address(grad_x), address(grad_gate)
        args.grad_initial, args.workspace = address(grad_initial), address(workspace)
        call("gs_gated_scan_backward", device, ctypes.byref(args))
        return grad_x, grad_gate, grad_initial, None, None


def gated_scan(x: torch.Tensor, gate: torch.Tensor, packed: PackedSequences | None = None, *,
               initial: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The recurrence over ``x`` and ``gate`` [tokens, channels] (one type:
    float32, bfloat16 or float16; rows may be strided, as slices of one
    projection are). ``packed`` says which rows form which sequence (None: all
    rows are one); ``initial`` [sequences, channels] float32 is the state each
    sequence starts from (None: zeros). Returns ``y`` [tokens, channels], the
    states in the type of ``x``, and ``last`` [sequences, channels] float32, the
    final ones (of an empty sequence, its initial state).

    The state is held in float32 throughout. Differentiable in x, gate and
    initial, through y and last; deterministic in both directions."""
    what = "gated_scan"
    device = check_cuda(what, x=x, gate=gate, initial=initial)
    dtype = _check_pair(what, x, gate, "tokens")
    tokens, channels = x.shape
    check_tokens(tokens, what)
    check_packed(packed, tokens, device, what)
    if initial is not None:
        expected = (1 if packed is None else len(packed), channels)
        if initial.dtype != torch.float32 or tuple(initial.shape) != expected:
            raise ValueError(f"{what}: initial must be float32 {expected}, got {initial.dtype} "
                             f"{tuple(initial.shape)}")
    return _GatedScan.apply(x, gate, initial, packed, dtype)


def gated_scan_step(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
    """One step of each stream: updates ``state`` [batch, channels] float32 in
    place from ``x`` and ``gate`` [batch, channels] and returns it in the type of
    ``x``. No gradient."""
    what = "gated_scan_step"
    device = check_cuda(what, x=x, gate=gate, state=state)
    dtype = _check_pair(what, x, gate, "batch")
    if state.dtype != torch.float32 or state.shape != x.shape or not state.is_contiguous():
        raise ValueError(f"{what}: state must be a contiguous float32 tensor of shape "
                         f"{tuple(x.shape)}, got {state.dtype} {tuple(state.shape)}"
                         f"{'' if state.is_contiguous() else ' (not contiguous)'}")
    x, gate = _rows(x), _rows(gate)
    y = x.new_empty(x.shape)
    call("gs_gated_scan_step", device, x.shape[0], x.shape[1], dtype, address(x), x.stride(0),
         address(gate), gate.stride(0), address(state), address(y))
    changed_in_place(state)
    return y
