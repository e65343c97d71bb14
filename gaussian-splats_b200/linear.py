"""A linear layer with what usually follows it in its epilogue.

:func:`linear` computes ``act(x @ weight.T + bias) + residual`` in one kernel: the
product's sums are biased, activated and added to the residual stream before they
are rounded and written. Differentiable; the forward of a training pass also
keeps the activation's slope, so that the backward needs neither the sums nor
another product to make them again.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from . import native
from .attention import _whole
from .norm import _rows
from .sequences import address, call, check_cuda, check_tokens, element_type

ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "silu": 3}  # GS_IDENTITY, ...
_TYPES = (torch.bfloat16, torch.float16)
_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # GS_FLOAT32, ...

# Rows of no whole 16-byte words are read in place by the kernel up to so many inputs, and
# aligned first beyond (100,000 x 59 -> 256: 25 us against 26; 251 inputs: 51 against 46; a
# backward needs them aligned).
_GATHERED = 128


def _operand(t: torch.Tensor) -> torch.Tensor:
    """``t`` [rows, channels] as the kernels read a product's operand: rows of contiguous
    channels that start on 16-byte borders. ``t`` itself if it lies so, else a copy."""
    (row, channel), (rows, channels) = t.stride(), t.shape
    if channel == 1 and row % 8 == 0 and row >= channels and t.data_ptr() % 16 == 0:
        return t
    if channel != 1:
        t = t.contiguous()
        if rows and channels % 8 == 0:  # a new one, then, and whole words
            return t
    copy = t.new_empty((rows, -(-channels // 8) * 8))
    call("gs_align_rows", t.device, rows, channels, t.data_ptr(), t.stride(0), copy.data_ptr())
    return copy[:, :channels]


def _arguments(x, weight, bias, **values):
    """``gs_linear_args`` of operands ``x`` and ``weight``."""
    dtype, (rows, inputs) = _CODES[x.dtype], x.shape
    return native.LinearArgs(
        rows=rows, inputs=inputs, outputs=weight.shape[0], dtype=dtype,
        bias_dtype=dtype if bias is None else _CODES[bias.dtype], x=x.data_ptr(),
        weight=weight.data_ptr(), bias=address(bias), x_stride=x.stride(0),
        weight_stride=weight.stride(0), **values)


def _forward(x, weight, bias, residual, activation, train):
    """The result, and what the backward keeps."""
    outputs, inputs = weight.shape
    rows, w = x if x.dim() == 2 else x.reshape(-1, inputs), _operand(weight)
    if train or inputs > _GATHERED or rows.stride(1) != 1:
        rows = _operand(rows)
    b = None if bias is None else bias.contiguous()
    if residual is None:
        y, res, stride = x.new_empty(x.shape[:-1] + (outputs,)), None, 0
    else:
        y, res = residual.new_empty(residual.shape), _rows(residual)
        stride = res.stride(0)
    slope = None
    if train and activation:
        exact = b is not None and b.dtype == torch.float32
        slope = x.new_empty((rows.shape[0], -(-outputs // 8) * 8),
                            dtype=torch.float32 if exact else torch.int16)
    args = _arguments(rows, w, b, activation=activation, residual_dtype=_CODES[y.dtype],
                      residual=address(res), residual_stride=stride, y=y.data_ptr(),
                      slope=address(slope))
    if slope is not None:
        args.slope_float = slope.dtype == torch.float32
    call("gs_linear", x.device, ctypes.byref(args))
    return y, (rows, w, b, slope)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        y, kept = _forward(x, weight, bias, residual, activation, True)
        ctx.save_for_backward(*kept)
        ctx.activation, ctx.shape = activation, x.shape
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y):
        x, weight, bias, slope = ctx.saved_tensors
        # A saved-tensor hook may have brought back tensors that lie differently.
        x, weight = _operand(x), _operand(weight)
        slope = None if slope is None else _whole(slope)
        want_x, want_weight, want_bias, want_residual = ctx.needs_input_grad[:4]
        grads = [x.new_empty(ctx.shape) if want_x else None,
                 weight.new_empty(weight.shape) if want_weight else None,
                 torch.empty_like(bias) if want_bias else None]
        if want_x or want_weight or want_bias:
            rows = _whole(grad_y.reshape(x.shape[0], weight.shape[0]))
            args = _arguments(x, weight, bias, activation=ctx.activation,
                              residual_dtype=_CODES[rows.dtype], slope=address(slope),
                              grad_y=address(rows), grad_x=address(grads[0]),
                              grad_weight=address(grads[1]), grad_bias=address(grads[2]))
            if slope is not None:
                args.slope_float = slope.dtype == torch.float32
            size = native.lib().gs_linear_workspace_size(ctypes.byref(args))
            workspace = x.new_empty((size,), dtype=torch.uint8)
            args.workspace, args.workspace_size = address(workspace), size
            call("gs_linear_backward", x.device, ctypes.byref(args))
        return (*grads, grad_y if want_residual else None, None)


def _check_added(what, name, t, shape, dtype):
    if t.shape != shape:
        raise ValueError(f"{what}: {name} {tuple(t.shape)} is not {shape}")
    if t.dtype != dtype and t.dtype != torch.float32:
        raise ValueError(f"{what}: the {name} must be {dtype} or float32, got {t.dtype}")


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
           residual: torch.Tensor | None = None, *, activation: str | None = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual`` for ``x`` [..., inputs] and ``weight``
    [outputs, inputs], any number of rows. ``activation`` is None, ``"relu"``,
    ``"gelu"`` (``z`` times the normal distribution function of ``z``) or ``"silu"``.

    x and weight are bfloat16 or float16 (one type), the bias [outputs] in their type
    or float32, the residual [..., outputs] too; the result has the residual's type, or
    x's where there is none: a float32 residual stream stays one. Sums, bias, activation
    and the residual's addition are in float32, rounded once.

    Differentiable in x, weight, bias and residual (in reverse mode; a forward-mode
    tangent is refused), and deterministic in both directions. The backward rounds the
    gradient of the sums, ``grad * act'``, to the inputs' type, as its products need;
    float16 gradients below 6e-8 vanish there, as in any float16 tensor (scale the loss).
    Operands are read in place if their rows are contiguous and start on 16-byte borders
    (any slice of a projection does whose channels are multiples of 8) and copied
    otherwise."""
    what = "linear"
    device = check_cuda(what, x=x, weight=weight, bias=bias, residual=residual)
    element_type(x.dtype, what, _TYPES)
    if weight.dtype != x.dtype:
        raise ValueError(f"{what}: weight of {weight.dtype} for x of {x.dtype}")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"{what}: weight {tuple(weight.shape)} does not go with x "
                         f"{tuple(x.shape)}")
    outputs, inputs = weight.shape
    if not (1 <= inputs <= native.MAX_LINEAR_FEATURES and
            1 <= outputs <= native.MAX_LINEAR_FEATURES):
        raise ValueError(f"{what}: 1 to {native.MAX_LINEAR_FEATURES} inputs and outputs are "
                         f"supported, got {inputs} and {outputs}")
    check_tokens(x.numel() // inputs, what)
    if activation not in ACTIVATIONS:
        raise ValueError(f"{what}: activation must be one of {tuple(ACTIVATIONS)}, got "
                         f"{activation!r}")
    if bias is not None:
        _check_added(what, "bias", bias, (outputs,), x.dtype)
    if residual is not None:
        _check_added(what, "residual", residual, (*x.shape[:-1], outputs), x.dtype)
    # Within a level of forward-mode differentiation any of them may carry a tangent, which
    # the function's call refuses.
    if forward_ad._current_level >= 0 or torch.is_grad_enabled() and (
            x.requires_grad or weight.requires_grad or
            (bias is not None and bias.requires_grad) or
            (residual is not None and residual.requires_grad)):
        return _Linear.apply(x, weight, bias, residual, ACTIVATIONS[activation])
    return _forward(x, weight, bias, residual, ACTIVATIONS[activation], False)[0]
