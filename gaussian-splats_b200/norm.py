"""Root-mean-square norm of a token's channels with the residual's addition.

:func:`rms_norm` adds the residual stream, norms the sum and returns both
(differentiable); :func:`rms_norm_e4m3` does the same for serving with an 8-bit
output, one scale a token, as the next matrix product takes it.
"""

from __future__ import annotations

import ctypes

import torch

from . import native
from .sequences import address, call, check_cuda, element_type


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as rows with contiguous channels: a view where it has them, else a copy."""
    t = t.reshape(-1, t.shape[-1]) if t.dim() != 2 else t
    return t if t.stride(1) == 1 and t.stride(0) >= 0 else t.contiguous()


def _check(what, x, weight, residual, eps):
    check_cuda(what, x=x, weight=weight, residual=residual)
    if x.dim() < 1 or x.shape[-1] < 1 or x.shape[-1] > native.MAX_NORM_CHANNELS:
        raise ValueError(f"{what}: x {tuple(x.shape)} must have 1 to "
                         f"{native.MAX_NORM_CHANNELS} channels in its last axis")
    element_type(x.dtype, what)
    element_type(weight.dtype, f"{what} weight")
    if weight.shape != x.shape[-1:]:
        raise ValueError(f"{what}: weight {tuple(weight.shape)} for {x.shape[-1]} channels")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"{what}: residual {tuple(residual.shape)} does not match x "
                             f"{tuple(x.shape)}")
        if residual.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"{what}: the residual must be {x.dtype} or float32, got "
                             f"{residual.dtype}")
    eps = float(eps)
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"{what}: eps must be >= 0 and finite, got {eps}")
    return eps


def _arguments(x, weight, residual, eps, **outputs):
    """``gs_rms_norm_args`` of rows ``x`` and ``residual``, and its codes of types."""
    dtype = element_type(x.dtype, "")
    return native.RmsNormArgs(
        rows=x.shape[0], channels=x.shape[1], dtype=dtype,
        residual_dtype=dtype if residual is None else element_type(residual.dtype, ""),
        weight_dtype=element_type(weight.dtype, ""), eps=eps, x=address(x),
        residual=address(residual), weight=address(weight), x_stride=x.stride(0),
        residual_stride=0 if residual is None else residual.stride(0),
        **{name: address(t) for name, t in outputs.items()})


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        shape = x.shape
        rows, weight = _rows(x), weight.contiguous()
        res = None if residual is None else _rows(residual)
        y = x.new_empty(shape)
        total = None if res is None else res.new_empty(shape)
        args = _arguments(rows, weight, res, eps, y=y, sum=total)
        call("gs_rms_norm", x.device, ctypes.byref(args))
        # The sum itself where it lost nothing, else what it was made of.
        again = res is not None and res.dtype != torch.float32
        ctx.save_for_backward(rows if res is None or again else total, weight, res if again else None)
        ctx.args, ctx.has_residual, ctx.x_dtype, ctx.shape = args, res is not None, x.dtype, shape
        ctx.set_materialize_grads(False)
        return y if res is None else (y, total)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y, grad_sum=None):
        z, weight, residual = ctx.saved_tensors
        # A saved-tensor hook may have brought back tensors that lie differently.
        z, weight = _rows(z), weight.contiguous()
        shape = ctx.shape
        grad_y = z.new_zeros(shape, dtype=ctx.x_dtype) if grad_y is None \
            else grad_y.contiguous()
        grad_sum = None if grad_sum is None else grad_sum.contiguous()
        grad_x = z.new_empty(shape, dtype=ctx.x_dtype)
        grad_residual = None
        if ctx.has_residual and residual is None and z.dtype != ctx.x_dtype:
            grad_residual = z.new_empty(shape)
        grad_weight = torch.empty_like(weight)
        args = native.RmsNormArgs.from_buffer_copy(ctx.args)  # sizes and types
        args.x = args.residual = args.y = args.sum = None
        args.x_stride = args.residual_stride = args.sum_stride = 0
        if residual is None:
            args.sum, args.sum_stride = address(z), z.stride(0)
        else:
            residual = _rows(residual)
            args.x, args.x_stride = address(z), z.stride(0)
            args.residual, args.residual_stride = address(residual), residual.stride(0)
        args.weight = address(weight)
        args.grad_y, args.grad_sum = address(grad_y), address(grad_sum)
        args.grad_x, args.grad_residual = address(grad_x), address(grad_residual)
        args.grad_weight = address(grad_weight)
        lib = native.lib()
        size = lib.gs_rms_norm_workspace_size(ctypes.byref(args))
        workspace = z.new_empty((size,), dtype=torch.uint8)
        args.workspace, args.workspace_size = address(workspace), size
        call("gs_rms_norm_backward", z.device, ctypes.byref(args))
        if ctx.has_residual and grad_residual is None:
            grad_residual = grad_x
        return grad_x, grad_weight, grad_residual, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *,
             eps: float = 1e-6):
    """``z / sqrt(mean(z**2) + eps) * weight`` over the last axis of ``z = x +
    residual``. Without a residual returns the norm, in the type of ``x``; with
    one (in the type of ``x``, or float32) returns the norm and ``z`` in the
    residual's type, the residual stream for the next layer.

    float32, bfloat16 or float16, at most 16,384 channels; the sum and the norm
    are computed in float32, and the norm and its gradients are those of the
    unrounded sum, for which a 16-bit residual's call keeps x and the residual for
    the backward. Differentiable in x, weight and residual, through both results;
    deterministic in both directions."""
    eps = _check("rms_norm", x, weight, residual, eps)
    return _RmsNorm.apply(x, weight, residual, eps)


def rms_norm_e4m3(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *,
                  eps: float = 1e-6):
    """:func:`rms_norm` with an 8-bit result: returns ``q`` (float8_e4m3fn, the
    shape of ``x``) and ``scale`` (float32, one a token), with ``q * scale`` the
    norm and ``scale = max|norm| / 448`` (1 for a token of zeros); with a
    residual, also the sum. No gradient."""
    eps = _check("rms_norm_e4m3", x, weight, residual, eps)
    rows, res = _rows(x), None if residual is None else _rows(residual)
    q = x.new_empty(x.shape, dtype=torch.float8_e4m3fn)
    scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
    total = None if res is None else res.new_empty(x.shape)
    weight = weight.contiguous()
    args = _arguments(rows, weight, res, eps, q=q, scale=scale, sum=total)
    call("gs_rms_norm", x.device, ctypes.byref(args))
    return (q, scale) if res is None else (q, scale, total)
