"""Attention in a sliding window with a few first tokens that stay visible.

For Gaussians along a space-filling order, a token's neighbours in the sequence
are its neighbours in space, so a refiner attends in a window of them, and to a
few first tokens that stand for the scene or the camera. Three entry points:

:func:`window_attention`
    whole sequences, packed, differentiable: training, and inference over a
    scene.
:func:`window_attention_step`
    one new token of each of a batch of streams against a cache of fixed size
    (:func:`window_cache`): the first tokens keep their slots, later tokens
    take the others in turn.
:func:`window_attention_step_4bit`
    the same against a cache that holds keys and values in 4 bits
    (:func:`window_cache_4bit`): a quarter of the memory, and of the reading.

Query ``i`` of a sequence sees key ``j`` if the key is valid, ``j <= i + right``,
and ``j >= i - left`` or ``j < first``. A query that sees nothing gets zeros, and
no gradient flows through it.
"""

from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch

from . import native
from .sequences import (PackedSequences, address, call, changed_in_place, check_cuda,
                        check_packed, check_tokens, element_type, tile_arguments)

MAX_HEAD_DIM = 128
_TYPES = (torch.bfloat16, torch.float16)
_WIDEST = 2 ** 31 - 1  # of a window's sides: no window


def _heads(what, q, k, v, rows_name):
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError(f"{what}: expected [{rows_name}, heads, dim] tensors, got "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    (rows, heads, dim), (k_rows, kv_heads, k_dim) = q.shape, k.shape
    if k.shape != v.shape or k_rows != rows or k_dim != dim:
        raise ValueError(f"{what}: q {tuple(q.shape)} does not go with k {tuple(k.shape)} and v "
                         f"{tuple(v.shape)}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"{what}: {heads} query heads are not a multiple of {kv_heads} "
                         "key-value heads")
    if dim < 8 or dim % 8 or dim > MAX_HEAD_DIM:
        raise ValueError(f"{what}: head dim {dim} is not a multiple of 8 in [8, {MAX_HEAD_DIM}]")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"{what}: q, k and v have different types: {q.dtype}, {k.dtype}, "
                         f"{v.dtype}")
    return element_type(q.dtype, what, _TYPES)


def _scale(what, scale, dim):
    scale = dim ** -0.5 if scale is None else float(scale)
    if not (0.0 < scale < math.inf):
        raise ValueError(f"{what}: scale must be positive and finite, got {scale}")
    return scale


def _strided(t: torch.Tensor) -> torch.Tensor:
    """``t`` itself where the kernels can read it in place (rows of whole,
    aligned 16-byte words), else a contiguous copy."""
    row, head, channel = t.stride()
    if channel == 1 and row % 8 == 0 and head % 8 == 0 and row > 0 and head > 0 and \
            t.data_ptr() % 16 == 0:
        return t
    return t.contiguous() if not t.is_contiguous() else t.clone(
        memory_format=torch.contiguous_format)


def _whole(t: torch.Tensor) -> torch.Tensor:
    """``t`` contiguous and 16-byte aligned."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _place(q, k, v):
    """The fields of an operator's arguments that say where q, k and v lie."""
    (q_stride, q_head, _), (k_stride, k_head, _), (v_stride, v_head, _) = \
        q.stride(), k.stride(), v.stride()
    return dict(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_stride=q_stride,
                q_head_stride=q_head, k_stride=k_stride, k_head_stride=k_head,
                v_stride=v_stride, v_head_stride=v_head)


def _arguments(kind, q, k, v, **values):
    return kind(**_place(q, k, v), **values)


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, packed, left, right, first, valid, scale, dtype, need_grad):
        q, k, v = _strided(q), _strided(k), _strided(v)
        tokens, heads, dim = q.shape
        out = q.new_empty((tokens, heads, dim))
        lse = q.new_empty((heads, tokens), dtype=torch.float32) if need_grad else None
        args = _arguments(native.WindowAttentionArgs, q, k, v, tokens=tokens,
                          **tile_arguments(packed, tokens), heads=heads, kv_heads=k.shape[1], dim=dim, dtype=dtype,
                          left=left, right=right, first=first, scale=scale, valid=address(valid),
                          out=out.data_ptr(), lse=address(lse))
        call("gs_window_attention", q.device, ctypes.byref(args))
        if need_grad:
            ctx.save_for_backward(q, k, v, out, lse, valid)
            ctx.packed, ctx.args = packed, args  # sizes, the layout's table
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        q, k, v, out, lse, valid = ctx.saved_tensors
        # A saved-tensor hook (offloading to the host, say) may have brought back
        # tensors that lie differently than the forward's did.
        q, k, v, out, grad_out = _strided(q), _strided(k), _strided(v), _whole(out), _whole(grad_out)
        lse, valid = lse.contiguous(), None if valid is None else valid.contiguous()
        grad_q, grad_k, grad_v = (t.new_empty(t.shape) for t in (q, k, v))
        lib, args = native.lib(), native.WindowAttentionArgs.from_buffer_copy(ctx.args)
        for name, value in _place(q, k, v).items():
            setattr(args, name, value)
        args.out, args.lse, args.valid = out.data_ptr(), lse.data_ptr(), address(valid)
        size = lib.gs_window_attention_workspace_size(ctypes.byref(args))
        workspace = q.new_empty((size,), dtype=torch.uint8)
        args.grad_out, args.grad_q = grad_out.data_ptr(), grad_q.data_ptr()
        args.grad_k, args.grad_v = grad_k.data_ptr(), grad_v.data_ptr()
        args.workspace, args.workspace_size = workspace.data_ptr(), size
        call("gs_window_attention_backward", q.device, ctypes.byref(args))
        return (grad_q, grad_k, grad_v) + (None,) * 8


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                     packed: PackedSequences | None = None, *, left: int, right: int = 0,
                     first: int = 0, valid: torch.Tensor | None = None,
                     scale: float | None = None) -> torch.Tensor:
    """Attention of ``q`` [tokens, heads, dim] over ``k`` and ``v`` [tokens,
    kv_heads, dim] (``heads`` a multiple of ``kv_heads``; query head ``h`` uses
    key-value head ``h // (heads / kv_heads)``), each query to ``left`` keys
    before it, ``right`` after it, itself, and the ``first`` tokens of its
    sequence (at most 128) that do not come after its window. ``right=0`` is
    causal; a ``left`` or ``right`` of the sequence's length is no window.

    ``packed`` says which rows form which sequence (None: all rows are one).
    ``valid`` [tokens] bool leaves keys out, e.g. of dead splats; what invalid
    rows of k and v hold does not matter, and their gradient is zero. An invalid
    token still asks: its row of q counts like any other. What a query that sees
    nothing holds does not matter either. A non-finite value of a valid key or
    value reaches every query that sees it, one of a query or of its output's
    gradient the gradients of every key that it sees; both may reach others of
    the same sequence less than a window and 128 tokens away.
    ``scale`` multiplies the scores (default ``dim ** -0.5``).

    bfloat16 or float16, dim a multiple of 8 up to 128; scores, maxima and sums
    in float32. The probabilities, and in the backward the score gradients, are
    rounded to the inputs' type for their products (float16's are scaled into its
    range, whatever the gradients' size). q, k and v may be slices of one projection: they are read
    in place if rows and heads start on 16-byte boundaries, and copied
    otherwise. Returns [tokens, heads, dim]; differentiable in q, k and v, and
    deterministic in both directions."""
    what = "window_attention"
    device = check_cuda(what, q=q, k=k, v=v, valid=valid)
    dtype = _heads(what, q, k, v, "tokens")
    tokens = q.shape[0]
    check_tokens(tokens, what)
    check_packed(packed, tokens, device, what)
    left, right, first = int(left), int(right), int(first)
    if left < 0 or right < 0:
        raise ValueError(f"{what}: left and right must be >= 0, got {left} and {right}")
    if not 0 <= first <= native.MAX_FIRST_TOKENS:
        raise ValueError(f"{what}: first must be in [0, {native.MAX_FIRST_TOKENS}], got {first}")
    if valid is not None:
        if valid.dtype != torch.bool or valid.shape != (tokens,):
            raise ValueError(f"{what}: valid must be a bool tensor of {tokens} tokens, got "
                             f"{valid.dtype} {tuple(valid.shape)}")
        valid = valid.contiguous()
    need_grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or
                                             v.requires_grad)
    return _WindowAttention.apply(q, k, v, packed, min(left, _WIDEST), min(right, _WIDEST),
                                  first, valid, _scale(what, scale, q.shape[2]), dtype, need_grad)


def window_cache(batch: int, left: int, first: int, kv_heads: int, dim: int,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
    """An empty cache for ``batch`` streams with a window of ``left`` tokens
    before the new one and ``first`` first tokens: the tensors ``cache_k`` and
    ``cache_v`` [batch, first + left + 1, kv_heads, dim]. Their size does not
    grow with the streams."""
    if left < 0 or first < 0:
        raise ValueError(f"window_cache: left and first must be >= 0, got {left} and {first}")
    shape = (batch, first + left + 1, kv_heads, dim)
    return (torch.zeros(shape, dtype=dtype, device=device),
            torch.zeros(shape, dtype=dtype, device=device))


def _step_checks(what, batch, slots, positions, first, valid, cache_valid):
    """``first`` and ``valid`` of a step, as the kernels take them."""
    first = int(first)
    if not 0 <= first < slots:
        raise ValueError(f"{what}: first must be in [0, {slots}) for {slots} slots, got "
                         f"{first}")
    if positions.dtype != torch.int64 or positions.shape != (batch,):
        raise ValueError(f"{what}: positions must be int64 [{batch}], got {positions.dtype} "
                         f"{tuple(positions.shape)}")
    if cache_valid is None and valid is not None:
        raise ValueError(f"{what}: valid without cache_valid, which keeps it for the later tokens")
    if cache_valid is not None and (cache_valid.dtype != torch.bool or
                                    tuple(cache_valid.shape) != (batch, slots) or
                                    not cache_valid.is_contiguous()):
        raise ValueError(f"{what}: cache_valid must be a contiguous bool tensor {(batch, slots)}, got "
                         f"{cache_valid.dtype} {tuple(cache_valid.shape)}")
    if valid is not None:
        if valid.dtype != torch.bool or valid.shape != (batch,):
            raise ValueError(f"{what}: valid must be bool [{batch}], got {valid.dtype} "
                             f"{tuple(valid.shape)}")
        valid = valid.contiguous()
    return first, valid


def window_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                          cache_k: torch.Tensor, cache_v: torch.Tensor, positions: torch.Tensor,
                          *, first: int = 0, scale: float | None = None,
                          valid: torch.Tensor | None = None,
                          cache_valid: torch.Tensor | None = None) -> torch.Tensor:
    """One new token of each stream: writes ``k`` and ``v`` [batch, kv_heads,
    dim] to the caches [batch, slots, kv_heads, dim] in place and returns the
    attention of ``q`` [batch, heads, dim] over what the caches then hold, the
    row of :func:`window_attention` with ``left = slots - first - 1`` and
    ``right = 0`` for that token.

    ``positions`` [batch] int64 is each token's place in its stream, counted
    from zero; -1 marks an idle stream (zeros come back, its cache is left
    alone). Token ``p`` goes to slot ``p`` while ``p < first`` and then to
    ``first + (p - first) % (slots - first)``, so a stream's tokens must come in
    order.

    ``cache_valid`` [batch, slots] bool leaves slots out as
    :func:`window_attention`'s ``valid`` leaves keys out (None: none are); it goes
    with the caches and is updated in place from ``valid`` [batch] bool, which says
    whether the new tokens may be seen (None: all may). No gradient."""
    what = "window_attention_step"
    device = check_cuda(what, q=q, k=k, v=v, cache_k=cache_k, cache_v=cache_v,
                        positions=positions, valid=valid, cache_valid=cache_valid)
    dtype = _heads(what, q, k, v, "batch")
    batch, heads, dim = q.shape
    shape = tuple(cache_k.shape)
    if len(shape) != 4 or tuple(cache_v.shape) != shape or \
            (shape[0], shape[2], shape[3]) != tuple(k.shape):
        raise ValueError(f"{what}: caches {shape} and {tuple(cache_v.shape)} are not [batch, "
                         f"slots, kv_heads, dim] for k {tuple(k.shape)}")
    if cache_k.dtype != q.dtype or cache_v.dtype != q.dtype:
        raise ValueError(f"{what}: caches of {cache_k.dtype} and {cache_v.dtype} for {q.dtype} "
                         "tokens")
    if not (cache_k.is_contiguous() and cache_v.is_contiguous()) or cache_k.data_ptr() % 16 or \
            cache_v.data_ptr() % 16:
        raise ValueError(f"{what}: the caches must be contiguous and 16-byte aligned (they are "
                         "updated in place)")
    if batch * shape[1] > native.MAX_SEQUENCE_TOKENS:
        raise ValueError(f"{what}: caches of {batch} x {shape[1]} slots, at most "
                         f"{native.MAX_SEQUENCE_TOKENS} in all are supported")
    first, valid = _step_checks(what, batch, shape[1], positions, first, valid, cache_valid)
    positions = positions.contiguous()
    q, k, v = _strided(q), _strided(k), _strided(v)
    out = q.new_empty((batch, heads, dim))
    args = _arguments(native.WindowAttentionStepArgs, q, k, v, batch=batch, heads=heads,
                      kv_heads=k.shape[1], dim=dim, dtype=dtype, slots=shape[1], first=first,
                      scale=_scale(what, scale, dim), cache_k=cache_k.data_ptr(),
                      cache_v=cache_v.data_ptr(), positions=positions.data_ptr(),
                      out=out.data_ptr(), valid=address(valid), cache_valid=address(cache_valid))
    call("gs_window_attention_step", device, ctypes.byref(args))
    changed_in_place(cache_k, cache_v, cache_valid)
    return out


class FourBitCache(NamedTuple):
    """Keys and values of a batch of streams in 4 bits. Codes are uint8 [batch,
    kv_heads, slots, dim / 2], channel ``2i`` in the low half of byte ``i`` and
    ``2i + 1`` in the high one; ranges are [batch, kv_heads, slots, 2] in the
    tokens' type: code ``c`` of a row stands for ``(c - 7.5) * range[0] + range[1]``."""

    k_codes: torch.Tensor
    k_range: torch.Tensor
    v_codes: torch.Tensor
    v_range: torch.Tensor


def window_cache_4bit(batch: int, left: int, first: int, kv_heads: int, dim: int,
                      dtype: torch.dtype = torch.bfloat16, device="cuda") -> FourBitCache:
    """:func:`window_cache` in 4 bits: an empty cache for ``batch`` streams with a
    window of ``left`` tokens before the new one and ``first`` first tokens."""
    if left < 0 or first < 0:
        raise ValueError(f"window_cache_4bit: left and first must be >= 0, got {left} and {first}")
    if dim < 8 or dim % 8:
        raise ValueError(f"window_cache_4bit: dim must be a multiple of 8, got {dim}")
    shape = (batch, kv_heads, first + left + 1)
    codes = [torch.zeros((*shape, dim // 2), dtype=torch.uint8, device=device) for _ in range(2)]
    ranges = [torch.zeros((*shape, 2), dtype=dtype, device=device) for _ in range(2)]
    return FourBitCache(codes[0], ranges[0], codes[1], ranges[1])


def window_attention_step_4bit(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                               cache: FourBitCache, positions: torch.Tensor, *, first: int = 0,
                               scale: float | None = None, valid: torch.Tensor | None = None,
                               cache_valid: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`window_attention_step` against a :class:`FourBitCache`, which is
    updated in place: the new token's row ``x`` of each key-value head is held as
    16 even steps between its least and its greatest channel, ``range = ((max x - min
    x) / 15, (max x + min x) / 2)`` rounded to the tokens' type and codes ``(x -
    range[1]) / range[0] + 7.5`` rounded to the nearest, ties to even. The output is
    the attention over what the cache then holds, the new token as it is held
    included; scores and sums in float32, the weights times the values' steps rounded to
    11 bits (relative to the steps' largest where they are 2^21 apart). A row with a
    channel that is not finite is held as one that is not finite.

    q, k and v [batch, heads, dim], bfloat16 or float16, dim a multiple of 8 up to
    128; ``positions``, ``first``, ``scale``, ``valid`` and ``cache_valid`` as
    :func:`window_attention_step` takes them. No gradient."""
    what = "window_attention_step_4bit"
    k_codes, k_range, v_codes, v_range = cache
    device = check_cuda(what, q=q, k=k, v=v, k_codes=k_codes, k_range=k_range, v_codes=v_codes,
                        v_range=v_range, positions=positions, valid=valid,
                        cache_valid=cache_valid)
    dtype = _heads(what, q, k, v, "batch")
    batch, heads, dim = q.shape
    kv_heads = k.shape[1]
    slots = k_codes.shape[2] if k_codes.dim() == 4 else 0
    codes, ranges = (batch, kv_heads, slots, dim // 2), (batch, kv_heads, slots, 2)
    pointers = [t.data_ptr() for t in (k_codes, k_range, v_codes, v_range)]
    if slots < 1 or k_codes.shape != codes or v_codes.shape != codes or \
            k_range.shape != ranges or v_range.shape != ranges or \
            k_codes.dtype != torch.uint8 or v_codes.dtype != torch.uint8 or \
            k_range.dtype != q.dtype or v_range.dtype != q.dtype:
        given = ", ".join(f"{tuple(t.shape)} {t.dtype}" for t in cache)
        raise ValueError(f"{what}: a cache of {given} is not [batch, kv_heads, slots, dim / 2] "
                         f"uint8 codes and [..., 2] {q.dtype} ranges for k {tuple(k.shape)}")
    if any(p % 16 for p in pointers) or not (k_codes.is_contiguous() and k_range.is_contiguous() and
                                             v_codes.is_contiguous() and v_range.is_contiguous()):
        raise ValueError(f"{what}: the cache must be contiguous and 16-byte aligned (it is "
                         "updated in place)")
    if batch * slots > native.MAX_SEQUENCE_TOKENS:
        raise ValueError(f"{what}: caches of {batch} x {slots} slots, at most "
                         f"{native.MAX_SEQUENCE_TOKENS} in all are supported")
    first, valid = _step_checks(what, batch, slots, positions, first, valid, cache_valid)
    positions = positions.contiguous()
    q, k, v = _strided(q), _strided(k), _strided(v)
    out = q.new_empty((batch, heads, dim))
    args = _arguments(native.WindowAttentionStep4BitArgs, q, k, v, batch=batch, heads=heads,
                      kv_heads=kv_heads, dim=dim, dtype=dtype, slots=slots, first=first,
                      scale=_scale(what, scale, dim), positions=positions.data_ptr(),
                      out=out.data_ptr(), valid=address(valid), cache_valid=address(cache_valid),
                      k_codes=pointers[0], k_range=pointers[1], v_codes=pointers[2],
                      v_range=pointers[3])
    size = native.lib().gs_window_attention_step_4bit_workspace_size(ctypes.byref(args))
    workspace = q.new_empty((size,), dtype=torch.uint8)
    args.workspace, args.workspace_size = workspace.data_ptr(), size
    call("gs_window_attention_step_4bit", device, ctypes.byref(args))
    changed_in_place(k_codes, k_range, v_codes, v_range, cache_valid)
    return out
