"""Fused optimizer step for training splats on the GPU, and gradient clipping.

The reference trains with ``torch.optim.Adam`` over one parameter group per
splat tensor (``training/train.py:111-118``: mean, rotation, scale, opacity,
color; ``eps=1e-15``), calls ``optimizer.step()`` after every backward
(``training/train.py:151``) and then perturbs the means with
``noise_splats`` (``training/utils.py:50-62``). :class:`FusedAdam` is that
optimizer with both steps done by one sm_100a kernel (``gs_adam_step``): each
parameter, gradient and moment element is read once and written once,
instead of ~30 elementwise kernels re-reading them.

It subclasses ``torch.optim.Adam`` and keeps its state layout (per parameter:
``step``, ``exp_avg``, ``exp_avg_sq``), so code that edits optimizer state
-- ``relocate_splats`` (``training/utils.py:147-210``) zeroing moments of
relocated splats or growing them when densifying -- works unchanged.

:func:`clip_grad_norm` clips the gradients of any parameters (a refiner's, say)
to a global norm, :func:`grad_norm` only measures it, and
``FusedAdam.step(max_norm=...)`` clips the splats' gradients inside the step.
"""

from __future__ import annotations

import ctypes

from collections.abc import Iterable

import torch

from . import native
from .sequences import call, changed_in_place

GROUP_NAMES = ("mean", "rotation", "scale", "opacity", "color")
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # GS_FLOAT32, ...


def _dense(t: torch.Tensor) -> bool:
    """Whether the elements fill one run of memory, in whatever order."""
    if t.is_contiguous():
        return True
    size = 1
    for stride, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != size:
            return False
        size *= n
    return True


def _max_norm(what: str, max_norm: float) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"{what}: max_norm must be >= 0, got {max_norm}")
    return max_norm


def _norm(what: str, tensors: list[torch.Tensor], max_norm: float, scale: bool) -> torch.Tensor:
    """The norm of dense tensors on one device and the factor that clips it to
    ``max_norm``, two floats; with ``scale`` the tensors are multiplied by it."""
    device, words = tensors[0].device, []
    index = tensors[0].get_device()
    for t in tensors:
        dtype = _TYPES.get(t.dtype)
        if dtype is None or t.get_device() != index or index < 0 or t.layout != torch.strided:
            _refuse(what, t, device)
        words += (t.data_ptr(), t.numel(), dtype)
    entries = (ctypes.c_int64 * len(words))(*words)  # gs_gradient: three words each
    size = native.lib().gs_clip_grad_norm_workspace_size(len(tensors))
    result = torch.empty(2, dtype=torch.float32, device=device)
    workspace = torch.empty(size, dtype=torch.uint8, device=device)
    call("gs_clip_grad_norm", device, len(tensors), entries, max_norm, int(scale),
         result.data_ptr(), workspace.data_ptr(), size)
    return result


def _refuse(what: str, t: torch.Tensor, device: torch.device) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{what} runs on CUDA devices only (there is no CPU path); a gradient "
                           f"is on {t.device}")
    if t.layout != torch.strided or t.dtype not in _TYPES:
        raise ValueError(f"{what}: gradients must be dense and float32, bfloat16 or float16, got "
                         f"{t.dtype} ({t.layout})")
    raise RuntimeError(f"{what}: a gradient is on {t.device}, another on {device}")


def _check_finite(what: str, norm: torch.Tensor) -> None:
    if not torch.isfinite(norm):
        raise RuntimeError(f"{what}: the gradients' norm is {norm.item()}, so they cannot be "
                           "clipped")


def grad_norm(tensors: torch.Tensor | Iterable[torch.Tensor]) -> torch.Tensor:
    """The root of the sum of the squares of all elements of ``tensors``
    (float32, bfloat16 and float16, on one device, any strides and sizes) as a
    float32 scalar on their device, without a wait. One pass over the data; sums
    in float32 over 128 bytes of elements and in float64 beyond that, so that no
    finite norm overflows on the way; the same result every time. No gradient."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        raise ValueError("grad_norm needs at least one tensor")
    tensors = [t.detach() for t in tensors]
    tensors = [t if t.layout != torch.strided or _dense(t) else t.contiguous() for t in tensors]
    return _norm("grad_norm", tensors, float("inf"), False)[0]


def clip_grad_norm(parameters: torch.Tensor | Iterable[torch.Tensor], max_norm: float, *,
                   error_if_nonfinite: bool = False) -> torch.Tensor:
    """Multiplies the ``.grad`` of all ``parameters`` by ``min(1, max_norm / (norm
    + 1e-6))``, ``norm`` their :func:`grad_norm`, and returns the norm from before
    (``torch.nn.utils.clip_grad_norm_`` with the 2-norm). Parameters without a
    gradient are passed over, one listed twice counts once; where the norm is small
    enough, every gradient keeps its values (those that lie in one run of memory,
    apart from the others, are not written at all). An infinity makes the factor 0 and
    a NaN makes it NaN, for every gradient, as an infinity does where ``max_norm`` is
    one itself; ``error_if_nonfinite`` raises instead, before anything is written, which
    costs a wait for the norm. Gradients may be float32, bfloat16 or float16 in any
    mixture and of any strides, on one device; an element that two of them share counts
    twice and is multiplied once. No gradient."""
    what = "clip_grad_norm"
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    max_norm = _max_norm(what, max_norm)
    if not parameters:
        raise ValueError(f"{what} needs at least one parameter")
    grads = [g for p in {id(p): p for p in parameters}.values() if (g := p.grad) is not None]
    if not grads:
        return torch.zeros((), dtype=torch.float32, device=parameters[0].device)
    tensors, copies, spans = list(grads), [], []
    whole = True
    for g in grads:
        if g.layout != torch.strided or not g.is_contiguous():
            whole = False
            break
        at = g.data_ptr()
        spans.append((at, at + g.nbytes))
    if not whole or _overlap(spans):
        copies = _apart(what, tensors)
    if error_if_nonfinite:
        _check_finite(what, _norm(what, tensors, max_norm, False)[0])
    result = _norm(what, tensors, max_norm, True)
    for t, copy in copies:
        t.copy_(copy)
    changed_in_place(*grads)
    return result[0]


def _overlap(spans: list[tuple[int, int]]) -> bool:
    spans = sorted(s for s in spans if s[0] < s[1])
    return any(a[1] > b[0] for a, b in zip(spans, spans[1:]))


def _apart(what: str, tensors: list[torch.Tensor]) -> list[tuple[torch.Tensor, torch.Tensor]]:
    """Replaces gradients that do not fill one run of memory by contiguous copies, and
    all of them where what they span overlaps (slices of one tensor, say); returns
    those replaced and their copies."""
    spans = [(t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum(
        s * (n - 1) for s, n in zip(t.stride(), t.shape)))) for t in tensors
        if t.layout == torch.strided and t.numel()]
    woven, copies = _overlap(spans), []
    for i, t in enumerate(tensors):
        if t.layout == torch.strided and (woven or not _dense(t)):
            if 0 in (s for s, n in zip(t.stride(), t.shape) if n > 1):
                raise ValueError(f"{what}: a gradient of strides {t.stride()} shares memory "
                                 "between its elements")
            t = t.detach()
            tensors[i] = t.clone(memory_format=torch.contiguous_format)
            copies.append((t, tensors[i]))
    return copies


class FusedAdam(torch.optim.Adam):
    """``torch.optim.Adam`` for a splat's five parameter tensors, one kernel
    per step.

    Build it the way the reference builds its optimizer: one group per
    tensor, each with a ``"name"`` from :data:`GROUP_NAMES` and one CUDA
    float32 contiguous parameter, e.g. ``FusedAdam([{"params": [s.mean],
    "name": "mean", "lr": 1.6e-4}, ...], eps=1e-15)``. Plain Adam only
    (no weight decay, amsgrad or maximize); anything else raises
    ``ValueError``. There is no CPU path.
    """

    # Of the last step with a max_norm. Here, since copies are not made by __init__.
    grad_norm: torch.Tensor | None = None

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0):
        super().__init__(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                         foreach=False)
        names = [group.get("name") for group in self.param_groups]
        if sorted(map(str, names)) != sorted(GROUP_NAMES):
            raise ValueError(f"FusedAdam needs one group per name in {GROUP_NAMES}, got {names}")
        for group in self.param_groups:
            if len(group["params"]) != 1:
                raise ValueError(f"group {group['name']!r} must hold exactly one tensor")
            if group["weight_decay"] or group["amsgrad"] or group["maximize"]:
                raise ValueError("FusedAdam supports plain Adam only (no weight decay, amsgrad "
                                 "or maximize)")
            if group["betas"] != self.param_groups[0]["betas"] or \
                    group["eps"] != self.param_groups[0]["eps"]:
                raise ValueError("FusedAdam needs the same betas and eps in every group")

    def _groups(self):
        by_name = {group["name"]: group for group in self.param_groups}
        return [by_name[name] for name in GROUP_NAMES]

    @torch.no_grad()
    def step(self, closure=None, noise=None, max_norm=None):
        """One Adam step over the five groups (parameters without ``.grad``
        are skipped, as torch does). With ``noise=(noise_lr, position_lr)``
        the same kernel then adds noise_splats' position noise
        (``training/utils.py:50-62``) to the updated means, drawing its
        normal samples with ``torch.randn_like(mean)`` as the reference does.

        With ``max_norm`` the step is that of gradients clipped as
        :func:`clip_grad_norm` clips them, all five together: the factor is applied
        as the kernel reads them, the ``.grad`` tensors stay as they are, and
        ``self.grad_norm`` is their norm (a device scalar; None without gradients)."""
        if max_norm is not None:
            max_norm, self.grad_norm = _max_norm("FusedAdam", max_norm), None
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        groups = self._groups()
        params = [group["params"][0] for group in groups]
        mean = params[0]
        n = mean.shape[0]
        for name, p in zip(GROUP_NAMES, params):
            if not (p.is_cuda and p.dtype == torch.float32 and p.is_contiguous()):
                raise RuntimeError(f"FusedAdam: {name} must be a contiguous CUDA float32 tensor "
                                   "(there is no CPU path)")
            if p.shape[0] != n or p.device != mean.device:
                raise RuntimeError(f"FusedAdam: {name} has {p.shape[0]} rows on {p.device}, "
                                   f"mean has {n} on {mean.device}")
        color = params[4]
        if color.dim() != 3 or color.shape[2] != 3:
            raise RuntimeError(f"FusedAdam: color must be [N, K, 3], got {tuple(color.shape)}")
        steps, grads = [], []
        for p in params:
            state = self.state[p]
            if len(state) == 0:
                state["step"] = torch.tensor(0.0, dtype=torch.float32)
                state["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                state["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
            if p.grad is not None:
                if p.grad.is_sparse:
                    raise RuntimeError("FusedAdam does not support sparse gradients")
                state["step"] += 1
                grads.append(p.grad.contiguous())
            else:
                grads.append(None)
            steps.append(max(1.0, float(state["step"])))
        if all(g is None for g in grads) and noise is None:
            return loss
        beta1, beta2 = groups[0]["betas"]
        noise_lr, position_lr = noise if noise is not None else (0.0, 0.0)
        hyper = native.adam_params(steps, [float(g["lr"]) for g in groups], (beta1, beta2),
                                   groups[0]["eps"], noise_lr, position_lr)
        randn = torch.randn_like(mean) if noise is not None else None
        clip = None
        if max_norm is not None:
            present = [g for g in grads if g is not None]
            if present:
                clip = _norm("FusedAdam", present, max_norm, False)
                self.grad_norm = clip[0]

        def arrays(tensors):
            return native.SplatArrays(*(t.data_ptr() if t is not None else None
                                        for t in tensors))

        sets = (arrays(params), arrays(grads),
                arrays([self.state[p]["exp_avg"] for p in params]),
                arrays([self.state[p]["exp_avg_sq"] for p in params]))
        with torch.cuda.device(mean.device):
            stream = ctypes.c_void_p(torch.cuda.current_stream(mean.device).cuda_stream)
            arguments = (n, color.shape[1], *(ctypes.byref(s) for s in sets), ctypes.byref(hyper),
                         ctypes.c_void_p(randn.data_ptr() if randn is not None else None))
            if clip is None:
                native.check(native.lib().gs_adam_step(*arguments, stream), "gs_adam_step")
            else:
                native.check(native.lib().gs_adam_step_clipped(
                    *arguments, ctypes.c_void_p(clip.data_ptr() + 4), stream),
                    "gs_adam_step_clipped")
        return loss
