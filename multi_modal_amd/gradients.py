"""Global gradient norm over many tensors, and clipping by it (csrc/gradients.hip).

What a training step of an encoder with PatchEmbedLayer does between `loss.backward()` and `optimizer.step()`; the reference's loops
go straight to the optimizer (classification/vggsound/vanilla_single.py:75-80).  Semantics of torch.nn.utils.clip_grad_norm_, with
the sums in float64 and in a fixed order, two launches for about a hundred tensors, and an optional second set of tensors (of
another type, e.g. the float32 gradients an optimizer takes) that the clipped gradients go to.
"""
from __future__ import annotations

import ctypes
import math
from typing import Iterable, List, Optional, Sequence, Union

import torch

from . import _native as N
from .plans import OUT_CODES, require_gpu

_KINDS = {2.0: N.NORM_2, math.inf: N.NORM_MAX}


def _gradients(tensors: Union[torch.Tensor, Iterable[torch.Tensor]]) -> List[torch.Tensor]:
    """Gradients of a list of parameters (those that have one), or the tensors of the list themselves."""
    found = []
    for t in [tensors] if isinstance(tensors, torch.Tensor) else tensors:
        if isinstance(t, torch.nn.Parameter) or (t.requires_grad and t.is_leaf):
            t = t.grad
            if t is None:
                continue
        found.append(t)
    return found


def _dense(t: torch.Tensor) -> bool:
    """Every element of t's extent is t's, once (contiguous in some order of its dimensions): order does not matter to a norm."""
    if t.is_contiguous():
        return True
    need = 1
    for s, m in sorted((s, m) for s, m in zip(t.stride(), t.shape) if m != 1):
        if s != need:
            return False
        need *= m
    return True


def _check(grads: Sequence[torch.Tensor], what: str) -> torch.device:
    device = grads[0].device
    for t in grads:
        if t.layout != torch.strided:
            raise TypeError(f"{what}: sparse gradients are not supported")
        if t.dtype not in OUT_CODES:
            raise TypeError(f"{what}: float32, float16 or bfloat16 tensors, got {t.dtype}")
        if t.device != device:
            raise ValueError(f"{what}: the tensors are on {device} and {t.device}: clip each device's by itself")
    if device.type != "cuda":
        raise ValueError(f"{what}: the tensors must be on the GPU (there is no CPU path)")
    return device


def _run(grads, outs, kind, max_norm, device) -> torch.Tensor:
    norm = torch.empty((), dtype=torch.float32, device=device)
    n = len(grads)
    partials = torch.empty(N.grad_partials(n), dtype=torch.float64, device=device)
    N.grad_clip([t.data_ptr() for t in grads], [t.numel() for t in grads], [OUT_CODES[t.dtype] for t in grads],
                None if outs is None else [t.data_ptr() for t in outs], None if outs is None else [OUT_CODES[t.dtype] for t in outs],
                kind, max_norm, partials.data_ptr(), norm.data_ptr(), device.index, torch.cuda.current_stream(device).cuda_stream)
    return norm


def _kind(norm_type: float) -> int:
    try:
        return _KINDS[float(norm_type)]
    except KeyError:
        raise ValueError(f"norm_type is 2 or inf, got {norm_type}") from None


@torch.no_grad()
def grad_norm(tensors: Union[torch.Tensor, Iterable[torch.Tensor]], norm_type: float = 2.0) -> torch.Tensor:
    """Norm over all values of all tensors (of their gradients, where they are parameters): a float32 scalar on their device.
    float32, float16 and bfloat16 tensors of any shape on one GPU; norm_type 2 or inf.  Nothing given: 0."""
    kind = _kind(norm_type)
    require_gpu()
    grads = _gradients(tensors)
    if not grads:
        return torch.zeros((), device="cuda")
    device = _check(grads, "grad_norm")
    return _run([t if _dense(t) else t.contiguous() for t in grads], None, kind, 0.0, device)


@torch.no_grad()
def clip_grad_norm(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
                   error_if_nonfinite: bool = False, out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Scales the gradients of `parameters` (or the tensors themselves, where they are no parameters) by
    min(1, max_norm / (norm + 1e-6)), in place, and returns their norm, as torch.nn.utils.clip_grad_norm_ does; a NaN norm makes
    every gradient NaN.  With `out` (one contiguous tensor per gradient, same number of elements, any of the three types) the
    scaled gradients go there and the gradients stay as they are.  The tensors must not share memory.
    error_if_nonfinite=True waits for the norm and raises before anything is scaled."""
    kind = _kind(norm_type)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError("max_norm must be a number >= 0")
    require_gpu()
    grads = _gradients(parameters)
    if out is not None:
        out = list(out)
        if len(out) != len(grads):
            raise ValueError(f"out holds {len(out)} tensors for {len(grads)} gradients")
    if not grads:
        return torch.zeros((), device="cuda")
    device = _check(grads, "clip_grad_norm")
    if error_if_nonfinite:
        norm = grad_norm(grads, norm_type)
        if not bool(torch.isfinite(norm)):
            raise RuntimeError(f"the norm of the gradients is {float(norm)}: nothing was scaled")
    if out is not None:
        _check(out, "clip_grad_norm: out")
        for g, o in zip(grads, out):
            if o.device != device or o.numel() != g.numel() or not o.is_contiguous():
                raise ValueError(f"out: contiguous tensors on {device} with their gradient's number of elements")
        return _run([t.contiguous() for t in grads], out, kind, max_norm, device)
    if all(t.is_contiguous() or _dense(t) for t in grads):
        return _run(grads, grads, kind, max_norm, device)
    # views with gaps: their values pass through a packed copy
    for t in grads:
        if any(s == 0 and m > 1 for s, m in zip(t.stride(), t.shape)):
            raise ValueError("clip_grad_norm cannot write an expanded gradient")
    packed = [t if _dense(t) else t.contiguous() for t in grads]
    norm = _run(packed, packed, kind, max_norm, device)
    for t, p in zip(grads, packed):
        if p is not t:
            t.copy_(p)
    return norm
