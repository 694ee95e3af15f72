"""Global gradient norm over many tensors, and clipping by it (csrc/gradients.hip).

What a training step of an encoder with PatchEmbedLayer does between `loss.backward()` and `optimizer.step()`; the reference's loops
go straight to the optimizer (classification/vggsound/vanilla_single.py:75-80).  Semantics of torch.nn.utils.clip_grad_norm_, with
the sums in float64 and in a fixed order, two launches for about a hundred tensors, and an optional second set of tensors (of
another type, e.g. the float32 gradients an optimizer takes) that the clipped gradients go to.
"""
from __future__ import annotations

import math
from operator import attrgetter
from typing import Iterable, List, Optional, Sequence, Tuple, Union

import torch

from . import _native as N
from .plans import OUT_CODES, folded, mark_written, raw_stream, require_gpu

_KINDS = {2.0: N.NORM_2, math.inf: N.NORM_MAX}


def _gradients(tensors: Union[torch.Tensor, Iterable[torch.Tensor]]) -> List[torch.Tensor]:
    """Gradients of a list of parameters (those that have one), or the tensors of the list themselves."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    kinds = set(map(type, tensors))
    if kinds == _PLAIN and not any(map(_requires_grad, tensors)):        # the two usual lists, walked in C
        return tensors
    if kinds == _PARAMETERS:
        return [g for g in map(_grad, tensors) if g is not None]
    found = []
    for t in tensors:
        if (t.requires_grad and t.is_leaf) or isinstance(t, torch.nn.Parameter):
            t = t.grad
            if t is None:
                continue
        found.append(t)
    return found


_PLAIN, _PARAMETERS = {torch.Tensor}, {torch.nn.Parameter}
_dtype, _grad, _requires_grad = attrgetter("dtype"), attrgetter("grad"), attrgetter("requires_grad")


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


def _check(tensors: Sequence[torch.Tensor], what: str) -> Tuple[int, List[int], bool]:
    """(device index, type codes, all contiguous)"""
    codes = list(map(OUT_CODES.get, map(_dtype, tensors)))
    devices = set(map(torch.Tensor.get_device, tensors))
    if None in codes:
        raise TypeError(f"{what}: float32, float16 or bfloat16 tensors, got {tensors[codes.index(None)].dtype}")
    if -1 in devices:
        raise ValueError(f"{what}: the tensors must be on the GPU (there is no CPU path)")
    if len(devices) > 1:
        raise ValueError(f"{what}: the tensors are on GPUs {sorted(devices)}: clip each device's by itself")
    contiguous = all(map(torch.Tensor.is_contiguous, tensors))
    if not contiguous and any(t.layout != torch.strided for t in tensors):           # a sparse tensor is not contiguous
        raise TypeError(f"{what}: sparse gradients are not supported")
    return devices.pop(), codes, contiguous


def _run(grads, codes, outs, out_codes, kind, max_norm, device: int) -> torch.Tensor:
    n = len(grads)
    # the float32 norm stands behind the call's float64 partial sums
    work = torch.empty(N.grad_partials(n) + 1, dtype=torch.float64, device=grads[0].device)
    norm = work[-1:].view(torch.float32)[0]
    ptrs = map(torch.Tensor.data_ptr, grads)
    N.grad_clip(ptrs, map(torch.Tensor.numel, grads), codes, None if outs is None else ptrs if outs is grads else map(torch.Tensor.data_ptr, outs),
                out_codes, kind, max_norm, work.data_ptr(), norm.data_ptr(), device, raw_stream(device))
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
    grads = _gradients(tensors)
    if not grads:
        require_gpu()
        return torch.zeros((), device="cuda")
    device, codes, contiguous = _check(grads, "grad_norm")
    return _run(grads if contiguous else [t if _dense(t) else t.contiguous() for t in grads], codes, None, None, kind, 0.0, device)


@torch.no_grad()
def clip_grad_norm(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
                   error_if_nonfinite: bool = False, out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Scales the gradients of `parameters` (or the tensors themselves, where they are no parameters) by
    min(1, max_norm / (norm + 1e-6)), in place, and returns their norm, as torch.nn.utils.clip_grad_norm_ does: a NaN norm makes
    every gradient NaN, an infinite one finite gradients zero (NaN where max_norm is infinite too).  With `out` (one contiguous tensor
    per gradient, same number of elements, any of the three types) the
    scaled gradients go there and the gradients stay as they are.  The tensors must not share memory.
    error_if_nonfinite=True waits for the norm and raises before anything is scaled."""
    kind = _kind(norm_type)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError("max_norm must be a number >= 0")
    grads = _gradients(parameters)
    if out is not None:
        out = list(out)
        if len(out) != len(grads):
            raise ValueError(f"out holds {len(out)} tensors for {len(grads)} gradients")
    if not grads:
        require_gpu()
        return torch.zeros((), device="cuda")
    device, codes, contiguous = _check(grads, "clip_grad_norm")
    if error_if_nonfinite:
        norm = grad_norm(grads, norm_type)
        if not bool(torch.isfinite(norm)):
            raise RuntimeError(f"the norm of the gradients is {float(norm)}: nothing was scaled")
    if out is not None:
        out_device, out_codes, packed = _check(out, "clip_grad_norm: out")
        if out_device != device or not packed or list(map(torch.Tensor.numel, out)) != list(map(torch.Tensor.numel, grads)):
            raise ValueError(f"out: contiguous tensors on GPU {device} with their gradient's number of elements")
        norm = _run(grads if contiguous else [t.contiguous() for t in grads], codes, out, out_codes, kind, max_norm, device)
        mark_written(out)
        return norm
    if contiguous or all(map(_dense, grads)):
        norm = _run(grads, codes, grads, codes, kind, max_norm, device)
        mark_written(grads)
        return norm
    # views with gaps: their values pass through a packed copy, so the library does not see what they share
    if any(map(folded, grads)):
        raise ValueError("clip_grad_norm cannot write a gradient whose elements share memory (an expanded view)")
    starts = [t.data_ptr() for t in grads if t.numel()]
    if len(set(starts)) < len(starts):
        raise ValueError("clip_grad_norm: two of the gradients share memory (the same gradient given twice?)")
    packed = [t if _dense(t) else t.contiguous() for t in grads]
    norm = _run(packed, codes, packed, codes, kind, max_norm, device)
    mark_written(packed)
    for t, p in zip(grads, packed):
        if p is not t:
            t.copy_(p)
    return norm
