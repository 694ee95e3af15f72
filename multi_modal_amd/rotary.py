"""Rotary positions with several axes for the query and key heads of an encoder layer.

The tokens PatchEmbed makes sit on a grid - frequency and time for a spectrogram, height and width for an image, with a time axis
in front for video - and every axis turns its own share of each head's element pairs (csrc/rotary.hip):

    (x, y) -> (x cos phi - y sin phi, y cos phi + x sin phi)        phi = position[axis] * theta

The reference adds a learned table to the tokens instead (classification/vggsound/models/vit_model.py:384-385), which ties an
encoder to one clip length; there is no rotary code in it.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _native as N
from .plans import OUT_CODES, folded as _folded, mark_written, once_differentiable, raw_stream, refuse_forward_mode, require_gpu

_ARGS_SIZE = ctypes.sizeof(N.RotaryArgs)

_LADDERS = {"shared": N.ROTARY_SHARED, "axis": N.ROTARY_PER_AXIS}
_PAIRINGS = {"halves": N.ROTARY_HALVES, "adjacent": N.ROTARY_ADJACENT}


def grid_positions(*sizes: int, device=None) -> torch.Tensor:
    """Positions of the tokens of a grid, last axis fastest (the order of PatchEmbed's tokens: `grid_positions(H // 16, W // 16)`):
    (len(sizes), prod(sizes)) int32."""
    if not sizes or any(int(n) < 0 for n in sizes):
        raise ValueError("grid_positions takes one size >= 0 per axis")
    axes = torch.meshgrid(*[torch.arange(int(n), dtype=torch.int32, device=device) for n in sizes], indexing="ij")
    return torch.stack([a.reshape(-1) for a in axes])


def _gpu_index(device: Union[None, int, str, torch.device]) -> Optional[int]:
    """Index of a GPU, None for the current one."""
    if device is None:
        return None
    d = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
    if d.type != "cuda":
        raise ValueError(f"the frequency table lives on a GPU, not on {d}")
    return d.index


class Rotary:
    """Rotary(sections): sections[a] = element pairs of a head that axis a turns (1 to 4 axes, 2 * sum(sections) <= head size; the
    elements behind them pass through).

    ladder "shared": pair i of all R = sum(sections) turns with base ** (-i / R); "axis": the j-th pair of axis a with
    base ** (-j / sections[a]).  pairing "halves": elements (i, i + R) form a pair; "adjacent": elements (2 i, 2 i + 1).
    The frequency table lives on the GPU `device` (an index, "cuda", "cuda:1", a torch.device; default: the current one); the object may be shared between threads and streams."""

    def __init__(self, sections: Sequence[int], base: float = 10000.0, ladder: str = "axis", pairing: str = "halves",
                 device: Union[None, int, str, torch.device] = None):
        self.sections = tuple(int(s) for s in sections)
        if ladder not in _LADDERS or pairing not in _PAIRINGS:
            raise ValueError("ladder is 'shared' or 'axis', pairing is 'halves' or 'adjacent'")
        if not 1 <= len(self.sections) <= 4 or any(s < 0 for s in self.sections) or not 1 <= sum(self.sections) <= 512:
            raise ValueError(f"sections: 1 to 4 axes with 1 to 512 pairs together, got {self.sections}")
        if not 0.0 < float(base) < float("inf"):
            raise ValueError("base must be a positive number")
        index = _gpu_index(device)
        require_gpu()
        self.base, self.ladder, self.pairing = float(base), ladder, pairing
        self._pairs2 = 2 * sum(self.sections)
        self.device = torch.cuda.current_device() if index is None else index
        self._h = N.RotaryHandle(self.sections, _LADDERS[ladder], _PAIRINGS[pairing], self.base, self.device)

    def __call__(self, q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
                 inplace: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
        """q: (B, N, H, D); k: (B, N, K, D) of the same type, or None; float32, float16 or bfloat16, any strides (views of a packed
        projection are read where they are).  positions: (axes, N), the same for every batch entry, or (axes, B, N); integers of any
        sign and size.  Returns new contiguous tensors (q', k'), or q' alone when k is None; float32 arithmetic, rounded once, angles
        in float64.  Differentiable in q and k (once, in reverse mode).
        inplace=True writes the result over q and k (no gradients; the two must not share elements) and returns them.
        Tensors on the CPU are copied over and the results copied back."""
        origin = q.device
        dtype, shape = q.dtype, q.shape
        if len(shape) != 4 or (k is not None and k.dim() != 4):
            raise ValueError("q and k are (batch, tokens, heads, head size) tensors")
        if dtype not in OUT_CODES or (k is not None and (k.dtype != dtype or k.device != origin)):
            raise ValueError("q and k must both be float32, float16 or bfloat16 on one device")
        B, n, _, D = shape
        if k is not None and (k.shape[0] != B or k.shape[1] != n or k.shape[3] != D):
            raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} differ in batch, tokens or head size")
        if not self._pairs2 <= D <= 1024:
            raise ValueError(f"head size {D}: the sections {self.sections} need {self._pairs2} elements (1024 at most)")
        kind = positions.dtype
        if kind != torch.int32 and kind != torch.int64:
            if kind.is_floating_point or kind.is_complex or kind == torch.bool:
                raise TypeError("positions must be integers")
            positions = positions.to(torch.int64)
        A = len(self.sections)
        if tuple(positions.shape) not in ((A, n), (A, B, n)):
            raise ValueError(f"positions must be ({A}, {n}) or ({A}, {B}, {n}), got {tuple(positions.shape)}")
        given = (q,) if k is None else (q, k)
        refuse_forward_mode("Rotary", *given)
        if inplace:
            if torch.is_grad_enabled() and any(t.requires_grad for t in given):
                raise RuntimeError("inplace=True has no gradient: use it under torch.no_grad()")
            if not q.is_cuda:
                raise ValueError("inplace=True takes tensors on the GPU")
            if any(map(_folded, given)):
                raise ValueError("inplace=True cannot write a tensor whose elements share memory")
            if k is not None and _share(q, k):
                raise ValueError("inplace=True: q and k share elements")
            if any(t.stride(3) != 1 and D > 1 for t in given):
                raise ValueError("inplace=True needs a unit stride inside the heads")
        if not q.is_cuda:
            q, k = q.cuda(self.device), None if k is None else k.cuda(self.device)
        if q.get_device() != self.device:
            raise ValueError(f"tensors on {q.device} but the frequency table is on cuda:{self.device}")
        if positions.get_device() != self.device:
            positions = positions.to(q.device)
        if not inplace and torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
            out = _RotaryFn.apply(q, k, positions, self)
            yq, yk = out if k is not None else (out, None)
        else:
            yq, yk = self._run(q, k, positions, False, inplace)
            if inplace:
                mark_written(given)
        if q.device != origin:
            yq, yk = yq.to(origin), None if yk is None else yk.to(origin)
        return yq if yk is None else (yq, yk)

    forward = __call__

    def _run(self, q, k, positions, inverse: bool, inplace: bool = False):
        some = q if q is not None else k
        B, n, _, D = some.shape
        if q is not None and q.stride(3) != 1 and D > 1:
            q = q.contiguous()
        if k is not None and k.stride(3) != 1 and D > 1:
            k = k.contiguous()
        yq = q if inplace or q is None else torch.empty(q.shape, dtype=q.dtype, device=q.device)
        yk = k if inplace or k is None else torch.empty(k.shape, dtype=k.dtype, device=k.device)
        if B * n == 0:
            return yq, yk
        zero = (0, 0, 0)
        ps = positions.stride()
        qh, qp, yqp, qs, yqs = (0, 0, 0, zero, zero) if q is None else (q.shape[2], q.data_ptr(), yq.data_ptr(), q.stride()[:3], yq.stride()[:3])
        kh, kp, ykp, ks, yks = (0, 0, 0, zero, zero) if k is None else (k.shape[2], k.data_ptr(), yk.data_ptr(), k.stride()[:3], yk.stride()[:3])
        self._h.run(N.pack_rotary(_ARGS_SIZE, OUT_CODES[some.dtype], positions.dtype == torch.int64, inverse, qh, kh, D, 0, B, n, qp, yqp, kp, ykp,
                                  *qs, *yqs, *ks, *yks, positions.data_ptr(), *((ps[0], 0, ps[1]) if len(ps) == 2 else ps)), raw_stream(self.device))
        return yq, yk

    def close(self) -> None:
        self._h.close()


def _share(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two (B, N, H, D) tensors hold a common element: exact for views that differ in their head range only (cuts of one
    packed projection), by their extents otherwise."""
    def extent(t):
        return t.data_ptr(), t.data_ptr() + (sum((m - 1) * s for m, s in zip(t.shape, t.stride())) + 1) * t.element_size()
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = extent(a), extent(b)
    if a1 <= b0 or b1 <= a0:
        return False
    if a.stride()[:2] == b.stride()[:2] and all(s >= 0 for s in a.stride() + b.stride()):
        # per token, heads [first, last) of one row: disjoint when the rows' head ranges are, and fit into the token stride
        ra, rb = extent(a[0, 0]), extent(b[0, 0])
        row = min([s for s, m in zip(a.stride()[:2], a.shape[:2]) if m > 1], default=1 << 62) * a.element_size()
        return not ((ra[1] <= rb[0] or rb[1] <= ra[0]) and max(ra[1], rb[1]) - min(ra[0], rb[0]) <= row)
    return True


class _RotaryFn(torch.autograd.Function):
    """The gradient of a rotation is the rotation by the negative angle."""

    @staticmethod
    def forward(ctx, q, k, positions, rotary):
        ctx.rotary = rotary
        ctx.save_for_backward(positions)
        yq, yk = rotary._run(q, k, positions, False)
        return yq if k is None else (yq, yk)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        gq = grads[0] if ctx.needs_input_grad[0] else None
        gk = grads[1] if len(grads) > 1 and ctx.needs_input_grad[1] else None
        if gq is not None or gk is not None:
            gq, gk = ctx.rotary._run(gq, gk, ctx.saved_tensors[0], True)
        return gq, gk, None, None
