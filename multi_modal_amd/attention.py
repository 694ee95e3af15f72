"""Attention over the encoders' tokens on the device, forward and backward (csrc/attention.hip, csrc/attention_backward.hip).

Stands where the encoders' Attention.forward (classification/vggsound/models/vit_model.py:43-69) forms its score tensor, takes a softmax
and multiplies by the values, and adds what batches of clips need next to it: documents of different lengths (padded or packed),
causal and prefix masks, capped scores, a bias that falls with distance, key heads shared by query heads, and one or a few new tokens over
what a stream has kept.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch

from . import _native as N
from .plans import OUT_CODES, once_differentiable, raw_stream, refuse_forward_mode, require_gpu

_ARGS_SIZE = ctypes.sizeof(N.AttentionArgs)
_GRADS_SIZE = ctypes.sizeof(N.AttentionGrads)
_DTYPES = (torch.float16, torch.bfloat16)
_LARGEST = torch.finfo(torch.float32).max
_SCALES = (2.0 ** -90, 2.0 ** 126)


def _rows(t: torch.Tensor) -> Tuple[torch.Tensor, Tuple[int, int, int]]:
    """t itself when the kernels can read it where it is (unit stride inside the heads, 16-byte pieces), else a packed copy; and its
    (batch, row, head) strides, 0 where there is one entry."""
    if t.dim() == 4:
        b, n, h, e = t.stride()
        m = t.shape
        s = (b if m[0] > 1 else 0, n if m[1] > 1 else 0, h if m[2] > 1 else 0)
    else:
        n, h, e = t.stride()
        m = t.shape
        s = (0, n if m[0] > 1 else 0, h if m[1] > 1 else 0)
    if e == 1 and t.data_ptr() % 16 == 0 and (s[0] | s[1] | s[2]) % 8 == 0 and s[1] <= 1 << 24:
        return t, s
    return _dense(t), _packed_strides(t)


def _packed_strides(t: torch.Tensor) -> Tuple[int, int, int]:
    """Strides of a contiguous tensor of t's shape."""
    h, d = t.shape[-2], t.shape[-1]
    return (t.shape[-3] * h * d if t.dim() == 4 else 0, h * d, d)


def _dense(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """t, or a copy of it, contiguous and on a 16-byte boundary."""
    if t is None or (t.is_contiguous() and t.data_ptr() % 16 == 0):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _counts(x, name: str, n: int, device, limit: Optional[int] = None, rising: bool = False) -> Optional[torch.Tensor]:
    """Per-document integers as the int32 device tensor the kernels read; what the host holds is checked, what the device holds is
    clamped by the kernels."""
    if x is None:
        return None
    if type(x) is torch.Tensor and x.dtype == torch.int32 and x.is_cuda and x.device == device and x.shape == (n,) and x.is_contiguous():
        return x
    t = x if isinstance(x, torch.Tensor) else torch.tensor(x, dtype=None if len(x) else torch.int32)
    if t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
        raise TypeError(f"{name} must be integers")
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name} must hold {n} entries, got {tuple(t.shape)}")
    if not t.is_cuda and n > 0:
        if int(t.min()) < 0 or (limit is not None and int(t.max()) > limit):
            raise ValueError(f"{name} must lie in [0, {limit}]" if limit is not None else f"{name} must not be negative")
        if rising and bool((t[1:] < t[:-1]).any()):
            raise ValueError(f"{name} must not fall")
    if t.dtype != torch.int32 or t.device != device or not t.is_contiguous():
        if t.dtype == torch.int64:                         # entries past 32 bits are out of range, and stay so
            t = t.clamp(-1, 2**31 - 1)
        t = t.to(device=device, dtype=torch.int32).contiguous()
    return t


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


class _Call:
    """One checked call: what does not depend on its tensors.  `counts` are q_len, k_len, q_off, k_off, prefix and slopes; `strides`
    those of q, k and v as the forward pass reads them."""

    __slots__ = ("packed", "causal", "n_docs", "scale", "cap", "counts", "device", "strides", "backward_bytes")

    def args(self, q, k, v, out, rest, lse, counts, strides) -> bytes:
        H, n = q.shape[-2], q.shape[-3]
        return N.pack_attention(
            _ARGS_SIZE, OUT_CODES[q.dtype], self.n_docs, H, k.shape[-2], q.shape[-1], self.packed, self.causal, self.scale, self.cap, n, k.shape[-3],
            q.data_ptr(), k.data_ptr(), v.data_ptr(), *map(_ptr, counts), _ptr(out), _ptr(rest), _ptr(lse), *strides, *_packed_strides(q), H * n, n)

    def forward(self, q, k, v, want_lse: bool, gradients: bool = False):
        device = q.device
        out = torch.empty(q.shape, dtype=q.dtype, device=device)
        rest = lse = None
        if want_lse:
            shape = (q.shape[-2], q.shape[-3])
            lse = torch.empty(shape if self.packed else (q.shape[0],) + shape, dtype=torch.float32, device=device)
        args = self.args(q, k, v, out, None, lse, self.counts, self.strides)
        if gradients:
            self.backward_bytes = N.attention_workspace(args, backward=True)
            if self.backward_bytes:            # 0: the backward pass reads neither out nor its rest
                rest = torch.empty(q.shape, dtype=q.dtype, device=device)
                args = self.args(q, k, v, out, rest, lse, self.counts, self.strides)
        need = N.attention_workspace(args) if k.shape[-3] > 512 else 0
        work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        N.attention_forward(args, _ptr(work), self.device, raw_stream(self.device))
        return out, rest, lse


def _form(tensors) -> list:
    return [None if t is None else (t.shape, t.dtype, t.get_device(), t.stride()) for t in tensors]


class _AttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, call):
        out, rest, lse = call.forward(q, k, v, True, True)
        ctx.call = call
        # the counts too: autograd then notices when one of them has been changed before the backward pass
        saved = (q, k, v, out if call.backward_bytes else None, rest, lse, *call.counts)
        ctx.form = _form(saved)
        ctx.save_for_backward(*saved)
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)       # or every backward pass fills a gradient of lse's shape with zeros that nothing reads
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out, _):
        # Saved-tensor hooks (torch.autograd.graph.save_on_cpu, checkpoints) return equal values in any layout: every address below is taken
        # from what was unpacked, and the forward pass's strides serve only where they are still the tensors' own.
        saved, call = ctx.saved_tensors, ctx.call
        q, k, v, out, rest, lse, *counts = saved
        if grad_out is None:                   # an operation behind this one returned no gradient
            return tuple(torch.zeros_like(t) if needed else None for t, needed in zip((q, k, v), ctx.needs_input_grad)) + (None,)
        strides, form = call.strides, _form(saved)
        if form != ctx.form:
            for new, old in zip(form, ctx.form):
                if (new and new[:3]) != (old and old[:3]):
                    raise RuntimeError(f"attention: a saved-tensor hook returned {new} in place of {old} (shape, type, device, strides)")
            lse, *counts = (None if t is None else t.contiguous() for t in (lse, *counts))
        if form != ctx.form or (q.data_ptr() | k.data_ptr() | v.data_ptr()) % 16 or (out is not None and (out.data_ptr() | rest.data_ptr()) % 16):
            (q, q_stride), (k, k_stride), (v, v_stride) = _rows(q), _rows(k), _rows(v)
            strides = q_stride + k_stride + v_stride
            out, rest = _dense(out), _dense(rest)
        g, g_stride = _rows(grad_out)
        gq, gk, gv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        kv_stride = _packed_strides(gk)
        grads = N.pack_attention_grads(_GRADS_SIZE, 0, g.data_ptr(), gq.data_ptr(), gk.data_ptr(), gv.data_ptr(), *g_stride, *_packed_strides(gq), *kv_stride, *kv_stride)
        work = torch.empty(call.backward_bytes, dtype=torch.uint8, device=q.device) if call.backward_bytes else None
        N.attention_backward(call.args(q, k, v, out, rest, lse, counts, strides), grads, _ptr(work), call.device, raw_stream(call.device))
        need = ctx.needs_input_grad
        return gq if need[0] else None, gk if need[1] else None, gv if need[2] else None, None


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, lengths=None, kv_lengths=None, offsets=None, kv_offsets=None, causal: bool = False,
              prefix=None, slopes=None, cap: float = 0.0, scale: Optional[float] = None,
              return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """softmax(scores) v over the tokens of each document; float16 or bfloat16, differentiable in q, k and v.

    Padded: q (B, N, H, D), k and v (B, S, K, D), a document per batch entry; `lengths` (B,) valid rows of q (default: all),
    `kv_lengths` (B,) valid rows of k and v (default: `lengths` when S == N, else all).  K divides H: query head h reads key head
    h // (H // K).  D: a multiple of 8 up to 128.  Any strides (views of a packed projection are read where they are).
    Packed: q (T, H, D), k and v (S, K, D) with `offsets` (documents + 1,): document d holds rows offsets[d] .. offsets[d + 1] - 1, and
    of the keys those that `kv_offsets` (default: `offsets`) cuts out.

    Scores are scale * q . k (default scale: D ** -0.5); cap > 0 makes them cap * tanh(score / cap); `slopes` (H,) subtracts
    slopes[h] * |distance| (row i stands at key position i + len_k - len_q: the last row meets the last key).  causal=True hides the keys
    behind a row's position, except the first `prefix[d]` keys of a document when `prefix` (one per document) is given.
    Rows that see no key, and rows no document holds, give zeros, no gradients, and lse = -inf.

    `lengths`, `offsets` and `prefix` may be integer tensors on the GPU (not read back; entries out of range are clamped) or on the
    host (checked).  return_lse=True also returns the float32 log-sum-exp of each row's scores, (B, H, N) or (H, T), without gradient.
    Second derivatives and forward-mode derivatives are refused.  Tensors on the CPU are copied over and the result is copied back."""
    dtype = q.dtype
    if dtype not in _DTYPES or k.dtype != dtype or v.dtype != dtype:
        raise TypeError(f"attention takes float16 or bfloat16 tensors of one type, got {q.dtype}, {k.dtype}, {v.dtype}")
    packed = offsets is not None
    qs, ks = q.shape, k.shape
    dims = 3 if packed else 4
    if len(qs) != dims or len(ks) != dims or v.dim() != dims:
        raise ValueError("attention takes (batch, tokens, heads, head size) tensors, or (tokens, heads, head size) with offsets")
    if ks != v.shape or ks[-1] != qs[-1] or (not packed and ks[0] != qs[0]):
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit together")
    H, D, K = qs[-2], qs[-1], ks[-2]
    if K < 1 or H < 1 or H % K != 0:
        raise ValueError(f"{H} query heads cannot share {K} key heads")
    if D < 8 or D > 128 or D % 8 != 0:
        raise ValueError(f"head size {D}: a multiple of 8 up to 128")
    device = origin = q.device
    if k.device != device or v.device != device:
        raise ValueError("q, k and v must be on one device")
    call = _Call()
    call.cap = float(cap)
    call.scale = D ** -0.5 if scale is None else float(scale)
    # as the float32 that the kernels take: a cap that rounds to zero would be none, and below the least scale a row without keys would get weights
    if not (0.0 <= call.cap <= _LARGEST and (call.cap == 0.0 or ctypes.c_float(call.cap).value > 0.0)) or not _SCALES[0] <= call.scale <= _SCALES[1]:
        raise ValueError("cap must be 0 or a positive float32, and scale lie between 2^-90 and 2^126")
    if prefix is not None and not causal:
        raise ValueError("prefix belongs to causal=True")
    if packed and (lengths is not None or kv_lengths is not None):
        raise ValueError("lengths belong to the padded form: documents that are packed have offsets")
    if not packed and kv_offsets is not None:
        raise ValueError("kv_offsets needs offsets")
    n, s = qs[-3], ks[-3]
    if packed:
        m = len(offsets) - 1
        if m < 0:
            raise ValueError("offsets holds at least one entry")
        if kv_offsets is None and s != n:
            raise ValueError(f"{n} rows and {s} keys: kv_offsets says how the keys are cut")
    else:
        m = qs[0]
        if kv_lengths is None and s == n:
            kv_lengths = lengths
    refuse_forward_mode("attention", q, k, v)
    if not q.is_cuda:
        require_gpu()
        q, k, v = q.cuda(), k.cuda(), v.cuda()
        device = q.device
    call.device = device.index
    call.packed, call.causal, call.n_docs = packed, bool(causal), m
    q_len = k_len = q_off = k_off = None
    if packed:
        q_off = _counts(offsets, "offsets", m + 1, device, n, rising=True)
        k_off = q_off if kv_offsets is None else _counts(kv_offsets, "kv_offsets", m + 1, device, s, rising=True)
    else:
        q_len = _counts(lengths, "lengths", m, device, n)
        k_len = q_len if kv_lengths is lengths and s == n else _counts(kv_lengths, "kv_lengths", m, device, s)
    prefix = _counts(prefix, "prefix", m, device)
    if slopes is not None:
        t = torch.as_tensor(slopes)
        if tuple(t.shape) != (H,):
            raise ValueError(f"slopes must hold one entry per query head ({H}), got {tuple(t.shape)}")
        if t.requires_grad:
            raise ValueError("slopes have no gradient: detach them")
        slopes = t.to(device=device, dtype=torch.float32).contiguous()
    call.counts = (q_len, k_len, q_off, k_off, prefix, slopes)
    (q, q_stride), (k, k_stride), (v, v_stride) = _rows(q), _rows(k), _rows(v)
    call.strides = q_stride + k_stride + v_stride
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out, lse = _AttentionFn.apply(q, k, v, call)
    else:
        out, _, lse = call.forward(q, k, v, return_lse)
    if device != origin:
        out, lse = out.to(origin), None if lse is None else lse.to(origin)
    return (out, lse) if return_lse else out
