"""Refusals of the token operators that need no GPU: argument checks of the Python entry points and of the C entries, which look at
everything they can on the host before a device is touched."""
import ctypes
import math

import pytest
import torch


@pytest.fixture(scope="module")
def N():
    from multi_modal_amd import _native
    _native.load_library()
    return _native


@pytest.mark.parametrize("kw", [dict(sections=[]), dict(sections=[1] * 5), dict(sections=[0, 0]), dict(sections=[-1, 4]), dict(sections=[513]),
                                dict(sections=[4], ladder="both"), dict(sections=[4], pairing="third"), dict(sections=[4], base=0.0),
                                dict(sections=[4], base=math.inf), dict(sections=[4], base=math.nan)])
def test_rotary_constructor_refuses(N, kw):
    from multi_modal_amd.rotary import Rotary
    with pytest.raises(ValueError):
        Rotary(**kw)


def test_grid_positions():
    from multi_modal_amd.rotary import grid_positions
    p = grid_positions(2, 3)
    assert p.dtype == torch.int32 and p.tolist() == [[0, 0, 0, 1, 1, 1], [0, 1, 2, 0, 1, 2]]
    assert grid_positions(4, 0, 2).shape == (3, 0)
    with pytest.raises(ValueError):
        grid_positions()


def test_rotary_entries_refuse(N):
    lib = N.load_library()
    h = ctypes.c_void_p()
    def create(sections, ladder=0, pairing=0, base=10000.0):
        s = (ctypes.c_int32 * max(1, len(sections)))(*sections)
        return lib.mmfe_rotary_create(len(sections), s, ladder, pairing, base, 0, ctypes.byref(h))
    for args in (([],), ([1] * 5,), ([0],), ([-3, 5],), ([300, 300],), ([4], 2), ([4], 0, 2), ([4], 0, 0, -1.0), ([4], 0, 0, math.nan)):
        assert create(*args) == -1 and h.value is None, args
    assert lib.mmfe_rotary_create(1, None, 0, 0, 10000.0, 0, ctypes.byref(h)) == -1
    assert lib.mmfe_rotary_run(None, None, None) == -1
    assert lib.mmfe_rotary_destroy(None) == 0
    if not torch.cuda.is_available():
        assert create([4]) == -2                       # no device: no CPU path


def test_struct_sizes_match_header(N):
    """The ctypes structures have the C layout (8-byte members on 8-byte boundaries, no padding inside)."""
    assert ctypes.sizeof(N.RotaryArgs) == 8 * 4 + 2 * 8 + 4 * 8 + 12 * 8 + 8 + 3 * 8
    # ... and the packed bytes are those of the structures
    for cls, pack in ((N.RotaryArgs, N.pack_rotary), (N.AttentionArgs, N.pack_attention), (N.AttentionGrads, N.pack_attention_grads)):
        s, values = cls(), []
        for i, (name, kind) in enumerate(cls._fields_):
            n = getattr(kind, "_length_", 1)
            v = [float(i) + 0.5] if kind is ctypes.c_float else [1000 * i + j + 1 for j in range(n)]
            setattr(s, name, kind(*v) if n > 1 else v[0])
            values += v
        assert bytes(s) == pack(*values), cls.__name__


def clip(N, ptrs, numels, dtypes, outs=None, out_dtypes=None, kind=2, max_norm=1.0, partials=64, norm=64):
    lib, n = N.load_library(), len(ptrs)
    vp, i64, i32 = ctypes.c_void_p * max(1, n), ctypes.c_int64 * max(1, n), ctypes.c_int32 * max(1, n)
    return lib.mmfe_grad_clip(n, vp(*ptrs), i64(*numels), i32(*dtypes), None if outs is None else vp(*outs),
                              None if out_dtypes is None else i32(*out_dtypes), kind, max_norm, partials, norm, 99, None)


def test_clip_entry_refuses(N):
    """Every call names device 99: one that passes the checks is refused for that (-2 or -3), nothing is launched."""
    A, B = 1 << 20, 1 << 21
    ok = clip(N, [A, B], [100, 50], [0, 0], [A, B], [0, 0])
    assert ok not in (0, -1)
    assert clip(N, [A, B], [100, 50], [0, 2], [A, B], [0, 2], kind=0) == ok
    assert clip(N, [A, A + 200], [100, 50], [2, 0], [A, A + 200], [2, 0]) == ok          # behind one another
    bad = [
        clip(N, [A, B], [100, 50], [0, 0], [A, B], [0, 0], kind=1),
        clip(N, [A, B], [100, -1], [0, 0], [A, B], [0, 0]),
        clip(N, [A, B], [100, 50], [0, 3], [A, B], [0, 3]),
        clip(N, [A, None], [100, 50], [0, 0]),
        clip(N, [A, B + 2], [100, 50], [0, 0]),                                           # float32 off its alignment
        clip(N, [A, B], [100, 50], [0, 0], [A, B], [0, 0], max_norm=-1.0),
        clip(N, [A, B], [100, 50], [0, 0], [A, B], [0, 0], max_norm=math.nan),
        clip(N, [A, B], [100, 50], [0, 0], [A, None], [0, 0]),
        clip(N, [A, B], [100, 50], [0, 0], [A, B], None),
        clip(N, [A, A], [100, 100], [0, 0], [A, A], [0, 0]),                              # the same gradient twice
        clip(N, [A, A + 396], [100, 50], [0, 0], [A, A + 396], [0, 0]),                   # one element shared
        clip(N, [A], [100], [0], [A + 4], [0]),                                           # result shifted over its input
        clip(N, [A], [100], [0], [A], [1]),                                               # in place with another type
        clip(N, [A, B], [100, 50], [0, 0], partials=None),
        clip(N, [A, B], [100, 50], [0, 0], norm=None),
    ]
    assert bad == [-1] * len(bad)
    assert clip(N, [A, A], [100, 100], [0, 0]) == ok                                      # a norm alone may read a tensor twice
    assert N.load_library().mmfe_grad_partials(-1) == 0


def test_wrappers_refuse(N):
    from multi_modal_amd.gradients import clip_grad_norm, grad_norm
    x = torch.ones(4)
    with pytest.raises(ValueError, match="norm_type"):
        clip_grad_norm([x], 1.0, norm_type=1.0)
    with pytest.raises(ValueError, match="norm_type"):
        grad_norm([x], norm_type=3)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm([x], bad)
    with pytest.raises(ValueError, match="no CPU path"):
        clip_grad_norm([x], 1.0)
    if not torch.cuda.is_available():
        with pytest.raises(N.MmfeError):
            clip_grad_norm([], 1.0)


def test_share_of_views():
    """What inplace=True asks about its two tensors: cuts of one packed projection share nothing, overlapping cuts do."""
    from multi_modal_amd.rotary import _share
    qkv = torch.zeros(2, 5, 12, 8)
    assert not _share(qkv[:, :, :4], qkv[:, :, 4:8])
    assert _share(qkv[:, :, :5], qkv[:, :, 4:8])
    assert _share(qkv[:, :, :4], qkv[:, :, :4])
    assert not _share(torch.zeros(1, 2, 3, 4), torch.zeros(1, 2, 3, 4))
    assert _share(qkv[:, 1:, :4], qkv[:, :-1, :4])
    flat = torch.zeros(200)
    a = flat.as_strided((1, 5, 2, 8), (0, 16, 8, 1))
    b = flat.as_strided((1, 5, 2, 8), (0, 16, 8, 1), 16)      # the same tokens, one further on
    assert _share(a, b)


def test_clip_entry_takes_empty_tensors(N):
    """Tensors without elements have no address: two of them share nothing, whatever their types."""
    assert clip(N, [None, 1 << 20, None], [0, 10, 0], [0, 0, 1], [None, 1 << 20, None], [1, 0, 1]) not in (0, -1)


@pytest.mark.parametrize("opts", [dict(), dict(cap=2.0), dict(slope=0.3), dict(causal=True, prefix=3), dict(causal=True, cap=1.0, slope=0.1)])
def test_oracle_gradients_against_differences(opts):
    """The formulas the kernels' gradients are held to, against central differences in float64."""
    from oracle import token_oracle as O
    gen = torch.Generator().manual_seed(1)
    q, k, v, g = (torch.randn(n, 8, generator=gen, dtype=torch.float64) for n in (5, 7, 7, 5))
    r = O.attention_head(q, k, v, 0.4, g=g, **opts)
    for name, x in (("dq", q), ("dk", k), ("dv", v)):
        for _ in range(6):
            d = torch.randn(x.shape, generator=gen, dtype=torch.float64)
            h = 1e-5
            def loss(s):
                a = dict(dq=q, dk=k, dv=v)
                a[name] = x + s * d
                return float((O.attention_head(*a.values(), 0.4, **opts)["o"] * g).sum())
            assert abs((loss(h) - loss(-h)) / (2 * h) - float((r[name] * d).sum())) <= 1e-8 * (1 + float((r[name] * d).abs().sum()))
    # and against torch's own differentiation of softmax
    if not opts:
        qq, kk, vv = (t.clone().requires_grad_() for t in (q, k, v))
        o = torch.softmax(0.4 * qq @ kk.T, 1) @ vv
        assert torch.allclose(o, r["o"]) and all(torch.allclose(a, r[n]) for a, n in zip(torch.autograd.grad(o, [qq, kk, vv], g), ("dq", "dk", "dv")))


def test_attention_wrapper_refuses(N):
    """Checks that come before a device is asked for."""
    from multi_modal_amd.attention import attention as fn
    q = torch.zeros(2, 10, 4, 64, dtype=torch.bfloat16)
    for call, error in [
        (lambda: fn(q, q[:, :, :3], q[:, :, :3]), ValueError), (lambda: fn(q.float(), q.float(), q.float()), TypeError),
        (lambda: fn(q[..., :12], q[..., :12], q[..., :12]), ValueError), (lambda: fn(q, q, q, offsets=[0, 10]), ValueError),
        (lambda: fn(q, q, q, prefix=[1, 1]), ValueError), (lambda: fn(q, q, q, cap=math.inf), ValueError), (lambda: fn(q, q, q, scale=-1.0), ValueError),
        (lambda: fn(q[0], q[0], q[0], offsets=[]), ValueError),
    ]:
        with pytest.raises(error):
            call()


def test_attention_entries_refuse(N):
    """The C entries check sizes, types, alignment and pointers on the host; device 99 is what a good call is refused for."""
    lib = N.load_library()
    A = 1 << 20

    def args(**kw):
        a = dict(struct_size=ctypes.sizeof(N.AttentionArgs), dtype=2, n_docs=2, heads=4, kv_heads=2, dim=64, packed=0, causal=0, scale=0.1, cap=0.0, q_rows=10,
                 k_rows=10, q=A, k=A, v=A, out=A, lse=A)
        a.update(kw)
        s = N.AttentionArgs(**{n: v for n, v in a.items() if "stride" not in n})
        for n in ("q_stride", "k_stride", "v_stride", "out_stride"):
            setattr(s, n, (ctypes.c_int64 * 3)(*a.get(n, (2560, 256, 64))))
        s.lse_stride = (ctypes.c_int64 * 2)(40, 10)
        return s

    def forward(**kw):
        return lib.mmfe_attention_forward(ctypes.byref(args(**kw)), A, 99, None)

    def backward(grads=None, work=A, **kw):
        g = dict(struct_size=ctypes.sizeof(N.AttentionGrads), grad_out=A, grad_q=A, grad_k=A, grad_v=A)
        g.update(grads or {})
        s = N.AttentionGrads(**{n: v for n, v in g.items() if "stride" not in n})
        for n in ("grad_out_stride", "grad_q_stride", "grad_k_stride", "grad_v_stride"):
            setattr(s, n, (ctypes.c_int64 * 3)(*g.get(n, (2560, 256, 64))))
        return lib.mmfe_attention_backward(ctypes.byref(args(**kw)), ctypes.byref(s), work, 99, None)
    good = forward()
    assert good not in (0, -1) and backward() == good
    wrong = [dict(struct_size=8), dict(dtype=0), dict(dim=12), dict(dim=136), dict(dim=0), dict(n_docs=-1), dict(q_rows=-1), dict(k_rows=1 << 31), dict(heads=3),
             dict(kv_heads=0), dict(scale=0.0), dict(scale=math.inf), dict(cap=-1.0), dict(cap=math.nan), dict(cap=1e-39), dict(packed=1), dict(packed=1, n_docs=0), dict(prefix=A), dict(q=None), dict(k=None),
             dict(v=None), dict(out=None), dict(q=A + 8), dict(k_stride=(2560, 260, 64)), dict(v_stride=(2560, 256, 65)), dict(out_stride=(4, 256, 64)),
             dict(k_stride=(0, 1 << 25, 64)), dict(q_stride=(-8, 256, 64)), dict(slopes=A, k_rows=1 << 25)]
    assert lib.mmfe_attention_forward(ctypes.byref(args(k_rows=10 ** 6)), None, 99, None) == -1          # 10 rows over many keys: a workspace
    assert lib.mmfe_attention_forward(ctypes.byref(args(k_rows=10 ** 6)), A + 8, 99, None) == -1
    assert lib.mmfe_attention_workspace(ctypes.byref(args(k_rows=10 ** 6))) > 0 and lib.mmfe_attention_workspace(ctypes.byref(args())) == 0
    assert lib.mmfe_attention_workspace(ctypes.byref(args(dim=12))) == -1
    wrong.append(dict(out_rest=A + 2))
    for kw in wrong:
        assert forward(**kw) == -1, kw
        assert backward(**kw) == -1, kw
    for kw in (dict(struct_size=4), dict(grad_out=None), dict(grad_q=None), dict(grad_k=None), dict(grad_v=None), dict(grad_q=A + 2),
               dict(grad_k_stride=(2560, 256, 4))):
        assert backward(grads=kw) == -1, kw
    assert backward(lse=None) == -1 and backward(work=None) == -1 and backward(work=A + 4) == -1
    assert lib.mmfe_attention_backward_workspace(ctypes.byref(args(kv_heads=4))) == 0                     # short documents: no workspace, no out
    assert backward(kv_heads=4, work=None, out=None) == good and backward(kv_heads=4, lse=None) == -1
    assert lib.mmfe_attention_backward_workspace(ctypes.byref(args())) > 0 and lib.mmfe_attention_backward_workspace(ctypes.byref(args(dim=9))) == -1
    assert lib.mmfe_attention_forward(None, None, 0, None) == -1 and lib.mmfe_attention_backward(None, None, None, 0, None) == -1
    assert forward(n_docs=0, q=None, k=None, v=None, out=None) == 0 and forward(q_rows=0, q=None, out=None) == 0


def test_attention_counts():
    """Entries past 32 bits stay out of range (they must not wrap round into it); an empty list fits an empty batch."""
    from multi_modal_amd.attention import _counts
    cpu = torch.device("cpu")
    assert _counts([2 ** 32 + 5], "prefix", 1, cpu).tolist() == [2 ** 31 - 1]
    assert _counts(torch.tensor([7, 0], dtype=torch.uint8), "lengths", 2, cpu, 7).tolist() == [7, 0]
    assert _counts([], "lengths", 0, cpu, 5).shape == (0,)
    for bad, limit, error in (([2 ** 32], 9, ValueError), ([-1], None, ValueError), ([True], 9, TypeError), ([1.0], 9, TypeError), ([1, 2], 9, ValueError)):
        with pytest.raises(error):
            _counts(bad, "lengths", 1, cpu, limit)
    with pytest.raises(ValueError, match="must not fall"):
        _counts([0, 3, 2], "offsets", 3, cpu, 9, rising=True)


def test_folded_views():
    """What inplace=True refuses to write: views whose elements share memory."""
    from multi_modal_amd.rotary import _folded
    x = torch.zeros(2, 5, 12, 8)
    assert not any(map(_folded, (x, x[:, :, 2:5], x[:, ::2], x.transpose(1, 2), x[:0], x[:, :1], x[..., :3])))
    assert _folded(x[:, :1].expand(2, 5, 12, 8)) and _folded(x.view(-1).as_strided((1, 9, 2, 8), (0, 8, 8, 1)))


# What a saved-tensor hook may make of a tensor: equal values in another layout.
RELAID = {
    "same": lambda t: t,
    "packed": lambda t: torch.empty(t.size(), dtype=t.dtype).copy_(t),                     # what offloading to the host does
    "clone": lambda t: t.clone(),
    "gaps": lambda t: torch.empty(t.shape[:-1] + (t.shape[-1] + 8,), dtype=t.dtype)[..., :t.shape[-1]].copy_(t),
    "turned": lambda t: t.transpose(0, -1).contiguous().transpose(0, -1),                  # no unit stride inside the heads
}


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("kv", [2, 4])
@pytest.mark.parametrize("relay", RELAID)
def test_attention_backward_addresses_what_was_unpacked(N, monkeypatch, relay, kv, packed):
    """Pointers and strides of the backward call belong together, whatever layout a saved-tensor hook returns; counts are the saved ones."""
    from multi_modal_amd import attention as A
    seen, calls = {}, []

    def unpack(t):
        t = RELAID[relay](t)
        seen[t.data_ptr()] = t
        return t
    monkeypatch.setattr(A, "require_gpu", lambda: None)
    monkeypatch.setattr(A, "raw_stream", lambda device: 0)
    monkeypatch.setattr(torch.Tensor, "cuda", lambda self: self)
    monkeypatch.setattr(A.N, "attention_forward", lambda args, work, device, stream: None)
    monkeypatch.setattr(A.N, "attention_backward", lambda args, grads, work, device, stream: calls.append(
        (N.AttentionArgs.from_buffer_copy(args), N.AttentionGrads.from_buffer_copy(grads))))
    qkv = torch.zeros(2, 300, 3, 4, 64, dtype=torch.float16)
    q, k, v = (t.detach() for t in qkv.unbind(2))
    k, v = k[:, :, :kv], v[:, :, :kv]
    counts = torch.tensor([0, 100, 290] if packed else [300, 20], dtype=torch.int32)
    if packed:
        q, k, v = q[0], k[0], v[0]
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    prefix = torch.tensor([3, 4], dtype=torch.int32)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(memory_format=torch.preserve_format) if t.dtype == torch.int32 else t.detach(), unpack):
        out = A.attention(q, k, v, causal=True, prefix=prefix, **(dict(offsets=counts) if packed else dict(lengths=counts)))
    prefix.fill_(7)                                    # after the forward pass: a hook has its copy, and autograd notices nothing
    torch.autograd.grad(out, [q, k, v], torch.zeros_like(out))
    (args, grads), = calls
    for name, t in (("q", q), ("k", k), ("v", v)):
        at, strides = getattr(args, name), tuple(getattr(args, name + "_stride"))
        if relay == "turned":                          # the kernels cannot read it where it is
            assert at not in seen and strides == A._packed_strides(t), (name, strides)
        else:
            assert seen[at].shape == t.shape and strides == A._rows(seen[at])[1], (name, strides, seen[at].stride())
    dense = A._packed_strides(q)
    assert tuple(args.out_stride) == dense
    for at, of in ((args.out, q.shape), (args.out_rest, q.shape), (args.lse, (4, 300) if packed else (2, 4, 300))):
        assert not at or at not in seen or (seen[at].shape == torch.Size(of) and seen[at].is_contiguous())
    for at, want in ((args.prefix, [3, 4]), (args.q_off if packed else args.q_len, counts.tolist())):
        assert (ctypes.c_int32 * len(want)).from_address(at)[:] == want


def test_attention_backward_refuses_other_tensors(N, monkeypatch):
    """A hook that returns another shape or type than it was given would make the kernels read past it."""
    from multi_modal_amd import attention as A
    monkeypatch.setattr(A, "require_gpu", lambda: None)
    monkeypatch.setattr(A, "raw_stream", lambda device: 0)
    monkeypatch.setattr(torch.Tensor, "cuda", lambda self: self)
    monkeypatch.setattr(A.N, "attention_forward", lambda *a: None)
    monkeypatch.setattr(A.N, "attention_backward", lambda *a: pytest.fail("launched"))
    for change in (lambda t: t.float() if t.dtype == torch.float16 else t, lambda t: t[:1] if t.dim() == 4 else t, lambda t: t[..., :1] if t.dtype == torch.float32 else t,
                   lambda t: t[:1] if t.dtype == torch.int32 else t, lambda t: t.long() if t.dtype == torch.int32 else t):
        q = torch.zeros(2, 300, 4, 64, dtype=torch.float16, requires_grad=True)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), change):
            out = A.attention(q, q, q, lengths=torch.tensor([5, 300], dtype=torch.int32))
        with pytest.raises(RuntimeError, match="saved-tensor hook"):
            torch.autograd.grad(out, [q], torch.zeros_like(out))


def test_forward_mode_is_refused(N, monkeypatch):
    """A dual tensor's tangent must not be dropped in silence."""
    import torch.autograd.forward_ad as fwd
    from multi_modal_amd import attention as A, rotary as R
    for m in (A, R):
        monkeypatch.setattr(m, "require_gpu", lambda: None)
        monkeypatch.setattr(m, "raw_stream", lambda device: 0)
    monkeypatch.setattr(torch.Tensor, "cuda", lambda self, *a: self)
    monkeypatch.setattr(A.N, "attention_forward", lambda *a: None)
    monkeypatch.setattr(R.N, "RotaryHandle", lambda *a: type("H", (), {"run": lambda *a: None, "close": lambda self: None})())
    q, pos = torch.zeros(1, 3, 2, 8, dtype=torch.float16), torch.zeros(1, 3, dtype=torch.int32)
    rot = R.Rotary([2], device=0)
    rot.device = -1                                    # the CPU's number
    with fwd.dual_level():
        dual = fwd.make_dual(q, torch.ones_like(q))
        for args in ((dual, q, q), (q, dual, q), (q, q, dual)):
            with pytest.raises(NotImplementedError, match="attention"):
                A.attention(*args)
        for args in ((dual, None), (q, dual), (dual, q)):
            with pytest.raises(NotImplementedError, match="Rotary"):
                rot(*args, pos)
        leaf = q.clone().requires_grad_()
        for out in (A.attention(leaf, leaf, leaf), rot(leaf, None, pos)):
            with pytest.raises(NotImplementedError, match="gradient"):
                torch.autograd.grad(out, [leaf], dual)
        assert A.attention(q, q, q).shape == q.shape and rot(q, q, pos)[1].shape == q.shape       # tensors without a tangent
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda x: A.attention(x, q, q), (q,), (q,))


def test_rotary_devices(N, monkeypatch):
    """Devices by index, name and object; a missing index is the current GPU, and what is no GPU is refused."""
    from multi_modal_amd import rotary as R
    for device in ("cpu", "cpu:0", torch.device("cpu"), torch.device("meta")):
        with pytest.raises(ValueError, match="GPU"):
            R.Rotary([4], device=device)
    monkeypatch.setattr(R, "require_gpu", lambda: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(R.N, "RotaryHandle", lambda *a: a)
    for device, index in ((None, 3), ("cuda", 3), (torch.device("cuda"), 3), (0, 0), (2, 2), ("cuda:1", 1), (torch.device("cuda", 1), 1)):
        assert R.Rotary([4], device=device)._h[4] == index == R.Rotary([4], device=device).device


def test_attention_rows_of_empty_and_strided_tensors():
    """Every layout ends in one that the kernels read: a tensor without elements counts as contiguous whatever its strides."""
    from multi_modal_amd import attention as A
    x = torch.arange(2 * 10 * 3 * 32, dtype=torch.float16).view(2, 10, 3, 32)
    for t in (x[..., ::2][:, :0], x[:, :0, :, :12], x[:0, ..., 1:9], x[:0, :, ::2, ::4], x[0, :0, :, ::4], torch.zeros(2, 0, 3, 12, dtype=torch.float16)[..., :8],
              x, x[..., ::2], x[..., 1:17], x[..., 8:16], x.transpose(1, 2), x[0], x[0, :, :, 4:12], x[:, :1, :, 2:10], x.transpose(1, 3)[..., 0:1].expand(-1, -1, -1, 8)):
        r, strides = A._rows(t)
        assert torch.equal(r, t) and r.shape == t.shape
        used = [(s, g) for s, g, n in zip(r.stride()[:-1], strides[-(r.dim() - 1):], r.shape) if n > 1 and r.numel()]
        assert all(s == g for s, g in used) and all(s % 8 == 0 for s in strides) and r.data_ptr() % 16 == 0 and (r.stride(-1) == 1 or not r.numel())


def test_attention_scales_and_caps_past_float32(N):
    """Numbers that float32 does not hold, or holds as zero, are refused rather than rounded to another meaning."""
    from multi_modal_amd.attention import attention as fn
    q = torch.zeros(2, 10, 4, 64, dtype=torch.bfloat16)
    for kw in (dict(cap=1e300), dict(cap=1e-60), dict(scale=1e300), dict(scale=1e-60), dict(scale=1e-28), dict(scale=3e38), dict(cap=math.nan)):
        with pytest.raises(ValueError, match="scale"):
            fn(q, q, q, **kw)
    lib, A = N.load_library(), 1 << 20

    def forward(scale, cap):
        s = N.AttentionArgs(struct_size=ctypes.sizeof(N.AttentionArgs), dtype=2, n_docs=2, heads=4, kv_heads=4, dim=64, scale=scale, cap=cap, q_rows=10, k_rows=10,
                            q=A, k=A, v=A, out=A)
        return lib.mmfe_attention_forward(ctypes.byref(s), None, 99, None)
    good = forward(0.1, 0.0)
    assert good not in (0, -1)
    assert forward(2.0 ** -90, 0.0) == forward(2.0 ** 126, 0.0) == forward(0.1, 3e38) == forward(0.1, 1e-30) == good
    assert forward(2.0 ** -91, 0.0) == forward(2.0 ** 127, 0.0) == forward(-0.1, 0.0) == forward(math.nan, 0.0) == forward(0.1, math.inf) == -1


def test_attention_grids_past_the_launch_limit(N):
    """More blocks than a launch takes (2^32 - 1 threads) are refused before anything is launched; device 99 is what a good call is refused for."""
    lib, A = N.load_library(), 1 << 20

    def args(**kw):
        a = dict(struct_size=ctypes.sizeof(N.AttentionArgs), dtype=2, n_docs=2, heads=4, kv_heads=4, dim=64, scale=0.1, cap=0.0, q_rows=10, k_rows=10, q=A, k=A, v=A, out=A, lse=A)
        a.update(kw)
        s = N.AttentionArgs(**a)
        s.lse_stride = (ctypes.c_int64 * 2)(a["heads"] * a["q_rows"], a["q_rows"])
        return s

    def both(**kw):
        g = N.AttentionGrads(struct_size=ctypes.sizeof(N.AttentionGrads), grad_out=A, grad_q=A, grad_k=A, grad_v=A)
        return (lib.mmfe_attention_forward(ctypes.byref(args(**kw)), A, 99, None),
                lib.mmfe_attention_backward(ctypes.byref(args(**kw)), ctypes.byref(g), A, 99, None))
    good = both()[0]
    assert both() == (good, good) and good not in (0, -1)
    assert both(n_docs=2 ** 20, heads=16, kv_heads=16) == (-1, -1)                    # 2^24 blocks of 256
    assert both(n_docs=2 ** 20, heads=15, kv_heads=15, dim=72) == (good, -1)          # the preparing launch of the gradients has 2 x 15 x 2^20
    assert both(n_docs=2 ** 19, heads=15, kv_heads=15) == (good, good)
    assert both(n_docs=2 ** 19, heads=16, kv_heads=16) == (good, -1)                  # short documents: 2^23 blocks of 512
    assert both(n_docs=2 ** 17, heads=8, kv_heads=8, q_rows=1, k_rows=4000) == (good, -1)
    assert both(n_docs=2 ** 21, heads=64, kv_heads=8, q_rows=1, k_rows=4000)[0] == good   # one chunk a key head: 2^24 blocks of 128
    assert both(n_docs=2 ** 22, heads=64, kv_heads=8, q_rows=1, k_rows=4000)[0] == -1
    assert both(packed=1, q_off=A, k_off=A, n_docs=2 ** 23, heads=2, kv_heads=2) == (-1, -1)


def test_attention_backward_takes_a_dense_lse_only(N):
    """Statistics of the rows lie in the workspace as lse does: strides of a larger array would lead out of it."""
    lib, A = N.load_library(), 1 << 20

    def backward(stride, **kw):
        a = dict(struct_size=ctypes.sizeof(N.AttentionArgs), dtype=2, n_docs=2, heads=4, kv_heads=2, dim=64, scale=0.1, cap=0.0, q_rows=10, k_rows=10, q=A, k=A, v=A, out=A, lse=A)
        a.update(kw)
        s = N.AttentionArgs(**a)
        s.lse_stride = (ctypes.c_int64 * 2)(*stride)
        g = N.AttentionGrads(struct_size=ctypes.sizeof(N.AttentionGrads), grad_out=A, grad_q=A, grad_k=A, grad_v=A)
        return lib.mmfe_attention_backward(ctypes.byref(s), ctypes.byref(g), A, 99, None)
    good = backward((40, 10))
    assert good not in (0, -1)
    assert backward((80, 10)) == backward((40, 20)) == backward((10, 20)) == backward((40, -10)) == backward((80, 10), kv_heads=4) == -1
    packed = dict(packed=1, q_off=A, k_off=A)
    assert backward((0, 10), **packed) == backward((7, 10), **packed) == backward((7, 10), n_docs=1) == backward((10, 3), heads=1, kv_heads=1) == good
    assert backward((0, 12), **packed) == -1


def test_attention_backward_fills_no_gradient_of_lse(N, monkeypatch):
    """lse has no gradient: nothing is allocated and zeroed for one; an undefined gradient of the output still gives zeros."""
    from torch.utils._python_dispatch import TorchDispatchMode
    from multi_modal_amd import attention as A
    monkeypatch.setattr(A, "require_gpu", lambda: None)
    monkeypatch.setattr(A, "raw_stream", lambda device: 0)
    monkeypatch.setattr(torch.Tensor, "cuda", lambda self: self)
    monkeypatch.setattr(A.N, "attention_forward", lambda *a: None)
    monkeypatch.setattr(A.N, "attention_backward", lambda *a: None)
    seen = []

    class Record(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))
    q = torch.zeros(2, 30, 4, 64, dtype=torch.float16, requires_grad=True)
    out, lse = A.attention(q, q, q, return_lse=True)
    assert not lse.requires_grad
    with Record():
        torch.autograd.grad(out, [q], torch.ones_like(out))
    assert not any("zero" in name for name in seen) and any("empty" in name for name in seen), seen

    class Nothing(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x.clone()

        @staticmethod
        def backward(ctx, g):
            return None
    (g,) = torch.autograd.grad(Nothing.apply(A.attention(q, q, q)), [q], torch.ones_like(out), allow_unused=True)
    assert (g == 0).all()
