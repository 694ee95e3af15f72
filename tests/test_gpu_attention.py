"""Attention (csrc/attention.hip, csrc/attention_backward.hip) against the float64 oracle (oracle/token_oracle.py), which gives a bound
for each element: half a step of the 16-bit type for the result, half a step for each rounded softmax value or score gradient that
enters it, and the float32 errors of the scores, taken through the formulas."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mm():
    import multi_modal_amd as m
    m.load_library()
    assert torch.cuda.is_available()
    return m


@pytest.fixture(scope="module")
def O():
    from oracle import token_oracle
    return token_oracle


BF, HF = torch.bfloat16, torch.float16


def limits(dtype):
    i = torch.finfo(dtype)
    return dict(eps=i.eps, tiny=i.smallest_normal * i.eps / 2)


def within(name, got, ref, tol):
    got = got.detach().double()
    bad = ~((got - ref).abs() <= tol) & ~((got == ref))
    assert not bad.any(), (name, int(bad.sum()), float(((got - ref).abs() / tol.clamp_min(1e-300))[bad].max()), bad.nonzero()[:4].tolist())


def slopes_of(H):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)])


def docs_padded(lens, kv, N, S):
    return [(b * N, n, b * S, m) for b, (n, m) in enumerate(zip(lens, kv))]


def check(mm, O, q, k, v, docs, opts, g=None, scale=None, flat=lambda t: t, lse_flat=lambda t: t, host=None):
    """q, k, v (any form) on the GPU; `flat` brings a result to (rows, heads, dim), `lse_flat` a lse to (heads, rows)."""
    host = host or {}
    fn = mm.attention.attention
    ref, tol = O.attention(flat(q.detach()), flat(k.detach()), flat(v.detach()), docs, scale=scale, cap=opts.get("cap", 0.0), slopes=host.get("slopes"),
                           causal=opts.get("causal", False), prefix=host.get("prefix"), g=None if g is None else flat(g), **limits(q.dtype))
    with torch.no_grad():
        out, lse = fn(q, k, v, scale=scale, return_lse=True, **opts)
    assert out.dtype == q.dtype and out.shape == q.shape and lse.dtype == torch.float32
    within("out", flat(out), ref["o"], tol["o"])
    within("lse", lse_flat(lse), ref["lse"], tol["lse"])
    if g is None:
        return out
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    o2 = fn(q, k, v, scale=scale, **opts)
    assert torch.equal(o2, out)
    dq, dk, dv = torch.autograd.grad(o2, [q, k, v], g)
    for name, got in (("dq", dq), ("dk", dk), ("dv", dv)):
        assert got.dtype == q.dtype and got.shape == (q if name == "dq" else k).shape
        within(name, flat(got), ref[name], tol[name])
    again = torch.autograd.grad(fn(q, k, v, scale=scale, **opts), [q, k, v], g)
    assert all(torch.equal(a, b) for a, b in zip(again, (dq, dk, dv)))          # no atomics on values: the same bits
    return out


def flat4(t):
    return t.reshape(-1, *t.shape[2:])


def lse4(t):
    return t.transpose(0, 1).reshape(t.shape[1], -1)


PADDED = [
    # lens, N, kv, S, H, K, D, dtype, causal, prefix, bias, cap
    ([1], 1, [1], 1, 1, 1, 8, HF, False, False, False, 0.0),
    ([257], 257, [257], 257, 3, 3, 64, HF, False, False, False, 0.0),
    ([193, 1, 0, 64, 65, 192], 193, None, 193, 4, 2, 64, BF, False, False, False, 0.0),
    ([128, 127, 129], 129, None, 129, 2, 1, 128, HF, True, False, False, 0.0),
    ([300, 31], 300, None, 300, 6, 2, 72, BF, True, True, True, 0.0),
    ([150, 90], 150, None, 150, 2, 2, 32, HF, False, False, True, 8.0),
    ([260], 260, None, 260, 2, 2, 128, BF, True, True, False, 5.0),
    ([33, 64, 10], 64, [200, 10, 0], 201, 4, 2, 64, BF, True, False, False, 0.0),    # more rows than keys: rows that see nothing
    ([5, 40], 40, [500, 333], 512, 3, 1, 96, HF, False, False, True, 0.0),           # cross attention
    ([70, 70], 70, [70, 3], 70, 2, 2, 16, HF, True, True, False, 0.0),
    ([600], 600, None, 600, 1, 1, 40, HF, True, False, True, 30.0),
    ([0, 0], 5, [3, 0], 9, 2, 2, 64, BF, False, False, False, 0.0),
]


@pytest.mark.parametrize("case", PADDED, ids=lambda c: f"{c[0]}x{c[4]}x{c[6]}")
def test_padded(mm, O, case):
    lens, N, kv, S, H, K, D, dtype, causal, prefix, bias, cap = case
    B = len(lens)
    gen = torch.Generator().manual_seed(N * 7 + D)
    q = torch.randn(B, N, H, D, generator=gen).to(dtype).cuda()
    k, v = (torch.randn(B, S, K, D, generator=gen).to(dtype).cuda() for _ in "kv")
    g = torch.randn(B, N, H, D, generator=gen).to(dtype).cuda()
    host = {}
    opts = dict(causal=causal, cap=cap, lengths=lens)
    if kv is not None:
        opts["kv_lengths"] = kv
    m = kv or lens
    if prefix:
        host["prefix"] = [x // 3 + 1 for x in m]
        opts["prefix"] = torch.tensor(host["prefix"], device="cuda")
    if bias:
        host["slopes"] = opts["slopes"] = slopes_of(H)
    # what no document holds is never read as a value
    for b in range(B):
        for t, n in ((q, lens[b]), (g, lens[b]), (k, m[b]), (v, m[b])):
            t[b, n:] = math.nan
    out = check(mm, O, q, k, v, docs_padded(lens, m, N, S), opts, g=g, flat=flat4, lse_flat=lse4, host=host)
    # lengths on the device, and views of a packed projection with heads in front: the same bits
    opts["lengths"] = torch.tensor(lens, dtype=torch.int64, device="cuda")
    big = torch.full((B, H, N, D + 24), math.nan, dtype=dtype, device="cuda")
    big[..., 8:8 + D] = q.transpose(1, 2)
    assert torch.equal(mm.attention.attention(big[..., 8:8 + D].transpose(1, 2), k, v, **opts), out)
    odd = torch.empty(q.numel() + 1, dtype=dtype, device="cuda")[1:].view(q.shape).copy_(q)
    assert torch.equal(mm.attention.attention(odd, k, v, **opts), out)


PACKED = [
    # lens, lead, tail, H, K, D, dtype, causal, prefix, bias, cap
    ([5], 0, 0, 1, 1, 64, HF, False, False, False, 0.0),
    ([1, 200, 0, 64, 129, 1, 1, 33], 0, 7, 4, 2, 64, BF, True, False, False, 30.0),
    ([100, 0, 128, 300], 131, 140, 2, 1, 128, HF, False, False, True, 0.0),
    ([7] * 150, 3, 0, 2, 2, 32, BF, True, True, False, 0.0),
    ([0, 0], 4, 9, 2, 1, 64, HF, True, False, False, 0.0),
    ([], 0, 130, 2, 1, 64, BF, True, False, False, 0.0),
    ([3, 0, 130] * 60 + [257], 0, 300, 2, 1, 64, HF, True, False, False, 0.0),
    ([0, 200, 1, 0] * 40, 200, 0, 2, 2, 32, BF, False, False, True, 0.0),
    ([60, 61, 300, 2, 0, 128, 129], 1, 1, 12, 2, 128, BF, True, True, True, 9.0),
    ([700, 40], 0, 0, 8, 2, 64, HF, True, False, True, 0.0),          # a key head's query heads on blocks of their own
]


@pytest.mark.parametrize("case", PACKED, ids=lambda c: f"{c[0][:8]}x{c[3]}x{c[5]}")
def test_packed(mm, O, case):
    lens, lead, tail, H, K, D, dtype, causal, prefix, bias, cap = case
    off = [lead]
    for n in lens:
        off.append(off[-1] + n)
    T = off[-1] + tail
    gen = torch.Generator().manual_seed(T + D)
    q, g = (torch.randn(T, H, D, generator=gen).to(dtype).cuda() for _ in "qg")
    k, v = (torch.randn(T, K, D, generator=gen).to(dtype).cuda() for _ in "kv")
    for t in (q, k, v, g):
        t[:lead] = math.nan
        t[off[-1]:] = math.inf
    host, opts = {}, dict(causal=causal, cap=cap, offsets=torch.tensor(off, dtype=torch.int32, device="cuda"))
    if prefix:
        host["prefix"] = opts["prefix"] = [n // 2 for n in lens]
    if bias:
        host["slopes"] = opts["slopes"] = slopes_of(H)
    docs = [(off[d], n, off[d], n) for d, n in enumerate(lens)]
    out = check(mm, O, q, k, v, docs, opts, g=g, host=host)
    opts["offsets"] = off
    assert torch.equal(mm.attention.attention(q, k, v, **opts), out)


TOKENS = [
    # q rows, lens of keys, room, H, K, D, dtype, causal, prefix, bias, cap
    (1, [1, 0, 31, 32, 33, 4000], 4096, 8, 2, 128, BF, True, False, False, 0.0),
    (1, [500], 512, 12, 12, 64, HF, True, False, True, 0.0),
    (5, [5, 3000, 129, 2], 3001, 6, 2, 72, BF, True, True, False, 20.0),
    (64, [700, 64], 700, 4, 1, 32, HF, True, False, True, 0.0),
    (33, [9000, 40], 9001, 4, 4, 64, BF, False, False, False, 0.0),
    (2, [1025, 1024, 1023], 1025, 16, 1, 8, HF, False, False, False, 0.0),
    (1, [70000], 70001, 3, 1, 64, BF, True, False, False, 0.0),
]


@pytest.mark.parametrize("case", TOKENS, ids=lambda c: f"{c[0]}x{c[1][-1]}x{c[3]}x{c[5]}")
def test_few_rows_over_many_keys(mm, O, case):
    n, kv, room, H, K, D, dtype, causal, prefix, bias, cap = case
    B = len(kv)
    gen = torch.Generator().manual_seed(room)
    lens = [n] * (B - 1) + [max(1, n - 1)]
    q, g = (torch.randn(B, n, H, D, generator=gen).to(dtype).cuda() for _ in "qg")
    k, v = (torch.randn(B, room, K, D, generator=gen).to(dtype).cuda() for _ in "kv")
    for b in range(B):
        k[b, kv[b]:] = math.nan
        v[b, kv[b]:] = math.nan
        q[b, lens[b]:] = math.nan
        g[b, lens[b]:] = math.nan
    host, opts = {}, dict(causal=causal, cap=cap, lengths=lens, kv_lengths=torch.tensor(kv, device="cuda"))
    if prefix:
        host["prefix"] = opts["prefix"] = [m // 2 for m in kv]
    if bias:
        host["slopes"] = opts["slopes"] = slopes_of(H)
    out = check(mm, O, q, k, v, docs_padded(lens, kv, n, room), opts, g=g, flat=flat4, lse_flat=lse4, host=host)
    for b in (0, B - 1):            # alone, with no more room than it needs
        m = max(kv[b], 1)
        o = dict(opts, lengths=lens[b:b + 1], kv_lengths=kv[b:b + 1])
        if prefix:
            o["prefix"] = opts["prefix"][b:b + 1]
        alone = mm.attention.attention(q[b:b + 1], k[b:b + 1, :m], v[b:b + 1, :m], **o)
        assert ((alone[0].double() - out[b].double()).abs() <= 2 * torch.finfo(dtype).eps * out[b].double().abs() + 1e-3).all()


def test_one_nan_key_reaches_its_rows(mm):
    """A NaN in a key that a row sees makes that row NaN, whichever chunk it lies in, and no other document's."""
    fn = mm.attention.attention
    k, v = (torch.randn(2, 3000, 1, 64, device="cuda").to(BF) for _ in "kv")
    q = torch.randn(2, 1, 4, 64, device="cuda").to(BF)
    want = fn(q, k, v)
    for at in (0, 31, 32, 1500, 2999):
        bad = k.clone()
        bad[0, at] = math.nan
        o = fn(q, bad, v)
        assert o[0].isnan().all() and torch.equal(o[1], want[1])
        o = fn(q, bad, v, kv_lengths=[at, 3000])
        assert o[0].isfinite().all() and torch.equal(o[1], want[1])


def test_one_key_has_no_score_gradient(mm):
    """A softmax over one key is constant: gradients of q and k are exactly zero, that of v is the incoming one."""
    fn = mm.attention.attention
    for n in (1, 3):
        q, g = (torch.randn(2, n, 2, 64, device="cuda").to(BF) for _ in "qg")
        k, v = (torch.randn(2, 1, 2, 64, device="cuda").to(BF) for _ in "kv")
        q, k, v = (t.requires_grad_() for t in (q, k, v))
        o = fn(q, k, v)
        assert torch.equal(o, v.expand(2, n, 2, 64))
        dq, dk, dv = torch.autograd.grad(o, [q, k, v], g)
        assert (dq == 0).all() and (dk == 0).all() and (n > 1 or torch.equal(dv, g))


def test_documents_do_not_touch_each_other(mm):
    """A document full of NaN and infinities changes no other document's rows or gradients, and each document is what it is alone."""
    gen = torch.Generator().manual_seed(4)
    lens = [70, 50, 130]
    off = [0, 70, 120, 250]
    q, g = (torch.randn(250, 4, 64, generator=gen).to(BF).cuda() for _ in "qg")
    k, v = (torch.randn(250, 2, 64, generator=gen).to(BF).cuda() for _ in "kv")
    fn = mm.attention.attention

    def run(q, k, v, g, **kw):
        q, k, v = (t.detach().clone().requires_grad_() for t in (q, k, v))
        o = fn(q, k, v, causal=True, **kw)
        return (o.detach(),) + torch.autograd.grad(o, [q, k, v], g)
    clean = run(q, k, v, g, offsets=off)
    for d in range(3):
        s = slice(off[d], off[d + 1])
        alone = run(q[None, s], k[None, s], v[None, s], g[None, s])
        assert all(torch.equal(a[s], b[0]) for a, b in zip(clean, alone))
    dirty = [t.clone() for t in (q, k, v, g)]
    for t, x in zip(dirty, (math.nan, math.inf, -math.inf, math.nan)):
        t[70:120] = x
    r = run(*dirty, offsets=off)
    for a, b in zip(r, clean):
        assert torch.equal(a[:70], b[:70]) and torch.equal(a[120:], b[120:])


@pytest.mark.parametrize("dtype", [HF, BF])
def test_extreme_scores(mm, O, dtype):
    """Scores of thousands (one key takes all), all keys alike, and scores that rise and fall along the keys past the point where the running
    maximum is raised."""
    gen = torch.Generator().manual_seed(6)
    T, D = 400, 64
    q = torch.randn(1, T, 2, D, generator=gen)
    k, v = torch.randn(1, T, 2, D, generator=gen), torch.randn(1, T, 2, D, generator=gen)
    ramp = torch.linspace(-6, 6, T)[None, :, None, None]
    docs = [(0, T, 0, T)]
    for a, b in ((q * 30, k * 30), (torch.zeros_like(q), k), (q.abs(), ramp.expand(k.shape) * 3), (q.abs(), -ramp.expand(k.shape) * 3)):
        check(mm, O, a.to(dtype).cuda(), b.to(dtype).cuda(), v.to(dtype).cuda(), docs, dict(causal=False), flat=flat4, lse_flat=lse4)


@pytest.mark.parametrize("size", [1e-4, 1.0, 1e3])
def test_float16_gradients_of_every_size(mm, O, size):
    """Incoming gradients down to 1e-4 over 2000 keys: p (dp - delta) is far below float16's range, its scaled form is not."""
    gen = torch.Generator().manual_seed(8)
    T, D = 2000, 64
    q, k, v = (torch.randn(1, T, 1, D, generator=gen).to(HF).cuda() for _ in "qkv")
    g = (torch.randn(1, T, 1, D, generator=gen) * size).to(HF).cuda()
    if size > 1:
        v = v * 0.01                                            # gradients of q and k stay in float16's own range
    check(mm, O, q, k, v, [(0, T, 0, T)], dict(causal=True), g=g, flat=flat4, lse_flat=lse4)


def test_value_differences(mm):
    """o is linear in v: <g, o(v + h) - o(v)> is <dv, h> up to the roundings of o."""
    gen = torch.Generator().manual_seed(11)
    q, k, v, g, h = (torch.randn(2, 200, 2, 64, generator=gen).to(HF).cuda() for _ in range(5))
    fn = mm.attention.attention
    v = v.requires_grad_()
    w = (v.detach() + h)
    o = fn(q, k, v, causal=True)
    (dv,) = torch.autograd.grad(o, [v], g)
    d = (g.double() * (fn(q, k, w, causal=True).double() - o.detach().double())).sum()
    step = (w.double() - v.detach().double())
    size = (g.double().abs() * (fn(q, k, w.abs(), causal=True).double() + fn(q, k, v.detach().abs(), causal=True).double())).sum() \
        + (dv.double().abs() * step.abs()).sum()
    assert abs(float(d - (dv.double() * step).sum())) <= 3 * 2.0 ** -11 * float(size)


def test_partial_gradients_and_broadcast(mm):
    """Gradients of some inputs only, an expanded gradient, keys broadcast over the batch."""
    gen = torch.Generator().manual_seed(12)
    fn = mm.attention.attention
    q = torch.randn(3, 40, 2, 64, generator=gen).to(BF).cuda().requires_grad_()
    k, v = (torch.randn(1, 40, 2, 64, generator=gen).to(BF).cuda().requires_grad_() for _ in "kv")
    full = torch.autograd.grad(fn(q, k.expand(3, -1, -1, -1), v.expand(3, -1, -1, -1)).float().sum(), [q, k, v])
    each = [torch.autograd.grad(fn(q[b:b + 1], k, v).float().sum(), [q, k, v]) for b in range(3)]
    assert torch.equal(full[0], each[0][0] + each[1][0] + each[2][0])
    for i in (1, 2):
        total = sum(e[i].float() for e in each)
        assert ((full[i].float() - total).abs() <= 3 * 2.0 ** -8 * sum(e[i].float().abs() for e in each) + 1e-30).all()
    (only,) = torch.autograd.grad(fn(q, k.detach().expand(3, -1, -1, -1), v.detach().expand(3, -1, -1, -1)).float().sum(), [q])
    assert torch.equal(only, full[0])


def test_streams_and_graph(mm):
    fn = mm.attention.attention
    q, k, v, g = (torch.randn(2, 150, 2, 64, device="cuda").to(HF) for _ in range(4))
    lengths = torch.tensor([150, 77], dtype=torch.int32, device="cuda")

    def step(q, k, v):
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        o = fn(q, k, v, lengths=lengths, causal=True)
        return (o.detach(),) + torch.autograd.grad(o, [q, k, v], g)
    want = step(q, k, v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(q, k, v)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(q, k, v)
    for i in range(3):
        for t in (q, k, v, g):
            t.copy_(torch.randn(t.shape, device="cuda"))
        lengths.copy_(torch.tensor([150 - i, 60 + 30 * i]))
        graph.replay()
        want = step(q, k, v)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        torch.cuda.synchronize()


def test_bad_counts_on_the_device_are_clamped(mm):
    """Lengths past the rows read and write nothing past them: the tensors lie inside larger ones whose rest stays as it was."""
    fn = mm.attention.attention
    pool = torch.randn(3, 4, 100, 2, 64, device="cuda").to(BF)
    q, k, v = (pool[i, 1:3] for i in range(3))
    keep = pool.clone()
    full = fn(q, k, v)
    assert torch.equal(fn(q, k, v, lengths=torch.tensor([100000, 2 ** 31 - 1], device="cuda")), full)
    none = fn(q, k, v, lengths=torch.tensor([-5, -2 ** 31], device="cuda"))
    assert (none == 0).all()
    p = pool[0, 1], pool[1, 1], pool[2, 1]
    o = fn(*p, offsets=torch.tensor([0, 40, 10 ** 6], device="cuda"))
    assert torch.equal(o, fn(*p, offsets=[0, 40, 100]))
    assert torch.equal(pool, keep)


def test_refusals(mm):
    fn = mm.attention.attention
    q, k, v = (torch.randn(2, 10, 4, 64, device="cuda").to(BF) for _ in "qkv")
    for call, error in [
        (lambda: fn(q, k[:, :, :3], v[:, :, :3]), ValueError), (lambda: fn(q, k, v[:, :5]), ValueError), (lambda: fn(q, k[:1], v[:1]), ValueError),
        (lambda: fn(q.float(), k.float(), v.float()), TypeError), (lambda: fn(q, k.to(HF), v), TypeError), (lambda: fn(q[..., :20], k[..., :20], v[..., :20]), ValueError),
        (lambda: fn(q[0], k[0], v[0]), ValueError), (lambda: fn(q, k, v, offsets=[0, 10]), ValueError), (lambda: fn(q, k, v, lengths=[1]), ValueError),
        (lambda: fn(q, k, v, lengths=[1, 11]), ValueError), (lambda: fn(q, k, v, lengths=[1.0, 2.0]), TypeError), (lambda: fn(q, k, v, prefix=[1, 1]), ValueError),
        (lambda: fn(q, k, v, cap=-1.0), ValueError), (lambda: fn(q, k, v, scale=0.0), ValueError), (lambda: fn(q, k, v, scale=math.nan), ValueError),
        (lambda: fn(q, k, v, slopes=torch.ones(3)), ValueError), (lambda: fn(q, k, v, slopes=torch.ones(4, requires_grad=True)), ValueError),
        (lambda: fn(q, k, v, kv_offsets=[0, 1]), ValueError), (lambda: fn(q[0], k[0], v[0], offsets=[0, 5, 4]), ValueError),
        (lambda: fn(q[0], k[0], v[0], offsets=[0, 11]), ValueError), (lambda: fn(q[0], k[0, :5], v[0, :5], offsets=[0, 5]), ValueError),
        (lambda: fn(q[0], k[0], v[0], offsets=[0, 5], lengths=[1]), ValueError), (lambda: fn(q, k.cpu(), v), ValueError),
    ]:
        with pytest.raises(error):
            call()
    assert fn(q[:0], k[:0], v[:0]).shape == (0, 10, 4, 64)
    assert fn(q[:, :0], k, v).shape == (2, 0, 4, 64)
    assert (fn(q, k[:, :0], v[:, :0]) == 0).all()
    c = fn(q.cpu(), k.cpu(), v.cpu())
    assert not c.is_cuda and torch.equal(c, fn(q, k, v).cpu())


def test_empty_calls_and_their_gradients(mm):
    fn = mm.attention.attention
    for B, N, S in ((0, 5, 5), (2, 0, 7), (2, 7, 0), (2, 0, 0)):
        for dtype in (BF, HF):
            q = torch.randn(B, N, 4, 64, device="cuda", dtype=dtype).requires_grad_()
            k, v = (torch.randn(B, S, 2, 64, device="cuda", dtype=dtype).requires_grad_() for _ in "kv")
            o, lse = fn(q, k, v, return_lse=True)
            assert o.shape == q.shape and (o == 0).all() and lse.shape == (B, 4, N) and (S > 0 or (lse == -math.inf).all())
            for t, x in zip(torch.autograd.grad(o, [q, k, v], torch.ones_like(o)), (q, k, v)):
                assert t.shape == x.shape and (t == 0).all()


def test_changed_inputs_are_noticed(mm):
    """What the backward pass reads must be what the forward pass read; a second derivative is refused."""
    fn = mm.attention.attention
    lengths = torch.tensor([5, 9], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 9, 2, 64, device="cuda", dtype=BF).requires_grad_()
    o = fn(q, q, q, lengths=lengths)
    lengths.fill_(3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(o.sum(), [q])
    o = fn(q, q, q)
    (g,) = torch.autograd.grad(o.float().square().sum(), [q], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), [q])
    x = torch.randn(2, 9, 2, 64, device="cuda", dtype=BF).requires_grad_()
    y = x * 1.0
    z = (y * y).sum()
    rot = mm.Rotary([8])
    with torch.no_grad():
        rot(y, None, mm.grid_positions(9, device="cuda"), inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_cache_past_32_bits(mm):
    """Keys and values of 2.6e9 elements each: the last head of the last rows lies past 2^32 bytes and past 2^31 elements."""
    fn = mm.attention.attention
    S, K, D = 640_000, 32, 128
    k, v = (torch.empty(1, S, K, D, dtype=BF, device="cuda").normal_() for _ in "kv")
    q = torch.randn(1, 3, K, D, device="cuda").to(BF)
    o = fn(q, k, v, causal=True)
    far = fn(q[:, :1], k[:, -200:], v[:, -200:])                     # the end alone
    for h in (0, 31):
        for kk, vv, n, got in ((k[0, :, h], v[0, :, h], 3, o), (k[0, -200:, h], v[0, -200:, h], 1, far)):
            s = (q[0, :n, h].double() @ kk.double().T) * D ** -0.5
            if n == 3:
                s[0, -2:] = s[1, -1] = -math.inf
            p = torch.softmax(s, 1)
            ref, size = p @ vv.double(), p @ vv.double().abs()
            assert ((got[0, :n, h].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -14 * size + 2.0 ** -8 * (p * p @ vv.double().square()).sqrt() * 6).all()
    del k, v


def test_many_documents(mm):
    """70 000 documents of 0 to 3 tokens: each one is what it is in a batch of its own."""
    fn = mm.attention.attention
    gen = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 4, (70000,), generator=gen)
    off = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)]).to(torch.int32).cuda()
    T = int(off[-1])
    q, k, v = (torch.randn(T, 1, 64, generator=gen).to(BF).cuda() for _ in "qkv")
    o = fn(q, k, v, offsets=off, causal=True)
    first = torch.zeros(T, dtype=torch.bool, device="cuda")
    first[off[:-1][lens.cuda() > 0].long()] = True
    assert torch.equal(o[first], v[first])                            # a document's first row sees itself alone
    d = int((lens == 3).nonzero()[-1])
    s = slice(int(off[d]), int(off[d]) + 3)
    assert torch.equal(o[s], fn(q[None, s], k[None, s], v[None, s], causal=True)[0])


SHORT = [
    # lens, N, kv, S, H, D, dtype, causal, prefix, bias, cap: a key head per query head, up to 256 rows and keys
    ([256, 255, 129, 0], 256, None, 256, 2, 64, HF, True, False, False, 0.0),
    ([1, 20], 20, [256, 225], 256, 3, 64, BF, False, False, True, 0.0),
    ([250, 256], 256, [3, 32], 32, 2, 32, HF, True, True, False, 0.0),
    ([128, 97], 128, None, 128, 2, 64, HF, True, False, True, 12.0),
    ([33, 32, 31], 33, [64, 65, 128], 128, 1, 40, BF, True, True, False, 6.0),
    ([130, 7], 130, [129, 256], 256, 2, 8, BF, True, False, False, 0.0),
    ([160, 193], 193, None, 193, 2, 48, HF, False, False, True, 5.0),
    ([1, 0, 1], 1, [1, 1, 0], 1, 2, 64, HF, True, False, False, 0.0),
]


@pytest.mark.parametrize("case", SHORT, ids=lambda c: f"{c[0]}x{c[3]}x{c[5]}")
@pytest.mark.parametrize("size", [1e-4, 1.0, 1e2])
def test_short_documents(mm, O, case, size):
    """Around the sizes where one block does a head's gradients, with incoming gradients of every size."""
    lens, N, kv, S, H, D, dtype, causal, prefix, bias, cap = case
    B = len(lens)
    gen = torch.Generator().manual_seed(N * 5 + S + D)
    q = torch.randn(B, N, H, D, generator=gen).to(dtype).cuda()
    k, v = (torch.randn(B, S, H, D, generator=gen).to(dtype).cuda() for _ in "kv")
    g = (torch.randn(B, N, H, D, generator=gen) * size).to(dtype).cuda()
    m = kv or lens
    host, opts = {}, dict(causal=causal, cap=cap, lengths=lens, kv_lengths=m)
    if prefix:
        host["prefix"] = opts["prefix"] = [x // 2 for x in m]
    if bias:
        host["slopes"] = opts["slopes"] = slopes_of(H)
    for b in range(B):
        for t, n in ((q, lens[b]), (g, lens[b]), (k, m[b]), (v, m[b])):
            t[b, n:] = math.nan
    check(mm, O, q, k, v, docs_padded(lens, m, N, S), opts, g=g, flat=flat4, lse_flat=lse4, host=host)
    # one row or key more of room, which nothing uses: another launch, the same results within the bounds
    wide = (torch.cat([t, torch.full_like(t[:, :1], math.nan)], 1) for t in (q, k, v))
    ref, tol = O.attention(flat4(q), flat4(k), flat4(v), docs_padded(lens, m, N, S), cap=cap, slopes=host.get("slopes"), causal=causal, prefix=host.get("prefix"),
                           g=flat4(g), **limits(dtype))
    x = [t.requires_grad_() for t in wide]
    got = torch.autograd.grad(mm.attention.attention(*x, **opts), x, torch.cat([g, torch.full_like(g[:, :1], math.nan)], 1))
    for name, t, n in zip(("dq", "dk", "dv"), got, (N, S, S)):
        assert (t[:, n] == 0).all()
        within(name, flat4(t[:, :n]), ref[name], tol[name])


def test_counts_past_32_bits(mm):
    """64-bit counts on the device are clamped, not cut off; one list of lengths serves rows and fewer keys."""
    fn = mm.attention.attention
    q, k, v = (torch.randn(2, 40, 2, 64, device="cuda").to(BF) for _ in "qkv")
    assert torch.equal(fn(q, k, v, lengths=torch.tensor([2 ** 32 + 5, 2 ** 40], device="cuda")), fn(q, k, v))
    assert (fn(q, k, v, lengths=torch.tensor([-2 ** 40, -2 ** 32 + 9], device="cuda")) == 0).all()
    assert torch.equal(fn(q, k, v, causal=True, prefix=[2 ** 32, 2 ** 33]), fn(q, k, v))
    lens = [40, 3]
    with pytest.raises(ValueError):
        fn(q, k[:, :30], v[:, :30], lengths=lens, kv_lengths=lens)
    assert fn(q[:0], k[:0], v[:0], lengths=[]).shape == q[:0].shape


MANY = [
    # as TOKENS: keys in one chunk (shared heads, many streams), and rows of several tiles over many keys
    (1, [1, 0, 200, 129, 33, 150, 64] * 20, 200, 8, 2, 64, BF, True, False, False, 0.0),
    (3, [512, 500, 31] * 35, 512, 6, 1, 32, HF, True, False, True, 15.0),
    (300, [5000, 299, 1024], 5000, 2, 2, 64, HF, True, False, False, 0.0),
    (129, [2500], 2500, 6, 2, 128, BF, True, True, True, 0.0),
    (700, [3000, 20], 3000, 3, 1, 40, BF, False, False, False, 9.0),
]


@pytest.mark.parametrize("case", MANY, ids=lambda c: f"{c[0]}x{c[2]}x{c[3]}x{c[5]}")
def test_rows_over_kept_keys(mm, O, case):
    test_few_rows_over_many_keys(mm, O, case)


LONG = [
    # few blocks and long walks: both passes of the gradients in parts
    ("padded", ([1500, 3], 1500, None, 1500, 2, 1, 128, HF, True, False, False, 0.0)),
    ("padded", ([1100], 1100, None, 1100, 1, 1, 40, BF, False, False, True, 7.0)),
    ("padded", ([90, 2000], 2000, [2100, 0], 2100, 4, 2, 64, HF, True, True, False, 0.0)),
    ("packed", ([1300, 20, 0], 5, 140, 3, 1, 64, BF, True, True, False, 0.0)),
    ("packed", ([2050], 0, 0, 2, 2, 72, HF, False, False, False, 12.0)),
]


@pytest.mark.parametrize("form, case", LONG, ids=lambda c: c if isinstance(c, str) else f"{c[0]}x{c[-8]}x{c[-6]}")
def test_gradients_in_parts(mm, O, form, case):
    (test_padded if form == "padded" else test_packed)(mm, O, case)


def test_cut_walks_keep_nan_and_empty_rows(mm):
    """1200 rows over 1200 keys of one head: a NaN in any part of the keys reaches every row that sees it; rows that see no key are zeros."""
    fn = mm.attention.attention
    q, k, v = (torch.randn(1, 1200, 1, 64, device="cuda").to(HF) for _ in "qkv")
    want, lse = fn(q, k, v, lengths=[1000], kv_lengths=[700], causal=True, return_lse=True)        # the first 300 rows see nothing
    assert (want[0, :300] == 0).all() and (lse[0, 0, :300] == -math.inf).all() and want[0, 300:1000].abs().amin() >= 0
    assert lse[0, 0, 300:1000].isfinite().all() and (want[0, 1000:] == 0).all() and (lse[0, 0, 1000:] == -math.inf).all()
    for at in (0, 31, 32, 599, 600, 1199):
        x = k.clone()
        x[0, at, 0, 5] = math.nan
        assert fn(q, x, v).isnan().all()
        y, l = fn(q, x, v, causal=True, return_lse=True)
        assert y[0, at:].isnan().all() and l[0, 0, at:].isnan().all() and not y[0, :max(0, at - 63)].isnan().any()


@pytest.mark.parametrize("rows, keys, heads, kv", [(1200, 1200, 2, 1), (3, 5000, 4, 2), (200, 3000, 2, 2)])
def test_cut_walks_in_graphs(mm, rows, keys, heads, kv):
    """Two graphs of calls whose walks are cut, each with its workspaces, replayed in turn and between eager calls on another stream."""
    fn = mm.attention.attention

    def make(seed):
        gen = torch.Generator("cuda").manual_seed(seed)
        t = [torch.randn(2, n, h, 64, device="cuda", generator=gen).to(HF) for n, h in ((rows, heads), (keys, kv), (keys, kv), (rows, heads))]
        return t + [torch.tensor([keys, keys // 2], dtype=torch.int32, device="cuda")]

    def step(q, k, v, g, lens):
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        o = fn(q, k, v, kv_lengths=lens, causal=True)
        return (o.detach(),) + torch.autograd.grad(o, [q, k, v], g)
    sets = [make(0), make(1)]
    for s in sets:
        step(*s)
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step(*s)
        graphs.append((g, got))
    side = torch.cuda.Stream()
    for i in range(3):
        for s, fresh in zip(sets, (make(10 + i), make(20 + i))):
            for a, b in zip(s, fresh):
                a.copy_(b)
            s[4][1] = keys // 2 - i
        graphs[0][0].replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step(*sets[1])
        graphs[1][0].replay()
        torch.cuda.current_stream().wait_stream(side)
        for (_, got), s in zip(graphs, sets):
            assert all(torch.equal(a, b) for a, b in zip(got, step(*s)))
        assert all(torch.equal(a, b) for a, b in zip(other, graphs[1][1]))
        torch.cuda.synchronize()


def turned(t):
    return t.transpose(0, -1).contiguous().transpose(0, -1)


@pytest.mark.parametrize("B, n, s, H, K, packed", [(2, 193, 193, 4, 4, False), (2, 300, 300, 4, 2, False), (1, 1100, 1300, 2, 1, False), (2, 20, 3000, 4, 2, False),
                                                   (1, 260, 260, 4, 2, True), (1, 1500, 1500, 2, 2, True)])
@pytest.mark.parametrize("dtype", [HF, BF])
def test_gradients_under_saved_tensor_hooks(mm, dtype, B, n, s, H, K, packed):
    """Views of one packed projection whose saved tensors come back in other layouts (host copies, clones, recomputation), with counts that are
    changed in between: the bits of the plain run."""
    from torch.autograd.graph import save_on_cpu, saved_tensors_hooks
    from torch.utils.checkpoint import checkpoint
    fn = mm.attention.attention
    gen = torch.Generator().manual_seed(n + s)
    room = max(n, s)
    qkv = torch.randn(B, room, H + 2 * K, 64, generator=gen).to(dtype).cuda()
    q, k, v = qkv[:, :n, :H], qkv[:, :s, H:H + K], qkv[:, :s, H + K:]
    g = torch.randn(B, n, H, 64, generator=gen).to(dtype).cuda()
    if packed:
        q, k, v, g = q[0], k[0], v[0], g[0]
        cuts = [0, n // 3, n - 5]
    else:
        cuts = [n] * B
        cuts[-1] = n - 7

    def run(counts, prefix, hooks=None, again=False):
        x = [t.detach().requires_grad_() for t in (q, k, v)]
        call = lambda *x: fn(*x, causal=True, prefix=prefix, **(dict(offsets=counts) if packed else dict(lengths=counts)))
        if hooks is None:
            o = checkpoint(call, *x, use_reentrant=False) if again else call(*x)
        else:
            with hooks:
                o = call(*x)
            counts.fill_(0)
            prefix.fill_(0)
        return (o.detach(),) + torch.autograd.grad(o, x, g)

    def fresh():
        return torch.tensor(cuts, dtype=torch.int32, device="cuda"), torch.tensor([3] * (2 if packed else B), dtype=torch.int32, device="cuda")
    want = run(*fresh())
    keep = lambda t: t.detach().clone(memory_format=torch.preserve_format)
    for hooks in (save_on_cpu(pin_memory=True), save_on_cpu(), saved_tensors_hooks(keep, lambda t: t.contiguous().clone()), saved_tensors_hooks(keep, turned),
                  saved_tensors_hooks(keep, lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t))):
        got = run(*fresh(), hooks)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(run(*fresh(), again=True), want))


CAPPED = [
    # as PADDED: one block a head, two passes, cut walks, chunks of keys, every head size
    ([193, 30], 193, None, 193, 2, 2, 64, HF, False, False, False),
    ([100], 100, None, 100, 2, 2, 32, BF, True, False, True),
    ([300, 31], 300, None, 300, 4, 2, 64, BF, True, True, False),
    ([260], 260, None, 260, 2, 1, 128, HF, True, False, True),
    ([1100], 1100, None, 1100, 1, 1, 72, HF, False, False, False),
    ([1, 1], 1, [4000, 700], 4000, 4, 1, 64, HF, True, False, False),
    ([3], 3, [3000], 3000, 4, 2, 128, BF, True, False, True),
]


@pytest.mark.parametrize("cap, size", [(5.0, 4.0), (50.0, 20.0), (50.0, 1.0), (1e3, 1.0), (1e4, 1.0), (1e4, 60.0), (1e6, 1.0), (1e30, 1.0), (3e38, 1.0)])
@pytest.mark.parametrize("case", CAPPED, ids=lambda c: f"{c[0]}x{c[3]}x{c[6]}")
def test_capped_scores_of_any_cap(mm, O, case, cap, size):
    """The error of a capped score is bounded by the score, however large the cap; scores of a few units (size 1) and across half the cap."""
    class Relative:
        attention = staticmethod(lambda *a, **k: O.attention(*a, relative=True, **k))
    lens, N, kv, S, H, K, D, dtype, causal, prefix, bias = case
    B = len(lens)
    gen = torch.Generator().manual_seed(N + S + D)
    q = (size * torch.randn(B, N, H, D, generator=gen)).to(dtype).cuda()
    k, v = (torch.randn(B, S, K, D, generator=gen).to(dtype).cuda() for _ in "kv")
    g = torch.randn(B, N, H, D, generator=gen).to(dtype).cuda()
    m = kv or lens
    host, opts = {}, dict(causal=causal, cap=cap, lengths=lens, kv_lengths=m)
    if prefix:
        host["prefix"] = opts["prefix"] = [x // 2 for x in m]
    if bias:
        host["slopes"] = opts["slopes"] = slopes_of(H)
    for b in range(B):
        for t, n in ((q, lens[b]), (g, lens[b]), (k, m[b]), (v, m[b])):
            t[b, n:] = math.nan
    check(mm, Relative, q, k, v, docs_padded(lens, m, N, S), opts, g=g, flat=flat4, lse_flat=lse4, host=host)


def test_cut_walks_with_rows_that_see_nothing(mm, O):
    """1000 of 1200 rows over 700 of 1200 keys of one head, causal, walks cut: the rows that see keys, next to 300 that see none."""
    gen = torch.Generator().manual_seed(21)
    q, k, v, g = (torch.randn(1, 1200, 1, 64, generator=gen).to(HF).cuda() for _ in range(4))
    check(mm, O, q, k, v, docs_padded([1000], [700], 1200, 1200), dict(causal=True, lengths=[1000], kv_lengths=[700]), g=g, flat=flat4, lse_flat=lse4)


@pytest.mark.parametrize("rows, H, K, D, causal", [(2000, 2, 1, 64, False), (2000, 2, 2, 64, True), (1300, 4, 2, 128, True), (1100, 2, 1, 96, False), (1500, 1, 1, 32, True)])
@pytest.mark.parametrize("dtype", [HF, BF])
def test_long_documents_in_the_mean(mm, O, dtype, rows, H, K, D, causal):
    """The bounds of single elements add up worst cases over the keys, and would let a lost tile of 32 keys pass among 2000.  Roundings are independent:
    a result's mean square error is the sum of its terms' squares, (u p v)^2 over the keys for o, (u p g)^2 over the rows for dv, (u scale ds k)^2 and
    (u scale ds q)^2 for dq and dk, and (u x)^2 for its own rounding, u half a step of the type, at which a rounding's mean square is at most a third of u^2."""
    gen = torch.Generator().manual_seed(rows + D)
    q, g = (torch.randn(1, rows, H, D, generator=gen).to(dtype).cuda() for _ in "qg")
    k, v = (torch.randn(1, rows, K, D, generator=gen).to(dtype).cuda() for _ in "kv")
    x = [t.detach().requires_grad_() for t in (q, k, v)]
    o = mm.attention.attention(*x, causal=causal)
    dq, dk, dv = torch.autograd.grad(o, x, g)
    u, scale = torch.finfo(dtype).eps / 2, D ** -0.5
    ref = {n: torch.zeros(rows, h, D, dtype=torch.float64, device="cuda") for n, h in (("o", H), ("dq", H), ("dk", K), ("dv", K))}
    var = {n: torch.zeros_like(t) for n, t in ref.items()}
    for h in range(H):
        c = h // (H // K)
        a = [t.double() for t in (q[0, :, h], k[0, :, c], v[0, :, c], g[0, :, h])]
        r = O.attention_head(*a[:3], scale, causal=causal, g=a[3])
        p2, ds2 = r["p"].square(), (scale * r["ds"]).square()
        ref["o"][:, h], ref["dq"][:, h] = r["o"], r["dq"]
        ref["dk"][:, c] += r["dk"]
        ref["dv"][:, c] += r["dv"]
        var["o"][:, h] = p2 @ a[2].square()
        var["dq"][:, h] = ds2 @ a[1].square()
        var["dk"][:, c] += ds2.T @ a[0].square()
        var["dv"][:, c] += p2.T @ a[3].square()
    for name, got in (("o", o), ("dq", dq), ("dk", dk), ("dv", dv)):
        # in blocks of 100 rows, so that the few large ones do not cover the others
        err, bound = ((t.flatten(1).mean(1).split(100)) for t in ((got.detach()[0].double() - ref[name]).square(), u * u * (var[name] + ref[name].square())))
        for i, (e, b) in enumerate(zip(err, bound)):
            assert float(e.mean()) <= float(b.mean()), (name, i, float((e.mean() / b.mean()).sqrt()))


CROSS = [
    # rows of each document, keys of each, rows before and behind, keys before and behind, H, K, D, dtype, causal, prefix, bias, cap
    ([5, 200, 0, 64, 129], [300, 10, 7, 0, 129], (3, 9), (0, 40), 4, 2, 64, BF, True, True, False, 0.0),
    ([1, 1, 3, 1], [5000, 0, 1300, 31], (0, 0), (0, 0), 8, 2, 128, HF, True, False, True, 0.0),        # new tokens over packed keys, walks cut
    ([1500, 20], [40, 900], (0, 1), (130, 0), 2, 1, 72, BF, False, False, True, 9.0),
    ([3, 0, 7] * 30, [0, 5, 150] * 30, (2, 0), (0, 3), 2, 2, 32, HF, True, True, False, 100.0),        # more than 64 documents
    ([130, 1] * 40, [1, 257] * 40, (0, 0), (0, 0), 3, 1, 96, BF, False, False, False, 0.0),
]


@pytest.mark.parametrize("case", CROSS, ids=lambda c: f"{len(c[0])}x{c[4]}x{c[6]}")
def test_packed_rows_with_keys_of_their_own(mm, O, case):
    lens, kv, (lead, tail), (klead, ktail), H, K, D, dtype, causal, prefix, bias, cap = case
    off, koff = [lead], [klead]
    for n, m in zip(lens, kv):
        off.append(off[-1] + n)
        koff.append(koff[-1] + m)
    T, S = off[-1] + tail, koff[-1] + ktail
    gen = torch.Generator().manual_seed(T + S)
    q, g = (torch.randn(T, H, D, generator=gen).to(dtype).cuda() for _ in "qg")
    k, v = (torch.randn(S, K, D, generator=gen).to(dtype).cuda() for _ in "kv")
    for ts, o in (((q, g), off), ((k, v), koff)):
        for t in ts:
            t[:o[0]] = math.nan
            t[o[-1]:] = math.inf
    host, opts = {}, dict(causal=causal, cap=cap, offsets=off, kv_offsets=torch.tensor(koff, device="cuda"))
    if prefix:
        host["prefix"] = opts["prefix"] = [n // 3 + 5 for n in kv]                # past the keys of some documents
    if bias:
        host["slopes"] = opts["slopes"] = slopes_of(H)
    docs = [(off[d], lens[d], koff[d], kv[d]) for d in range(len(lens))]
    check(mm, O, q, k, v, docs, opts, g=g, host=host)


def test_broadcast_rows_and_gradients(mm):
    """Tensors and gradients that repeat one row (stride 0) give the bits of their written-out copies."""
    fn = mm.attention.attention
    gen = torch.Generator().manual_seed(31)
    for n, s, H, K in ((70, 70, 2, 2), (300, 300, 4, 2), (1200, 1300, 1, 1), (3, 3000, 4, 1)):
        q, k, v = (torch.randn(1, 1, h, 64, generator=gen).to(HF).cuda() for h in (H, K, K))
        g = torch.randn(64, generator=gen).to(HF).cuda()
        views = [q.expand(2, n, -1, -1), k.expand(2, s, -1, -1), v.expand(2, s, -1, -1), g.expand(2, n, H, 64)]

        def run(q, k, v, g):
            x = [t.detach().requires_grad_() for t in (q, k, v)]
            o = fn(*x, causal=True)
            return (o.detach(),) + torch.autograd.grad(o, x, g)
        assert all(torch.equal(a, b) for a, b in zip(run(*views), run(*(t.contiguous() for t in views))))
