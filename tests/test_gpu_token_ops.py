"""Rotary positions (csrc/rotary.hip) and gradient norm and clipping (csrc/gradients.hip) against float64 restatements.

Tolerances.  u = 2^-24.  Rotary: a float32 product pair with |cos| + |sin| <= sqrt(2); cosine and sine are within 2 u of the true
ones plus the angle's rounding (a turn in [-1/2, 1/2] rounded to float32: 2 pi 2^-26 = 1.6 u); two products and a sum add 2 u:
6 u (|x| + |y|) covers them, 8 is asserted.  Norm: float64 sums, rounded once: 1 u, 2 asserted.  Clipped values: the limit, the norm, norm + 1e-6, the quotient and
the product are rounded once each: 5 u relative, 6 asserted.  16-bit results add half a step: eps / 2 relative, or half the smallest subnormal."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def mm():
    import multi_modal_amd as m
    m.load_library()
    assert torch.cuda.is_available()
    return m


def half_step(ref, dtype):
    if dtype == torch.float32:
        return ref.abs() * U
    info = torch.finfo(dtype)
    return torch.maximum(ref.abs() * (info.eps / 2), torch.full_like(ref, info.smallest_normal * info.eps / 2))


def rotary_ref(x, pos, sections, base, ladder, pairing, sign=1.0):
    """float64, pair by pair; returns the rotated tensor and sum of magnitudes of each pair."""
    x = x.detach().cpu().double()
    pos = pos.cpu().double()
    if pos.dim() == 2:
        pos = pos[:, None]
    R = sum(sections)
    y, mag = x.clone(), torch.zeros_like(x)
    i = 0
    for a, n in enumerate(sections):
        for j in range(n):
            theta = base ** (-(i / R if ladder == "shared" else j / n))
            phi = (sign * pos[a] * theta)[..., None]
            u, w = (i, i + R) if pairing == "halves" else (2 * i, 2 * i + 1)
            y[..., u] = x[..., u] * phi.cos() - x[..., w] * phi.sin()
            y[..., w] = x[..., w] * phi.cos() + x[..., u] * phi.sin()
            mag[..., u] = mag[..., w] = x[..., u].abs() + x[..., w].abs()
            i += 1
    return y, mag


def check_rotary(got, x, pos, rot, sign=1.0):
    ref, mag = rotary_ref(x, pos, rot.sections, rot.base, rot.ladder, rot.pairing, sign)
    got = got.cpu()
    err = (got.double() - ref).abs()
    tol = 8 * U * mag
    if got.dtype != torch.float32:
        tol = tol + half_step(ref.abs() + tol, got.dtype)
    assert (err <= tol).all(), (err - tol).max()
    R2 = 2 * sum(rot.sections)
    assert torch.equal(got[..., R2:], x.detach().cpu()[..., R2:])


ROTARY = [
    # B, N, H, K, D, sections, ladder, pairing, dtype
    (1, 1, 1, 1, 2, [1], "axis", "halves", torch.float32),
    (8, 1, 12, 12, 64, [16, 16], "axis", "halves", torch.float16),
    (2, 37, 6, 2, 64, [8, 12, 12], "shared", "halves", torch.bfloat16),
    (3, 193, 4, 4, 72, [9, 10], "axis", "adjacent", torch.float16),
    (2, 50, 3, 1, 80, [7, 5, 11], "shared", "halves", torch.float32),       # odd sections: every vector off its alignment
    (2, 50, 3, 1, 80, [7, 5, 11], "axis", "adjacent", torch.bfloat16),
    (1, 1000, 2, 2, 128, [10, 20, 20, 14], "shared", "adjacent", torch.float32),
    (4, 9, 5, 3, 33, [0, 16], "axis", "halves", torch.float16),             # an empty section, an odd head size
    (1, 5, 1, 1, 1024, [512], "shared", "halves", torch.bfloat16),
    (33, 700, 6, 6, 32, [8, 8], "axis", "halves", torch.bfloat16),
]


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("case", ROTARY, ids=lambda c: "x".join(map(str, c[:5])))
def test_rotary(mm, case, wide):
    B, n, H, K, D, sections, ladder, pairing, dtype = case
    g = torch.Generator().manual_seed(n * 31 + D)
    rot = mm.Rotary(sections, ladder=ladder, pairing=pairing)
    q, k = torch.randn(B, n, H, D, generator=g).to(dtype), torch.randn(B, n, K, D, generator=g).to(dtype)
    pos = torch.randint(-50, 100000, (len(sections), B, n) if wide else (len(sections), n), generator=g)
    pos = pos.to(torch.int64 if wide else torch.int32).cuda()
    yq, yk = rot(q.cuda(), k.cuda(), pos)
    check_rotary(yq, q, pos, rot)
    check_rotary(yk, k, pos, rot)
    assert torch.equal(rot(q.cuda(), None, pos), yq)
    # in place, and from the CPU: the same bits
    q2, k2 = q.cuda(), k.cuda()
    r = rot(q2, k2, pos, inplace=True)
    assert r[0] is q2 and torch.equal(q2, yq) and torch.equal(k2, yk)
    zq, zk = rot(q, k, pos.cpu())
    assert not zq.is_cuda and torch.equal(zq, yq.cpu()) and torch.equal(zk, yk.cpu())


def test_rotary_far_positions(mm):
    """Positions of 2^40 and of both signs keep their phase to what float64 holds of it: 2^40 * 2^-53 radians at most."""
    rot = mm.Rotary([4, 4], ladder="axis")
    q = torch.randn(1, 6, 2, 16, generator=torch.Generator().manual_seed(1))
    pos = torch.tensor([[0, 1, -1, 2 ** 40 + 1, -2 ** 40, 2 ** 31 + 7], [2 ** 33, 5, 0, -7, 2 ** 39, 1]])
    y = rot(q.cuda(), None, pos.cuda())
    ref, mag = rotary_ref(q, pos, rot.sections, rot.base, rot.ladder, rot.pairing)
    assert ((y.cpu().double() - ref).abs() <= (8 * U + 4 * 2.0 ** -13) * mag).all()
    near = pos.abs().max(0).values < 2 ** 31
    assert ((y.cpu().double() - ref).abs() <= (8 * U + 1e-6) * mag)[:, near].all()


def test_rotary_strided_views_in_place(mm):
    """Queries and keys inside one packed projection, rotated where they are: values and everything else untouched."""
    rot = mm.Rotary([8, 8], pairing="halves")
    qkv = torch.randn(3, 20, 4 + 2 + 2, 40, generator=torch.Generator().manual_seed(2)).to(torch.float16).cuda()
    before = qkv.clone()
    pos = mm.grid_positions(4, 5, device="cuda")
    rot(qkv[:, :, :4], qkv[:, :, 4:6], pos, inplace=True)
    check_rotary(qkv[:, :, :4], before[:, :, :4], pos, rot)
    check_rotary(qkv[:, :, 4:6], before[:, :, 4:6], pos, rot)
    assert torch.equal(qkv[:, :, 6:], before[:, :, 6:])
    t = before.transpose(1, 2)[:, :4].transpose(1, 2)             # the same tensor through other strides
    assert torch.equal(rot(t, None, pos), qkv[:, :, :4])
    odd = torch.empty(3 * 20 * 4 * 40 + 1, dtype=torch.float16, device="cuda")[1:].view(3, 20, 4, 40).copy_(before[:, :, :4])     # off every alignment
    assert torch.equal(rot(odd, None, pos), qkv[:, :, :4])
    wide = before[:, :, :4].expand(3, 20, 4, 40)[:1].expand(3, 20, 4, 40)            # a broadcast batch
    assert torch.equal(rot(wide, None, pos)[2], rot(before[:1, :, :4], None, pos)[0])


@pytest.mark.parametrize("pairing", ["halves", "adjacent"])
@pytest.mark.parametrize("dtype", TYPES)
def test_rotary_gradient(mm, dtype, pairing):
    rot = mm.Rotary([5, 3, 4], ladder="shared", pairing=pairing)
    g = torch.Generator().manual_seed(3)
    q = torch.randn(2, 30, 4, 32, generator=g).to(dtype).cuda().requires_grad_()
    k = torch.randn(2, 30, 2, 32, generator=g).to(dtype).cuda().requires_grad_()
    gq, gk = torch.randn(2, 30, 4, 32, generator=g).to(dtype).cuda(), torch.randn(2, 30, 2, 32, generator=g).to(dtype).cuda()
    pos = torch.randint(0, 4000, (3, 2, 30), generator=g).cuda()
    yq, yk = rot(q, k, pos)
    dq, dk = torch.autograd.grad([yq, yk], [q, k], [gq, gk])
    check_rotary(dq, gq, pos, rot, sign=-1.0)
    check_rotary(dk, gk, pos, rot, sign=-1.0)
    # one of the two only, a broadcast gradient, and against differences: y is linear in q, so <g, y(q + d) - y(q)> = <dq, d>
    (only,) = torch.autograd.grad(rot(q, k.detach(), pos)[0].float().sum(), [q])
    check_rotary(only, torch.ones_like(gq), pos, rot, sign=-1.0)
    if dtype == torch.float32:
        d = torch.randn(q.shape, generator=g).cuda()
        with torch.no_grad():
            diff = (gq.double() * (rot(q + d, k, pos)[0].double() - rot(q, k, pos)[0].double())).sum()
        size = (gq.double().abs() * 2 * (q.double().abs() + d.double().abs())).sum()
        assert abs(float((diff - (dq.double() * d.double()).sum()).detach())) <= 32 * U * float(size.detach())


def test_rotary_streams_graph_and_refusals(mm):
    rot = mm.Rotary([8, 8])
    q = torch.randn(2, 30, 4, 32, device="cuda").to(torch.bfloat16)
    k = torch.randn(2, 30, 2, 32, device="cuda").to(torch.bfloat16)
    pos = mm.grid_positions(5, 6, device="cuda")
    want = rot(q, k, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rot(q, k, pos)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yq, yk = rot(q, k, pos)
    for i in range(3):
        q.copy_(torch.randn(q.shape, device="cuda"))
        pos.add_(i)
        graph.replay()
        want = rot(q, k, pos)
        assert torch.equal(yq, want[0]) and torch.equal(yk, want[1])
    for call, error in [
        (lambda: rot(q[0], k, pos), ValueError), (lambda: rot(q, k[:1], pos), ValueError), (lambda: rot(q, k.float(), pos), ValueError),
        (lambda: rot(q.double(), None, pos), ValueError), (lambda: rot(q[..., :16], None, pos), ValueError),
        (lambda: rot(q, k, pos[:1]), ValueError), (lambda: rot(q, k, pos[:, :7]), ValueError), (lambda: rot(q, k, pos.float()), TypeError),
        (lambda: rot(q, q, pos, inplace=True), ValueError), (lambda: rot(q[:1].expand(2, 30, 4, 32), None, pos, inplace=True), ValueError),
        (lambda: rot(q.clone().requires_grad_(), None, pos, inplace=True), RuntimeError), (lambda: rot(q.cpu(), None, pos, inplace=True), ValueError),
    ]:
        with pytest.raises(error):
            call()
    empty = rot(q[:, :0], k[:, :0], pos[:, :0])
    assert empty[0].shape == (2, 0, 4, 32) and empty[1].shape == (2, 0, 2, 32)


def clip_ref(grads, max_norm, kind):
    gs = [g.detach().cpu().double() for g in grads]
    if kind == math.inf:
        norm = max([float(g.abs().max()) for g in gs if g.numel()], default=0.0)
    else:
        norm = math.sqrt(sum(float((g * g).sum()) for g in gs))
    return norm, [g * min(1.0, max_norm / (norm + 1e-6)) for g in gs]


def check_clipped(got, ref, dtype):
    tol = 6 * U * ref.abs()
    if dtype != torch.float32:
        tol = tol + half_step(ref.abs() + tol, dtype)
    assert got.dtype == dtype and ((got.cpu().double() - ref).abs() <= tol).all()


SIZES = {"one": [1], "layer": [(768, 1, 16, 16), 768], "odd": [1, 3, 255, 16383, 16384, 16385, 70001, 0, 5],
         "many": [7 + 13 * i for i in range(400)], "large": [6_000_003, 9]}


@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("dtype", TYPES + ["mixed"])
@pytest.mark.parametrize("sizes", SIZES)
def test_clip(mm, sizes, dtype, kind):
    g = torch.Generator().manual_seed(5)
    grads = []
    for i, s in enumerate(SIZES[sizes]):
        t = TYPES[i % 3] if dtype == "mixed" else dtype
        grads.append((torch.randn(s, generator=g) * 0.01 * (1 + i % 5)).to(t).cuda())
    for factor in (0.3, 3.0):
        norm, _ = clip_ref(grads, 1.0, kind)
        limit = float(torch.tensor(norm * factor, dtype=torch.float32))
        _, ref = clip_ref(grads, limit, kind)
        assert abs(float(mm.grad_norm(grads, kind)) - norm) <= 2 * U * norm
        outs = [torch.full((x.numel(),), -1.0, dtype=TYPES[(i + 1) % 3], device="cuda") for i, x in enumerate(grads)]
        keep = [x.clone() for x in grads]
        got = mm.clip_grad_norm(grads, limit, kind, out=outs)
        assert abs(float(got) - norm) <= 2 * U * norm and all(torch.equal(a, b) for a, b in zip(grads, keep))
        for o, r in zip(outs, ref):
            check_clipped(o, r.reshape(-1), o.dtype)
        again = mm.clip_grad_norm(keep, limit, kind)
        assert torch.equal(again, got)                            # a fixed order of sums: the same bits
        for x, k, r in zip(grads, keep, ref):
            check_clipped(k, r, x.dtype)
            if factor > 1:
                assert torch.equal(x, k)


def test_clip_large_and_nonfinite_values(mm):
    big = [torch.full((1000,), 3e38, device="cuda"), torch.full((10,), 3e38, device="cuda").to(torch.bfloat16)]
    norm, ref = clip_ref(big, 1.0, 2.0)
    assert norm > 3.5e38 and math.isinf(float(mm.grad_norm(big)))            # past float32's range: infinite, as its float32 is
    small = [torch.full((1000,), 1e-30, device="cuda")]                       # squares below float32's range
    norm, _ = clip_ref(small, 1.0, 2.0)
    assert abs(float(mm.grad_norm(small)) - norm) <= 2 * U * norm
    assert abs(float(mm.grad_norm([torch.full((100,), 2e38, device="cuda") / 10])) - 2e38) <= 2e38 * 2.0 ** -22
    for kind in (2.0, math.inf):
        x = [torch.ones(5000, device="cuda"), torch.ones(40000, device="cuda").to(torch.float16)]
        x[1][39999] = math.inf
        assert math.isinf(float(mm.clip_grad_norm(x, 1.0, kind)))
        assert (x[0] == 0).all() and x[1][39999].isnan() and (x[1][:-1] == 0).all()
        x = [torch.ones(5000, device="cuda"), torch.ones(40000, device="cuda").to(torch.bfloat16)]
        x[1][20001] = math.nan
        keep = [t.clone() for t in x]
        with pytest.raises(RuntimeError):
            mm.clip_grad_norm(x, 1.0, kind, error_if_nonfinite=True)
        assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(x, keep))
        assert math.isnan(float(mm.clip_grad_norm(x, 1.0, kind))) and x[0].isnan().all() and x[1].isnan().all()
    z = [torch.zeros(100, device="cuda")]
    assert float(mm.clip_grad_norm(z, 0.5)) == 0.0 and (z[0] == 0).all()
    x = [torch.randn(100, device="cuda")]
    mm.clip_grad_norm(x, 0.0)
    assert (x[0] == 0).all()


def test_clip_parameters_layouts_and_refusals(mm):
    g = torch.Generator().manual_seed(9)
    lin = torch.nn.Linear(33, 17).cuda()
    lin.weight.grad = torch.randn(33, 17, generator=g).cuda().t()                             # dense, transposed
    keep = lin.weight.grad.clone()
    norm, ref = clip_ref([keep], 0.1, 2.0)
    assert abs(float(mm.clip_grad_norm(lin.parameters(), 0.1)) - norm) <= 2 * U * norm        # the bias has no gradient
    check_clipped(lin.weight.grad, ref[0], torch.float32)
    buf = torch.randn(10, 40, generator=g).cuda()
    rows = [buf[:, :7], buf[:, 9:30]]                                                          # views with gaps
    norm, ref = clip_ref(rows, 0.1, 2.0)
    rest = buf[:, 30:].clone()
    assert abs(float(mm.clip_grad_norm(rows, 0.1)) - norm) <= 2 * U * norm
    check_clipped(rows[0], ref[0], torch.float32)
    check_clipped(rows[1], ref[1], torch.float32)
    assert torch.equal(buf[:, 30:], rest)
    flat = torch.randn(1001, generator=g).to(torch.float16).cuda()
    cuts = [flat[:1], flat[1:4], flat[4:501], flat[501:]]                                      # every alignment
    norm, ref = clip_ref(cuts, 0.5, 2.0)
    mm.clip_grad_norm(cuts, 0.5)
    for c, r in zip(cuts, ref):
        check_clipped(c, r, torch.float16)
    assert float(mm.clip_grad_norm([], 1.0)) == 0.0 and float(mm.grad_norm([])) == 0.0
    x = torch.randn(10, device="cuda")
    for call, error in [
        (lambda: mm.clip_grad_norm([x, x], 1.0), mm.MmfeError), (lambda: mm.clip_grad_norm([x[:6], x[5:]], 1.0), mm.MmfeError),
        (lambda: mm.clip_grad_norm([x.double()], 1.0), TypeError), (lambda: mm.clip_grad_norm([x.cpu()], 1.0), ValueError),
        (lambda: mm.clip_grad_norm([x, x.cpu()], 1.0), ValueError), (lambda: mm.clip_grad_norm([x], 1.0, out=[]), ValueError),
        (lambda: mm.clip_grad_norm([x], 1.0, out=[x[:5]]), ValueError), (lambda: mm.clip_grad_norm([x], 1.0, out=[torch.empty(20, device="cuda")[::2]]), ValueError),
        (lambda: mm.clip_grad_norm([x[:1].expand(8)], 1.0), ValueError), (lambda: mm.clip_grad_norm([x], 1.0, out=[x.view(torch.int32)]), TypeError),
        (lambda: mm.clip_grad_norm([x.to_sparse()], 1.0), TypeError),
    ]:
        keep = x.clone()
        with pytest.raises(error):
            call()
        assert torch.equal(x, keep)
    assert abs(float(mm.grad_norm([x, x])) - math.sqrt(2) * float(x.double().norm())) <= 4 * U * 20


def test_clip_graph(mm):
    x = [torch.randn(50000, device="cuda"), torch.randn(77, device="cuda").to(torch.bfloat16)]
    mm.clip_grad_norm([t.clone() for t in x], 1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = mm.clip_grad_norm(x, 1.0)
    for _ in range(3):
        for t in x:
            t.copy_(torch.randn(t.shape, device="cuda"))
        want = [t.clone() for t in x]
        graph.replay()
        n = mm.clip_grad_norm(want, 1.0)
        assert torch.equal(n, norm) and all(torch.equal(a, b) for a, b in zip(x, want))


@pytest.mark.parametrize("case", [
    (3, 301, 5, 2, 128, [1, 4], "axis", "halves", torch.float16),           # fewer pairs than a vector, a long rest
    (3, 301, 5, 2, 64, [1, 2], "axis", "adjacent", torch.bfloat16),
    (2, 130, 2, 2, 64, [16, 15], "shared", "halves", torch.bfloat16),       # a rest of two elements
    (2, 130, 2, 1, 41, [5], "axis", "halves", torch.float32),
    (1, 9, 1, 1, 6, [3], "axis", "adjacent", torch.float16),                # a head smaller than a vector
    (2, 600, 16, 4, 128, [15, 21, 27], "shared", "halves", torch.float16),
], ids=lambda c: "x".join(map(str, c[:5])))
def test_rotary_sections_of_any_size(mm, case):
    test_rotary(mm, case, True)


def test_clipping_rounds_twice_and_infinite_norms_give_zeros(mm):
    """The factor is rounded once and the product once: 2 halves of 2^-23.  A norm past float32's range is infinite and leaves zeros."""
    g = [torch.randn(3000, device="cuda", generator=torch.Generator("cuda").manual_seed(i)) * 10.0 ** (i - 3) for i in range(6)]
    exact = math.sqrt(sum(float(t.double().square().sum()) for t in g))
    factor = 0.5 / (exact + 1e-6)
    want = [t.double() * factor for t in g]
    norm = mm.clip_grad_norm(g, 0.5)
    assert abs(float(norm) - exact) <= 2.0 ** -24 * exact
    for a, b in zip(g, want):
        assert ((a.double() - b).abs() <= 2.01 * 2.0 ** -24 * b.abs()).all()
    big = torch.full((8,), 3e38, device="cuda")
    assert mm.clip_grad_norm([big], 1.0).isinf() and (big == 0).all()


@pytest.mark.parametrize("kind", [2.0, math.inf])
def test_infinite_limits(mm, kind):
    """max_norm = inf measures the norm and leaves the gradients alone, unless the norm is infinite: NaN then, as torch's own has it."""
    for value, scaled in ((2.0, 1.0), (math.inf, math.nan), (math.nan, math.nan)):
        x = [torch.ones(5000, device="cuda"), torch.ones(70, device="cuda").to(torch.bfloat16)]
        x[1][3] = value
        want = [torch.nn.Parameter(t.float()) for t in x]
        for p, t in zip(want, x):
            p.grad = t.float().clone()
        norm = torch.nn.utils.clip_grad_norm_(want, math.inf, kind)
        outs = [torch.zeros(t.shape, device="cuda") for t in x]
        got = mm.clip_grad_norm(x, math.inf, kind, out=outs)
        assert torch.allclose(got, norm, rtol=2.0 ** -20, atol=0, equal_nan=True)
        mm.clip_grad_norm(x, math.inf, kind)
        for t, o, p in zip(x, outs, want):
            assert torch.equal(t.float().nan_to_num(7.0), p.grad.nan_to_num(7.0)) and torch.equal(o.nan_to_num(7.0), p.grad.nan_to_num(7.0))
            assert torch.equal(t[:3].float().nan_to_num(7.0), torch.full((3,), scaled, device="cuda").nan_to_num(7.0))
    if kind == 2.0:                                    # finite in float64, infinite in float32
        big = torch.full((1000,), 3e38, device="cuda")
        assert mm.clip_grad_norm([big], math.inf).isinf() and big.isnan().all()


def test_clip_views_that_share_memory(mm):
    """Views with gaps go through copies: the same view twice, and views that overlap themselves, are refused as dense ones are; neighbours are not."""
    buf = torch.randn(12, 40, device="cuda")
    keep = buf.clone()
    a = buf[:, :7]
    flat = buf.view(-1)
    for grads in ([a, a], [a, buf[:, 9:12], a], [buf[:, :7], buf[:, :5]], [flat.as_strided((5, 8), (4, 1)), buf[6:, :3]], [a[:1].expand(3, 7), buf[:, 9:12]]):
        with pytest.raises(ValueError, match="share memory"):
            mm.clip_grad_norm(grads, 0.1)
        assert torch.equal(buf, keep)
    _, ref = clip_ref([buf[:, :7], buf[:, 7:20]], 0.1, 2.0)
    mm.clip_grad_norm([buf[:, :7], buf[:0, :3], buf[:, 7:20], buf[:0, 1:4]], 0.1)
    check_clipped(buf[:, :7], ref[0], torch.float32)
    check_clipped(buf[:, 7:20], ref[1], torch.float32)
    assert torch.equal(buf[:, 20:], keep[:, 20:])
