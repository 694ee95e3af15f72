"""The token operators together, as a training step of an encoder uses them: waveforms -> spectrograms -> PatchEmbedLayer tokens -> packed
projection -> rotary positions of the (frequency, time) grid -> attention over clips of different lengths -> loss -> backward ->
clipping -> optimizer, and new tokens over what a stream has kept."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

H, D = 6, 64
E = H * D


@pytest.fixture(scope="module")
def mm():
    import multi_modal_amd as m
    m.load_library()
    assert torch.cuda.is_available()
    return m


class Layer(torch.nn.Module):
    def __init__(self, mm, img):
        super().__init__()
        from multi_modal_amd.patch_embed import PatchEmbedLayer
        self.mm, self.grid = mm, (img[0] // 16, img[1] // 16)
        self.patch_embed = PatchEmbedLayer(img, embed_dim=E, compute_dtype=torch.float16, out_dtype=torch.float16)
        self.qkv = torch.nn.Linear(E, 3 * E)
        self.proj = torch.nn.Linear(E, E)
        self.rotary = mm.Rotary([16, 16])

    def attend(self, tokens, lengths):
        B, N, _ = tokens.shape
        with torch.autocast("cuda", dtype=torch.float16):
            q, k, v = self.qkv(tokens).view(B, N, 3, H, D).unbind(2)
        q, k = self.rotary(q, k, self.mm.grid_positions(*self.grid, device=tokens.device))
        return self.mm.attention.attention(q, k, v, lengths=lengths)

    def forward(self, image, lengths):
        o = self.attend(self.patch_embed(image), lengths)
        with torch.autocast("cuda", dtype=torch.float16):
            return self.proj(o.flatten(2))


def reference(layer, tokens, lengths, g):
    """Gradients of sum(g * output) in float64 from the tokens on."""
    W = {n: p.detach().double().requires_grad_() for n, p in layer.named_parameters() if not n.startswith("patch")}
    x = tokens.detach().double().requires_grad_()
    B, N, _ = x.shape
    q, k, v = (x @ W["qkv.weight"].T + W["qkv.bias"]).view(B, N, 3, H, D).unbind(2)
    pos = layer.mm.grid_positions(*layer.grid, device="cuda").double()

    def rotate(t):
        theta = 10000.0 ** -(torch.arange(16, device="cuda", dtype=torch.float64) / 16)
        phi = torch.cat([pos[a][:, None] * theta for a in (0, 1)], 1)[:, None]           # (N, 1, 32)
        a, b = t[..., :32], t[..., 32:]
        return torch.cat([a * phi.cos() - b * phi.sin(), b * phi.cos() + a * phi.sin()], -1)
    q, k = rotate(q), rotate(k)
    o = torch.zeros_like(q)
    rows = []
    for b in range(B):
        n = int(lengths[b])
        s = torch.matmul(q[b, :n].transpose(0, 1), k[b, :n].permute(1, 2, 0).contiguous()) * D ** -0.5
        y = torch.matmul(torch.softmax(s, -1), v[b, :n].transpose(0, 1).contiguous()).transpose(0, 1)
        rows.append(torch.cat([y, y.new_zeros(N - n, H, D)]))
    out = torch.stack(rows).flatten(2) @ W["proj.weight"].T + W["proj.bias"]
    grads = torch.autograd.grad((out * g).sum(), [x] + list(W.values()))
    return out.detach(), dict(zip(["tokens"] + list(W), grads))


def test_training_step(mm):
    torch.manual_seed(0)
    B = 3
    layer = Layer(mm, (384, 128)).cuda()
    waves = 0.1 * torch.randn(B, 160000, device="cuda")
    image = mm.preprocessing_audio_batch(waves, dtype=torch.float16).unsqueeze(1)          # (B, 1, 384, 128)
    lengths = torch.tensor([192, 100, 33], dtype=torch.int32, device="cuda")
    # The loss is a sum over 3 x 192 tokens, gradients are 2200 in norm against weights of 16: a rate of 0.1 (clipped to a quarter) moves the
    # projection by 55, three times its own size, after which float16 gradients overflow; this one moves it by 0.01.
    optimizer = torch.optim.SGD(layer.parameters(), lr=2e-5)
    for step in range(2):
        out = layer(image, lengths)
        g = torch.randn(out.shape, device="cuda")
        optimizer.zero_grad()
        (out.float() * g).sum().backward()
        tokens = layer.patch_embed(image)
        ref, grads = reference(layer, tokens, lengths, g.double())
        # Between the tokens and a gradient lie at most 14 roundings to float16 (operands, projections, rotations, p, o, their gradients), each
        # 2^-11 of its value at most; values amplify by no more than about 4 from one to the next at initialisation, where a score
        # has a standard deviation of 0.15 (queries and keys 0.4 each, 64 of them, / 8): 14 * 4 * 2^-11 = 0.027.
        rel = {"out": float((out.detach().double() - ref).norm() / ref.norm())}
        for n, p in layer.named_parameters():
            if n in grads:
                rel[n] = float((p.grad.double() - grads[n]).norm() / grads[n].norm())
        assert all(v <= 0.027 for v in rel.values()), rel
        # the patch embedding's gradient, from the reference's gradient of its tokens
        gt = grads["tokens"].reshape(-1, E)
        patches = image.double().reshape(B, 24, 16, 8, 16).permute(0, 1, 3, 2, 4).reshape(-1, 256)
        want = (gt.T @ patches).view(E, 1, 16, 16)
        got = layer.patch_embed.proj.weight.grad.double()
        assert float((got - want).norm() / want.norm()) <= 0.035
        # clipping: the float64 norm of what backward left, and every gradient scaled by one factor
        before = [p.grad.clone() for p in layer.parameters()]
        norm = math.sqrt(sum(float(t.double().square().sum()) for t in before))
        got = mm.clip_grad_norm(layer.parameters(), 0.25 * norm)
        assert abs(float(got) - norm) <= 2.0 ** -22 * norm
        for p, t in zip(layer.parameters(), before):
            assert torch.allclose(p.grad, t * 0.25, rtol=2.0 ** -20, atol=0)
        assert abs(float(mm.grad_norm(layer.parameters())) - 0.25 * norm) <= 2.0 ** -19 * norm
        weight = layer.patch_embed.proj.weight.detach().clone()
        optimizer.step()
        assert not torch.equal(weight, layer.patch_embed.proj.weight)
        assert not torch.equal(tokens, layer.patch_embed(image))                            # the next forward pass has the new weights


def test_chain_gradient_is_its_parts(mm):
    """Autograd through rotary and attention, against the two run by hand: the gradient of a rotation is the rotation by the negative
    positions, bit for bit; q, k and v are views of one packed projection."""
    torch.manual_seed(1)
    rot = mm.Rotary([16, 16])
    pos = mm.grid_positions(10, 7, device="cuda")
    qkv = torch.randn(2, 70, 3, H, D, device="cuda").to(torch.bfloat16)
    g = torch.randn(2, 70, H, D, device="cuda").to(torch.bfloat16)
    q, k, v = (t.detach().requires_grad_() for t in qkv.unbind(2))
    o = mm.attention.attention(*rot(q, k, pos), v, causal=True)
    dq, dk, dv = torch.autograd.grad(o, [q, k, v], g)
    yq, yk = (t.requires_grad_() for t in rot(q.detach(), k.detach(), pos))
    w = v.detach().requires_grad_()
    eq, ek, ev = torch.autograd.grad(mm.attention.attention(yq, yk, w, causal=True), [yq, yk, w], g)
    eq, ek = rot(eq, ek, -pos)
    assert torch.equal(dv, ev) and torch.equal(dq, eq) and torch.equal(dk, ek)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_new_tokens_over_a_kept_prefix(mm, dtype):
    """A stream served token by token - rotated in place at its own position, attended over what is kept - gives the rows of one causal
    call over the whole, within the two forms' roundings of p and o: half a step of o and of p each."""
    torch.manual_seed(2)
    N, K = 300, 2
    rot = mm.Rotary([32], ladder="shared")
    q, k, v = torch.randn(1, N, H, D, device="cuda").to(dtype), torch.randn(1, N, K, D, device="cuda").to(dtype), torch.randn(1, N, K, D, device="cuda").to(dtype)
    fn = mm.attention.attention
    pos = mm.grid_positions(N, device="cuda")
    wq, wk = rot(q, k, pos)
    whole = fn(wq, wk, v, causal=True)
    size = fn(wq, wk, v.abs(), causal=True).double()
    keys, values = torch.full((1, 512, K, D), math.nan, device="cuda", dtype=dtype), torch.full((1, 512, K, D), math.nan, device="cuda", dtype=dtype)
    at = 0
    for n in [1, 5, 64, 100, 1, 1, 63, 1, 64]:
        s = slice(at, at + n)
        qn, kn = rot(q[:, s].clone(), k[:, s].clone(), pos[:, s], inplace=True)
        keys[:, s], values[:, s] = kn, v[:, s]
        at += n
        o = fn(qn, keys, values, causal=True, kv_lengths=torch.tensor([at], dtype=torch.int32, device="cuda"))
        eps = torch.finfo(dtype).eps
        assert ((o.double() - whole[:, s].double()).abs() <= eps * whole[:, s].double().abs() + 1.1 * eps * size[:, s] + 1e-6).all()
    assert at == N
