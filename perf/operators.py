"""Workloads of the token operators: rotary positions, attention, gradient norm and clipping.

A case is a dict of plain values (several numbers stand in one text).  `prepare` makes its inputs on the GPU from a seed, `run` makes one pass over them, either in
plain torch operations or (`own`) through this package, `exact` states the result in float64."""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _text(numbers):
    return ",".join(str(n) for n in numbers)


def _ints(text):
    return [int(n) for n in text.split(",")]


def listed():
    return [
        # one new token of each of 8 streams: the smallest call there is, latency counts
        dict(name="rotary_token", op="rotary", dtype="f16", batch=8, grid=_text([1, 1]), heads=12, kv_heads=12, dim=64, sections=_text([16, 16]), ladder="axis",
             pairing="halves", packed=True, train=False, far=3000, shared=False),
        # 64 spectrograms of 384 x 128 cut into 24 x 8 patches, queries and keys read out of the packed projection
        dict(name="rotary_clips", op="rotary", dtype="f16", batch=64, grid=_text([24, 8]), heads=12, kv_heads=12, dim=64, sections=_text([16, 16]), ladder="axis",
             pairing="halves", packed=True, train=False, far=0, shared=True),
        # two videos of 16 x 28 x 28 tokens with grouped heads, forward and backward of a training step
        dict(name="rotary_video_train", op="rotary", dtype="bf16", batch=2, grid=_text([16, 28, 28]), heads=16, kv_heads=4, dim=128, sections=_text([16, 24, 24]),
             ladder="shared", pairing="halves", packed=False, train=True, far=100000, shared=False),
        # one clip of 256 x 256 (16 x 16 patches and a class token) through a 6-head encoder layer: latency
        dict(name="attention_one_clip", op="attention", dtype="f16", lens="257", kv="257", padded=True, room=0, heads=6, kv_heads=6, dim=64, causal=False,
             prefix=False, bias=False, cap=0.0, train=False),
        # a training batch of 64 clips, 192 patches and a class token each, some cut short
        dict(name="attention_clips_train", op="attention", dtype="f16", lens=_text([193] * 48 + [181, 97, 49, 193, 145, 25, 120, 169] * 2), kv="", padded=True,
             room=0, heads=12, kv_heads=12, dim=64, causal=False, prefix=False, bias=False, cap=0.0, train=True),
        # recordings of very different lengths packed one behind the other, capped scores, training
        dict(name="attention_packed_train", op="attention", dtype="bf16", lens="1,2047,333,64,1500,4096,7,900,2500,65,129,3001,1000,17,1,700",
             kv="", padded=False, room=0, heads=12, kv_heads=4, dim=64, causal=True, prefix=False, bias=False, cap=30.0, train=True),
        # a long recording behind a prefix of tokens that everything sees, scores falling with distance, grouped heads
        dict(name="attention_prefix_long", op="attention", dtype="bf16", lens="8192", kv="8192", padded=True, room=0, heads=16, kv_heads=4, dim=128,
             causal=True, prefix=True, bias=True, cap=0.0, train=False),
        # one new token of each of 16 streams over what they have kept, up to 30001 tokens of it
        dict(name="attention_one_token", op="attention", dtype="bf16", lens=_text([1] * 16), kv=_text([30001, 20000, 16384, 12345, 8192, 4097, 2048, 1000] * 2), padded=True,
             room=32768, heads=16, kv_heads=4, dim=128, causal=True, prefix=False, bias=False, cap=0.0, train=False),
        # the same for one stream with little kept: latency
        dict(name="attention_one_token_short", op="attention", dtype="f16", lens="1", kv="500", padded=True, room=512, heads=12, kv_heads=12, dim=64,
             causal=True, prefix=False, bias=True, cap=0.0, train=False),
        # the two gradients of one patch embedding layer: latency
        dict(name="clip_layer", op="clip", depth=0, width=768, dtype="f32", mixed=False, into=False, norm="2"),
        # 12 encoder blocks and the embedding, a step whose norm stays below the limit (most steps)
        dict(name="clip_encoder", op="clip", depth=12, width=384, dtype="f32", mixed=False, into=False, norm="2"),
        # a large encoder with 16-bit gradients, clipped into the float32 ones that the optimizer takes
        dict(name="clip_large_into_f32", op="clip", depth=32, width=1280, dtype="bf16", mixed=True, into=True, norm="2"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "attention", "attention", "attention", "clip", "clip"])
    dtype = rng.choice(["f16", "bf16"])
    if op == "rotary":
        axes = rng.choice([1, 2, 3])
        dim = rng.choice([32, 64, 80, 128])
        left, sections = dim // 2, []
        for a in range(axes):
            s = rng.randint(1, max(1, left // (axes - a)))
            sections.append(s)
            left -= s
        kv = rng.choice([1, 2, 4, 6])
        heads = kv * rng.choice([1, 2, 4])
        batch = _log_int(rng, 1, 32)
        tokens = min(_log_int(rng, 1, 20000), 60_000_000 // (batch * (heads + kv) * dim) + 1)
        side = max(1, int(tokens ** (1 / axes)))
        grid = [side] * (axes - 1) + [max(1, tokens // side ** (axes - 1))]
        return dict(op=op, dtype=rng.choice(["f16", "bf16", "f32"]), batch=batch, grid=_text(grid), heads=heads, kv_heads=kv, dim=dim, sections=_text(sections),
                    ladder=rng.choice(["axis", "shared"]), pairing=rng.choice(["halves", "adjacent"]), packed=rng.random() < 0.5,
                    train=rng.random() < 0.5, far=_log_int(rng, 1, 500000), shared=rng.random() < 0.5)
    if op == "attention":
        kv = rng.choice([1, 2, 4, 6])
        heads = kv * rng.choice([1, 2, 3, 4])
        dim = rng.choice([32, 64, 72, 128])
        causal = rng.random() < 0.5
        base = dict(op=op, dtype=dtype, heads=heads, kv_heads=kv, dim=dim, causal=causal, prefix=causal and rng.random() < 0.4, bias=rng.random() < 0.4,
                    cap=rng.choice([0.0, 0.0, 20.0]))
        kind = rng.choice(["token", "chunk", "self", "self", "packed", "packed"])
        if kind in ("token", "chunk"):
            n = _log_int(rng, 1, 16)
            room = _log_int(rng, 40, 30000)
            q = 1 if kind == "token" else rng.randint(2, 33)
            return dict(base, lens=_text([q] * n), kv=_text([rng.randint(q, room) for _ in range(n)]), padded=True, room=room, train=False)
        if kind == "self":
            n = _log_int(rng, 1, 64)
            top = min(_log_int(rng, 1, 4000), max(1, int(math.sqrt(1.6e8 / (n * heads)))))
            return dict(base, lens=_text([top if rng.random() < 0.6 else rng.randint(0, top) for _ in range(n)]), kv="", padded=True, room=top, train=rng.random() < 0.5)
        n = rng.randint(1, 24)
        return dict(base, lens=_text([min(_log_int(rng, 1, 4000), int(math.sqrt(1.6e8 / (n * heads)))) for _ in range(n)]), kv="", padded=False, room=rng.choice([0, 0, 11]),
                    train=rng.random() < 0.5)
    width = rng.choice([96, 192, 200, 384, 640])
    return dict(op="clip", depth=_log_int(rng, 1, 24), width=width, dtype=rng.choice(["f16", "bf16", "f32"]), mixed=rng.random() < 0.3,
                into=rng.random() < 0.5, norm=rng.choice(["2", "2", "inf"]), shift=rng.randint(0, 5))


# ---- inputs --------------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _clip_shapes(case):
    """Gradients of a patch embedding and `depth` encoder blocks: matrices, and biases and norm weights between them."""
    w, shift = case["width"], case.get("shift", 0)
    shapes = [(w, 256), (w,)]
    for _ in range(case["depth"]):
        shapes += [(w,), (w,), (3 * w, w), (3 * w + shift,), (w, w), (w,), (w,), (w,), (4 * w + shift, w), (4 * w,), (w, 4 * w), (w,)]
    if case["depth"]:
        shapes += [(w,), (w,), (309, w), (309,)]
    return shapes


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "rotary":
        t = TYPES[case["dtype"]]
        B, N, H, K, D = case["batch"], math.prod(_ints(case["grid"])), case["heads"], case["kv_heads"], case["dim"]
        if case["packed"]:              # queries and keys are views of the projection's output
            qkv = torch.randn(B, N, H + 2 * K, D, generator=g, device="cuda").to(t)
            q, k = qkv[:, :, :H], qkv[:, :, H:H + K]
        else:
            q = torch.randn(B, N, H, D, generator=g, device="cuda").to(t)
            k = torch.randn(B, N, K, D, generator=g, device="cuda").to(t)
        axes = torch.meshgrid(*[torch.arange(n, device="cuda") for n in _ints(case["grid"])], indexing="ij")
        pos = torch.stack([a.reshape(-1) for a in axes])
        if not case["shared"]:          # every row of the batch starts somewhere else on the first axis
            start = torch.randint(0, case["far"] + 1, (B,), generator=g, device="cuda")
            pos = pos[:, None, :].repeat(1, B, 1)
            pos[0] += start[:, None]
        s = dict(case=case, q=q, k=k, pos=pos.to(torch.int32))
        if case["train"]:
            s["q"], s["k"] = q.detach().requires_grad_(), k.detach().requires_grad_()
            s["gq"] = torch.randn(B, N, H, D, generator=g, device="cuda").to(t)
            s["gk"] = torch.randn(B, N, K, D, generator=g, device="cuda").to(t)
        if own:
            from multi_modal_amd.rotary import Rotary
            s["rotary"] = Rotary(_ints(case["sections"]), ladder=case["ladder"], pairing=case["pairing"])
        return s
    if case["op"] == "attention":
        t = TYPES[case["dtype"]]
        H, K, D, lens = case["heads"], case["kv_heads"], case["dim"], _ints(case["lens"])
        kv = _ints(case["kv"]) if case["kv"] else lens
        n = len(lens)
        if case["padded"]:
            rows = max(1, max(lens), 0 if case["kv"] else case["room"])
            keys = max(1, max(kv), case["room"])
            lead_q, lead_k = (n, rows), (n, keys)
        else:
            lead_q = lead_k = (sum(lens) + case["room"],)
        q = torch.randn(*lead_q, H, D, generator=g, device="cuda").to(t)
        k = torch.randn(*lead_k, K, D, generator=g, device="cuda").to(t)
        v = torch.randn(*lead_k, K, D, generator=g, device="cuda").to(t)
        s = dict(case=case, q=q, k=k, v=v, lens=lens, kv=kv)
        s["opts"] = o = dict(causal=case["causal"], cap=case["cap"])
        if case["padded"]:
            o["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
            o["kv_lengths"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
        else:
            o["offsets"] = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
        if case["prefix"]:
            s["prefix"] = [(x * 7) // 32 for x in kv]
            o["prefix"] = torch.tensor(s["prefix"], dtype=torch.int32, device="cuda")
        if case["bias"]:
            o["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device="cuda")
        if case["train"]:
            for name in "qkv":
                s[name] = s[name].requires_grad_()
            s["go"] = torch.randn(q.shape, generator=g, device="cuda").to(t)
        return s
    # The gradients are views of one buffer for each type, behind one another as the parameters come (what a data-parallel step reduces)
    where, flat = [], {}
    for i, shape in enumerate(_clip_shapes(case)):
        t = torch.float32 if case["mixed"] and len(shape) == 1 else TYPES[case["dtype"]]
        where.append((t, flat.get(t, 0), shape, 1e-3 * (1 + i % 7)))
        flat[t] = flat.get(t, 0) + math.prod(shape)

    def views(buffers):
        return [buffers[t][at:at + math.prod(shape)].view(shape) for t, at, shape, _ in where]

    buffers = {t: torch.randn(n, generator=g, device="cuda").to(t) for t, n in flat.items()}
    grads = views(buffers)
    for x, (_, _, _, size) in zip(grads, where):
        x.mul_(size)
    limit = (0.01 if case["into"] else 10.0) * 5e-3 * math.sqrt(sum(flat.values()))
    s = dict(case=case, grads=grads, limit=limit, kind=float(case["norm"]), results=list(buffers.values()))
    if case["into"]:
        buffers = {t: torch.empty(n, device="cuda") for t, n in flat.items()}
        s["into"], s["results"] = views(buffers), list(buffers.values())
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------------

def _frequencies(case, xp):
    """theta of every pair, and the axis it turns with."""
    sections, theta, axis = _ints(case["sections"]), [], []
    R, at = sum(sections), 0
    for a, n in enumerate(sections):
        for j in range(n):
            theta.append(10000.0 ** (-(j / n) if case["ladder"] == "axis" else -((at + j) / R)))
            axis.append(a)
        at += n
    return xp.tensor(theta, dtype=torch.float64, device="cuda"), xp.tensor(axis, device="cuda")


def _rotate_plain(case, x, pos):
    theta, axis = _frequencies(case, torch)
    R = theta.numel()
    angle = pos.double()[axis] * theta.view(-1, *[1] * (pos.dim() - 1))         # (R, [B,] N): far positions need 64 bits
    cos, sin = angle.cos().float(), angle.sin().float()
    cos, sin = (c.movedim(0, -1).unsqueeze(-2) for c in (cos, sin))             # ([B,] N, 1, R)
    f = x.float()
    if case["pairing"] == "halves":
        a, b, rest = f[..., :R], f[..., R:2 * R], f[..., 2 * R:]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    else:
        a, b, rest = f[..., 0:2 * R:2], f[..., 1:2 * R:2], f[..., 2 * R:]
        y = torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)
    return y.to(x.dtype)


def _visible(case, nq, nk, prefix):
    i = torch.arange(nq, device="cuda")[:, None] + (nk - nq)
    j = torch.arange(nk, device="cuda")[None, :]
    see = torch.ones(nq, nk, dtype=torch.bool, device="cuda")
    if case["causal"]:
        see = j <= i
        if prefix is not None:
            see = see | (j < prefix)
    return see, (i - j).abs()


def _attend_plain(case, q, k, v, slopes, prefix):
    """One document: q (n, H, D), k and v (m, K, D) in float32 -> (n, H, D) in float32."""
    nq, H, D = q.shape
    nk, K, _ = k.shape
    if nq == 0:
        return q
    if nk == 0:
        return torch.zeros_like(q)
    qh = q.view(nq, K, H // K, D).permute(1, 2, 0, 3).reshape(K, H // K * nq, D)
    s = torch.matmul(qh, k.permute(1, 2, 0).contiguous()).view(H, nq, nk) * (1.0 / math.sqrt(D))
    if case["cap"]:
        s = torch.tanh(s / case["cap"]) * case["cap"]
    see, far = _visible(case, nq, nk, prefix)
    if slopes is not None:
        s = s - slopes[:, None, None] * far
    s = torch.where(see, s, torch.full((), -math.inf, device="cuda"))
    top = s.detach().amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total > 0, total, torch.ones_like(total))
    o = torch.matmul(p.view(K, H // K * nq, nk), v.permute(1, 0, 2).contiguous())
    return o.view(K, H // K, nq, D).permute(2, 0, 1, 3).reshape(nq, H, D)


def _attention_plain(s):
    case, lens, kv, o = s["case"], s["lens"], s["kv"], s["opts"]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    prefixes = s.get("prefix", [None] * len(lens))
    if case["padded"] and len(set(lens)) == len(set(kv)) == 1 and len(lens) == 1:
        return _attend_plain(case, q[0, :lens[0]], k[0, :kv[0]], v[0, :kv[0]], o.get("slopes"), prefixes[0])[None].to(s["q"].dtype)
    out, at = [], 0
    for d, (nq, nk) in enumerate(zip(lens, kv)):
        if case["padded"]:
            y = _attend_plain(case, q[d, :nq], k[d, :nk], v[d, :nk], o.get("slopes"), prefixes[d])
            out.append(torch.cat([y, y.new_zeros(q.shape[1] - nq, *y.shape[1:])]))
        else:
            out.append(_attend_plain(case, q[at:at + nq], k[at:at + nk], v[at:at + nk], o.get("slopes"), prefixes[d]))
            at += nq
    if case["padded"]:
        return torch.stack(out).to(s["q"].dtype)
    out.append(q.new_zeros(q.shape[0] - at, *q.shape[1:]))
    return torch.cat(out).to(s["q"].dtype)


def _clip_plain(s):
    if s["kind"] == math.inf:
        norm = torch.stack([x.float().abs().max().double() for x in s["grads"]]).max()
    else:
        norm = torch.stack([x.double().square().sum() for x in s["grads"]]).sum().sqrt()        # long sums
    norm = norm.float()
    factor = (s["limit"] / (norm + 1e-6)).clamp(max=1.0)
    for i, x in enumerate(s["grads"]):
        if "into" in s:
            s["into"][i].copy_(x.float() * factor)
        else:
            x.copy_(x.float() * factor)
    return norm


# ---- one pass ----------------------------------------------------------------------------------------------------------

def run(state):
    s, case = state, state["case"]
    if case["op"] == "rotary":
        if own:
            yq, yk = s["rotary"](s["q"], s["k"], s["pos"])
        else:
            yq, yk = _rotate_plain(case, s["q"], s["pos"]), _rotate_plain(case, s["k"], s["pos"])
        if not case["train"]:
            return {"q": yq, "k": yk}
        gq, gk = torch.autograd.grad([yq, yk], [s["q"], s["k"]], [s["gq"], s["gk"]])
        return {"q": yq.detach(), "k": yk.detach(), "grad_q": gq, "grad_k": gk}
    if case["op"] == "attention":
        if own:
            from multi_modal_amd.attention import attention
            out = attention(s["q"], s["k"], s["v"], **s["opts"])
        else:
            out = _attention_plain(s)
        if not case["train"]:
            return {"out": out}
        gq, gk, gv = torch.autograd.grad(out, [s["q"], s["k"], s["v"]], s["go"])
        return {"out": out.detach(), "grad_q": gq, "grad_k": gk, "grad_v": gv}
    if own:
        from multi_modal_amd.gradients import clip_grad_norm
        norm = clip_grad_norm(s["grads"], s["limit"], norm_type=s["kind"], out=s.get("into"))
    else:
        norm = _clip_plain(s)
    return {"norm": norm, "grads": s["results"]}


# ---- cost --------------------------------------------------------------------------------------------------------------

def _size(dtype):
    return 4 if dtype == "f32" else 2


def work(case):
    if case["op"] == "rotary":
        tokens, heads = case["batch"] * math.prod(_ints(case["grid"])), case["heads"] + case["kv_heads"]
        times = 2 if case["train"] else 1
        at = len(_ints(case["sections"])) * (tokens if not case["shared"] else math.prod(_ints(case["grid"]))) * 4
        return {"bytes": times * (2 * tokens * heads * case["dim"] * _size(case["dtype"]) + at), "flops": times * 6 * tokens * heads * sum(_ints(case["sections"]))}
    if case["op"] == "attention":
        lens = _ints(case["lens"])
        kv = _ints(case["kv"]) if case["kv"] else lens
        pairs = 0
        for nq, nk in zip(lens, kv):
            if not case["causal"]:
                pairs += nq * nk
                continue
            first, p = nk - nq + 1, (nk * 7) // 32 if case["prefix"] else 0     # row i sees max(first + i, p) keys, 0 to nk of them
            seen = np.clip(np.maximum(np.arange(nq, dtype=np.int64) + first, p), 0, nk)
            pairs += int(seen.sum())
        D, H, K = case["dim"], case["heads"], case["kv_heads"]
        tq, tk = sum(lens) * H * D * 2, 2 * sum(kv) * K * D * 2
        if case["train"]:           # forward: q k v in, o out; backward: q k v o do in, dq dk dv out
            return {"bytes": (2 * tq + tk) + (4 * tq + 2 * tk), "flops": 14 * D * pairs * H}
        return {"bytes": 2 * tq + tk, "flops": 4 * D * pairs * H}
    bytes_, flops = 0, 0
    for shape in _clip_shapes(case):
        n = math.prod(shape)
        e = 4 if case["mixed"] and len(shape) == 1 else _size(case["dtype"])
        bytes_ += n * (e + 4 if case["into"] else e)           # below the limit nothing has to be written
        flops += n * (3 if case["into"] else 2)
    return {"bytes": bytes_, "flops": flops}


# ---- the definition, in 64 bits ------------------------------------------------------------------------------------------

def _exact_rotary(case, x, pos, sign):
    """As complex numbers: (a + ib) e^(i phi)."""
    x = x.detach().double()
    sections = _ints(case["sections"])
    R = sum(sections)
    pos = pos.double() if pos.dim() == 3 else pos.double()[:, None, :]
    out = x.clone()
    done = 0
    for a, n in enumerate(sections):
        for j in range(n):
            i = done + j
            exponent = j / n if case["ladder"] == "axis" else i / R
            phi = sign * pos[a] / 10000.0 ** exponent
            turn = torch.polar(torch.ones_like(phi), phi)[..., None]
            u, w = (i, i + R) if case["pairing"] == "halves" else (2 * i, 2 * i + 1)
            z = torch.complex(x[..., u], x[..., w]) * turn
            out[..., u], out[..., w] = z.real, z.imag
        done += n
    return out


def _exact_head(case, q, k, v, slope, prefix, go):
    """One head of one document in float64: output and, where go is given, the three gradients from their formulas."""
    nq, nk, D = q.shape[0], k.shape[0], q.shape[1]
    raw = (q @ k.t()) / D ** 0.5
    t = torch.tanh(raw / case["cap"]) if case["cap"] else None
    s = case["cap"] * t if case["cap"] else raw
    rows = torch.arange(nq, device=q.device).view(-1, 1) + nk - nq
    cols = torch.arange(nk, device=q.device).view(1, -1)
    if slope:
        s = s - slope * (rows - cols).abs().double()
    if case["causal"]:
        hidden = (cols > rows) & (cols >= (0 if prefix is None else prefix))
        s = s.masked_fill(hidden, float("-inf"))
    lse = torch.logsumexp(s, 1, keepdim=True)
    p = torch.where(torch.isinf(lse), torch.zeros_like(s), torch.exp(s - lse))
    o = p @ v
    if go is None:
        return o, None, None, None
    dp = go @ v.t()
    ds = p * (dp - (p * dp).sum(1, keepdim=True))
    if case["cap"]:
        ds = ds * (1 - t * t)
    ds = ds / D ** 0.5
    return o, ds @ k, ds.t() @ q, p.t() @ go


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    if case["op"] == "rotary":
        r = {"q": _exact_rotary(case, s["q"], s["pos"], 1), "k": _exact_rotary(case, s["k"], s["pos"], 1)}
        if case["train"]:
            r["grad_q"], r["grad_k"] = _exact_rotary(case, s["gq"], s["pos"], -1), _exact_rotary(case, s["gk"], s["pos"], -1)
        return r
    if case["op"] == "attention":
        H, K, lens, kv = case["heads"], case["kv_heads"], s["lens"], s["kv"]
        q, k, v = (s[n].detach().double() for n in "qkv")
        go = s["go"].double() if case["train"] else None
        r = {"out": torch.zeros_like(q)}
        if case["train"]:
            r.update(grad_q=torch.zeros_like(q), grad_k=torch.zeros_like(k), grad_v=torch.zeros_like(v))
        at = 0
        for d, (nq, nk) in enumerate(zip(lens, kv)):
            iq, ik = ((d, slice(0, nq)), (d, slice(0, nk))) if case["padded"] else ((slice(at, at + nq),), (slice(at, at + nk),))
            at += nq
            if nq == 0 or nk == 0:
                continue
            for h in range(H):
                c = h // (H // K)
                slope = 2.0 ** (-8.0 * (h + 1) / H) if case["bias"] else 0.0
                if case["bias"]:
                    slope = float(np.float32(slope))
                prefix = s["prefix"][d] if case["prefix"] else None
                o, dq, dk, dv = _exact_head(case, q[iq][:, h], k[ik][:, c], v[ik][:, c], slope, prefix, go[iq][:, h] if case["train"] else None)
                r["out"][iq + (h,) if case["padded"] else (iq[0], h)] = o
                if case["train"]:
                    r["grad_q"][iq + (h,) if case["padded"] else (iq[0], h)] = dq
                    r["grad_k"][ik + (c,) if case["padded"] else (ik[0], c)] += dk
                    r["grad_v"][ik + (c,) if case["padded"] else (ik[0], c)] += dv
        return r
    if case["norm"] == "inf":
        norm = max(float(x.abs().max()) for x in s["grads"])
    else:
        norm = math.sqrt(sum(float((x.double() ** 2).sum()) for x in s["grads"]))
    factor = min(1.0, s["limit"] / (norm + 1e-6))
    types = dict.fromkeys(x.dtype for x in s["grads"])
    return {"norm": torch.tensor(norm, dtype=torch.float64),
            "grads": [torch.cat([x.double().reshape(-1) for x in s["grads"] if x.dtype == t]) * factor for t in types]}
