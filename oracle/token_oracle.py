"""Restatement of the token operators in float64, one document and one head at a time (test infrastructure)."""
import math

import torch


def attention_head(q, k, v, scale, cap=0.0, slope=0.0, causal=False, prefix=0, g=None, relative=False):
    """One head of one document: q (n, D), k and v (m, D), all float64.  Returns a dict with o, lse, and with g the gradients dq, dk, dv
    by their formulas; next to each result what its tolerance is made of (see attention_tolerances).

    relative: a capped score's error is bounded by the score and not by the cap.  With z = s / cap and steps of u = 2^-24: up to |z| = 1/2 the series in z^2 and its
    products are off by at most 1 step for z, 2 for the square (which count z^2 / 3 times at most), 1 for each of 3 products; beyond, 1 - 2 / (e^(2 z) + 1) has the
    exponential's 2 steps and its argument's 2 |z|, taken by r (1 - r) <= 1/4, the reciprocal's 2 and the sum's 1, taken by r <= 1, twice, and 1 of the result:
    2 (1/4 (2 + 2 |z|) + 3) + 1, where |z| r (1 - r) <= 0.23, is at most 9 steps of cap, and |s| >= 0.46 cap: 20 steps of |s| hold both."""
    n, m = q.shape[0], k.shape[0]
    raw = scale * (q @ k.T)
    t = torch.tanh(raw / cap) if cap else None
    s = cap * t if cap else raw
    i = torch.arange(n, device=q.device)[:, None] + (m - n)
    j = torch.arange(m, device=q.device)[None, :]
    if slope:
        s = s - slope * (i - j).abs()
    see = torch.ones(n, m, dtype=torch.bool, device=q.device)
    if causal:
        see = (j <= i) | (j < prefix)
    s = torch.where(see, s, torch.full_like(s, -math.inf))
    top = s.amax(1, keepdim=True) if m else s.new_zeros(n, 1)
    e = torch.where(see, torch.exp(s - top), torch.zeros_like(s))
    total = e.sum(1, keepdim=True)
    p = torch.where(total > 0, e / total, torch.zeros_like(e))
    r = {"o": p @ v, "lse": torch.where(total > 0, top + total.log(), torch.full_like(total, -math.inf))[:, 0]}
    # rounding errors of a score in float32: the products' sum, the multiplications behind it, tanh, the distance
    D = q.shape[1]
    u = 2.0 ** -24
    capped = (cap * t).abs() if cap else 0.0
    es = u * ((D + 4) * scale * (q.abs() @ k.T.abs()) + 4 * torch.where(see, s.abs(), torch.zeros_like(s)) + (20 * capped if relative else 16 * cap))
    es = torch.where(see, es, torch.zeros_like(es))
    es = es + (es.amax(1, keepdim=True) if m else 0.0)              # of the score, and of the row's normaliser
    r["p"], r["es"], r["see"] = p, es, see
    r["A"] = (p * 1.0) @ v.abs()
    r["Ae"] = (p * es) @ v.abs()
    r["sv"] = see.double() @ v.abs()
    if g is not None:
        dp = g @ v.T
        delta = (g * r["o"]).sum(1, keepdim=True)
        f = (1 - t * t) if cap else torch.ones_like(s)
        ds = p * (dp - delta) * f
        r.update(dv=p.T @ g, dq=scale * (ds @ k), dk=scale * (ds.T @ q), ds=ds, f=f, delta=delta, gv=g.abs() @ v.abs().T)
    return r


def attention_tolerances(r, q, k, v, g, scale, eps, tiny):
    """Bounds on |kernel - exact| of o (and dq, dk, dv).  u = eps / 2 is half a step of the 16-bit type, `tiny` half its smallest
    subnormal.  p is rounded to 16 bits (u relative, or tiny against a largest value of at least 1; with the kernels' scaling of
    float16 gradients the subnormals are 2^-8 of that and left in); p itself carries its score's float32 error es; results are
    rounded once.  delta is formed from the rounded o.
    bfloat16 has float32's exponents, so its subnormals are those of the arithmetic itself, which the exponential and the matrix
    instructions take as zeros: p, ds and results below 2^-126 may be lost whole.  A lost p is an error of at most 2^-126 in o's and dv's
    terms and of 2^-126 |dp - delta| <= 2^-126 (|g||v| + |delta|) in ds, a lost ds one of 2^-126."""
    u, u32, lost = eps / 2, 2.0 ** -24, 2.0 ** -126
    tiny = max(tiny, lost)
    ep = 1.02 * u + 64 * u32                                        # relative error of a rounded p, without its score's
    tol = {"o": u * r["o"].abs() * 1.01 + ep * r["A"] + 1.1 * r["Ae"] + tiny * (r["sv"] + 1)}
    if g is None:
        return tol
    p, es = r["p"], r["es"]
    D = q.shape[1]
    tol["dv"] = 1.01 * u * r["dv"].abs() + (p * (ep + 1.1 * es)).T @ g.abs() + tiny * (r["see"].double().T @ g.abs() + 1)
    edelta = (g.abs() * tol["o"]).sum(1, keepdim=True) + (D + 2) * u32 * (g.abs() * r["o"].abs()).sum(1, keepdim=True)
    edp = (D + 2) * u32 * r["gv"]
    eds = r["ds"].abs() * (ep + 1.1 * es) + p * r["f"] * (edelta + edp) + p * (r["gv"] + r["delta"].abs()) * 16 * u32
    # subnormal ds of float16: relative to the largest possible |g||v| of the document, 2^-29 of it is still a normal number
    eds = eds + r["see"].double() * (tiny * 2.0 ** -3 * float(g.norm(dim=1).max() if g.numel() else 0) * float(v.norm(dim=1).max() if v.numel() else 0))
    eds = eds + r["see"].double() * lost * (1 + r["gv"] + r["delta"].abs())
    tol["dq"] = 1.01 * u * r["dq"].abs() + scale * (eds @ k.abs()) + tiny
    tol["dk"] = 1.01 * u * r["dk"].abs() + scale * (eds.T @ q.abs()) + tiny
    return tol


def attention(q, k, v, docs, scale=None, cap=0.0, slopes=None, causal=False, prefix=None, g=None, eps=0.0, tiny=0.0, relative=False):
    """q (T, H, D), k and v (S, K, D); docs: (first row, rows, first key, keys) of each document.  Returns ({o, lse, dq, dk, dv}, the same of
    tolerances), zeros (lse -inf) in rows that no document holds."""
    T, H, D = q.shape
    K = k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    z = {"o": torch.zeros(T, H, D, dtype=torch.float64, device=q.device), "lse": torch.full((H, T), -math.inf, dtype=torch.float64, device=q.device)}
    if g is not None:
        z.update(dq=torch.zeros_like(z["o"]), dk=torch.zeros(k.shape, dtype=torch.float64, device=q.device), dv=torch.zeros(k.shape, dtype=torch.float64, device=q.device))
    w = {n: torch.zeros_like(t) for n, t in z.items()}
    w["lse"] = torch.zeros_like(z["lse"])
    for d, (q0, n, k0, m) in enumerate(docs):
        if n == 0 or m == 0:
            continue
        for h in range(H):
            c = h // (H // K)
            a = (q[q0:q0 + n, h].double(), k[k0:k0 + m, c].double(), v[k0:k0 + m, c].double())
            gg = None if g is None else g[q0:q0 + n, h].double()
            r = attention_head(*a, scale, cap, 0.0 if slopes is None else float(slopes[h]), causal, 0 if prefix is None else int(prefix[d]), gg, relative)
            t = attention_tolerances(r, *a, gg, scale, eps, tiny)
            z["o"][q0:q0 + n, h], w["o"][q0:q0 + n, h] = r["o"], t["o"]
            z["lse"][h, q0:q0 + n] = r["lse"]
            w["lse"][h, q0:q0 + n] = 1.1 * r["es"].amax(1) + 2.0 ** -22 * (torch.nan_to_num(r["lse"], neginf=0.0).abs() + 4)
            if g is not None:
                z["dq"][q0:q0 + n, h], w["dq"][q0:q0 + n, h] = r["dq"], t["dq"]
                for name in ("dk", "dv"):
                    z[name][k0:k0 + m, c] += r[name]
                    w[name][k0:k0 + m, c] += t[name]
    return z, w
