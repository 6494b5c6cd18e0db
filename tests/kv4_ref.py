"""Plain 64-bit forms of the 4-bit key/value cache's operators (torch on the CPU), written from their definitions."""
import math

import torch

GRID = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
MIN_EXP, MAX_EXP = -120, 125


def stored(x):
    """What the cache holds of rows [n][heads][dim]: [heads][n][dim], float64."""
    x = x.to("cpu", torch.float64).permute(1, 0, 2)
    b = x.reshape(*x.shape[:2], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    fin = torch.isfinite(top)
    m, e = torch.frexp(torch.where(fin, top, torch.ones_like(top)))  # 0.5 <= m < 1
    e = e - 3 + (m >= 0.875).to(e.dtype)
    e = torch.where(top == 0, torch.full_like(e, MIN_EXP), e.clamp(MIN_EXP, MAX_EXP))
    a = torch.ldexp(torch.where(fin.expand_as(b), b, torch.zeros_like(b)).abs(), -e)
    dist = (a[..., None] - GRID).abs()
    near = dist.argmin(-1)  # the lower of two equally near; the even code is wanted
    up = (near + 1).clamp(max=7)
    tie = (dist.gather(-1, near[..., None]) == dist.gather(-1, up[..., None]))[..., 0] & (up > near)
    code = torch.where(tie & (near % 2 == 1), up, near)
    v = torch.sign(b).nan_to_num() * GRID[code] * torch.ldexp(torch.ones_like(top), e)
    v = torch.where(fin.expand_as(b), v, torch.full_like(v, math.nan))
    return v.reshape(x.shape)


def attend(q, k, v, scale=None):
    """(out [n][heads][dim], weights [kv heads][len], bound) of queries q [n][heads][dim] over values k, v [kv heads][len][dim]
    in float64.  bound: how far an f32 evaluation of out may be off, sums in any order: a score of D products is off by at
    most (D + 4) 2^-24 of its terms' sizes, which exp turns into a relative error, the exponential, the products and the
    sums of up to len terms add (len + 16) 2^-24, the division and the maximum's cancellation are within the 16.  wbound: the same for the weights."""
    n, nq, d = q.shape
    nkv, length = k.shape[:2]
    grp = nq // nkv
    q = q.to("cpu", torch.float64)
    scale = 1 / math.sqrt(d) if scale is None else scale
    out = torch.empty(n, nq, d, dtype=torch.float64)
    bound = torch.empty_like(out)
    w = torch.zeros(nkv, length, dtype=torch.float64)
    wb = torch.zeros_like(w)
    seen = torch.arange(length)[None] <= torch.arange(length - n, length)[:, None]
    u = 2.0 ** -24
    for h in range(nq):
        g = h // grp
        s = (q[:, h] @ k[g].T) * scale
        es = (q[:, h].abs() @ k[g].abs().T) * abs(scale) * (d + 4) * u
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        p = torch.softmax(s, 1)
        rel = 2 * torch.where(seen, es, torch.zeros_like(es)).amax(1, keepdim=True) + (length + 16) * u
        # a value that is not seen takes no part, be it a NaN
        for i in range(n):
            vis = v[g][:length - n + i + 1]
            out[i, h] = p[i, :length - n + i + 1] @ vis
            bound[i, h] = rel[i] * (p[i, :length - n + i + 1] @ vis.abs())
        w[g] += torch.where(seen, p, torch.zeros_like(p)).sum(0)
        wb[g] += torch.where(seen, p * (rel + 2 * n * grp * u), torch.zeros_like(p)).sum(0)
    return out, w, bound, wb


def evict(w, keep, recent):
    """Indices kept [kv heads][min(keep, len)] of weights w [kv heads][len]."""
    w = w.to("cpu", torch.float64)
    length = w.shape[1]
    m = min(keep, length)
    recent = min(recent, length)
    out = []
    for row in w:
        old = [(-math.inf if math.isnan(x) else x + 0.0, math.isnan(x)) for x in row[:length - recent].tolist()]
        order = sorted(range(len(old)), key=lambda i: (old[i][1], -old[i][0], i))[:m - recent]
        out.append(sorted(order) + list(range(length - recent, length)))
    return torch.tensor(out, dtype=torch.int32).reshape(w.shape[0], m)


def logprobs(x, tokens, top):
    """(logp, entropy, ids, top_logp, bounds) of logits x [n][vocab] in float64; the bounds of logp and entropy hold for f32 sums
    in any order: sums of vocab positive terms (vocab + 8) 2^-24 relative, the logarithm and the differences 4 2^-24."""
    x = x.to("cpu", torch.float64)
    n, vocab = x.shape
    u = 2.0 ** -24
    m = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x).amax(1, keepdim=True)
    d = x - m
    z = torch.exp(d).sum(1, keepdim=True)
    lse = torch.log(z)
    ok = (tokens >= 0) & (tokens < vocab)
    lp = torch.gather(d, 1, torch.where(ok, tokens, torch.zeros_like(tokens)).long()[:, None])[:, 0] - lse[:, 0]
    lp = torch.where(ok, lp, torch.full_like(lp, math.nan))
    ed = torch.where(d == -math.inf, torch.zeros_like(d), torch.exp(d) * d)
    ent = lse[:, 0] - ed.sum(1) / z[:, 0]
    key = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    ids = torch.empty(n, top, dtype=torch.int32)
    for i in range(n):
        nan = torch.isnan(x[i]).tolist()
        order = sorted(range(vocab), key=lambda j: (nan[j], -key[i, j].item(), j)) if vocab <= 4096 else \
            torch.sort(key[i], descending=True, stable=True).indices.tolist()
        ids[i] = torch.tensor(order[:top], dtype=torch.int32)
    tl = torch.gather(d, 1, ids.long()) - lse
    rel = (vocab + 8) * u
    lb = rel + 4 * u * (lp.abs() + lse[:, 0].abs()).nan_to_num()
    eb = 2 * rel + 2 * rel * (ed.abs().sum(1) / z[:, 0]) + 4 * u * (lse[:, 0].abs() + ent.abs())
    tb = rel + 4 * u * (tl.abs() + lse.abs())
    return lp, ent, ids, tl, lb, eb, tb
