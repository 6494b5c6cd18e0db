"""Workloads of the 4-bit key/value cache and of the log probabilities, in plain torch and through daiza_amd.

A case is a dict of plain values; `op` names the operator:
  append    n rows of keys and values behind `start` cached ones (dz_kv4_append_dev), and the stored values of the new rows
            (dz_kv4_read_dev)
  attend    n queries, the newest n of `len` cached rows theirs (dz_kv4_attend_dev); with `weights` the attention that each
            row received is added to the row's weight
  evict     the `keep` rows of a cache of `len` that stay, the newest `recent` and those of the largest weights among the
            others (dz_kv4_evict_dev), and their stored values
  logprobs  log probabilities of given tokens, entropies and the `top` best alternatives of n rows of logits
            (dz_logprobs_dev)

A cached row holds, per head, blocks of 32 values as 4-bit floats (a sign and 0, 0.5, 1, 1.5, 2, 3, 4 or 6) times a power of
two: the smallest one at which the block's largest value does not round past 6.  Shapes are those of the 27B configuration
(24 heads on 4 of 256, a vocabulary of 248320, contexts up to 262144) and generic ones.
"""
import math

import torch

own = False

KEYS, VALUES = 1.5, 0.5  # sizes of the rows; unit queries then give scores of a spread of about 2
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one decoded token with its alternatives
        dict(name="logprobs_token", op="logprobs", n=1, vocab=248320, top=20, type="f32"),
        # a long prompt's scores from 16-bit logits
        dict(name="logprobs_prompt_1024_bf16", op="logprobs", n=1024, vocab=248320, top=20, type="bf16"),
        # the row that a decoded token adds
        dict(name="append_token", op="append", n=1, start=4096, kv_heads=4, head_dim=256, type="f32"),
        # a long prompt's rows
        dict(name="append_prompt_1024", op="append", n=1024, start=0, kv_heads=4, head_dim=256, type="f32"),
        # a decoded token at an ordinary context
        dict(name="attend_token_4096", op="attend", n=1, len=4096, heads=24, kv_heads=4, head_dim=256, type="f32", weights=False),
        # one at a long context whose rows are evicted by their weights
        dict(name="attend_token_32768_weights", op="attend", n=1, len=32768, heads=24, kv_heads=4, head_dim=256, type="f32",
             weights=True),
        # one at the model's whole context length
        dict(name="attend_token_262144", op="attend", n=1, len=262144, heads=24, kv_heads=4, head_dim=256, type="f32",
             weights=False),
        # the eight drafts of a verify step
        dict(name="attend_verify_8_at_8192", op="attend", n=8, len=8200, heads=24, kv_heads=4, head_dim=256, type="f32",
             weights=False),
        # the next turn of a conversation: a ragged number of tokens behind a long prefix, with weights
        dict(name="attend_333_at_7000_weights", op="attend", n=333, len=7333, heads=24, kv_heads=4, head_dim=256, type="f32",
             weights=True),
        # a prompt into an empty cache in 16 bits, narrower heads
        dict(name="attend_prompt_1024_bf16", op="attend", n=1024, len=1024, heads=32, kv_heads=8, head_dim=128, type="bf16",
             weights=False),
        # a long cache cut to a quarter
        dict(name="evict_32768_to_8192", op="evict", len=32768, keep=8192, recent=256, kv_heads=4, head_dim=256),
        # a short one that has grown past its bound by a few rows
        dict(name="evict_1100_to_1024", op="evict", len=1100, keep=1024, recent=64, kv_heads=4, head_dim=256),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# (query heads, key/value heads, head size)
_HEADS = [(24, 4, 256), (24, 4, 256), (6, 1, 256), (8, 8, 256), (16, 2, 256), (32, 8, 128), (12, 4, 128), (7, 1, 128),
          (16, 4, 64), (10, 2, 64)]


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "evict", "logprobs"])
    heads, kv, hd = rng.choice(_HEADS)
    if op == "logprobs":
        n = _log_int(rng, 1, 1024)
        vocab = _log_int(rng, 1000, 248320)
        return dict(op=op, n=n, vocab=vocab, top=rng.randint(0, 32),
                    type=rng.choice(["f32", "f16", "bf16"] if n <= 512 else ["f16", "bf16"]))
    if op == "append":
        return dict(op=op, n=_log_int(rng, 1, 1024), start=rng.randint(0, 4096), kv_heads=kv, head_dim=hd,
                    type=rng.choice(["f32", "f16", "bf16"]))
    if op == "evict":
        length = _log_int(rng, 64, 32768)
        keep = rng.randint(1, length)
        return dict(op=op, len=length, keep=keep, recent=rng.randint(0, min(keep, 1024)), kv_heads=kv, head_dim=hd)
    n = _log_int(rng, 1, 1024)
    # no more pairs of a query and a row than the largest listed case has
    most = max(n, 333 * 7000 * 24 * 256 // (n * heads * hd))
    length = n + _log_int(rng, 1, min(131072, most)) - 1
    return dict(op=op, n=n, len=length, heads=heads, kv_heads=kv, head_dim=hd, type=rng.choice(["f32", "f32", "f16", "bf16"]),
                weights=rng.random() < 0.4)


# ---------------------------------------------------------------- inputs


def _gen(seed, tag):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + tag * 7919) & 0x7FFFFFFFFFFF)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _rows(case, seed, tag, n, scale):
    """n rows [n][kv heads][head size] whose channels differ in size and mean, as keys' and values' do."""
    g = _gen(seed, tag)
    channel = torch.exp(_normal(g, case["kv_heads"], case["head_dim"]) * 0.5) * scale
    mean = _normal(g, case["kv_heads"], case["head_dim"]) * 0.5
    return ((_normal(g, n, case["kv_heads"], case["head_dim"]) + mean) * channel).to(TYPES[case.get("type", "f32")])


def _queries(case, seed):
    return _normal(_gen(seed, 3), case["n"], case["heads"], case["head_dim"]).to(TYPES[case["type"]])


def _row_weights(case, seed):
    """Weights as attention leaves them: many small ones, few large; some rows alike, some never attended to."""
    g = _gen(seed, 4)
    w = torch.exp(_normal(g, case["kv_heads"], case["len"]) * 2.0)
    w = torch.where(w < 0.3, torch.zeros_like(w), w)
    return torch.where(w > 4.0, torch.round(w), w)


def _logits(case, seed):
    """Logits of a spread that lets some tokens stand out, and the tokens that are asked about, mostly likely ones."""
    g = _gen(seed, 5)
    x = (_normal(g, case["n"], case["vocab"]) * 2.5).to(TYPES[case["type"]])
    tokens = torch.randint(0, case["vocab"], (case["n"],), generator=g, device="cuda", dtype=torch.int64)
    best = x.argmax(1)
    return x, torch.where(torch.rand(case["n"], generator=g, device="cuda") < 0.6, best, tokens).to(torch.int32)


def prepare(case, seed):
    op = case["op"]
    if own:
        import daiza_amd as dz
        if dz.lib().dz_device_init(torch.cuda.current_device()) != 0:
            raise dz.DaizaError(dz.DZ_ERR_DEVICE, dz.lib().dz_last_error().decode())
    if op == "logprobs":
        x, tokens = _logits(case, seed)
        s = dict(case, x=x, tokens=tokens)
        if own:
            n, k = case["n"], case["top"]
            s.update(logp=torch.empty(n, device="cuda"), entropy=torch.empty(n, device="cuda"),
                     top_ids=torch.empty(n, k, dtype=torch.int32, device="cuda"), top_logp=torch.empty(n, k, device="cuda"))
        return s
    hkv, hd = case["kv_heads"], case["head_dim"]
    cached = case["start"] if op == "append" else case["len"]
    k, v = _rows(case, seed, 1, cached, KEYS), _rows(case, seed, 2, cached, VALUES)
    s = dict(case)
    if own:
        cache = dz.Kv4Cache(hkv, hd, cached + case.get("n", 0))
        if cached:
            cache.append_dev(k, v, stream=_stream())
        s["cache"] = cache
    else:
        s["k"], s["v"] = _pack(k), _pack(v)
    if op == "append":
        s["new_k"], s["new_v"] = _rows(case, seed, 6, case["n"], KEYS), _rows(case, seed, 7, case["n"], VALUES)
        if own:
            s["out_k"], s["out_v"] = (torch.empty(hkv, case["n"], hd, device="cuda") for _ in range(2))
    elif op == "attend":
        s["q"] = _queries(case, seed)
        s["w"] = _row_weights(case, seed) if case["weights"] else None
        if own:
            s["out"] = torch.empty_like(s["q"])
    else:
        s["w"] = _row_weights(case, seed)
        if own:
            s["to"] = dz.Kv4Cache(hkv, hd, case["keep"])
            s["to_w"] = torch.empty(hkv, case["keep"], device="cuda")
            s["kept"] = torch.empty(hkv, case["keep"], dtype=torch.int32, device="cuda")
            s["out_k"], s["out_v"] = (torch.empty(hkv, case["keep"], hd, device="cuda") for _ in range(2))
    del k, v
    return s


def _stream():
    return torch.cuda.current_stream().cuda_stream


# ---------------------------------------------------------------- the plain forms


def _pack(x):
    """Rows [n][heads][size] as (codes [heads][n][size / 2], two a byte, and scale bytes [heads][n][size / 32])."""
    x = x.to(torch.float32).transpose(0, 1).unflatten(2, (-1, 32))
    big = x.abs().amax(3, keepdim=True)
    m, e = torch.frexp(big)  # big = m 2^e, 0.5 <= m < 1
    e = torch.clamp(e - 3 + (m >= 0.875).to(e.dtype), min=-120)
    e = torch.where(big == 0, torch.full_like(e, -120), e)
    a = torch.ldexp(x.abs(), -e)
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    code = code | ((x < 0) & (code > 0)).to(torch.uint8) << 3
    code = code.flatten(2)
    scale = torch.where(torch.isfinite(big), e + 127, torch.full_like(e, 255)).to(torch.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, scale[..., 0].flatten(2)


def _values(packed):
    """The float32 values [heads][n][size] that packed rows stand for."""
    codes, scale = packed
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(2)
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0.0, -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    unit = torch.ldexp(torch.ones_like(scale, dtype=torch.float32), scale.to(torch.int32) - 127)
    unit = torch.where(scale == 255, torch.full_like(unit, math.nan), unit)
    return grid[code.to(torch.int32)] * unit.repeat_interleave(32, 2)


def _attend(s):
    n, hd = s["n"], s["head_dim"]
    kv, length = s["kv_heads"], s["len"]
    group = s["heads"] // kv
    k, v = _values(s["k"]), _values(s["v"])
    q = s["q"].to(torch.float32).view(n, kv, group, hd).permute(1, 0, 2, 3).reshape(kv, n * group, hd)
    x = torch.matmul(q, k.transpose(1, 2)) * (1.0 / math.sqrt(hd))
    last = torch.arange(length - n, length, device=x.device).repeat_interleave(group)
    hidden = torch.arange(length, device=x.device)[None] > last[:, None]
    x = x.masked_fill(hidden, -math.inf)
    p = torch.exp(x - x.amax(2, keepdim=True))
    p = p / p.sum(2, keepdim=True)
    out = torch.matmul(p, v).view(kv, n, group, hd).permute(1, 0, 2, 3).reshape(n, s["heads"], hd).to(s["q"].dtype)
    return (out, s["w"] + p.sum(1)) if s["weights"] else out


def _evict(s):
    length, keep, recent = s["len"], s["keep"], s["recent"]
    order = torch.sort(s["w"][:, :length - recent], dim=1, descending=True, stable=True).indices[:, :keep - recent]
    newest = torch.arange(length - recent, length, device="cuda").expand(s["kv_heads"], recent)
    kept = torch.cat([torch.sort(order, dim=1).values, newest], 1)

    def rows(packed):
        return tuple(torch.gather(t, 1, kept[..., None].expand(-1, -1, t.shape[2])) for t in packed)

    return kept.to(torch.int32), torch.gather(s["w"], 1, kept), _values(rows(s["k"])), _values(rows(s["v"]))


def _logprobs(s):
    x = s["x"].to(torch.float32)
    d = x - x.amax(1, keepdim=True)
    e = torch.exp(d)
    z = e.sum(1, keepdim=True)
    lse = torch.log(z)
    logp = torch.gather(d, 1, s["tokens"].to(torch.int64)[:, None]) - lse
    entropy = lse - (e * d).sum(1, keepdim=True) / z
    # the largest values first, the lowest id first among equal ones: one whole number that orders both
    bits = (x + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64) * 4294967296
    ids = torch.topk(order - torch.arange(s["vocab"], device="cuda"), s["top"], dim=1).indices
    return logp[:, 0], entropy[:, 0], ids.to(torch.int32), torch.gather(d, 1, ids) - lse


def run(s):
    op = s["op"]
    if own:
        import daiza_amd as dz
        if op == "append":
            c = s["cache"]
            c.truncate(s["start"])
            c.append_dev(s["new_k"], s["new_v"], stream=_stream())
            c.read_dev(s["start"], s["out_k"], s["out_v"], stream=_stream())
            return s["out_k"], s["out_v"]
        if op == "attend":
            w = s["w"].clone() if s["weights"] else None
            s["cache"].attend_dev(s["q"], s["out"], weights=w, stream=_stream())
            return (s["out"], w) if s["weights"] else s["out"]
        if op == "evict":
            s["cache"].evict_dev(s["to"], s["keep"], s["recent"], s["w"], s["to_w"], s["kept"], stream=_stream())
            s["to"].read_dev(0, s["out_k"], s["out_v"], stream=_stream())
            return s["kept"], s["to_w"], s["out_k"], s["out_v"]
        dz.logprobs_dev(s["x"], s["tokens"], s["logp"], s["entropy"], s["top_ids"], s["top_logp"], stream=_stream())
        return s["logp"], s["entropy"], s["top_ids"], s["top_logp"]
    if op == "append":
        return _values(_pack(s["new_k"])), _values(_pack(s["new_v"]))
    return {"attend": _attend, "evict": _evict, "logprobs": _logprobs}[op](s)


# ---------------------------------------------------------------- the work of a pass


def work(case):
    op = case["op"]
    size = {"f32": 4, "f16": 2, "bf16": 2}[case.get("type", "f32")]
    if op == "logprobs":
        n, vocab = case["n"], case["vocab"]
        return {"bytes": n * vocab * size + n * (12 + 8 * case["top"]), "flops": 6 * n * vocab}
    row = case["kv_heads"] * case["head_dim"]  # values of a row of keys or of values
    held = 2 * row * 17 // 32  # bytes that the cache holds of a row
    if op == "append":
        n = case["n"]
        return {"bytes": n * (2 * row * size + held + 2 * row * 4), "flops": 20 * n * row}
    if op == "evict":
        keep = case["keep"]
        return {"bytes": 4 * case["kv_heads"] * (case["len"] + 2 * keep) + keep * (2 * held + 2 * row * 4), "flops": keep * 2 * row}
    n, length = case["n"], case["len"]
    pairs = sum(length - n + i + 1 for i in range(n)) * case["heads"]
    weights = 2 * 4 * case["kv_heads"] * length if case["weights"] else 0
    return {"bytes": length * held + 2 * n * case["heads"] * case["head_dim"] * size + weights,
            "flops": 4 * pairs * case["head_dim"]}


# ---------------------------------------------------------------- the same in 64 bits


def _stored64(x):
    """What the cache holds of rows [n][heads][size], in 64 bits: [heads][n][size]."""
    x = x.double().permute(1, 0, 2)
    blocks = x.reshape(*x.shape[:2], -1, 32)

    def two(power):
        return torch.ldexp(torch.ones_like(power), power.to(torch.int32))

    top = blocks.abs().max(-1, keepdim=True).values
    step = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
    step = torch.where(top >= two(step + 1), step + 1, torch.where(top < two(step), step - 1, step))
    step = torch.where(top > 0, step - 2 + (top >= 1.75 * two(step)), torch.full_like(step, -120)).clamp(min=-120)
    unit = two(step)
    a = blocks.abs() / unit
    # whole halves below 2, whole numbers below 4, even numbers above: the nearest, the even one of two as near
    near = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a), torch.round(a / 2) * 2)).clamp(max=6)
    return (torch.sign(blocks) * near * unit).reshape(x.shape)


def _exact_attend(case, seed):
    n, length, hd = case["n"], case["len"], case["head_dim"]
    group = case["heads"] // case["kv_heads"]
    q = _queries(case, seed).double()
    k, v = _stored64(_rows(case, seed, 1, length, KEYS)), _stored64(_rows(case, seed, 2, length, VALUES))
    out = torch.empty(n, case["heads"], hd, dtype=torch.float64, device="cuda")
    w = _row_weights(case, seed).double() if case["weights"] else None
    seen = torch.arange(length, device="cuda")[None, :] <= torch.arange(length - n, length, device="cuda")[:, None]
    for h in range(case["heads"]):
        g = h // group
        score = (q[:, h] @ k[g].t().contiguous()) / math.sqrt(hd)
        p = torch.softmax(torch.where(seen, score, torch.full_like(score, -math.inf)), 1)
        out[:, h] = p @ v[g]
        if w is not None:
            w[g] += p.sum(0)
    return (out, w) if case["weights"] else out


def _exact_evict(case, seed):
    length, keep, recent = case["len"], case["keep"], case["recent"]
    w = _row_weights(case, seed)
    # a row stays if fewer than keep - recent of the older rows come before it: larger ones, and equal ones of a lower index
    rank = torch.argsort(torch.argsort(-w[:, :length - recent].double(), dim=1, stable=True), dim=1)
    stays = torch.cat([rank < keep - recent, torch.ones_like(w[:, :recent], dtype=torch.bool)], 1)
    kept = torch.nonzero(stays)[:, 1].view(case["kv_heads"], keep)

    def rows(tag, scale):
        x = _stored64(_rows(case, seed, tag, length, scale))
        return torch.stack([x[g, kept[g]] for g in range(case["kv_heads"])])

    return (kept.to(torch.int32), torch.stack([w[g, kept[g]] for g in range(case["kv_heads"])]).double(), rows(1, KEYS),
            rows(2, VALUES))


def _exact_logprobs(case, seed):
    x, tokens = _logits(case, seed)
    outs = []
    for i in range(0, case["n"], 64):
        y = x[i:i + 64].double()
        lp = torch.log_softmax(y, 1)
        p = torch.exp(lp)
        top, ids = torch.sort(lp, dim=1, descending=True, stable=True)
        # equal logits give equal log probabilities, so the order is that of the logits
        outs.append((lp.gather(1, tokens[i:i + 64].long()[:, None])[:, 0], -(p * lp).sum(1), ids[:, :case["top"]].to(torch.int32),
                     top[:, :case["top"]]))
    return tuple(torch.cat(t) for t in zip(*outs))


def exact(case, seed):
    op = case["op"]
    if op == "append":
        return _stored64(_rows(case, seed, 6, case["n"], KEYS)), _stored64(_rows(case, seed, 7, case["n"], VALUES))
    return {"attend": _exact_attend, "evict": _exact_evict, "logprobs": _exact_logprobs}[op](case, seed)
