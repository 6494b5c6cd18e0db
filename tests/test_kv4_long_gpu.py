"""Long caches, many rows and large vocabularies, where calls take other forms of the kernels than the short ones of
test_kv4_gpu.py and test_logprobs_gpu.py, against the same 64-bit plain forms (kv4_ref.py)."""
import math

import pytest
import torch

import kv4_ref as ref
from test_kv4_gpu import TYPES, _cache, _check_attend, _check_evict, _normal, _rows, _same
from test_logprobs_gpu import _check, _logits

pytestmark = pytest.mark.gpu


# Eight waves on a row tile (beyond 32768 positions times key/value heads and row tiles), and chunks by the dozen: at one
# key/value head 20000 and 40000 positions go in 157 chunks, of four and of eight waves.
@pytest.mark.parametrize("nq,nkv,hd,length,n", [(24, 4, 256, 9000, 1), (24, 4, 256, 9000, 2), (24, 4, 256, 9001, 8), (2, 1, 64, 20000, 1),
                                                (2, 1, 64, 40000, 1), (7, 1, 128, 33000, 3), (16, 8, 128, 4500, 7)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_long(dz, nq, nkv, hd, length, n, dtype):
    _check_attend(dz, nq, nkv, hd, length, n, dtype, True)


# 17 to 112 query rows: the weights' pass has two tiles of 16 positions a wave from 400 blocks of 64 positions and heads on, and
# four from 800.
@pytest.mark.parametrize("nq,nkv,hd,length,n", [(16, 8, 64, 3300, 9), (16, 8, 64, 3271, 56), (16, 8, 64, 6500, 20), (8, 4, 128, 6410, 13),
                                                (8, 4, 64, 12801, 50), (16, 8, 256, 3300, 20), (8, 8, 256, 6405, 17)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_weights_of_few_tokens_behind_many_rows(dz, nq, nkv, hd, length, n, dtype):
    _check_attend(dz, nq, nkv, hd, length, n, dtype, True)


@pytest.mark.parametrize("nq,nkv,hd,length,n,at", [(24, 4, 256, 9000, 8, 8996), (24, 4, 256, 9000, 1, 31), (2, 1, 64, 40000, 3, 39998),
                                                   (16, 8, 64, 3300, 20, 3290), (16, 8, 64, 6500, 20, 6485), (8, 4, 128, 6410, 13, 6397)])
@pytest.mark.parametrize("where", ["k", "v"])
def test_later_rows_stay_out_of_long_calls(dz, nq, nkv, hd, length, n, at, where):
    """A row with a NaN: queries before it are as without it, bit for bit, those that see it get NaN, and the weights of other
    heads' rows and, of a value, all weights are untouched."""
    k, v = _rows(80, length, nkv, hd), _rows(81, length, nkv, hd)
    q = _normal(82, n, nq, hd).cuda()
    got = []
    for bad in (False, True):
        if bad:
            (k if where == "k" else v)[at, 0, 37] = math.nan
        c = _cache(dz, k, v)
        out, w = torch.empty_like(q), torch.zeros(nkv, length, device="cuda")
        c.attend_dev(q, out, weights=w)
        got.append((out.cpu(), w.cpu()))
    (want, ww), (out, w) = got
    first, grp = max(0, at - (length - n)), nq // nkv
    assert torch.equal(out[:first], want[:first]) and torch.equal(out[:, grp:], want[:, grp:]) and torch.equal(w[1:], ww[1:])
    if where == "k":
        assert bool(torch.isnan(out[first:, :grp]).all())
        # every row that a query with a NaN sees gets its share of it; the first such query sees the rows up to `seen`
        seen = length - n + first + 1
        assert bool(torch.isnan(w[0, :seen]).all())
    else:
        assert bool(torch.isnan(out[first:, :grp, 32:64]).all()) and torch.equal(out[..., :32], want[..., :32])
        assert torch.equal(w, ww)


# More than 32768 rows to choose from: the keys are read anew for each pass instead of staying in registers.
@pytest.mark.parametrize("kind", ["spread", "equal", "zeros", "special"])
@pytest.mark.parametrize("nkv,length,keep,recent", [(2, 32769, 1, 0), (1, 32868, 32868, 99), (1, 32869, 20000, 100), (2, 40001, 10000, 256),
                                                    (1, 100000, 33333, 0), (1, 100000, 99999, 64)])
def test_evict_long(dz, kind, nkv, length, keep, recent):
    g = torch.Generator().manual_seed(length + keep)
    w = torch.exp(torch.randn(nkv, length, generator=g) * 3)
    if kind == "equal":
        w[:] = 0.75
    elif kind == "zeros":
        w = torch.where(torch.rand(w.shape, generator=g) < 0.95, torch.zeros_like(w), w)
        w[0, ::3] = -0.0
    elif kind == "special":
        r = torch.rand(w.shape, generator=g)
        w = torch.where(r < 0.4, torch.full_like(w, math.nan), torch.where(r < 0.5, torch.full_like(w, math.inf), w))
        w = torch.where((r > 0.6) & (r < 0.9), torch.floor(w), w)
    _check_evict(dz, w, keep, recent, 64)


# More than 1024 groups of 256 logits: they are looked through in batches.
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab,top", [(262144, 20), (262145, 20), (300001, 64), (600000, 3)])
def test_large_vocabularies(dz, dtype, vocab, top):
    _check(dz, *_logits(vocab, 2, vocab, dtype), top)


@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "last", "masked"])
def test_orders_over_large_vocabularies(dz, kind):
    vocab = 300001
    i = torch.arange(vocab, dtype=torch.float32)
    x = {"equal": torch.full((vocab,), 0.5), "rising": i * 1e-4, "falling": -i * 1e-4, "last": torch.where(i > vocab - 30, 4.0, 0.0),
         "masked": torch.where(i < 270000, -math.inf, 1.0)}[kind].reshape(1, -1)
    if kind == "masked":
        x[0, 270005:] = -math.inf
    _check(dz, x, torch.tensor([270001], dtype=torch.int32), 40)


def test_more_rows_than_a_launch_takes(dz):
    _check(dz, *_logits(9, 70000, 7), 2)


def test_codes_past_32_bits(dz):
    """34 million rows of 128 bytes of codes: rows of zeros, on which every score is 0, and a few others at either end of them."""
    n, hd, nq = (1 << 25) + (1 << 20), 256, 6
    c = dz.Kv4Cache(1, hd, n + 8)
    k, v = _rows(92, 8, 1, hd), _rows(93, 8, 1, hd)
    c.append_dev(k[:3].cuda(), v[:3].cuda())
    zeros = torch.zeros(n, 1, hd, dtype=torch.bfloat16, device="cuda")
    c.append_dev(zeros, zeros)
    del zeros
    c.append_dev(k[3:].cuda(), v[3:].cuda())
    ks, vs = ref.stored(k)[0], ref.stored(v)[0]
    gk, gv = (torch.empty(1, 6, hd, device="cuda") for _ in range(2))
    c.read_dev(n + 2, gk, gv)
    assert torch.equal(gk[0, 1:].cpu().double(), ks[3:]) and torch.equal(gv[0, 1:].cpu().double(), vs[3:])
    assert not gk[0, 0].any() and not gv[0, 0].any()
    q = _normal(94, 2, nq, hd) * 8.0  # the last rows' scores against millions of zeros
    out, w = torch.empty(2, nq, hd, device="cuda"), torch.zeros(1, n + 8, device="cuda")
    c.attend_dev(q.cuda(), out, weights=w)
    s = (q.double() @ ks.T) / math.sqrt(hd)  # [2][heads][8]
    s[0, :, 7] = -math.inf
    m = s.amax(2, keepdim=True).clamp(min=0)
    p, z0 = torch.exp(s - m), torch.exp(-m[..., 0])
    z = p.sum(2) + n * z0
    want = (p @ vs) / z[..., None]
    # f32 sums of 34 million terms in 256 chunks of eight waves with 8 terms a tile and lane: partial sums of at most
    # 34e6 / 2048 / 32 = 520 tiles' totals, joined over waves and chunks, each addition 2^-24; scores and exponentials as
    # in kv4_ref.attend (hd + 4 and 16 units on scores of at most |s| + |m|)
    u = 2.0 ** -24
    terms = (q.double().abs() @ ks.abs().T).amax(2) / math.sqrt(hd)
    rel = (520 + 8 + 8 + 256 + 16) * u + 2 * (hd + 4) * u * terms
    assert bool(((out.cpu().double() - want).abs() <= rel[..., None] * ((p @ vs.abs()) / z[..., None]) + u * want.abs()).all())
    ww, got = (p / z[..., None]).sum((0, 1)), w[0].cpu().double()
    ends = torch.cat([got[:3], got[-5:]])
    assert bool(((ends - ww).abs() <= rel.max() * ww + 12 * u * ww).all())
    each = (z0 / z).sum()
    assert bool(((got[3:-5] - each).abs() <= (rel.max() + 12 * u) * each).all())
    # the three best of all but the newest two rows
    small = dz.Kv4Cache(1, hd, 5)
    kept, dw = torch.empty(1, 5, dtype=torch.int32, device="cuda"), torch.empty(1, 5, device="cuda")
    c.evict_dev(small, 5, 2, w, dw, kept)
    order = torch.sort(w[0, :-2], descending=True, stable=True).indices[:3].sort().values
    assert torch.equal(kept[0].cpu().long(), torch.cat([order.cpu(), torch.tensor([n + 6, n + 7])]))
    rk = torch.empty(1, 5, hd, device="cuda")
    small.read_dev(0, rk)
    assert torch.equal(rk[0, 3:].cpu().double(), ks[6:]) and torch.equal(dw[0], w[0, kept[0].long()])


def test_logits_past_32_bits(dz):
    """9000 rows of 248320 bf16 logits are 2^31 elements and more: the last rows by themselves give the same."""
    n, vocab = 9000, 248320
    x = torch.randn(64, vocab, generator=torch.Generator().manual_seed(12)).bfloat16().cuda()
    big = torch.empty(n, vocab, dtype=torch.bfloat16, device="cuda")
    for i in range(0, n, 64):
        big[i:i + 64] = x[:min(64, n - i)].roll(i // 64, 1)
    tokens = (torch.arange(n, device="cuda") * 27).to(torch.int32)

    def run(x, t):
        out = [torch.empty(x.shape[0], device="cuda"), torch.empty(x.shape[0], device="cuda"),
               torch.empty(x.shape[0], 5, dtype=torch.int32, device="cuda"), torch.empty(x.shape[0], 5, device="cuda")]
        dz.logprobs_dev(x, t, *out)
        return out

    whole = run(big, tokens)
    _check(dz, big[-2:].clone(), tokens[-2:].cpu(), 5)
    for r in (0, 4000, 8640, n - 100):
        part = run(big[r:r + 100].clone(), tokens[r:r + 100].clone())
        # more parts of a row with fewer rows: sums in another order
        assert torch.equal(whole[2][r:r + 100], part[2])
        assert all(torch.allclose(whole[i][r:r + 100], part[i], rtol=0, atol=1e-4) for i in (0, 1, 3))


def test_eight_million_rows(dz):
    """More rows than a launch of the join has threads for: every row against torch's own log softmax in 64 bits."""
    n = (1 << 23) + 77
    x = torch.randn(n, 3, generator=torch.Generator().manual_seed(10)).cuda()
    tokens = (torch.arange(n, device="cuda") % 3).to(torch.int32)
    lp, ent = torch.full((n,), 9.0, device="cuda"), torch.full((n,), 9.0, device="cuda")
    ids, tl = torch.full((n, 1), -1, dtype=torch.int32, device="cuda"), torch.full((n, 1), 9.0, device="cuda")
    dz.logprobs_dev(x, tokens, lp, ent, ids, tl)
    y = x.double()
    want = y - torch.logsumexp(y, 1, keepdim=True)
    best, at = want.max(1)
    # three terms and a logarithm in f32: the bounds of kv4_ref.logprobs at a vocabulary of 3, |log p| and the entropy under 16
    u = 2.0 ** -24
    assert ((lp.double() - want.gather(1, tokens.long()[:, None])[:, 0]).abs() <= 11 * u + 4 * u * 18).all()
    assert ((tl[:, 0].double() - best).abs() <= 11 * u + 4 * u * 18).all() and torch.equal(ids[:, 0].long(), at)
    assert ((ent.double() + (want.exp() * want).sum(1)).abs() <= 2 * 11 * u * 17 + 8 * u * 2).all()


def test_rows_in_and_out_of_a_long_cache(dz):
    n, nkv, hd = 70001, 1, 64
    k, v = _rows(90, n, nkv, hd), _rows(91, n, nkv, hd)
    c = _cache(dz, k, v)
    gk, gv = (torch.empty(nkv, n, hd, device="cuda") for _ in range(2))
    c.read_dev(0, gk, gv)
    assert _same(gk.cpu().double(), ref.stored(k)) and _same(gv.cpu().double(), ref.stored(v))
