"""The key/value cache held in 4 bits against 64-bit plain forms (kv4_ref.py): rows in and out, attention, the weights that rows
receive, eviction, the calls in sequence, under graph capture and on other streams, and what is refused."""
import ctypes
import math

import pytest
import torch

import kv4_ref as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _rows(seed, n, nkv, hd, scale=1.0, dtype="f32"):
    ch = torch.exp(_normal(seed, nkv, hd) * 0.7) * scale
    return ((_normal(seed + 1, n, nkv, hd) + 0.3 * _normal(seed + 2, nkv, hd)) * ch).to(TYPES[dtype])


def _cache(dz, k, v, capacity=None):
    n, nkv, hd = k.shape
    c = dz.Kv4Cache(nkv, hd, capacity or max(1, n))
    c.append_dev(k.cuda(), v.cuda())
    return c


def _read(c, start, n):
    k, v = (torch.empty(c.kv_heads, n, c.head_dim, device="cuda") for _ in range(2))
    c.read_dev(start, k, v)
    return k.cpu().double(), v.cpu().double()


def _same(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(), b.nan_to_num())


# ---------------------------------------------------------------- rows in and out


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("nkv,hd,start,n", [(4, 256, 0, 1), (1, 256, 31, 2), (2, 256, 33, 65), (3, 128, 0, 40), (1, 64, 17, 100)])
def test_rows_are_held_as_defined(dz, dtype, nkv, hd, start, n):
    k, v = _rows(1, start + n, nkv, hd, 2.0, dtype), _rows(5, start + n, nkv, hd, 0.01, dtype)
    c = dz.Kv4Cache(nkv, hd, start + n + 3)
    c.append_dev(k[:start].cuda(), v[:start].cuda())
    # new rows out of a wider array, at an odd offset
    wide = torch.zeros(n, 2 * nkv * hd + 3).to(TYPES[dtype])
    wide[:, 1:1 + nkv * hd] = k[start:].flatten(1)
    wide[:, 2 + nkv * hd:2 + 2 * nkv * hd] = v[start:].flatten(1)
    wide = wide.cuda()
    c.append_dev(wide[:, 1:1 + nkv * hd].unflatten(1, (nkv, hd)), wide[:, 2 + nkv * hd:2 + 2 * nkv * hd].unflatten(1, (nkv, hd)))
    assert len(c) == start + n
    gk, gv = _read(c, 0, start + n)
    assert torch.equal(gk, ref.stored(k)) and torch.equal(gv, ref.stored(v))
    if n > 1:
        pk, pv = _read(c, start + 1, n - 1)
        assert torch.equal(pk, gk[:, start + 1:]) and torch.equal(pv, gv[:, start + 1:])


def test_blocks_at_the_edges_of_the_format(dz):
    """Ties of every step, the largest value at every mantissa that decides the scale, zeros, the smallest and largest numbers,
    infinities and NaN; f32 rows that hold them read back as defined, and written again they stay as they are."""
    rows = []
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.0])
    eps = 2.0 ** -20
    blk = torch.cat([ties, -ties, ties * (1 + eps), ties * (1 - eps)])
    blk[7] = 6.0  # fixes the scale at 1
    for e in (0, -30, 60, -118, 125):
        rows.append(blk * 2.0 ** e)
    for top in (1.0, 1.49, 1.5, 1.7499999, 1.75, 1.7500001, 1.9999999):
        rows.append(torch.linspace(-1, 1, 32) * top)
    rows += [torch.zeros(32), torch.full((32,), -0.0), torch.full((32,), 1e-45), torch.full((32,), 2.0 ** -121),
             torch.full((32,), 2.0 ** -126), torch.full((32,), 3.4028234e38), torch.full((32,), -1.7e38)]
    for bad in (math.inf, -math.inf, math.nan):
        b = torch.linspace(-2, 3, 32)
        b[13] = bad
        rows.append(b)
    n = 4  # rows of 8 blocks
    while len(rows) % 8:
        rows.append(torch.linspace(0, len(rows), 32))
    x = torch.stack(rows).reshape(-1, 1, 256)
    n = x.shape[0]
    c = _cache(dz, x, x.flip(0), n)
    gk, gv = _read(c, 0, n)
    assert _same(gk, ref.stored(x)) and _same(gv, ref.stored(x.flip(0)))
    again = _cache(dz, gk.permute(1, 0, 2).float(), gv.permute(1, 0, 2).float(), n)
    hk, hv = _read(again, 0, n)
    assert _same(hk, gk) and _same(hv, gv)


def test_truncate_and_rows_behind(dz):
    k, v = _rows(7, 100, 2, 128), _rows(8, 100, 2, 128)
    c = _cache(dz, k, v, 100)
    c.truncate(200)
    assert len(c) == 100
    c.truncate(37)
    assert len(c) == 37
    nk, nv = _rows(9, 5, 2, 128), _rows(10, 5, 2, 128)
    c.append_dev(nk.cuda(), nv.cuda())
    gk, gv = _read(c, 0, 42)
    assert torch.equal(gk, torch.cat([ref.stored(k)[:, :37], ref.stored(nk)], 1))
    assert torch.equal(gv, torch.cat([ref.stored(v)[:, :37], ref.stored(nv)], 1))


# ---------------------------------------------------------------- attention


def _check_attend(dz, nq, nkv, hd, length, n, dtype, weights, kscale=1.0, seed=20):
    k, v = _rows(seed, length, nkv, hd, kscale), _rows(seed + 3, length, nkv, hd, 0.5)
    c = _cache(dz, k, v)
    q = _normal(seed + 9, n, nq, hd).to(TYPES[dtype])
    out = torch.full((n, nq, hd), 7.0, dtype=TYPES[dtype], device="cuda")
    w0 = _normal(seed + 11, nkv, length + 5).abs()
    w = w0.cuda()
    c.attend_dev(q.cuda(), out, weights=w if weights else None)
    want, ww, bound, wb = ref.attend(q, ref.stored(k), ref.stored(v))
    half = torch.finfo(TYPES[dtype]).eps / 2
    err = (out.cpu().double() - want).abs()
    assert bool((err <= bound * (1 + half) + half * want.abs() + 1e-30 + (6e-8 if dtype == "f16" else 0)).all()), \
        (err / bound).max()  # f16: half its smallest step beside the relative one
    if weights:
        got = w.cpu().double()
        assert torch.equal(got[:, length:], w0[:, length:].double())
        assert bool(((got[:, :length] - w0[:, :length].double() - ww).abs() <= wb + 2.0 ** -24 * (w0[:, :length] + ww)).all())


@pytest.mark.parametrize("nq,nkv,hd,length,n", [
    (24, 4, 256, 1, 1), (6, 1, 256, 31, 1), (6, 1, 256, 33, 1), (24, 4, 256, 700, 1), (8, 8, 256, 129, 1), (16, 1, 256, 64, 1),
    (32, 1, 256, 300, 1), (7, 1, 128, 257, 1), (12, 4, 128, 511, 1), (16, 4, 64, 96, 1), (10, 2, 64, 1000, 1),
    (6, 1, 256, 2, 2), (6, 1, 256, 200, 3), (24, 4, 256, 520, 8), (6, 1, 256, 47, 11), (2, 2, 256, 65, 65), (6, 1, 256, 333, 100),
    (3, 1, 128, 130, 43), (16, 2, 128, 400, 129), (16, 4, 64, 333, 70), (5, 5, 64, 64, 64), (40, 1, 128, 75, 5),
])
@pytest.mark.parametrize("dtype,weights", [("f32", True), ("bf16", False)])
def test_attend(dz, nq, nkv, hd, length, n, dtype, weights):
    _check_attend(dz, nq, nkv, hd, length, n, dtype, weights)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attend_types(dz, dtype):
    _check_attend(dz, 6, 1, 256, 300, 1, dtype, True)
    _check_attend(dz, 12, 4, 128, 300, 40, dtype, True)
    _check_attend(dz, 4, 2, 64, 100, 9, dtype, True)


@pytest.mark.parametrize("nq,nkv,hd,length,n", [(24, 4, 256, 700, 60), (6, 1, 256, 250, 250), (8, 2, 128, 600, 77), (16, 1, 128, 41, 13),
                                                (4, 2, 64, 260, 129), (12, 1, 64, 90, 33), (2, 2, 64, 2400, 200), (16, 2, 128, 4200, 30)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_attend_many_rows(dz, nq, nkv, hd, length, n, dtype):
    _check_attend(dz, nq, nkv, hd, length, n, dtype, True)


def test_attend_in_chunks_to_fill_the_last_round(dz):
    # 300 row tiles of 64 rows for 256 workgroups, 600 for 512, behind positions enough for chunks of their own
    _check_attend(dz, 75, 75, 64, 4200, 193, "f32", False)
    _check_attend(dz, 150, 150, 64, 4200, 193, "bf16", True)


@pytest.mark.parametrize("n", [1, 30, 70])
@pytest.mark.parametrize("hd", [64, 256])
def test_attend_queries_of_uneven_size(dz, n, hd):
    # one dim in every 32 a thousand times the others, whose keys are small: a query of many rows is held to 2^-29 of its
    # block's largest (the bound below), a key's 4 bits take the rest
    k, v = _rows(56, 150, 1, hd), _rows(57, 150, 1, hd)
    k[:, :, 7::32] *= 1e-3
    q = _normal(58, n, 4, hd)
    q[:, :, 7::32] *= 1e3
    c = _cache(dz, k, v)
    out, w = torch.empty(n, 4, hd, device="cuda"), torch.zeros(1, 150, device="cuda")
    c.attend_dev(q.cuda(), out, weights=w)
    ks, vs = ref.stored(k), ref.stored(v)
    want, ww, bound, wb = ref.attend(q, ks, vs)
    big = q.double().abs().reshape(n, 4, -1, 32).amax(-1)  # [n][heads][blocks]
    held = (big @ ks[0].abs().reshape(150, -1, 32).sum(-1).T).amax(-1) * 2.0 ** -29 / math.sqrt(hd)  # of a score, absolute
    more = 2 * held[..., None] * vs.abs().amax()
    assert bool(((out.cpu().double() - want).abs() <= bound + more + 2.0 ** -24 * want.abs()).all())
    assert bool(((w.cpu().double() - ww).abs() <= wb + 4 * held.amax() * ww + 2.0 ** -24 * ww).all())


@pytest.mark.parametrize("n", [1, 30, 70])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attend_f32_queries_beside_outliers(dz, n, hd):
    """One dim in every 32 a million times the others, whose keys are held as 0: the other dims' bits count as in any f32 product,
    by one query and by many, in the outputs and in the weights."""
    k, v = _rows(59, 150, 1, hd), _rows(63, 150, 1, hd)
    k[:, :, 7::32] *= 1e-6
    q = _normal(64, n, 4, hd)
    q[:, :, 7::32] *= 2.0 ** 20
    ks, vs = ref.stored(k), ref.stored(v)
    assert bool((ks[:, :, 7::32] == 0).all())
    c = _cache(dz, k, v)
    out, w = torch.empty(n, 4, hd, device="cuda"), torch.zeros(1, 150, device="cuda")
    c.attend_dev(q.cuda(), out, weights=w)
    want, ww, bound, wb = ref.attend(q, ks, vs)
    assert bool(((out.cpu().double() - want).abs() <= bound + 2.0 ** -24 * want.abs()).all())
    assert bool(((w.cpu().double() - ww).abs() <= wb + 2.0 ** -24 * ww).all())


@pytest.mark.parametrize("n,nkv", [(512, 4), (8, 256)])
def test_attend_errors_have_no_sign(dz, n, nkv):
    """The relative errors of a million positive f16 outputs average out, by many rows a head and by few.

    An output's rounding is off by up to 2^-11 to either side, so the mean of N = 2^20 of them stays under
    2^-10 sqrt(ln(2 / 1e-9) / 2N) = 3.1e-6 but for one run in 1e9 (Hoeffding); the f32 evaluation gets 16 half steps, 2^-20."""
    nq, hd, length = 4 * nkv, 128, 600
    k, v = _rows(65, length, nkv, hd), _rows(66, length, nkv, hd).abs() + 0.1
    q = _normal(67, n, nq, hd).half().cuda()
    c = _cache(dz, k, v)
    out = torch.empty_like(q)
    c.attend_dev(q, out)
    ks, vs, grp = ref.stored(k).cuda(), ref.stored(v).cuda(), nq // nkv
    hidden = torch.arange(length, device="cuda")[None] > torch.arange(length - n, length, device="cuda")[:, None]
    mean = torch.zeros((), dtype=torch.float64, device="cuda")
    for h in range(nq):
        s = (q[:, h].double() @ ks[h // grp].t().contiguous()) * hd ** -0.5
        want = torch.softmax(s.masked_fill(hidden, -math.inf), 1) @ vs[h // grp]
        mean += ((out[:, h].double() - want) / want).sum()
    assert out.numel() == 2 ** 20 and abs(mean.item() / out.numel()) < 3.1e-6 + 2.0 ** -20, mean.item() / out.numel()


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_query_that_is_not_a_number_among_many(dz, value, hd):
    k, v = _rows(50, 110, 1, hd), _rows(51, 110, 1, hd)
    q = _normal(52, 90, 3, hd)
    c = _cache(dz, k, v)
    want, got = torch.empty(90, 3, hd, device="cuda"), torch.empty(90, 3, hd, device="cuda")
    ww, gw = torch.zeros(1, 110, device="cuda"), torch.zeros(1, 110, device="cuda")
    c.attend_dev(q.cuda(), want, weights=ww)
    q[41, 1, hd - 3] = value
    c.attend_dev(q.cuda(), got, weights=gw)
    assert bool(torch.isnan(got[41, 1]).all())
    got[41, 1] = want[41, 1]
    assert torch.equal(got, want)
    assert bool(torch.isnan(gw[0, :20 + 42]).all()) and torch.equal(gw[0, 20 + 42:], ww[0, 20 + 42:])


@pytest.mark.parametrize("kscale", [1e-6, 30.0])
def test_attend_flat_and_peaked(dz, kscale):
    """Scores all but equal, and scores whose largest takes all the weight."""
    _check_attend(dz, 6, 1, 256, 500, 1, "f32", True, kscale)
    _check_attend(dz, 4, 2, 128, 200, 50, "f32", True, kscale)


def test_attend_strided_and_scaled(dz):
    k, v = _rows(30, 90, 2, 128), _rows(31, 90, 2, 128)
    c = _cache(dz, k, v)
    wide = torch.zeros(7, 2 * 4 * 128 + 1)
    q = _normal(33, 7, 4, 128)
    wide[:, 3:3 + 512] = q.flatten(1)
    dst = torch.full((7, 4 * 128 + 5), 3.0, device="cuda")
    c.attend_dev(wide.cuda()[:, 3:3 + 512].unflatten(1, (4, 128)), dst[:, 2:2 + 512].unflatten(1, (4, 128)), scale=0.02)
    want, _, bound, _ = ref.attend(q, ref.stored(k), ref.stored(v), 0.02)
    got = dst.cpu()
    assert bool(((got[:, 2:514].reshape(7, 4, 128).double() - want).abs() <= bound + 2.0 ** -24 * want.abs()).all())
    assert bool((got[:, :2] == 3).all()) and bool((got[:, 514:] == 3).all())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n", [1, 9, 120])
def test_attend_at_odd_addresses(dz, dtype, n):
    """16-bit queries and outputs out of wider arrays, two bytes off any alignment, by one tile of rows a workgroup and by four."""
    k, v = _rows(34, 300, 2, 128), _rows(35, 300, 2, 128)
    c = _cache(dz, k, v)
    q = _normal(36, n, 4, 128).to(TYPES[dtype])
    want, w0, w1 = torch.empty(n, 4, 128, dtype=TYPES[dtype], device="cuda"), *(torch.zeros(2, 300, device="cuda") for _ in range(2))
    c.attend_dev(q.cuda(), want, weights=w0)
    src, dst = (torch.full((n, 4 * 128 + 7), 3.0, dtype=TYPES[dtype], device="cuda") for _ in range(2))
    src[:, 1:513] = q.flatten(1).cuda()
    c.attend_dev(src[:, 1:513].unflatten(1, (4, 128)), dst[:, 3:515].unflatten(1, (4, 128)), weights=w1)
    assert torch.equal(dst[:, 3:515].unflatten(1, (4, 128)), want) and torch.equal(w0, w1)
    assert bool((dst[:, :3] == 3).all()) and bool((dst[:, 515:] == 3).all())


@pytest.mark.parametrize("nq,nkv,hd,length,n,at", [(6, 1, 256, 70, 20, 60), (4, 2, 128, 300, 120, 200), (2, 1, 64, 40, 40, 0),
                                                   (6, 1, 256, 700, 5, 697), (24, 4, 256, 40, 1, 12)])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_later_rows_stay_out(dz, nq, nkv, hd, length, n, at, where, value):
    """A row with an infinity or a NaN: queries before it are as without it, bit for bit; those that see it get NaN (of a
    value only in its block), and the weights of the rows that only earlier queries see are untouched."""
    k, v = _rows(40, length, nkv, hd), _rows(41, length, nkv, hd)
    q = _normal(42, n, nq, hd).cuda()

    def run(k, v):
        c = _cache(dz, k, v)
        out, w = torch.empty_like(q), torch.zeros(nkv, length, device="cuda")
        c.attend_dev(q, out, weights=w)
        return out.cpu(), w.cpu()

    want, ww = run(k, v)
    k2, v2 = k.clone(), v.clone()
    (k2 if where == "k" else v2)[at, 0, 37] = value
    got, gw = run(k2, v2)
    first = max(0, at - (length - n))  # the first query that sees row `at`
    grp = nq // nkv
    assert torch.equal(got[:first], want[:first])
    assert torch.equal(got[:, grp:], want[:, grp:])
    if where == "k":
        assert bool(torch.isnan(got[first:, :grp]).all())
        assert torch.equal(gw[1:], ww[1:])
        assert bool(torch.isnan(gw[0]).any())
    else:
        assert bool(torch.isnan(got[first:, :grp, 32:64]).all())
        assert torch.equal(got[first:, :grp, :32], want[first:, :grp, :32])
        assert torch.equal(got[first:, :grp, 64:], want[first:, :grp, 64:])
        assert torch.equal(gw, ww)


def test_query_with_nan(dz):
    k, v = _rows(50, 50, 1, 128), _rows(51, 50, 1, 128)
    q = _normal(52, 20, 3, 128)
    c = _cache(dz, k, v)
    want, got = torch.empty(20, 3, 128, device="cuda"), torch.empty(20, 3, 128, device="cuda")
    c.attend_dev(q.cuda(), want)
    q[4, 1, 5] = math.nan
    c.attend_dev(q.cuda(), got)
    assert bool(torch.isnan(got[4, 1]).all())
    got[4, 1] = want[4, 1]
    assert torch.equal(got, want)


@pytest.mark.parametrize("n", [2, 40])
def test_scores_past_f32(dz, n):
    # every score of head 0 is -inf in f32: its softmax is 0 / 0 in what each query sees, and nothing elsewhere
    k, v = torch.full((70, 1, 64), 2.0 ** 100), _rows(54, 70, 1, 64)
    c = _cache(dz, k, v)
    q = _normal(55, n, 2, 64)
    q[:, 0] = -2.0 ** 100
    q[:, 1] = 0
    out, w = torch.empty(n, 2, 64, device="cuda"), torch.zeros(1, 75, device="cuda")
    c.attend_dev(q.cuda(), out, weights=w)
    assert bool(torch.isnan(out[:, 0]).all()) and bool(torch.isfinite(out[:, 1]).all())
    assert bool(torch.isnan(w[0, :70]).all()) and bool((w[0, 70:] == 0).all())


def test_same_results_every_time(dz):
    k, v = _rows(60, 3000, 4, 256), _rows(61, 3000, 4, 256)
    c = _cache(dz, k, v)
    for n in (1, 8, 50):
        q = _normal(62, n, 24, 256).cuda()
        got = []
        for _ in range(3):
            out, w = torch.empty_like(q), torch.zeros(4, 3000, device="cuda")
            c.attend_dev(q, out, weights=w)
            got.append((out, w))
        assert all(torch.equal(a, got[0][0]) and torch.equal(b, got[0][1]) for a, b in got)


# ---------------------------------------------------------------- eviction


def _check_evict(dz, w, keep, recent, hd=64, spare=0):
    nkv, length = w.shape
    k, v = _rows(70, length, nkv, hd), _rows(71, length, nkv, hd)
    c = _cache(dz, k, v)
    m = min(keep, length)
    dst = dz.Kv4Cache(nkv, hd, max(1, m + spare))
    kept = torch.full((nkv, m), -1, dtype=torch.int32, device="cuda")
    dw = torch.full((nkv, m + 2), 9.0, device="cuda")
    c.evict_dev(dst, keep, recent, w.cuda(), dw, kept)
    want = ref.evict(w, keep, recent)
    assert torch.equal(kept.cpu(), want)
    assert len(dst) == m and len(c) == length
    idx = want.long()
    assert _same(dw.cpu()[:, :m], torch.gather(w, 1, idx)) and bool((dw[:, m:] == 9).all())
    if m:
        gk, gv = _read(dst, 0, m)
        ii = idx[..., None].expand(-1, -1, hd)
        assert torch.equal(gk, torch.gather(ref.stored(k), 1, ii)) and torch.equal(gv, torch.gather(ref.stored(v), 1, ii))


@pytest.mark.parametrize("length,keep,recent", [(1, 1, 0), (1, 1, 1), (5, 0, 0), (64, 10, 3), (100, 100, 7), (100, 300, 200), (100, 40, 40),
                                                (1000, 999, 0), (1025, 512, 64), (3000, 1, 0), (5000, 2500, 100)])
@pytest.mark.parametrize("nkv,hd", [(1, 256), (3, 128), (2, 64)])
def test_evict(dz, length, keep, recent, nkv, hd):
    w = torch.exp(_normal(length + keep, nkv, length) * 3)
    _check_evict(dz, w, keep, recent, hd)


@pytest.mark.parametrize("kind", ["equal", "zeros", "few", "neighbours", "special", "negative"])
@pytest.mark.parametrize("length,keep,recent", [(200, 50, 8), (2100, 1111, 0)])
def test_evict_ties_and_odd_weights(dz, kind, length, keep, recent):
    g = torch.Generator().manual_seed(length)
    w = torch.rand(2, length, generator=g)
    if kind == "equal":
        w[:] = 0.75
    elif kind == "zeros":
        w = torch.where(w < 0.9, torch.zeros_like(w), w) * torch.where(torch.rand(w.shape, generator=g) < 0.5, -0.0, 1.0).abs()
        w[0, ::3] = -0.0
        w[0, 1::3] = 0.0
    elif kind == "few":
        w = torch.floor(w * 4)
    elif kind == "neighbours":  # values that differ in their last bits only
        w = (torch.full_like(w, 1.0).view(torch.int32) + torch.randint(0, 5, w.shape, generator=g).to(torch.int32)).view(torch.float32)
    elif kind == "special":
        r = torch.rand(w.shape, generator=g)
        w = torch.where(r < 0.4, torch.full_like(w, math.nan), torch.where(r < 0.5, torch.full_like(w, math.inf), w))
        w = torch.where((r > 0.6) & (r < 0.7), torch.full_like(w, -math.inf), w)
    else:
        w = -w
    _check_evict(dz, w, keep, recent, spare=40)


# ---------------------------------------------------------------- in sequence


def test_append_attend_evict_and_on(dz):
    """A cache that a conversation fills, bounded twice, the weights carried along, against the same in 64 bits."""
    nq, nkv, hd, bound_rows = 6, 2, 128, 96
    a, b = dz.Kv4Cache(nkv, hd, 200), dz.Kv4Cache(nkv, hd, 200)
    wa, wb = torch.zeros(nkv, 200, device="cuda"), torch.zeros(nkv, 200, device="cuda")
    rk = rv = None
    seed = 100
    slack = torch.zeros(nkv, 0, dtype=torch.float64)
    for step, n in enumerate([70, 1, 1, 60, 1, 33, 90, 1]):
        k, v, q = _rows(seed, n, nkv, hd), _rows(seed + 1, n, nkv, hd), _normal(seed + 2, n, nq, hd)
        seed += 10
        a.append_dev(k.cuda(), v.cuda())
        wa[:, len(a) - n:len(a)] = 0
        out = torch.empty(n, nq, hd, device="cuda")
        a.attend_dev(q.cuda(), out, weights=wa)
        rk = ref.stored(k) if rk is None else torch.cat([rk, ref.stored(k)], 1)
        rv = ref.stored(v) if rv is None else torch.cat([rv, ref.stored(v)], 1)
        want, ww, bnd, wbnd = ref.attend(q, rk, rv)
        assert bool(((out.cpu().double() - want).abs() <= bnd + 2.0 ** -24 * want.abs()).all()), step
        length = len(a)
        if length > bound_rows:
            kept = torch.empty(nkv, bound_rows, dtype=torch.int32, device="cuda")
            a.evict_dev(b, bound_rows, 16, wa, wb, kept)
            # the choice is checked on the weights that the device holds
            assert torch.equal(kept.cpu(), ref.evict(wa[:, :length], bound_rows, 16)), step
            ii = kept.cpu().long()[..., None].expand(-1, -1, hd)
            rk, rv = torch.gather(rk, 1, ii), torch.gather(rv, 1, ii)
            a, b, wa, wb = b, a, wb, wa


def test_captured_calls_replay(dz):
    """Append, attend with weights, evict and read captured once, replayed with other inputs between eager work."""
    nq, nkv, hd = 6, 1, 256
    k, v = _rows(200, 600, nkv, hd).cuda(), _rows(201, 600, nkv, hd).cuda()
    c, dst = dz.Kv4Cache(nkv, hd, 700), dz.Kv4Cache(nkv, hd, 300)
    c.append_dev(k, v)
    nk, nv, q = torch.zeros(1, nkv, hd, device="cuda"), torch.zeros(1, nkv, hd, device="cuda"), torch.zeros(1, nq, hd, device="cuda")
    out, w = torch.empty_like(q), torch.zeros(nkv, 700, device="cuda")
    kept, dw = torch.empty(nkv, 300, dtype=torch.int32, device="cuda"), torch.empty(nkv, 300, device="cuda")
    rk, rv = (torch.empty(nkv, 300, hd, device="cuda") for _ in range(2))

    def step():
        c.truncate(600)
        c.append_dev(nk, nv)
        c.attend_dev(q, out, weights=w)
        c.evict_dev(dst, 300, 20, w, dw, kept)
        dst.read_dev(0, rk, rv)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        nk.copy_(_rows(300 + i, 1, nkv, hd))
        nv.copy_(_rows(310 + i, 1, nkv, hd))
        q.copy_(_normal(320 + i, 1, nq, hd))
        w.copy_(torch.rand(nkv, 700, generator=torch.Generator().manual_seed(i)))
        w0 = w.clone()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (out, w, kept, dw, rk, rv)]
        w.copy_(w0)
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (out, w, kept, dw, rk, rv))), i


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_captured_attention_of_many_rows(dz, dtype):
    """Two captured calls of many query rows, replayed at once on two streams, against the eager calls."""
    nq, nkv, hd, n, length = 8, 2, 128, 80, 900
    c = _cache(dz, _rows(210, length, nkv, hd), _rows(211, length, nkv, hd))
    q = [torch.zeros(n, nq, hd, dtype=TYPES[dtype], device="cuda") for _ in range(2)]
    out, w = [torch.empty_like(x) for x in q], [torch.zeros(nkv, length, device="cuda") for _ in range(2)]
    streams, graphs = [torch.cuda.Stream() for _ in range(2)], [torch.cuda.CUDAGraph() for _ in range(2)]
    for i in range(2):
        c.attend_dev(q[i], out[i], weights=w[i])
        torch.cuda.synchronize()
        with torch.cuda.graph(graphs[i]):
            c.attend_dev(q[i], out[i], weights=w[i])
    for r in range(3):
        for i in range(2):
            q[i].copy_(_normal(330 + 2 * r + i, n, nq, hd))
            w[i].zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            want, ww = torch.empty_like(q[i]), torch.zeros_like(w[i])
            c.attend_dev(q[i], want, weights=ww)
            torch.cuda.synchronize()
            assert torch.equal(out[i], want) and torch.equal(w[i], ww), (r, i)


def test_on_another_stream(dz):
    """Calls given a stream explicitly run there, in order, and their work memory outlives the call."""
    k, v = _rows(400, 500, 4, 256).cuda(), _rows(401, 500, 4, 256).cuda()
    q = _normal(402, 3, 24, 256).cuda()
    want = torch.empty_like(q)
    _c = dz.Kv4Cache(4, 256, 500)
    _c.append_dev(k, v)
    _c.attend_dev(q, want)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    c = dz.Kv4Cache(4, 256, 500)
    outs = [torch.zeros_like(q) for _ in range(8)]
    s.wait_stream(torch.cuda.current_stream())
    c.append_dev(k, v, stream=s)
    for o in outs:
        c.attend_dev(q, o, stream=s.cuda_stream)
        torch.full((1 << 18,), 5.0, device="cuda")  # the current stream's allocations must not take the call's memory
    s.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_work_memory_of_calls_without_weights(dz):
    """A call that adds to no weights has no use for its scores, 25 MB of a token's 24 heads at 262144 rows."""
    c = dz.Kv4Cache(4, 256, 262144)
    x = _rows(420, 40, 4, 256).cuda()
    c.append_dev(x, x)
    q = _normal(421, 1, 24, 256).cuda()
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    c.attend_dev(q, out)
    assert torch.cuda.max_memory_allocated() - before < 8 << 20


@pytest.mark.parametrize("nq,nkv,hd,length,n,dtype", [(24, 4, 256, 5000, 1, "f32"), (24, 4, 256, 2000, 2, "f32"), (6, 1, 256, 40, 3, "f32"),
                                                      (24, 4, 256, 900, 21, "f32"), (8, 2, 128, 3000, 80, "bf16"),
                                                      (8, 1, 64, 20000, 1, "f16"), (4, 4, 64, 600, 200, "f32")])
@pytest.mark.parametrize("weights", [False, True])
def test_work_memory_is_enough(dz, nq, nkv, hd, length, n, dtype, weights):
    """The sizes that the library gives hold what calls write: nothing behind them changes."""
    c = _cache(dz, _rows(422, length, nkv, hd), _rows(423, length, nkv, hd))
    q = _normal(424, n, nq, hd).to(TYPES[dtype]).cuda()
    want, out = torch.empty_like(q), torch.empty_like(q)
    ww, w = (torch.zeros(nkv, length, device="cuda") for _ in range(2))
    c.attend_dev(q, want, weights=ww if weights else None)
    L = dz.lib()
    size = (L.dz_kv4_attend_work_bytes if weights else L.dz_kv4_attend_only_work_bytes)(c._h, nq, n)
    work = torch.full((size + (1 << 24),), 0xA5, dtype=torch.uint8, device="cuda")
    rc = L.dz_kv4_attend_dev(c._h, q.data_ptr(), nq * hd, {"f32": 0, "f16": 1, "bf16": 30}[dtype], nq, n, hd ** -0.5,
                             w.data_ptr() if weights else None, length, out.data_ptr(), nq * hd, work.data_ptr(),
                             torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert rc == dz.DZ_OK and torch.equal(out, want) and torch.equal(w, ww if weights else torch.zeros_like(w))
    assert bool((work[size:] == 0xA5).all())


@pytest.mark.parametrize("handle", [False, True])
def test_work_memory_while_the_current_stream_is_busy(dz, handle):
    """A call on a stream of its own takes no block that queued work of the current stream still uses, though its tensor is gone."""
    k, v = _rows(410, 900, 4, 256), _rows(411, 900, 4, 256)
    c = _cache(dz, k, v)
    q = _normal(412, 2, 24, 256).cuda()
    x, tokens = (_normal(413, 4, 30000) * 3).cuda(), torch.tensor([1, 2, 3, 4], dtype=torch.int32, device="cuda")
    want, lwant = torch.empty_like(q), torch.empty(4, device="cuda")
    c.attend_dev(q, want)
    dz.logprobs_dev(x, tokens, lwant)
    got, lgot = torch.zeros_like(q), torch.zeros(4, device="cuda")
    sizes = (dz.lib().dz_kv4_attend_only_work_bytes(c._h, 24, 2), dz.lib().dz_logprobs_work_bytes(4, 30000, 0))
    s, big = torch.cuda.Stream(), torch.ones(1 << 27, device="cuda")
    for _ in range(3):
        got.zero_()
        lgot.zero_()
        torch.cuda.synchronize()
        for _ in range(40):  # some milliseconds
            big.mul_(1.0)
        kept = []
        for n in sizes:
            tmp = torch.full((n,), 7, dtype=torch.uint8, device="cuda")
            kept.append(tmp.clone())
            del tmp
        on = s.cuda_stream if handle else s
        c.attend_dev(q, got, stream=on)
        dz.logprobs_dev(x, tokens, lgot, stream=on)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(lgot, lwant)
        assert all(bool((t == 7).all()) for t in kept)


@pytest.mark.parametrize("handle", [False, True])
def test_captured_on_a_forked_stream(dz, handle):
    """A call given another stream of the capture, forked from the capturing one and joined again, replays with memory of the
    graph's own."""
    k, v = _rows(430, 900, 4, 256), _rows(431, 900, 4, 256)
    c = _cache(dz, k, v)
    q, x = torch.zeros(2, 24, 256, device="cuda"), torch.zeros(3, 30000, device="cuda")
    tokens = torch.tensor([5, 6, 7], dtype=torch.int32, device="cuda")
    out, w, lp = torch.empty_like(q), torch.zeros(4, 900, device="cuda"), torch.empty(3, device="cuda")
    ids, tl = torch.empty(3, 9, dtype=torch.int32, device="cuda"), torch.empty(3, 9, device="cuda")
    side = torch.cuda.Stream()

    def step(stream):
        c.attend_dev(q, out, weights=w, stream=stream)
        dz.logprobs_dev(x, tokens, lp, None, ids, tl, stream=stream)

    step(None)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        step(side.cuda_stream if handle else side)
        torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        q.copy_(_normal(440 + i, 2, 24, 256))
        x.copy_(_normal(450 + i, 3, 30000))
        w.zero_()
        junk = [torch.full((1 << 22,), 3.0, device="cuda") for _ in range(8)]  # whatever is free is written to
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (out, w, lp, ids, tl)]
        w.zero_()
        step(None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (out, w, lp, ids, tl))), i
        del junk


def test_two_caches_at_once(dz):
    """Two caches on two streams do not touch each other's work."""
    q = _normal(500, 2, 24, 256).cuda()
    caches, wants, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(2):
        c = _cache(dz, _rows(510 + i, 900 + i, 4, 256), _rows(520 + i, 900 + i, 4, 256))
        o = torch.empty_like(q)
        c.attend_dev(q, o)
        caches.append(c)
        wants.append(o)
    torch.cuda.synchronize()
    outs = [[torch.empty_like(q) for _ in range(6)] for _ in range(2)]
    for j in range(6):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                caches[i].attend_dev(q, outs[i][j])
    torch.cuda.synchronize()
    assert all(torch.equal(o, wants[i]) for i in range(2) for o in outs[i])


# ---------------------------------------------------------------- refusals


def test_refusals(dz):
    E = dz.DaizaError
    c = dz.Kv4Cache(2, 64, 10)
    x = torch.zeros(4, 2, 64, device="cuda")
    with pytest.raises(E):
        c.append_dev(x.double(), x.double())
    with pytest.raises(E):
        c.append_dev(x, x.half())
    with pytest.raises(E):
        c.append_dev(x, x[:3])
    with pytest.raises(E):
        c.append_dev(x.cpu(), x)
    with pytest.raises(E):
        c.append_dev(x.transpose(1, 2).contiguous().transpose(1, 2), x)
    with pytest.raises(E):
        c.append_dev(x[:1].expand(4, 2, 64), x)
    with pytest.raises(E, match="full"):
        c.append_dev(torch.zeros(11, 2, 64, device="cuda"), torch.zeros(11, 2, 64, device="cuda"))
    assert len(c) == 0
    q, out = torch.zeros(1, 4, 64, device="cuda"), torch.zeros(1, 4, 64, device="cuda")
    with pytest.raises(E):
        c.attend_dev(q, out)  # no rows
    c.append_dev(x, x)
    with pytest.raises(E):
        c.attend_dev(torch.zeros(5, 4, 64, device="cuda"), torch.zeros(5, 4, 64, device="cuda"))  # more queries than rows
    with pytest.raises(E):
        c.attend_dev(torch.zeros(1, 3, 64, device="cuda"), torch.zeros(1, 3, 64, device="cuda"))  # heads on kv heads
    with pytest.raises(E):
        c.attend_dev(q, out, weights=torch.zeros(2, 3, device="cuda"))
    with pytest.raises(E):
        c.attend_dev(q, out[:, :2])
    with pytest.raises(E):
        c.read_dev(2, torch.zeros(2, 3, 64, device="cuda"))
    with pytest.raises(E):
        c.read_dev(-1, torch.zeros(2, 1, 64, device="cuda"))
    with pytest.raises(E):
        c.truncate(-1)
    w, kept = torch.zeros(2, 4, device="cuda"), torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    with pytest.raises(E):
        c.evict_dev(c, 2, 1, w, None, kept)  # onto itself
    with pytest.raises(E):
        c.evict_dev(dz.Kv4Cache(2, 128, 10), 2, 1, w, None, kept)
    with pytest.raises(E):
        c.evict_dev(dz.Kv4Cache(2, 64, 1), 2, 1, w, None, kept)  # no room
    with pytest.raises(E):
        c.evict_dev(dz.Kv4Cache(2, 64, 10), 2, 3, w, None, kept)
    with pytest.raises(E):
        c.evict_dev(dz.Kv4Cache(2, 64, 10), 2, 1, w[:, :3], None, kept)
    with pytest.raises(E):
        c.evict_dev(dz.Kv4Cache(2, 64, 10), 2, 1, w, None, kept.long())
    # the C entries: host memory and null arrays
    L = dz.lib()
    host = torch.zeros(4, 2, 64)
    assert L.dz_kv4_append_dev(c._h, host.data_ptr(), 128, host.data_ptr(), 128, 0, 1, None) == dz.DZ_ERR_TENSOR
    assert L.dz_kv4_attend_dev(c._h, q.data_ptr(), 256, 0, 4, 1, 1.0, None, 0, out.data_ptr(), 256, None, None) == dz.DZ_ERR_MODEL
    assert L.dz_kv4_attend_dev(c._h, q.data_ptr(), 255, 0, 4, 1, 1.0, None, 0, out.data_ptr(), 256, x.data_ptr(), None) == dz.DZ_ERR_TENSOR
    assert L.dz_kv4_append_dev(c._h, x.data_ptr(), 128, x.data_ptr(), 128, 5, 1, None) == dz.DZ_ERR_UNSUPPORTED
    assert L.dz_kv4_append_dev(c._h, x.data_ptr() + 2, 128, x.data_ptr(), 128, 0, 1, None) == dz.DZ_ERR_TENSOR
    assert len(c) == 4
