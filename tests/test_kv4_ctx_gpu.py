"""Contexts whose key/value cache is held in 4 bits, against the float64 decoder (npref.py) attending to the rows that the
device holds: prefill, single tokens, verify and commit, eviction by the weights that the forwards summed, and the state calls."""
import numpy as np
import pytest
import torch

import kv4_ref as ref
from conftest import normwise_rel
from npref import K_ATT_K, K_ATT_KNORM, K_ATT_O, K_ATT_Q, K_ATT_QNORM, K_ATT_V, K_ATTN_NORM, NpDecoder, rmsnorm, rope_quirk, sigmoid

pytestmark = pytest.mark.gpu

SEED = 0xDA1A0031
BAR = 1e-4  # normwise, of logits whose own f32 rounding the other tests hold to 2e-5 a layer


class Kv4Decoder(NpDecoder):
    """NpDecoder whose attention reads the rows that a device context holds, and sums the weights that they receive."""

    def __init__(self, om, cfg, seed):
        super().__init__(om, cfg, seed)
        self.held = 0  # rows before the current token's
        self.w = {l: np.zeros((cfg.n_head_kv, 0)) for l in self.K}
        self.sum_weights = True
        self.own = {}  # layer -> the rows that this decoder itself would store

    def take_rows(self, ctx, n):
        """The first n rows of every attention layer of ctx."""
        for l in self.K:
            k, v = ctx.get_kv(l, n)
            self.K[l], self.V[l] = k.astype(np.float64), v.astype(np.float64)
            have = self.w[l].shape[1]
            if have < n:
                self.w[l] = np.concatenate([self.w[l], np.zeros((self.c.n_head_kv, n - have))], 1)

    def attention(self, l, h, cs):
        c = self.c
        hd, nq, nkv = c.head_dim, c.n_head, c.n_head_kv
        grp = nq // nkv
        n = rmsnorm(h, self.v(K_ATTN_NORM, l), c.rms_eps)
        qg = (self.W(K_ATT_Q, l) @ n).reshape(nq, 2, hd)
        k = (self.W(K_ATT_K, l) @ n).reshape(nkv, hd)
        v = (self.W(K_ATT_V, l) @ n).reshape(nkv, hd)
        qn, kn = self.v(K_ATT_QNORM, l), self.v(K_ATT_KNORM, l)
        q = np.stack([rope_quirk(rmsnorm(qg[i, 0], qn, c.rms_eps), *cs) for i in range(nq)]) / np.sqrt(hd)
        self.own[l] = (np.stack([rope_quirk(rmsnorm(k[i], kn, c.rms_eps), *cs) for i in range(nkv)]), v)
        o = np.zeros((nq, hd))
        seen = self.held + 1
        for qh in range(nq):
            g = qh // grp
            sc = self.K[l][g][:seen] @ q[qh]
            p = np.exp(sc - sc.max())
            p /= p.sum()
            if self.sum_weights:
                self.w[l][g][:seen] += p
            o[qh] = p @ self.V[l][g][:seen]
        o = o * sigmoid(qg[:, 1])
        return h + self.W(K_ATT_O, l) @ o.reshape(-1)

    def token(self, t):
        out = self.forward(int(t))
        self.held += 1
        return out


def _setup(dz, oracle, track=True, kv_rows=0, **kw):
    cfg = dz.Config.small(**{"n_layers": 4, "max_ctx": 256, "vocab": 512, **kw})
    om = oracle.Model(cfg, SEED)
    model = dz.Model.synthetic(cfg, SEED)
    return cfg, om, model, dz.Context(model, kv4=True, kv_rows=kv_rows, track=track)


def _attn(cfg):
    return [i for i in range(cfg.n_layers) if cfg.is_full_attention(i)]


def _check_own_rows(d, layer, row):
    """The row that the device stored is the one that the decoder would store, but for values next to a border."""
    k, v = d.own[layer]
    for mine, held in ((k, d.K[layer][:, row]), (v, d.V[layer][:, row])):
        want = ref.stored(torch.from_numpy(mine[None]))[:, 0].numpy()
        assert (want != held).mean() < 0.02
        # a neighbouring code: at most two of the block's steps, a step being half the least and a third of the largest
        top = np.abs(held.reshape(held.shape[0], -1, 32)).max(-1, keepdims=True)
        assert (np.abs(want - held).reshape(*top.shape[:2], 32) <= top).all()


def _batch(ctx, d, ids):
    got = ctx.forward_batch(ids, per_pos_logits=True)
    d.take_rows(ctx, d.held + len(ids))
    for i, t in enumerate(ids):
        assert normwise_rel(got[i], d.token(t)) < BAR, i
        for l in d.K:
            _check_own_rows(d, l, d.held - 1)


def _single(ctx, d, t):
    am, got = ctx.forward_single_token(int(t))
    d.take_rows(ctx, d.held + 1)
    want = d.token(t)
    assert normwise_rel(got, want) < BAR and am == int(np.argmax(got))
    for l in d.K:
        _check_own_rows(d, l, d.held - 1)


def test_prefill_tokens_verify(dz, oracle):
    cfg, om, model, ctx = _setup(dz, oracle)
    assert not ctx.token_kernel
    d = Kv4Decoder(om, cfg, SEED)
    rng = np.random.default_rng(1)
    ids = rng.integers(0, cfg.vocab, 100)
    _batch(ctx, d, ids[:40])          # the chunked delta rule, several row tiles
    for t in ids[40:43]:
        _single(ctx, d, t)
    _batch(ctx, d, ids[43:48])        # few tokens
    # five drafts of which two are kept
    got = ctx.verify_forward(ids[48:53])
    before = {l: d.w[l].copy() for l in d.w}
    d.take_rows(ctx, d.held + 5)
    d.sum_weights = False
    save = {l: d.S[l].copy() for l in d.S}, {l: d.ring[l].copy() for l in d.ring}, dict(d.head), d.pos, d.held
    for i, t in enumerate(ids[48:53]):
        assert normwise_rel(got[i], d.token(t)) < BAR, i
    d.S, d.ring, d.head, d.pos, d.held = save
    for t in ids[48:50]:
        d.token(t)
    d.sum_weights = True
    d.w = before
    ctx.verify_commit(2)
    assert ctx.pos == 50 and ctx.kv_len(_attn(cfg)[0]) == 50
    _single(ctx, d, ids[50])
    for l in _attn(cfg):
        w = ctx.kv_weights(l)
        assert w.shape == (cfg.n_head_kv, 51)
        # a weight sums up to 51 x 2 probabilities of attentions that agree to the bar
        assert np.abs(w - d.w[l][:, :51]).max() < 51 * 2 * BAR


def test_rows_are_the_f32_contexts_rounded(dz, oracle):
    """In the first layer the inputs are the same: the rows of an f32 context, each block rounded to its 4-bit values."""
    cfg, om, model, ctx = _setup(dz, oracle, n_layers=1, full_attn_interval=1, max_ctx=80)
    plain = dz.Context(model)
    ids = np.random.default_rng(2).integers(0, cfg.vocab, 70)
    plain.forward_batch(ids)
    ctx.forward_batch(ids)
    for a, b in zip(plain.get_kv(0, 70), ctx.get_kv(0, 70)):
        want = ref.stored(torch.from_numpy(a).permute(1, 0, 2)).numpy()
        assert np.array_equal(want, b.astype(np.float64))


def test_evict_and_go_on(dz, oracle):
    """A context that runs past its cache's rows by evicting, positions going on."""
    cfg, om, model, ctx = _setup(dz, oracle, kv_rows=50)
    attn = _attn(cfg)
    d = Kv4Decoder(om, cfg, SEED)
    rng = np.random.default_rng(3)
    ids = rng.integers(0, cfg.vocab, 160)
    at = 0
    for n, keep, recent in ((44, 20, 6), (25, 20, 0), (20, 39, 39), (9, 16, 16), (30, 100, 5)):
        _batch(ctx, d, ids[at:at + n])
        at += n
        rows = ctx.kv_len(attn[0])
        assert rows == d.held
        before = {l: (ctx.kv_weights(l), ctx.get_kv(l, rows)) for l in attn}
        for l in attn:
            assert np.abs(before[l][0] - d.w[l][:, :rows]).max() < 2 * at * BAR
        kept = ctx.kv_evict(keep, recent)
        m = min(keep, rows)
        assert kept.shape == (len(attn), cfg.n_head_kv, m) and ctx.kv_len(attn[0]) == m and ctx.pos == at
        for i, l in enumerate(attn):
            w, kv = before[l]
            assert np.array_equal(kept[i], ref.evict(torch.from_numpy(w), keep, recent).numpy())
            assert np.array_equal(ctx.kv_weights(l), np.take_along_axis(w, kept[i], 1))
            for a, b in zip(kv, ctx.get_kv(l, m)):
                assert np.array_equal(b, np.take_along_axis(a, kept[i][:, :, None], 1))
            d.w[l] = np.take_along_axis(d.w[l], kept[i].astype(np.int64), 1)
        d.held = m
        _single(ctx, d, ids[at])
        at += 1


def test_full_and_going_back(dz, oracle, tmp_path):
    cfg, om, model, ctx = _setup(dz, oracle, kv_rows=40)
    E = dz.DaizaError
    ids = np.random.default_rng(4).integers(0, cfg.vocab, 60)
    with pytest.raises(E, match="full"):
        ctx.forward_batch(ids[:41])
    ctx.forward_batch(ids[:40])
    for call in (lambda: ctx.forward_single_token(1), lambda: ctx.verify_forward(ids[:1]), lambda: ctx.decode_greedy(1, 1),
                 lambda: ctx.forward_logprobs(ids[:1]), lambda: ctx.mixer_step(_attn(cfg)[0], np.zeros(cfg.hidden))):
        with pytest.raises(E, match="full"):
            call()
    assert ctx.pos == 40
    ctx.kv_truncate(30)
    ctx.forward_batch(ids[40:45])
    ctx.save(str(tmp_path / "s"))
    ctx.kv_evict(20, 5)
    assert ctx.pos == 35 and ctx.kv_len(_attn(cfg)[0]) == 20
    ctx.forward_batch(ids[45:50])
    ctx.kv_truncate(36)
    with pytest.raises(E, match="eviction"):
        ctx.kv_truncate(34)
    with pytest.raises(E, match="eviction"):
        ctx.set_pos(10)
    with pytest.raises(E):
        ctx.set_pos(56)  # 41 rows
    with pytest.raises(E):
        ctx.save(str(tmp_path / "t"))
    with pytest.raises(E):
        ctx.kv_evict(3, 4)
    with pytest.raises(E):
        ctx.set_kv(_attn(cfg)[0], *(np.zeros((cfg.n_head_kv, 41, 256), np.float32) for _ in range(2)))
    a = ctx.logits()
    ctx.reset()
    assert ctx.pos == 0 and ctx.kv_len(_attn(cfg)[0]) == 0
    ctx.load(str(tmp_path / "s"))
    assert ctx.pos == 35
    small = dz.Context(model, kv4=True, kv_rows=34, track=True)
    with pytest.raises(E):
        small.load(str(tmp_path / "s"))
    plain = dz.Context(model, kv4=True)
    with pytest.raises(E):
        plain.kv_evict(3, 1)
    with pytest.raises(E):
        plain.kv_weights(_attn(cfg)[0])
    with pytest.raises(E):
        plain.copy_state_from(ctx)
    with pytest.raises(E):
        dz.Context(model).copy_state_from(ctx)
    with pytest.raises(E):
        dz.Context(model).kv_evict(3, 1)
    with pytest.raises(E):
        dz.Context(model, kv4=True, kv_rows=cfg.max_ctx + 1)
    assert np.isfinite(a).all()


def test_state_calls(dz, oracle, tmp_path):
    """copy_state, save and load, set and get of rows: a context that goes on from them gives the same logits, bit for bit."""
    cfg, om, model, a = _setup(dz, oracle)
    rng = np.random.default_rng(5)
    ids = rng.integers(0, cfg.vocab, 90)
    a.forward_batch(ids[:70])
    a.kv_evict(50, 10)
    b = dz.Context(model, kv4=True, kv_rows=64, track=True)
    b.forward_batch(ids[:33])
    b.copy_state_from(a)
    assert b.pos == 70 and b.kv_len(_attn(cfg)[0]) == 50
    la, lb = a.forward_batch(ids[70:77]), b.forward_batch(ids[70:77])
    assert np.array_equal(la, lb)
    for l in _attn(cfg):
        assert np.array_equal(a.kv_weights(l), b.kv_weights(l))
    assert np.array_equal(a.kv_evict(30, 4), b.kv_evict(30, 4))
    assert np.array_equal(a.forward_single_token(3)[1], b.forward_single_token(3)[1])
    c = dz.Context(model, kv4=True)
    c.forward_batch(ids[:60])
    c.save(str(tmp_path / "s"), history=ids[:60])
    e = dz.Context(model, kv4=True, kv_rows=100)
    hist, _, _ = e.load(str(tmp_path / "s"))
    assert np.array_equal(hist, ids[:60])
    assert np.array_equal(c.forward_batch(ids[60:70], per_pos_logits=True), e.forward_batch(ids[60:70], per_pos_logits=True))
    # an f32 context takes the file too, with the values that the rows stand for
    f = dz.Context(model)
    f.load(str(tmp_path / "s"))
    l = _attn(cfg)[0]
    assert all(np.array_equal(x, y) for x, y in zip(f.get_kv(l, 60), c.get_kv(l, 60)))


def test_token_loop(dz, oracle):
    """The greedy and sampled loops and the layer step on a 4-bit context follow its single tokens."""
    cfg, om, model, a = _setup(dz, oracle, track=False)
    b = dz.Context(model, kv4=True)
    ids = np.random.default_rng(6).integers(0, cfg.vocab, 20)
    first = int(np.argmax(a.forward_batch(ids)))
    b.forward_batch(ids)
    toks = a.decode_greedy(first, 8)
    t = first
    for i in range(8):
        am, lg = b.forward_single_token(t)
        assert am == toks[i], i
        t = am
    assert np.array_equal(a.logits(), b.logits())
    ra, rb = dz.LcgRng(7), dz.LcgRng(7)
    sp = dz.SamplingParams(0.9, 10, 0.9)
    drawn = a.decode_sample(5, 6, sp, ra)
    t = 5
    for i in range(6):
        t = dz.sample_top_k_top_p(b.forward_single_token(t)[1], sp, rb)
        assert t == drawn[i], i
    layer = _attn(cfg)[0]
    h = np.random.default_rng(8).standard_normal(cfg.hidden).astype(np.float32) * 0.1
    assert np.array_equal(a.mixer_step(layer, h), b.mixer_step(layer, h)) and a.pos == b.pos


@pytest.mark.parametrize("kv4", [False, True])
def test_log_probabilities_of_a_prompt(dz, oracle, kv4):
    """forward_logprobs against the log softmax of the same forward's logits (both take up to 128 tokens at once)."""
    cfg, om, model, a = _setup(dz, oracle, track=False)
    make = (lambda: dz.Context(model, kv4=True)) if kv4 else (lambda: dz.Context(model))
    a, b = make(), make()
    rng = np.random.default_rng(9)
    ids = rng.integers(0, cfg.vocab, 150)
    targets = np.append(ids[1:], -1).astype(np.int32)
    for i0, n in ((0, 1), (1, 100), (101, 49)):
        lg = a.forward_batch(ids[i0:i0 + n], per_pos_logits=True)
        logp, ent, tid, tlp = b.forward_logprobs(ids[i0:i0 + n], targets[i0:i0 + n], top=7)
        t = torch.from_numpy(targets[i0:i0 + n])
        wl, we, wi, wt, lb, eb, tb = ref.logprobs(torch.from_numpy(lg), t, 7)
        assert np.array_equal(tid, wi.numpy())
        fin = t >= 0
        assert bool(((torch.from_numpy(logp).double() - wl).abs() <= lb)[fin].all()) and bool(np.isnan(logp[~fin.numpy()]).all())
        assert bool(((torch.from_numpy(ent).double() - we).abs() <= eb).all())
        assert bool(((torch.from_numpy(tlp).double() - wt).abs() <= tb).all())
        assert b.pos == i0 + n
        one = b.logprobs(int(tid[-1, 2]), top=7)
        assert one[0] == tlp[-1, 2] and one[1] == ent[-1] and np.array_equal(one[2], tid[-1]) and np.array_equal(one[3], tlp[-1])
    assert np.array_equal(a.logits(), b.logits())
    logp, ent, tid, tlp = make().forward_logprobs(ids[:5])
    assert logp is None and ent.shape == (5,) and tid.shape == (5, 0)
    E = dz.DaizaError
    with pytest.raises(E):
        b.forward_logprobs(ids[:2], targets[:1])
    with pytest.raises(E):
        b.forward_logprobs(ids[:2], top=65)
    with pytest.raises(E):
        b.forward_logprobs([cfg.vocab])
    with pytest.raises(E):
        b.forward_logprobs([])
    with pytest.raises(E):
        b.logprobs(top=-1)
    assert b.pos == 150


def test_log_probabilities_over_chunks(dz, oracle):
    """A prompt longer than one forward's 1024 tokens is scored as its parts are."""
    cfg, om, model, a = _setup(dz, oracle, track=False, max_ctx=1100)
    b = dz.Context(model, kv4=True)
    ids = np.random.default_rng(11).integers(0, cfg.vocab, 1051)
    whole = a.forward_logprobs(ids[:1050], ids[1:], top=3)
    parts = [b.forward_logprobs(ids[i:j], ids[i + 1:j + 1], top=3) for i, j in ((0, 1024), (1024, 1050))]
    for w, p in zip(whole, zip(*parts)):
        assert np.array_equal(w, np.concatenate(p)) and np.isfinite(w).all()
    assert a.pos == b.pos == 1050 and np.array_equal(a.logits(), b.logits())


def test_non_finite_row_of_a_context(dz, oracle):
    """set_kv with a NaN in one value: the outputs become NaN, and truncating before the row makes them whole again."""
    cfg, om, model, a = _setup(dz, oracle, track=False, n_layers=1, full_attn_interval=1)
    rng = np.random.default_rng(10)
    k, v = (rng.standard_normal((cfg.n_head_kv, 50, 256)).astype(np.float32) for _ in range(2))
    a.set_kv(0, k, v)
    a.set_pos(40)
    want = a.forward_single_token(3)[1]
    v[0, 45, 9] = np.nan
    a.set_pos(0)
    a.set_kv(0, k, v)
    a.set_pos(50)
    assert np.isnan(a.forward_single_token(3)[1]).all()
    a.kv_truncate(40)
    assert np.array_equal(a.forward_single_token(3)[1], want)


@pytest.mark.parametrize("k,a", [(5, 2), (3, 2), (1, 1), (8, 8), (4, 0), (40, 30)])
def test_accepted_drafts_count_in_the_weights(dz, oracle, k, a):
    """track=2: verify and commit leave the weights that a forward of the accepted drafts alone leaves, and the same eviction."""
    cfg, om, model, x = _setup(dz, oracle, track=2, kv_rows=150)
    y = dz.Context(model, kv4=True, kv_rows=150, track=True)
    ids = np.random.default_rng(20).integers(0, cfg.vocab, 100)
    x.forward_batch(ids[:50])
    x.kv_evict(40, 8)  # rows and positions differ
    y.copy_state_from(x)
    before = {l: x.kv_weights(l) for l in _attn(cfg)}
    x.verify_forward(ids[50:50 + k])
    for l in _attn(cfg):
        assert np.array_equal(x.kv_weights(l), before[l])
    x.verify_commit(a)
    if a:
        y.forward_batch(ids[50:50 + a])
    assert x.pos == y.pos == 50 + a
    for l in _attn(cfg):
        wx, wy = x.kv_weights(l), y.kv_weights(l)
        assert wx.shape == wy.shape == (cfg.n_head_kv, 40 + a)
        # sums of a x (heads of a group) probabilities of attentions that agree to the bar
        assert np.abs(wx - wy).max() <= a * (cfg.n_head // cfg.n_head_kv) * BAR
        total = a * cfg.n_head // cfg.n_head_kv
        assert np.allclose(wx.sum(1) - before[l].sum(1), total, atol=1e-4 * max(1, total))
    # k and a tokens take their products in forms that round in other orders
    assert normwise_rel(x.forward_single_token(3)[1], y.forward_single_token(3)[1]) < BAR
    z = dz.Context(model, kv4=True, kv_rows=150, track=True)  # without it the commit adds none
    z.forward_batch(ids[:50])
    z.verify_forward(ids[50:50 + k])
    w = {l: z.kv_weights(l) for l in _attn(cfg)}
    z.verify_commit(a)
    for l in _attn(cfg):
        assert np.array_equal(z.kv_weights(l)[:, :50], w[l]) and not z.kv_weights(l)[:, 50:].any()


def test_speculative_steps_count_in_the_weights(dz, oracle):
    """dz_spec_verify on a track=2 context: every forwarded token's attention is in the weights once."""
    cfg, om, model, x = _setup(dz, oracle, track=2)
    ids = np.random.default_rng(21).integers(0, cfg.vocab, 30)
    t = int(np.argmax(x.forward_batch(ids)))
    y = dz.Context(model, kv4=True)
    y.forward_batch(ids)
    greedy = y.decode_greedy(t, 6)
    draft = np.append([t], greedy[:3]).astype(np.uint32)
    draft[-1] = (draft[-1] + 1) % cfg.vocab  # three right ones and a wrong one
    n, bonus = x.spec_verify(draft, None, dz.SamplingParams(0.0, 0, 1.0), dz.LcgRng(1))[:2]
    assert n == 3 and bonus == greedy[2] and x.pos == 33
    grp = cfg.n_head // cfg.n_head_kv
    for l in _attn(cfg):
        assert np.allclose(x.kv_weights(l).sum(1), 33 * grp, atol=1e-4 * 33 * grp)


def test_weights_after_going_back(dz, oracle):
    """What dropped tokens gave stays in the rows that remain; forwarded again, they give it again and their rows start from 0."""
    cfg, om, model, x = _setup(dz, oracle, n_layers=1, full_attn_interval=1)
    ids = np.random.default_rng(22).integers(0, cfg.vocab, 52)
    x.forward_batch(ids[:40])
    w0 = x.kv_weights(0)
    x.forward_batch(ids[40:])
    w1 = x.kv_weights(0)
    x.kv_truncate(40)
    assert np.array_equal(x.kv_weights(0), w1[:, :40])
    x.forward_batch(ids[40:])
    w2 = x.kv_weights(0)
    # an attention layer alone: the same tokens at the same positions give the same; two f32 additions of sums up to 52 x group
    assert np.allclose(w2[:, :40] - w1[:, :40], w1[:, :40] - w0, atol=2 * 52 * (cfg.n_head // cfg.n_head_kv) * 2.0 ** -24)
    assert np.array_equal(w2[:, 40:], w1[:, 40:])


def test_a_token_allocates_nothing(dz, oracle):
    """The work memory of a token's attention, which keeps its scores for the weights (16 MB here), is there before the first
    token: a failed allocation between its layers would leave some of them a token ahead."""
    shape = dict(n_layers=2, full_attn_interval=2, max_ctx=1 << 20, rope_dim=16)
    cfg, om, model, small = _setup(dz, oracle, kv_rows=64, **shape)
    ctx = dz.Context(model, kv4=True, track=True)
    for layer in range(2):  # what the runtime keeps for the kernels' first launches
        small.mixer_step(layer, np.zeros(cfg.hidden, np.float32))
    small.reset()
    small.forward_single_token(3)
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    ctx.forward_single_token(3)
    ctx.decode_greedy(5, 3)
    ctx.mixer_step(1, np.zeros(cfg.hidden, np.float32))
    torch.cuda.synchronize()
    assert torch.cuda.mem_get_info()[0] == before


def test_small_caches_and_empty_evictions(dz, oracle):
    """One row at a time, evictions that leave nothing or take nothing, and going on after each."""
    cfg, om, model, x = _setup(dz, oracle, kv_rows=1)
    a, n = _attn(cfg)[0], cfg.n_head // cfg.n_head_kv
    lg = x.forward_single_token(3)[1]
    assert np.allclose(x.kv_weights(a), n, atol=n * 2.0 ** -22)
    with pytest.raises(dz.DaizaError, match="full"):
        x.forward_single_token(4)
    assert x.kv_evict(1, 1).tolist() == [[[0]] * cfg.n_head_kv] * len(_attn(cfg))  # all stay
    assert x.kv_evict(0, 0).shape == (len(_attn(cfg)), cfg.n_head_kv, 0) and x.kv_len(a) == 0 and x.pos == 1
    for t in (4, 5, 6):  # each token sees itself alone
        x.forward_single_token(t)
        assert np.allclose(x.kv_weights(a), n, atol=n * 2.0 ** -22) and x.kv_len(a) == 1
        x.kv_evict(0, 0)
    assert x.pos == 4
    x.reset()
    assert np.array_equal(x.forward_single_token(3)[1], lg)
