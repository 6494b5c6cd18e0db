"""Log probabilities of given tokens, entropies and alternatives against the same in 64 bits (kv4_ref.py)."""
import math

import pytest
import torch

import kv4_ref as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _run(dz, x, tokens, top, **kw):
    n = x.shape[0]
    lp, ent = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    ids, tl = torch.empty(n, top, dtype=torch.int32, device="cuda"), torch.empty(n, top, device="cuda")
    dz.logprobs_dev(x, tokens.cuda(), lp, ent, ids, tl, **kw)
    return lp.cpu().double(), ent.cpu().double(), ids.cpu(), tl.cpu().double()


def _close(a, b, bound):
    assert torch.equal(torch.isnan(a), torch.isnan(b))
    same = a.nan_to_num() == b.nan_to_num()
    assert bool((same | ((a - b).abs() <= bound) | torch.isnan(a)).all()), ((a - b).abs() / bound).nan_to_num().max()


def _check(dz, x, tokens, top):
    lp, ent, ids, tl = _run(dz, x.cuda() if not x.is_cuda else x, tokens, top)
    wl, we, wi, wt, lb, eb, tb = ref.logprobs(x, tokens, top)
    assert torch.equal(ids, wi)
    _close(lp, wl, lb)
    _close(ent, we, eb)
    _close(tl, wt, tb)


def _logits(seed, n, vocab, dtype="f32", spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, vocab, generator=g) * spread).to(TYPES[dtype]), torch.randint(0, vocab, (n,), generator=g).to(torch.int32)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,vocab,top", [(1, 1, 1), (1, 2, 2), (3, 63, 5), (2, 64, 64), (5, 257, 20), (1, 1000, 0), (7, 4095, 64), (2, 4097, 33),
                                         (1, 20000, 20), (300, 517, 3), (2000, 130, 1)])
def test_against_64_bits(dz, dtype, n, vocab, top):
    _check(dz, *_logits(n + vocab, n, vocab, dtype), top)


def test_the_27b_vocabulary(dz):
    _check(dz, *_logits(1, 3, 248320), 20)
    _check(dz, *_logits(2, 1, 248320, "bf16"), 64)


@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "two", "zeros", "runs"])
@pytest.mark.parametrize("vocab,n", [(9000, 2), (9000, 300), (300, 2)])
def test_orders_and_ties(dz, kind, vocab, n):
    """Rows in which every value ties, keeps rising past all before it, or falls; ties go to the lowest id."""
    i = torch.arange(vocab, dtype=torch.float32)
    x = {"equal": torch.full((vocab,), 0.5), "rising": i * 1e-3, "falling": -i * 1e-3, "two": (i % 2) * 2.0,
         "zeros": torch.where(i % 3 == 0, -0.0, 0.0), "runs": torch.floor(i / 100) * 0.25}[kind]
    x = x.repeat(n, 1)
    x[0] = x[0].roll(17)
    _check(dz, x, torch.arange(n, dtype=torch.int32) % vocab, 40)


def test_masked_and_non_finite(dz):
    x, tokens = _logits(3, 8, 5000)
    x[0, 100:] = -math.inf                        # most of the vocabulary masked
    x[1] = -math.inf                              # all of it
    x[2] = -math.inf
    x[2, 4321] = 5.0                              # all but one
    x[3, 7] = math.nan
    x[4, 7] = math.inf
    x[5, 5:4000] = torch.finfo(torch.float32).min  # the type's lowest value as a mask
    x[6] = torch.finfo(torch.float32).min
    x[7, ::2] = 3e38
    tokens[0], tokens[2] = 50, 4321
    _check(dz, x, tokens, 12)
    y = x[0:1].clone()
    tokens = torch.tensor([200], dtype=torch.int32)  # a masked token
    lp, _, _, _ = _run(dz, y.cuda(), tokens, 0)
    assert lp.item() == -math.inf


def test_tokens_outside_the_vocabulary(dz):
    x, _ = _logits(4, 4, 100)
    lp, ent, _, _ = _run(dz, x.cuda(), torch.tensor([-1, 100, 99, 2 ** 31 - 1], dtype=torch.int32), 0)
    assert torch.isnan(lp).tolist() == [True, True, False, True] and bool(torch.isfinite(ent).all())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("off", [0, 1, 3])
def test_strided_rows(dz, dtype, off):
    x, tokens = _logits(5, 9, 777, dtype)
    wide = torch.full((9, 777 + 8), 50.0).to(TYPES[dtype])
    wide[:, off:off + 777] = x
    d = wide.cuda()[:, off:off + 777]
    assert d.stride(0) == 785
    _check(dz, d, tokens, 9)


def test_outputs_left_out(dz):
    x, tokens = _logits(6, 5, 3333)
    d = x.cuda()
    full = _run(dz, d, tokens, 4)
    lp = torch.empty(5, device="cuda")
    dz.logprobs_dev(d, tokens.cuda(), lp)
    assert torch.equal(lp.cpu().double(), full[0])
    ent = torch.empty(5, device="cuda")
    dz.logprobs_dev(d, entropy=ent)
    assert torch.equal(ent.cpu().double(), full[1])
    ids = torch.empty(5, 4, dtype=torch.int32, device="cuda")
    dz.logprobs_dev(d, top_ids=ids)
    assert torch.equal(ids.cpu(), full[2])
    dz.logprobs_dev(d[:0], top_ids=ids[:0])


def test_captured_and_on_two_streams(dz):
    x, tokens = _logits(7, 2, 30000)
    d, t = x.cuda(), tokens.cuda()
    out = [torch.empty(2, device="cuda"), torch.empty(2, device="cuda"), torch.empty(2, 20, dtype=torch.int32, device="cuda"),
           torch.empty(2, 20, device="cuda")]
    dz.logprobs_dev(d, t, *out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dz.logprobs_dev(d, t, *out)
    for i in range(4):
        d.copy_(_logits(20 + i, 2, 30000)[0])
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        dz.logprobs_dev(d, t, *out)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, out)), i
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[torch.empty_like(o) for o in out] for _ in range(8)]
    for i, o in enumerate(outs):
        s[i % 2].wait_stream(torch.cuda.current_stream())
        dz.logprobs_dev(d, t, *o, stream=s[i % 2])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, out))


def test_refusals(dz):
    E = dz.DaizaError
    x, tokens = _logits(8, 3, 70)
    d, t = x.cuda(), tokens.cuda()
    lp = torch.empty(3, device="cuda")
    for bad in (lambda: dz.logprobs_dev(x, t, lp), lambda: dz.logprobs_dev(d.double(), t, lp), lambda: dz.logprobs_dev(d, t.long(), lp),
                lambda: dz.logprobs_dev(d, t[:2], lp), lambda: dz.logprobs_dev(d, None, lp), lambda: dz.logprobs_dev(d.t(), t, lp),
                lambda: dz.logprobs_dev(d[:1].expand(3, 70), t, lp),
                lambda: dz.logprobs_dev(d, top_ids=torch.empty(3, 65, dtype=torch.int32, device="cuda")),
                lambda: dz.logprobs_dev(d[:, :4], top_ids=torch.empty(3, 5, dtype=torch.int32, device="cuda")),
                lambda: dz.logprobs_dev(d, t, lp.cpu())):
        with pytest.raises(E):
            bad()
    L = dz.lib()
    assert L.dz_logprobs_dev(x.data_ptr(), 70, 0, 3, 70, t.data_ptr(), 0, lp.data_ptr(), None, None, None, d.data_ptr(), None) == dz.DZ_ERR_TENSOR
    assert L.dz_logprobs_dev(d.data_ptr(), 70, 0, 3, 70, t.data_ptr(), 0, lp.data_ptr(), None, None, None, None, None) == dz.DZ_ERR_MODEL
