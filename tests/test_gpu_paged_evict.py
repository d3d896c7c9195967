"""Keys that are weighed, chosen and evicted (paged.weights, choose, evict, PagedKVCache.weigh and evict)
against tests/shared_oracle.py."""
import random

import numpy as np
import pytest
import torch

from polyhedral_amd import paged
from polyhedral_amd.polyattn import masks as pm
from polyhedral_amd.spec import MaskSpec
from tests import paged_oracle as po
from tests import shared_oracle as so
from tests.test_gpu_paged import RAGGED, TYPES, Batch
from tests.test_gpu_paged_shared import MASKS, dev, f64, falling, host

pytestmark = pytest.mark.gpu

I32 = torch.int32
NAN, INF = float("nan"), float("inf")


# ---- weights ---------------------------------------------------------------------------------------
def _weigh(b, mask, first=None, scale=None, max_fresh=None, lse=None, seed=0, pad=5):
    """Scores of a Batch's step against float64; the rows of scores lie apart."""
    spec = paged._paged_mask(mask).spec
    g = torch.Generator().manual_seed(seed)
    wide = torch.rand(b.pages, b.Hkv, b.P + pad, generator=g).to(b.gpu)
    scores = wide[:, :, :b.P]
    t, n, s = b.dev()
    if lse is None:
        lse = torch.empty(b.T, b.Hq, device=b.gpu)
        paged.attention(b.q, b.k, b.v, t, n, s, mask, scale, lse=lse)
    lse[int(b.n.sum()):] = NAN       # (rows of no request)
    f = np.zeros(len(b.n), dtype=int) if first is None else first
    old = wide.clone()
    want, bound = so.weights(f64(b.q), f64(b.k), b.tables, b.lengths, b.q_start, f64(lse), f64(scores), spec.live,
                             b.D ** -0.5 if scale is None else scale, f)
    # the new tokens' scores start from 0, whatever is there
    for r, (L, m) in enumerate(zip(b.lengths, b.n)):
        p = np.arange(max(L - m, f[r]), L)
        page = b.tables[r, p // b.P]
        ok = (page >= 0) & (page < b.pages)
        scores[torch.as_tensor(page[ok], device=b.gpu), :, torch.as_tensor((p % b.P)[ok], device=b.gpu)] = NAN
    got = paged.weights(b.q, b.k, t, n, s, lse, scores, mask, scale, None if first is None else dev(first, b.gpu), max_fresh)
    torch.cuda.synchronize()
    assert got is scores and torch.equal(wide[:, :, b.P:], old[:, :, b.P:])
    off = np.abs(f64(scores) - want)
    over = ~(off <= bound)
    assert not over.any(), f"{int(over.sum())} over the bound, first at {np.argwhere(over)[0]}: {off[over][0]:.3e} > {bound[over][0]:.3e}"
    return scores


@pytest.mark.parametrize("P", [16, 64, 256])
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 2), (3, 1), (16, 1), (20, 1)])
@pytest.mark.parametrize("dtype,D", TYPES)
def test_weights_of_a_ragged_batch(gpu, dtype, D, Hq, Hkv, P):
    b = Batch(gpu, dtype, D, P, Hq, Hkv, RAGGED, seed=P + Hq)
    _weigh(b, pm.Causal())
    _weigh(b, pm.Causal(), first=np.array([0, 1, 5, 3, 16, 9, 40, 17, -4, 0, 4, 128, 100]), max_fresh=1)


@pytest.mark.parametrize("mask", MASKS, ids=lambda m: getattr(m, "name", str(getattr(m, "include", m))))
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64)])
def test_weights_under_masks(gpu, dtype, D, mask):
    sizes = [(1, 200), (4, 131), (9, 9), (1, 1), (20, 300), (150, 410), (3, 33), (1, 500)]
    _weigh(Batch(gpu, dtype, D, 32, 8, 2, sizes, seed=5), mask)


@pytest.mark.parametrize("dtype,D", TYPES)
@pytest.mark.parametrize("Hq,Hkv", [(2, 2), (8, 2), (5, 1)])
def test_weights_of_chunks(gpu, dtype, D, Hq, Hkv):
    sizes = [(100, 100), (33, 400), (1, 700), (257, 513), (64, 64), (0, 10), (128, 1000), (31, 95), (2, 2)]
    b = Batch(gpu, dtype, D, 16, Hq, Hkv, sizes, seed=Hq)
    _weigh(b, pm.Causal(), scale=0.2)
    _weigh(b, pm.SinksWindow(5, 100), first=np.array([5] * 9))
    _weigh(b, pm.LocalStrided(60, 16), max_fresh=3)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64)])
@pytest.mark.parametrize("mask", [pm.SinksWindow(100, 300), pm.SinksWindow(1, 64), pm.SlidingWindow(5), pm.TwoBand(30, 700, 90),
                                  pm.Union(pm.SlidingWindow(70), pm.SinksWindow(300, 2)),
                                  pm.Difference(pm.SlidingWindow(400), pm.SlidingWindow(130))], ids=str)
def test_weights_under_windows_that_leave_blocks_dead(gpu, dtype, D, mask):
    """Blocks of keys that no new token sees keep their scores; new keys that nothing sees get 0."""
    sizes = [(1, 3000), (2, 1025), (40, 2500), (1, 64), (9, 70), (7, 1400), (130, 1300), (1, 2049), (300, 300), (1, 511)]
    b = Batch(gpu, dtype, D, 32, 8, 4, sizes, seed=9)
    _weigh(b, mask)
    _weigh(b, mask, first=np.array([64, 1000, 200, 64, 3, 1390, 900, 2040, 0, 400]))
    _weigh(b, mask, first=np.array([2900, 3, 2400, 1, 65, 700, 100, 1, 256, 511]), max_fresh=1)


def test_weights_of_many_requests_and_long_ones(gpu):
    rng = np.random.default_rng(1)
    for R in (63, 64, 65, 300):
        sizes = [(int(rng.integers(0, 3)), int(rng.integers(2, 90))) for _ in range(R)]
        _weigh(Batch(gpu, torch.bfloat16, 64, 16, 4, 2, sizes, seed=R), pm.Causal())
    _weigh(Batch(gpu, torch.bfloat16, 128, 64, 4, 1, [(1, 20001), (1, 3)]), pm.Causal())
    _weigh(Batch(gpu, torch.float16, 64, 64, 8, 2, [(300, 9000), (1, 3000)]), pm.Causal())


@pytest.mark.parametrize("dtype,D", TYPES)
@pytest.mark.parametrize("R", [65, 130, 300])
def test_weights_of_chunks_among_many_requests(gpu, dtype, D, R):
    """More requests than lanes: chunks before and behind the 64th, whose shares are merged, tokens beside them, some of
    none; and the same bits again."""
    rng = np.random.default_rng(R)
    sizes = [(int(n), int(n + x)) for n, x in zip(rng.integers(0, 3, R), rng.integers(1, 60, R))]
    for r in {0, 5, 63, 64, R - 1, int(rng.integers(65, R + 1)) - 1, int(rng.integers(R))}:
        n = int(rng.integers(33, 90))
        sizes[r] = (n, n + int(rng.integers(0, 300)))
    sizes[62], sizes[R - 1] = (500, 700), (610, 610)
    b = Batch(gpu, dtype, D, 16, 8, 2, sizes, seed=R)
    first = np.where(rng.random(R) < 0.3, rng.integers(0, 50, R), 0)
    got = _weigh(b, pm.Causal(), first=first)
    assert torch.equal(_weigh(b, pm.Causal(), first=first), got)
    _weigh(b, pm.SinksWindow(3, 100))
    # starts that fall back are taken as the ones that they stand for
    t, n, s = b.dev()
    lse, scores = torch.empty(b.T, b.Hq, device=gpu), [torch.zeros(b.pages, b.Hkv, b.P, device=gpu) for _ in range(2)]
    paged.attention(b.q, b.k, b.v, t, n, s, pm.Causal(), lse=lse)
    lse[int(b.n.sum()):] = NAN
    for x, at in zip(scores, (s, dev(falling(b.q_start, b.n, rng), gpu))):
        paged.weights(b.q, b.k, t, n, at, lse, x, pm.Causal())
    assert torch.equal(*scores)


def test_weights_sum_to_the_rows(gpu):
    """Over all keys a step's weights sum to its rows: new tokens times heads of the group."""
    sizes = [(1, 3000), (40, 700), (7, 7)]
    b = Batch(gpu, torch.float32, 128, 16, 8, 2, sizes, poison=0.0)
    scores = torch.zeros(b.pages, b.Hkv, b.P, device=gpu)
    t, n, s = b.dev()
    lse = torch.empty(b.T, b.Hq, device=gpu)
    paged.attention(b.q, b.k, b.v, t, n, s, pm.Causal(), lse=lse)
    paged.weights(b.q, b.k, t, n, s, lse, scores, pm.Causal())
    for r, (m, L) in enumerate(sizes):
        p = np.arange(L)
        mine = f64(scores)[b.tables[r, p // 16], :, p % 16].sum(axis=0)
        assert np.abs(mine / (4 * m) - 1).max() <= 2.0 ** -14


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float32, 64)])
@pytest.mark.parametrize("n", [1, 40])
def test_weights_of_what_is_dead(gpu, dtype, D, n):
    """Infinities and NaN in masked keys, rows without weight, keys without a page."""
    b = Batch(gpu, dtype, D, 16, 4, 2, [(n, 150), (2, 60)])
    mask = pm.SlidingWindow(30)
    page = int(b.tables[0, 3])
    lse = torch.empty(b.T, b.Hq, device=gpu)
    paged.attention(b.q, b.k, b.v, *b.dev(), mask, lse=lse)
    lse[0, 1] = -INF
    want = _weigh(b, mask, lse=lse.clone())
    b.k[page, :, 5] = NAN if n == 1 else INF         # (position 53: no row of n = 1 or 40 sees it)
    got = _weigh(b, mask, lse=lse.clone())
    assert torch.equal(got, want)
    b.tables[0, 7] = -1
    b.tables[1, 2] = 1 << 30
    _weigh(b, mask, lse=lse.clone())


def test_a_live_key_that_is_not_finite_has_its_own_weight(gpu):
    """.. and the others theirs."""
    b = Batch(gpu, torch.float16, 64, 16, 4, 2, [(3, 100)], poison=0.0)
    lse = torch.empty(b.T, b.Hq, device=gpu)
    paged.attention(b.q, b.k, b.v, *b.dev(), pm.Causal(), lse=lse)
    scores = [torch.zeros(b.pages, 2, 16, device=gpu) for _ in range(2)]
    paged.weights(b.q, b.k, *b.dev(), lse, scores[0], pm.Causal())
    page = int(b.tables[0, 2])
    b.k[page, :, 4] = NAN
    paged.weights(b.q, b.k, *b.dev(), lse, scores[1], pm.Causal())
    assert torch.isnan(scores[1][page, :, 4]).all()
    scores[1][page, :, 4] = scores[0][page, :, 4]
    assert torch.equal(*scores)


@pytest.mark.parametrize("mask", [pm.Causal(), pm.SinksWindow(3, 70), pm.LocalStrided(40, 16), pm.Full()], ids=str)
@pytest.mark.parametrize("dtype,D", TYPES)
def test_a_row_whose_lse_is_not_finite_weighs_its_live_keys_alone(gpu, dtype, D, mask):
    """NaN, infinities and the largest numbers as lse of some rows, in requests of few and of many rows: a key
    that such a row does not see has the other rows' weights."""
    b = Batch(gpu, dtype, D, 16, 8, 2, [(300, 700), (1, 60), (40, 150), (3, 100), (64, 64), (129, 400)], seed=3, poison=0.0)
    spec = paged._paged_mask(mask).spec
    t, n, s = b.dev()
    lse = torch.empty(b.T, b.Hq, device=gpu)
    paged.attention(b.q, b.k, b.v, t, n, s, mask, lse=lse)
    rng = np.random.default_rng(0)
    odd = [NAN, INF, -INF, -3.4e38, 3.4e38, -2.5e38]
    where = [(r, int(i), int(h), odd[int(rng.integers(len(odd)))]) for r in range(len(b.n))
             for i, h in zip(rng.integers(0, b.n[r], 5), rng.integers(0, b.Hq, 5))]
    for r, i, h, x in where:
        lse[b.q_start[r] + i, h] = x
    # (those without weight: the others' weights and what these may be off by)
    plain = f64(lse)
    plain[~(np.abs(plain) < 1e30)] = -INF
    want, bound = so.weights(f64(b.q), f64(b.k), b.tables, b.lengths, b.q_start, plain, np.zeros((b.pages, b.Hkv, b.P)), spec.live,
                             D ** -0.5, np.zeros(len(b.n), dtype=int))
    for r, i, h, _ in where:
        x = float(lse[b.q_start[r] + i, h])
        if np.isnan(x) or x < -1e30 and x != -INF:
            L = b.lengths[r]
            p = np.flatnonzero(spec.live(np.array([[L - b.n[r] + i]]), np.arange(L)[None, :])[0])
            want[b.tables[r, p // 16], h // 4, p % 16] += NAN if np.isnan(x) else INF
    scores = torch.zeros(b.pages, b.Hkv, b.P, device=gpu)
    got = f64(paged.weights(b.q, b.k, t, n, s, lse, scores, mask))
    assert np.isnan(want).any() and np.isinf(want).any()
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want))
    ok = np.isfinite(want)
    assert (np.abs(got[ok] - want[ok]) <= bound[ok]).all()


def test_weights_with_nothing_to_weigh(gpu):
    q = torch.ones(3, 4, 64, dtype=torch.float16, device=gpu)
    k, s = torch.zeros(2, 2, 16, 64, dtype=torch.float16, device=gpu), torch.full((2, 2, 16), 7.0, device=gpu)
    i32 = lambda *x: torch.tensor(x, dtype=I32, device=gpu)  # noqa: E731
    lse, some = torch.zeros(3, 4, device=gpu), torch.zeros(1, 2, dtype=I32, device=gpu)
    paged.weights(q, k, some, i32(20), i32(0, 0), lse, s, pm.Causal())
    paged.weights(q, k, some, i32(0), i32(0, 3), lse, s, pm.Causal())
    paged.weights(q, k, some, i32(20), i32(0, 3), lse, s, pm.Causal(), first=i32(20))
    paged.weights(q[:0], k, some, i32(20), i32(0, 0), lse[:0], s, pm.Causal())
    paged.weights(q, k[:0], some, i32(20), i32(0, 3), lse, s[:0], pm.Causal())
    paged.weights(q, k, some[:0], i32(), i32(0), lse, s, pm.Causal())
    paged.weights(q, k, some[:, :0], i32(20), i32(0, 3), lse, s, pm.Causal())
    assert (s == 7).all()


# ---- which stay -------------------------------------------------------------------------------------
def _pool(rng, lengths, P, spare=3):
    held = -(-lengths // P)
    tables = np.full((len(lengths), int(held.max(initial=0)) + 2), -1, dtype=np.int64)
    pages = int(held.sum()) + spare
    tables[np.arange(tables.shape[1])[None, :] < held[:, None]] = rng.permutation(pages)[:int(held.sum())]
    return tables, pages


def _choose(gpu, scores, tables, lengths, keep, recent, limit, first=None):
    """scores: numpy float32 [(layers,) pages, H, P]."""
    wide = torch.full((*scores.shape[:-1], scores.shape[-1] + 3), NAN, device=gpu)    # rows of any alignment
    wide[..., :scores.shape[-1]] = torch.as_tensor(scores, device=gpu)
    rest = dev(tables, gpu), dev(lengths, gpu), keep, recent, limit, None if first is None else dev(first, gpu)
    got = paged.choose(wide[..., :scores.shape[-1]], *rest)
    again = paged.choose(torch.as_tensor(scores, device=gpu), *rest)
    assert torch.equal(got.kept, again.kept) and torch.equal(got.lengths, again.lengths)
    f = np.zeros(len(lengths), dtype=int) if first is None else first
    for i, s in enumerate(scores if scores.ndim == 4 else scores[None]):
        kept, after = so.choose(s, tables, lengths, keep, recent, keep if limit is None else limit, f)
        assert np.array_equal(host(got.kept)[i] if scores.ndim == 4 else host(got.kept), kept), i
    assert np.array_equal(host(got.lengths), after)
    return got


@pytest.mark.parametrize("keep,recent,limit", [(1, 0, None), (1, 1, None), (16, 5, 20), (40, 40, None), (64, 0, 64), (100, 37, 130),
                                               (1000, 100, None)])
@pytest.mark.parametrize("P,H", [(16, 3), (256, 1)])
def test_choose_against_numpy(gpu, keep, recent, limit, P, H):
    rng = np.random.default_rng(keep)
    lengths = np.concatenate([[0, 1, 2, 15, 16, 17, keep - 1, keep, keep + 1, keep + 21], rng.integers(1, 3 * keep + 50, 9)])
    tables, pages = _pool(rng, lengths, P)
    scores = rng.standard_normal((2, pages, H, P)).astype(np.float32)
    _choose(gpu, scores, tables, lengths, keep, recent, limit)
    first = rng.integers(-2, 40, len(lengths))
    _choose(gpu, scores, tables, lengths, keep, recent, limit, first)
    _choose(gpu, np.round(np.maximum(scores, 0) * 3).astype(np.float32)[0], tables, lengths, keep, recent, limit, first)   # many ties


@pytest.mark.parametrize("L", [4096, 4097, 16384, 16385, 32768, 32769, 70000])
def test_choose_of_long_requests(gpu, L):
    rng = np.random.default_rng(L)
    lengths = np.array([L, 300])
    tables, pages = _pool(rng, lengths, 64)
    scores = np.exp(2 * rng.standard_normal((pages, 2, 64))).astype(np.float32)
    scores[rng.random(scores.shape) < 0.3] = 0
    for keep, recent in ((L // 3, 64), (L - 1, 0), (1, 0), (L * 4 // 5, 1)):
        _choose(gpu, scores, tables, lengths, keep, recent, None)
    _choose(gpu, np.zeros_like(scores), tables, lengths, 1000, 10, None)


def test_choose_of_odd_scores(gpu):
    """Infinities, NaN of either sign, zeros of either sign, the smallest and largest, keys without a page."""
    P, lengths = 16, np.array([160, 160, 160])
    rng = np.random.default_rng(0)
    tables, pages = _pool(rng, lengths, P)
    odd = np.array([INF, -INF, NAN, -0.0, 0.0, 1e-45, -1e-45, 3.4e38, -3.4e38, 1.0], dtype=np.float32)
    scores = rng.choice(odd, (pages, 2, P))
    scores.view(np.uint32)[np.isnan(scores) & (rng.random(scores.shape) < 0.5)] = 0xffc00001
    tables[1, 3], tables[1, 5], tables[2, :] = -1, 1 << 30, -1
    for keep in (1, 5, 20, 50, 100, 140, 159):
        _choose(gpu, scores, tables, lengths, keep, min(3, keep), None)


def test_choose_with_nothing_to_choose(gpu):
    s = torch.zeros(2, 1, 16, device=gpu)
    none = paged.choose(s, torch.zeros(0, 1, dtype=I32, device=gpu), torch.zeros(0, dtype=I32, device=gpu), 4, 1)
    assert none.kept.shape == (0, 1, 4)
    got = paged.choose(s[:0], torch.zeros(1, 0, dtype=I32, device=gpu), torch.full((1,), 50, dtype=I32, device=gpu), 4, 1)
    assert (got.kept == -1).all() and host(got.lengths).tolist() == [50]
    got = paged.choose(torch.zeros(0, 2, 1, 16, device=gpu), torch.zeros(1, 3, dtype=I32, device=gpu), torch.full((1,), 40, dtype=I32, device=gpu), 4, 1)
    assert got.kept.shape == (0, 1, 1, 4)


def test_choose_of_no_layers_says_how_long_requests_are(gpu):
    s = torch.zeros(0, 20, 3, 16, device=gpu)
    lengths, first = np.array([100, 40, 90, 0]), np.array([0, 3, 50, 0])
    t, n = torch.zeros(4, 9, dtype=I32, device=gpu), dev(lengths, gpu)
    want = so.choose(np.zeros((20, 1, 16)), host(t), lengths, 30, 5, 39, first)[1]
    out = (torch.empty(0, 4, 3, 30, dtype=I32, device=gpu), dev([-7] * 4, gpu))
    got = paged.choose(s, t, n, 30, 5, 39, dev(first, gpu), out=out)
    assert got.lengths is out[1] and np.array_equal(host(got.lengths), want) and want.tolist() == [30, 40, 80, 0]
    t[0, 3], flag = -1, dev([0], gpu)
    assert host(paged.choose(s, t, n, 30, 5, 39, dev(first, gpu), missing=flag).lengths).tolist() == [100, 40, 80, 0] and int(flag) == 1


# ---- their move ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,D", TYPES)
@pytest.mark.parametrize("P,layers,keep,first", [(16, 2, 50, 0), (64, None, 300, 3), (32, 1, 129, 40), (256, 3, 1000, 1)])
def test_evict_against_numpy(gpu, dtype, D, P, layers, keep, first):
    rng = np.random.default_rng(keep + D)
    g = torch.Generator().manual_seed(keep)
    lengths = np.concatenate([[0, 1, keep, keep + 1, keep + first, keep + first + 1], rng.integers(1, 3 * keep, 4)])
    tables, pages = _pool(rng, lengths, P)
    lead = () if layers is None else (layers,)
    k, v = (torch.randn(*lead, pages, 2, P, D, generator=g).to(dtype).to(gpu) for _ in range(2))
    scores = torch.rand(*lead, pages, 2, P, generator=g).to(gpu)
    f = rng.integers(0, first + 1, len(lengths))
    t, n, fd = dev(tables, gpu), dev(lengths, gpu), dev(f, gpu)
    choice = paged.choose(scores, t, n, keep, keep // 8, None, fd)
    want = [[so.evict(kept, y, tables, lengths, f) for kept, y in zip(host(choice.kept).reshape(-1, len(lengths), 2, keep),
                                                                      f64(x).reshape(-1, pages, 2, P, *x.shape[len(lead) + 3:]))]
            for x in (k, v, scores)]
    k2, v2 = k.clone(), v.clone()
    got = paged.evict(choice.kept, k, v, scores, t, n, fd)
    for x, w in zip(got, want):
        assert np.array_equal(f64(x).reshape(np.array(w).shape), np.array(w))
    paged.evict(choice.kept, k2, v2, None, t, n, fd)        # without scores
    assert torch.equal(k2, k) and torch.equal(v2, v)


@pytest.mark.parametrize("dtype,D", TYPES)
@pytest.mark.parametrize("R,H,layers", [(16, 4, 2), (9, 7, 3), (16, 8, 2), (33, 8, 2), (64, 2, 4), (511, 1, 1), (43, 3, 4)])
def test_evict_of_many_heads(gpu, dtype, D, R, H, layers):
    """From work-groups that cut rows into slices to those of 512 threads: R H layers on both sides of each rule."""
    P, keep = 16, 33
    rng = np.random.default_rng(R)
    g = torch.Generator().manual_seed(R)
    lengths = rng.integers(1, 4 * keep, R)
    tables, pages = _pool(rng, lengths, P)
    k, v = (torch.randn(layers, pages, H, P, D, generator=g).to(dtype).to(gpu) for _ in range(2))
    scores = torch.rand(layers, pages, H, P, generator=g).to(gpu)
    f = rng.integers(0, 9, R)
    t, n, fd = dev(tables, gpu), dev(lengths, gpu), dev(f, gpu)
    choice = paged.choose(scores, t, n, keep, 5, None, fd)
    kept = host(choice.kept)
    want = [[so.evict(kept[i], x[i], tables, lengths, f) for i in range(layers)] for x in (f64(k), f64(v), f64(scores))]
    for x, w in zip(paged.evict(choice.kept, k, v, scores, t, n, fd), want):
        assert np.array_equal(f64(x), np.array(w))


def test_evict_of_odd_lists(gpu):
    """Lists out of order, with entries below their place, past the table or without a page: each moves what
    the formula says, or nothing."""
    P, keep, H = 16, 60, 2
    rng = np.random.default_rng(4)
    lengths = np.array([200, 90, 130])
    tables, pages = _pool(rng, lengths, P)
    tables[0, 9], tables[1, 1], tables[2, 4] = -1, 1 << 30, -7
    k = torch.randn(pages, H, P, 64, device=gpu).half()
    v, s = torch.randn(pages, H, P, 64, device=gpu).half(), torch.rand(pages, H, P, device=gpu)
    first = np.array([0, 5, 7])
    place = first[:, None, None] + np.arange(keep)[None, None, :]
    kept = place + rng.integers(0, 60, (3, H, keep))
    kept[0, 0, ::7] = -1
    kept[1, 1, ::5] = place[1, 0, ::5] - 1
    kept[2, 0, 3::9] = 1 << 30
    want = [so.evict(kept, f64(x), tables, lengths, first) for x in (k, v, s)]
    got = paged.evict(dev(kept, gpu), k, v, s, dev(tables, gpu), dev(lengths, gpu), dev(first, gpu))
    for x, w in zip(got, want):
        assert np.array_equal(f64(x), w)


def test_evict_of_lists_longer_than_the_table(gpu):
    """The longest list there can be, 4 GiB, of a request at the largest positions: places past the table take
    nothing."""
    P, D, keep, cols = 256, 64, paged.MAX_POSITION, paged.MAX_POSITION // 256
    x = torch.randn(2, 3, 1, P, D, device=gpu).half()
    t = torch.full((1, cols), -1, dtype=I32, device=gpu)
    t[0, -2:] = dev([2, 0], gpu)
    reach, first = cols * P, cols * P - 300
    kept = torch.zeros(1, 1, keep, dtype=I32, device=gpu)
    kept[0, 0, :290] = torch.arange(first + 10, first + 300, dtype=I32, device=gpu)
    kept[0, 0, 290:400] = torch.arange(reach - 55, reach + 55, dtype=I32, device=gpu)
    kept[0, 0, -5000:] = reach - 1
    want = x.clone()
    flat = torch.cat([x[:, 2, 0], x[:, 0, 0]], dim=1)          # the last 512 places
    flat[:, 212:502] = flat[:, 222:512].clone()
    want[:, 2, 0], want[:, 0, 0] = flat[:, :P], flat[:, P:]
    paged.evict(kept, x[0], x[1], None, t, dev([reach], gpu), dev([first], gpu))
    assert torch.equal(x, want)


def test_evict_of_layouts(gpu):
    """K and V in one buffer, rows before heads, layers innermost."""
    P, keep, H, D, layers = 16, 40, 3, 64, 2
    rng = np.random.default_rng(4)
    lengths = np.array([100, 77])
    tables, pages = _pool(rng, lengths, P)
    s = torch.rand(layers, pages, H, P, device=gpu)
    t, n = dev(tables, gpu), dev(lengths, gpu)
    kept = paged.choose(s, t, n, keep, 4).kept
    x = torch.randn(2, layers, pages, H, P, D, device=gpu)
    want = x.clone()
    paged.evict(kept, want[0], want[1], None, t, n)
    for order in ((1, 0, 2, 3, 4, 5), (2, 0, 1, 4, 3, 5), (1, 2, 4, 3, 0, 5), (0, 2, 1, 3, 4, 5)):
        back = [order.index(i) for i in range(6)]
        y = x.permute(*order).contiguous().permute(*back)
        paged.evict(kept, y[0], y[1], None, t, n)
        assert torch.equal(y, want), order


def test_offsets_past_32_bits(gpu):
    """Keys, and scores, whose bytes lie past 4 GiB."""
    far, P, H, D = 8400, 256, 8, 128                    # pages of 512 KiB: 4.1 GiB
    b = Batch(gpu, torch.bfloat16, D, P, 16, H, [(1, 900), (40, 600), (1, 30)])
    t, n, s = b.dev()
    lse = torch.empty(b.T, b.Hq, device=gpu)
    paged.attention(b.q, b.k, b.v, t, n, s, pm.Causal(), lse=lse)
    near = torch.zeros(b.pages, H, P, device=gpu)
    paged.weights(b.q, b.k, t, n, s, lse, near, pm.Causal())
    k, v = (torch.empty(far + b.pages, H, P, D, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    k[far:], v[far:] = b.k, b.v
    wide = torch.empty(far + b.pages, H, 64 * P, device=gpu)[:, :, :P]      # 4.1 GiB of scores
    wide[far:] = 0
    ft = torch.where(t >= 0, t + far, t)
    paged.weights(b.q, k, ft, n, s, lse, wide, pm.Causal())
    assert torch.equal(wide[far:], near)
    kept, after = paged.choose(near, t, n, 300, 20)
    got = paged.choose(wide, ft, n, 300, 20)
    assert torch.equal(got.kept, kept) and torch.equal(got.lengths, after)
    paged.evict(kept, b.k, b.v, near, t, n)
    paged.evict(kept, k, v, wide, ft, n)
    assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in ((k[far:], b.k), (v[far:], b.v)))
    assert torch.equal(wide[far:], near)


def test_launches_that_run_again_and_at_once(gpu):
    """Two launches of weights with shares to merge, each captured and replayed on a stream of its own."""
    sizes = [(300, 2000), (1, 900), (90, 90)]
    made = []
    for seed in (1, 2):
        b = Batch(gpu, torch.bfloat16, 128, 16, 8, 2, sizes, seed=seed)
        lse = torch.empty(b.T, b.Hq, device=gpu)
        paged.attention(b.q, b.k, b.v, *b.dev(), pm.Causal(), lse=lse)
        scores = torch.zeros(b.pages, 2, 16, device=gpu)
        launch = paged.prepare_weights(b.q, b.k, *b.dev(), lse, scores, pm.Causal())
        want = launch().clone()
        scores.zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            launch()
        made.append((graph, launch, scores, want, b, lse))
    streams = [torch.cuda.Stream() for _ in made]
    for _ in range(4):
        torch.cuda.synchronize()
        for s, (graph, *_) in zip(streams, made):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, scores, want, *_ in made:
            assert torch.equal(scores, want)
            scores.zero_()


def test_refusals(gpu):
    k = torch.zeros(4, 2, 16, 64, dtype=torch.float16, device=gpu)
    v, s = torch.zeros_like(k), torch.zeros(4, 2, 16, device=gpu)
    t, n = torch.zeros(1, 4, dtype=I32, device=gpu), torch.full((1,), 60, dtype=I32, device=gpu)
    start = torch.tensor([0, 2], dtype=I32, device=gpu)
    q, lse = torch.zeros(2, 4, 64, dtype=torch.float16, device=gpu), torch.zeros(2, 4, device=gpu)
    kept = torch.zeros(1, 2, 8, dtype=I32, device=gpu)
    weights = lambda **kw: paged.weights(**{**dict(q=q, k=k, tables=t, lengths=n, q_start=start, lse=lse, scores=s, mask=pm.Causal()), **kw})  # noqa: E731
    choose = lambda **kw: paged.choose(**{**dict(scores=s, tables=t, lengths=n, keep=8, recent=2), **kw})  # noqa: E731
    evict = lambda **kw: paged.evict(**{**dict(kept=kept, k=k, v=v, scores=s, tables=t, lengths=n), **kw})  # noqa: E731
    weights(), choose(), evict()
    for call, bad in ((weights, dict(scores=s.half())), (weights, dict(scores=s[:3])), (weights, dict(scores=s.transpose(1, 2))),
                      (weights, dict(lse=lse[:1])), (weights, dict(scale=-1.0)), (weights, dict(first=n[:0])), (weights, dict(max_fresh=-1)),
                      (weights, dict(q=q[:, :3])), (weights, dict(mask=MaskSpec(((8, 0, 0, 0),)))),
                      (choose, dict(keep=0)), (choose, dict(recent=9)), (choose, dict(recent=-1)), (choose, dict(limit=7)),
                      (choose, dict(scores=s[0])), (choose, dict(scores=s[..., :15])), (choose, dict(first=n[:0])),
                      (choose, dict(out=(kept[..., :7], n.clone()))),
                      (evict, dict(v=v[:3])), (evict, dict(kept=kept[:, :1])), (evict, dict(kept=kept[None])), (evict, dict(scores=s[:3])),
                      (evict, dict(k=k[..., :32], v=v[..., :32]))):
        with pytest.raises(ValueError):
            call(**bad)
    for call, bad in ((weights, dict(first=n.long())), (choose, dict(lengths=n.long())), (evict, dict(kept=kept.long()))):
        with pytest.raises(TypeError):
            call(**bad)
    for call, bad in ((weights, dict(scores=s.cpu())), (choose, dict(scores=s.cpu())), (evict, dict(k=k.cpu())), (evict, dict(v=k)),
                      (weights, dict(scores=k.view(torch.float32).view(-1)[:128].view(4, 2, 16))),
                      (choose, dict(out=(s.view(-1)[:16].view(torch.int32).view(1, 2, 8), n.clone()))),
                      (choose, dict(out=(kept, n)))):
        with pytest.raises((RuntimeError, ValueError)):
            call(**bad)


# ---- the cache ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,D,P,G", [(torch.bfloat16, 128, 16, 4), (torch.float32, 64, 32, 1), (torch.float16, 64, 16, 2)])
def test_serving_a_cache_that_forgets(gpu, dtype, D, P, G):
    """Prompts, chunks and tokens, each step weighed, requests evicted, finished and begun anew, one prompt
    shared: the tables, the scores and the keys against a copy on the host that does the same with rows."""
    R, H, layers, keep, recent, limit, sinks = 5, 2, 2, 40, 8, 48, 3
    cache = paged.PagedKVCache(R, 320, 5 * 320 // P, H, D, dtype, P, layers, gpu, weigh=True)
    g = torch.Generator().manual_seed(P)
    rows = [[np.zeros((0, H, D)) for _ in range(R)] for _ in range(layers)]        # keys of each request
    pinned, prefix = [0] * R, 2 * P
    plan = [[prefix + 4, 30, 0, 0, 2], "share", [1, 30, 9, 1, 0], "evict", [1, 1, 1, 1, 50], "evict", [9, 1, 60, 1, 1], "evict", [1] * 5,
            "evict", "finish", [3, 70, 0, 2, 1], "evict", [1] * 5]
    for what in plan:
        if what == "share":
            cache.share(0, [2, 3], prefix)
            for layer in rows:
                layer[2] = layer[3] = layer[0][:prefix]
            pinned[0] = pinned[2] = pinned[3] = prefix
        elif what == "finish":
            cache.finish([False, True, True, True, False])
            for layer in rows:
                layer[1] = layer[2] = layer[3] = np.zeros((0, H, D))
            pinned[1] = pinned[2] = pinned[3] = 0
        elif what == "evict":
            tables, lengths = host(cache.tables), host(cache.lengths)
            first = np.maximum(pinned, sinks)
            chosen = [so.choose(f64(s), tables, lengths, keep, recent, limit, first) for s in cache.scores]
            cache.evict(keep, recent, limit, sinks)
            after = chosen[0][1]
            assert np.array_equal(host(cache.lengths), after)
            for layer, (kept, _) in zip(rows, chosen):
                for r in np.flatnonzero(after != lengths):
                    layer[r] = np.concatenate([layer[r][:first[r]], np.stack([layer[r][kept[r, h], h] for h in range(H)], axis=1)])
        else:
            T = sum(what) + 1
            step = cache.begin(what, T)
            for i in range(layers):
                kn, vn, q = (torch.randn(T, x, D, generator=g).to(dtype).to(gpu) for x in (H, H, H * G))
                cache.append(kn, vn, step, i)
                lse = torch.zeros(T, H * G, device=gpu)
                cache.attend(q, pm.Causal(), step, i, lse=lse)
                tables, lengths, starts = (host(x) for x in (cache.tables, step.lengths, step.q_start))
                want, bound = so.weights(f64(q), f64(cache.k[i]), tables, lengths, starts, f64(lse), f64(cache.scores[i]),
                                         lambda x, y: y <= x, D ** -0.5, np.array(pinned))
                cache.weigh(q, lse, pm.Causal(), step, i)
                assert (np.abs(f64(cache.scores[i]) - want) <= bound).all(), what
                for r in range(R):
                    rows[i][r] = np.concatenate([rows[i][r], f64(kn)[starts[r]:starts[r + 1]]])
        tables, lengths = host(cache.tables), host(cache.lengths)
        for i in range(layers):
            for r in range(R):
                t = np.arange(lengths[r])
                assert np.array_equal(f64(cache.k[i])[tables[r, t // P], :, t % P], rows[i][r]), (what, i, r)
        used = np.unique(tables[tables >= 0])
        free = host(cache.free_list)[:int(cache.free_count)]
        assert sorted(np.concatenate([used, free]).tolist()) == list(range(cache.pages))
        assert (tables[np.arange(tables.shape[1])[None, :] >= -(-lengths // P)[:, None]] < 0).all()
    cache.check()


def test_a_cache_without_scores_refuses(gpu):
    c = paged.PagedKVCache(2, 100, 20, 2, 64, torch.float16, 16, device=gpu)
    with pytest.raises(RuntimeError, match="weigh=True"):
        c.evict(10, 2)
    with pytest.raises(RuntimeError, match="weigh=True"):
        c.weigh(None, None, pm.Causal(), None)
    with pytest.raises(ValueError):
        paged.PagedKVCache(2, 100, 20, 2, 64, torch.float16, 16, device=gpu, weigh=True).evict(10, 2, sinks=-1)


def test_a_trimmed_cache_does_not_evict(gpu):
    c = paged.PagedKVCache(2, 100, 20, 2, 64, torch.float16, 16, device=gpu, weigh=True)
    c.begin([80, 3])
    c.trim(window=20)
    with pytest.raises(RuntimeError, match="trimmed"):
        c.evict(10, 2)


def test_requests_that_lack_pages_stay_whole_where_asked(gpu):
    """choose with missing: of requests past the limit those that lack a page from first on keep all."""
    rng = np.random.default_rng(0)
    P, lengths = 16, np.array([100, 100, 100, 100, 20, 0, 100])
    tables, pages = _pool(rng, lengths, P)
    first = np.array([0, 33, 32, 0, 0, 0, 48])
    tables[1, 2], tables[2, 1], tables[3, 6], tables[4, 0], tables[6, 3] = -1, -1, 1 << 30, -1, -7
    scores = rng.standard_normal((2, pages, 3, P)).astype(np.float32)
    whole = np.array([1, 3, 6])                     # (2 lacks one in front of first, 4 is within the limit)
    want = [so.choose(s, tables, lengths, 30, 4, 40, first) for s in scores]
    s, t, n, f = torch.as_tensor(scores, device=gpu), dev(tables, gpu), dev(lengths, gpu), dev(first, gpu)
    for layers in (slice(None), 0):
        bits = dev([3], gpu)
        got = paged.choose(s[layers], t, n, 30, 4, 40, f, missing=bits, missing_bits=64)
        kept, after = (np.stack([k for k, _ in want]) if layers != 0 else want[0][0]).copy(), want[0][1].copy()
        kept[..., whole, :, :], after[whole] = -1, lengths[whole]
        assert np.array_equal(host(got.kept), kept) and np.array_equal(host(got.lengths), after) and int(bits) == 67
        none = dev([3], gpu)
        paged.choose(s[layers], t[[0, 2, 4, 5]], n[[0, 2, 4, 5]], 30, 4, 40, f[[0, 2, 4, 5]], missing=none)
        assert int(none) == 3
    with pytest.raises(ValueError):
        paged.choose(s, t, n, 30, 4, 40, f, missing=n)
    with pytest.raises(RuntimeError, match="overlap"):
        paged.choose(s, t, n, 30, 4, 40, f, missing=n[:1])


def test_an_eviction_captured_before_a_trim_and_replayed_after(gpu):
    """Requests without pages in front stay as they are, the others are evicted, no page is lost, and check tells."""
    g = torch.Generator().manual_seed(0)
    c = paged.PagedKVCache(4, 200, 40, 2, 64, torch.float16, 16, 2, gpu, weigh=True)
    c.begin([100, 40, 90, 30])
    for x in (c.k, c.v, c.scores):
        x.copy_(torch.rand(x.shape, generator=g))
    out = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(out):
        c.evict(30, 5)
    c.trim(window=45)
    tables, k, v, scores = host(c.tables), f64(c.k), f64(c.v), f64(c.scores)
    assert (tables[[0, 2], 0] == -1).all() and (tables[1, :3] >= 0).all()
    only, none = np.array([0, 40, 0, 0]), np.zeros(4, dtype=int)
    kept = [so.choose(s, tables, only, 30, 5, 30, none)[0] for s in scores]
    want = [[so.evict(kept[i], x[i], tables, only, none) for i in range(2)] for x in (k, v, scores)]
    for i in range(2):                               # (the second has nothing left to do)
        out.replay()
        torch.cuda.synchronize()
        assert host(c.lengths).tolist() == [100, 30, 90, 30]
        tables[1, 2] = -1
        assert np.array_equal(host(c.tables), tables)
        ids = np.concatenate([tables[tables >= 0], host(c.free_list)[:int(c.free_count)]])
        assert sorted(ids.tolist()) == list(range(40))
    for x, w in zip((c.k, c.v, c.scores), want):
        assert np.array_equal(f64(x), np.array(w))
    with pytest.raises(RuntimeError, match="pages in front"):
        c.check()


def test_captured_steps_and_evictions(gpu):
    """A step with its weights and an eviction in graphs, replayed, against a second cache without."""
    R, H, G, D, P = 4, 2, 2, 64, 16
    a, e = (paged.PagedKVCache(R, 400, 80, H, D, torch.bfloat16, P, 2, gpu, weigh=True) for _ in range(2))
    gen = torch.Generator().manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=gen).to(torch.bfloat16).to(gpu)  # noqa: E731
    prompt = [90, 70, 3, 64]
    kp, vp, qp = rnd(227, H, D), rnd(227, H, D), rnd(227, H * G, D)
    ones = torch.ones(R, dtype=I32, device=gpu)
    q, kn, vn = rnd(R, H * G, D), rnd(R, H, D), rnd(R, H, D)

    def a_step(c, n, q, kn, vn, tokens=None):
        step = c.begin(n, tokens)
        for i in range(2):
            c.append(kn, vn, step, i)
            lse = torch.zeros(q.shape[:2], device=gpu)
            c.attend(q, pm.Causal(), step, i, lse=lse)
            c.weigh(q, lse, pm.Causal(), step, i)
    for c in (a, e):
        a_step(c, prompt, qp, kp, vp)
    torch.cuda.synchronize()
    step, out = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(step):
        a_step(a, ones, q, kn, vn, R)
    with torch.cuda.graph(out):
        a.evict(48, 8, 60, 2)
    for i in range(24):
        for x, n in ((q, H * G), (kn, H), (vn, H)):
            x.copy_(rnd(R, n, D))
        step.replay()
        a_step(e, ones, q, kn, vn, R)
        if i % 5 == 4:
            out.replay()
            e.evict(48, 8, 60, 2)
        torch.cuda.synchronize()
        for name in ("lengths", "tables", "k", "v", "scores", "free_count"):
            assert torch.equal(getattr(a, name), getattr(e, name)), (i, name)
    e.check()


@pytest.mark.parametrize("seed", range(8))
def test_lives_of_a_cache_at_random(gpu, seed):
    """Steps, shares (some refused), evictions and finishes in any order, against rows on the host: attention, scores,
    keys, holders, what check knows, and no page twice or lost."""
    rng = random.Random(seed)
    for _ in range(10):
        R, P, H, G, D = rng.randint(1, 9), rng.choice([16, 32]), rng.choice([1, 2]), rng.choice([1, 4]), 64
        dtype, cap = rng.choice([torch.float32, torch.bfloat16]), rng.choice([100, 300])
        c = paged.PagedKVCache(R, cap, R * -(-cap // P) + 2, H, D, dtype, P, 1, gpu, weigh=True)
        rows, holder, shared, failed, log = [np.zeros((0, H, D))] * R, [-1] * R, [0] * R, 0, []
        for _ in range(rng.randint(5, 25)):
            what, n = rng.choice(["step"] * 5 + ["share"] * 2 + ["evict", "finish"]), [len(x) for x in rows]
            if what == "step":
                fresh = [min(rng.choice([0, 1, 1, 2, 5, rng.randint(0, 60)]), c.max_length - n[r]) for r in range(R)]
                m, T = sum(fresh), sum(fresh) + rng.randint(1, 2)
                step = c.begin(fresh, T)
                kn, vn, q = (torch.randn(T, x, D, generator=torch.Generator().manual_seed(m)).to(dtype).to(gpu) for x in (H, H, H * G))
                c.append(kn, vn, step)
                lse = torch.zeros(T, H * G, device=gpu)
                o = c.attend(q, pm.Causal(), step, lse=lse, out=torch.zeros_like(q))
                at = host(c.tables), host(step.lengths), host(step.q_start)
                want, _, eo, _ = po.attention(f64(q), f64(c.k[0]), f64(c.v[0]), *at, lambda x, y: y <= x, D ** -0.5, dtype)
                assert (np.abs(f64(o)[:m] - want[:m]) <= eo[:m]).all(), log
                want, bound = so.weights(f64(q), f64(c.k[0]), *at, f64(lse), f64(c.scores[0]), lambda x, y: y <= x, D ** -0.5,
                                         np.array(shared))
                c.weigh(q, lse, pm.Causal(), step)
                assert (np.abs(f64(c.scores[0]) - want) <= bound).all(), log
                rows = [np.concatenate([x, f64(kn)[a:b]]) for x, a, b in zip(rows, at[2], at[2][1:])]
                log.append((what, fresh))
            elif what == "share":
                h, t = rng.randrange(R), P * rng.randint(1, max(c.max_length // P // 2, 1))
                members = [x for x in range(R) if x != h and rng.random() < 0.4]
                c.share(h, members, t)
                root = holder[h] if holder[h] not in (-1, h) else h
                can = n[h] >= t and (root == h or shared[h] >= t)
                for m in members:
                    if can and n[m] == 0 and holder[m] < 0:
                        rows[m], holder[m], shared[m] = rows[h][:t], root, t
                        holder[root], shared[root] = root, max(shared[root], t)
                    else:
                        failed |= paged.SHARED
                log.append((what, h, members, t))
            elif what == "evict":
                keep, sinks = rng.randint(1, 60), rng.randint(0, 20)
                recent, limit = rng.randint(0, keep), keep + rng.randint(0, 30)
                first = np.maximum(shared, sinks)
                kept, after = so.choose(f64(c.scores[0]), host(c.tables), np.array(n), keep, recent, limit, first)
                c.evict(keep, recent, limit, sinks)
                for r in np.flatnonzero(after != n):
                    rows[r] = np.concatenate([rows[r][:first[r]], np.stack([rows[r][kept[r, h], h] for h in range(H)], axis=1)])
                log.append((what, keep, recent, limit, sinks))
            else:
                done = [rng.random() < 0.4 for _ in range(R)]
                busy = [any(holder[m] == r != m and not done[m] for m in range(R)) for r in range(R)]
                c.finish(done)
                for r in np.flatnonzero(done):
                    if busy[r]:
                        failed |= paged.SHARED
                    else:
                        rows[r], holder[r], shared[r] = rows[r][:0], -1, 0
                log.append((what, done))
            tables, lengths = host(c.tables), host(c.lengths)
            assert lengths.tolist() == [len(x) for x in rows], log
            assert host(c.holders).tolist() == holder and host(c.shared).tolist() == shared and int(c.failed) == failed, log
            for r, L in enumerate(lengths):
                t = np.arange(L)
                assert np.array_equal(f64(c.k[0])[tables[r, t // P], :, t % P], rows[r]), log
            free = host(c.free_list)[:int(c.free_count)]
            assert sorted(np.concatenate([np.unique(tables[tables >= 0]), free]).tolist()) == list(range(c.pages)), log
