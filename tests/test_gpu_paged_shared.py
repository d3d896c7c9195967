"""Requests that share a prefix (paged.sharing, paged.shared_attention, PagedKVCache.share) against
tests/shared_oracle.py and tests/paged_oracle.py."""
import numpy as np
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from polyhedral_amd import paged
from polyhedral_amd.polyattn import masks as pm
from polyhedral_amd.spec import MaskSpec
from tests import paged_oracle as po
from tests import shared_oracle as so

pytestmark = pytest.mark.gpu

I32 = torch.int32
NAN, INF = float("nan"), float("inf")
TYPES = [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 64),
         (torch.float32, 128)]


def dev(x, gpu):
    return torch.as_tensor(np.ascontiguousarray(x), dtype=I32).to(gpu)


def host(t):
    return t.detach().cpu().numpy().astype(np.int64)


def f64(t):
    return t.float().cpu().numpy().astype(np.float64)


# ---- which tokens share a prefix ---------------------------------------------------------------
def _sharing(gpu, lengths, q_start, holders, shared, P, T):
    got = paged.sharing(dev(lengths, gpu), dev(q_start, gpu), dev(holders, gpu), dev(shared, gpu), P, T)
    for g, w, name in zip(got, so.sharing(lengths, q_start, holders, shared, P, T), paged.Sharing._fields):
        assert np.array_equal(host(g), w), name
    return got


@pytest.mark.parametrize("R,groups,fresh,P", [(1, 1, 3, 16), (2, 1, 1, 64), (5, 2, 4, 16), (64, 1, 1, 64), (63, 9, 7, 32),
                                              (256, 30, 2, 16), (600, 3, 40, 128), (1024, 200, 1, 16), (1025, 5, 2, 16),
                                              (2500, 700, 3, 64)])
def test_sharing_against_numpy(gpu, R, groups, fresh, P):
    rng = np.random.default_rng(R)
    lengths = rng.integers(0, 9 * P, R)
    n = np.minimum(rng.integers(0, fresh + 1, R), lengths)
    holders = rng.integers(-1, groups, R) * (R // groups)
    shared = rng.integers(0, 9 * P, R)
    q_start = np.concatenate([[0], np.cumsum(n)])
    _sharing(gpu, lengths, q_start, holders, shared, P, int(n.sum()) + int(rng.integers(0, 5)))


def test_sharing_of_odd_entries(gpu):
    """Holders and shares out of range, tokens past lengths, no tokens, nobody."""
    lengths, n = np.array([100, 40, 64, 7, 900, 64]), np.array([1, 2, 0, 3, 5, 64])
    q_start = np.concatenate([[0], np.cumsum(n)])
    for holders, shared in (([2, 2, 2, 2, 2, 2], [64, 32, 64, 64, 1 << 30, 64]), ([6, -5, 1 << 30, 0, 0, 0], [64] * 6),
                            ([4, 4, 4, 4, 4, 4], [15, 16, 17, 16, -3, 0]), ([0, 1, 2, 3, 4, 5], [16] * 6)):
        _sharing(gpu, lengths, q_start, np.array(holders), np.array(shared), 16, 80)
    _sharing(gpu, np.zeros(0, dtype=int), np.array([0]), np.zeros(0, dtype=int), np.zeros(0, dtype=int), 16, 3)
    _sharing(gpu, lengths, np.zeros(7, dtype=int), np.full(6, 2), np.full(6, 16), 16, 0)


def _plan(lengths, q_start, holders, shared, P, T):
    """so.sharing for many requests, all in range: a stable sort by holder."""
    R, n = len(lengths), np.diff(q_start)
    some = np.minimum(shared, lengths) // P * P
    own = np.where((n > 0) & (some > 0), holders, -1)
    big = 1 << 40
    count, prefix, low, high = np.zeros(R, dtype=np.int64), np.full(R, big), np.full(R, big), np.zeros(R, dtype=np.int64)
    who = np.flatnonzero(own >= 0)
    np.add.at(count, own[who], 1)
    np.minimum.at(prefix, own[who], some[who])
    np.minimum.at(low, own[who], (lengths - n)[who])
    np.maximum.at(high, own[who], lengths[who] - 1)
    for x in (prefix, low, high):
        x[count < 2] = 0
    who = who[count[own[who]] > 1]
    first = np.zeros(R, dtype=np.int64)
    first[who] = prefix[own[who]]
    who = who[np.argsort(own[who], kind="stable")]
    start = np.zeros(R + 1, dtype=np.int64)
    np.add.at(start, own[who] + 1, n[who])
    i = np.arange(int(n[who].sum())) - np.repeat(np.cumsum(n[who]) - n[who], n[who])
    fill = np.full(T - len(i), -1)
    return (np.cumsum(start), np.concatenate([np.repeat(q_start[who], n[who]) + i, fill]),
            np.concatenate([np.repeat((lengths - n)[who], n[who]) + i, fill]), prefix, low, high, first)


def _many(R, groups, seed):
    rng = np.random.default_rng(seed)
    lengths = rng.integers(0, 300, R)
    n = np.minimum(rng.integers(0, 3, R), lengths)
    return lengths, np.concatenate([[0], np.cumsum(n)]), rng.integers(-1, groups, R) * (R // groups), rng.integers(0, 300, R)


@pytest.mark.parametrize("R,groups", [(40, 7), (1025, 1), (2048, 2048), (20000, 300), (200000, 1), (200000, 50000), (1 << 20, 5)])
def test_sharing_of_many_requests(gpu, R, groups):
    """Work that does not grow with the square of the requests."""
    for x, y in zip(_plan(*_many(300, 20, R), 16, 900), so.sharing(*_many(300, 20, R), 16, 900)):
        assert np.array_equal(x, y)
    args = _many(R, groups, R)
    T = int(args[1][-1]) + 3
    got = paged.sharing(*(dev(x, gpu) for x in args), 16, T)
    for g, w, name in zip(got, _plan(*args, 16, T), paged.Sharing._fields):
        assert np.array_equal(host(g), w), name


def falling(q_start, n, rng):
    """Starts that are the given ones once those that fall back are taken as the largest before."""
    raw = q_start.copy()
    at = 1 + np.flatnonzero(n == 0)
    raw[at] -= rng.integers(0, 50, len(at))
    raw[0] -= 4
    assert np.array_equal(np.maximum.accumulate(np.maximum(raw, 0)), q_start) and (np.diff(raw) < 0).any()
    return raw


@pytest.mark.parametrize("R,groups", [(6, 2), (64, 3), (65, 9), (1000, 40), (1024, 5), (1025, 5), (5000, 99)])
def test_sharing_of_starts_that_fall_back(gpu, R, groups):
    lengths, q_start, holders, shared = _many(R, groups, R)
    T, rng = int(q_start[-1]) + 2, np.random.default_rng(R)
    raw = falling(q_start, np.diff(q_start), rng)
    got = paged.sharing(dev(lengths, gpu), dev(raw, gpu), dev(holders, gpu), dev(shared, gpu), 16, T)
    for g, w, name in zip(got, so.sharing(lengths, q_start, holders, shared, 16, T), paged.Sharing._fields):
        assert np.array_equal(host(g), w), name
    raw[R // 2:] = T + 9 - np.arange(R + 1 - R // 2)      # (and past the rows, falling from there)
    want = np.maximum.accumulate(np.clip(raw, 0, T))
    lengths = lengths + np.diff(want)
    got = paged.sharing(dev(lengths, gpu), dev(raw, gpu), dev(holders, gpu), dev(shared, gpu), 16, T)
    for g, w, name in zip(got, so.sharing(lengths, want, holders, shared, 16, T), paged.Sharing._fields):
        assert np.array_equal(host(g), w), name


# ---- attention ------------------------------------------------------------------------------------
class Shared:
    """groups: (prefix tokens, [(new tokens, own tokens with them), ..]); alone: the same of requests without
    a prefix.  The prefixes' holders are requests without new tokens, in front; the others in a random
    order."""

    def __init__(self, gpu, dtype, D, P, Hq, Hkv, groups, alone=(), seed=0, pad=3, poison=NAN, spread=1.0, holder_goes_on=False):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.gpu, self.dtype, self.D, self.P, self.Hq, self.Hkv = gpu, dtype, D, P, Hq, Hkv
        rows = [(i, n, L) for i, (_, m) in enumerate(groups) for n, L in m] + [(-1, n, L) for n, L in alone]
        rng.shuffle(rows)
        first = [p for p, _ in groups]
        self.lengths = np.array([p + 5 * holder_goes_on for p in first] + [(first[i] if i >= 0 else 0) + L for i, _, L in rows])
        self.n = np.array([int(holder_goes_on)] * len(groups) + [n for _, n, _ in rows])
        self.holders = np.array([i if holder_goes_on else -1 for i in range(len(groups))] + [i for i, _, _ in rows])
        self.shared = np.array([p * holder_goes_on for p in first] + [first[i] if i >= 0 else 0 for i, _, _ in rows])
        R = len(self.lengths)
        own = self.shared // P * np.array([r >= len(groups) for r in range(R)])      # columns of another's pages
        held = -(-self.lengths // P)
        col = np.arange(int(held.max()) + 1)[None, :]
        mine = (col >= own[:, None]) & (col < held[:, None])
        self.pages = int(mine.sum()) + 3
        self.tables = np.full(mine.shape, -1, dtype=np.int64)
        self.tables[mine] = rng.permutation(self.pages)[:int(mine.sum())]
        self.tables = np.where(col < own[:, None], self.tables[self.holders], self.tables)
        self.q_start = np.concatenate([[0], np.cumsum(self.n)])
        self.T = int(self.n.sum()) + pad
        self.q = torch.randn(self.T, Hq + 2, D, generator=g).mul_(spread).to(dtype).to(gpu)[:, 1:-1]
        k, v = (torch.randn(self.pages, Hkv, P, D, generator=g).to(dtype) for _ in range(2))
        used = torch.zeros(self.pages, P, dtype=torch.bool)
        for r, L in enumerate(self.lengths):
            t = np.arange(L)
            used[self.tables[r, t // P], t % P] = True
        for x in (k, v):
            x.masked_fill_(~used[:, None, :, None], poison)
        self.k, self.v = k.to(gpu), v.to(gpu)

    def args(self):
        return dev(self.tables, self.gpu), dev(self.lengths, self.gpu), dev(self.q_start, self.gpu)

    def launch(self, mask, **kw):
        args = self.args()
        sharing = _sharing(self.gpu, self.lengths, self.q_start, self.holders, self.shared, self.P, self.T)
        o = torch.full((self.T, self.Hq, self.D), 7.0, dtype=self.dtype, device=self.gpu)
        lse = torch.full((self.Hq, self.T), 7.0, device=self.gpu).t()
        return paged.prepare_shared_attention(self.q, self.k, self.v, *args, sharing, mask, out=o, lse=lse, **kw), o, lse

    def run(self, mask, launches=1, **kw):
        launch, o, lse = self.launch(mask, **kw)
        for _ in range(launches):
            assert launch() is o
        torch.cuda.synchronize()
        return o, lse

    def check(self, mask, scale=None, **kw):
        spec = paged._paged_mask(mask).spec
        o, lse = self.run(mask, scale=scale, **kw)
        want, wl, eo, el = po.attention(f64(self.q), f64(self.k), f64(self.v), self.tables, self.lengths, self.q_start, spec.live,
                                        self.D ** -0.5 if scale is None else scale, self.dtype)
        n = int(self.n.sum())
        assert (f64(o[n:]) == 7).all() and (f64(lse[n:]) == 7).all(), "rows of no request were written"
        off = np.abs(f64(o[:n]) - want[:n])
        over = ~(off <= eo[:n])
        assert not over.any(), (f"o: {int(over.sum())} of {over.size} over the bound, first at {np.argwhere(over)[0]}, "
                                f"{off[over][0]:.3e} > {eo[:n][over][0]:.3e}")
        dead, gl = np.isinf(wl[:n]), f64(lse[:n])
        assert np.array_equal(np.isinf(gl), dead) and (gl[dead] < 0).all() and (f64(o[:n])[dead] == 0).all()
        assert (np.abs(gl[~dead] - wl[:n][~dead]) <= el[:n][~dead]).all()
        return o, lse


def _tokens(n, lo, hi, seed, fresh=1):
    rng = np.random.default_rng(seed)
    return [(fresh, int(x)) for x in rng.integers(max(lo, fresh), hi, n)]


@pytest.mark.parametrize("P", [16, 64, 256])
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 2), (3, 1), (16, 1)])
@pytest.mark.parametrize("dtype,D", TYPES)
def test_groups_of_tokens(gpu, dtype, D, Hq, Hkv, P):
    groups = [(2 * P, _tokens(9, 1, 70, 1)), (P, [(1, 1), (2, 17)]), (4 * P, _tokens(3, 1, 40, 2)), (P, [(1, 30)]), (3 * P, [])]
    Shared(gpu, dtype, D, P, Hq, Hkv, groups, [(1, 1), (3, 50), (0, 20)], seed=P + Hq).check(pm.Causal())


@pytest.mark.parametrize("dtype,D,Hq,Hkv,prefix", [(torch.bfloat16, 128, 8, 2, 6016), (torch.float16, 64, 4, 4, 3008),
                                                   (torch.float32, 64, 4, 2, 2000), (torch.bfloat16, 128, 4, 4, 400)])
def test_a_long_prefix_is_split(gpu, dtype, D, Hq, Hkv, prefix):
    Shared(gpu, dtype, D, 16, Hq, Hkv, [(prefix, _tokens(40, 1, 300, 5))], _tokens(4, 1, 2000, 6)).check(pm.Causal())
    Shared(gpu, dtype, D, 16, Hq, Hkv, [(prefix, _tokens(3, 1, 300, 5))]).check(pm.Causal())


@pytest.mark.parametrize("dtype,D", TYPES)
def test_chunks_behind_prefixes(gpu, dtype, D):
    groups = [(320, [(100, 100), (33, 40), (1, 7), (64, 300)]), (64, [(257, 260), (1, 1), (5, 5)])]
    Shared(gpu, dtype, D, 32, 8, 2, groups, [(70, 90), (1, 400)]).check(pm.Causal())
    Shared(gpu, dtype, D, 32, 8, 2, groups, [(70, 90), (1, 400)]).check(pm.Causal(), scale=0.3)


MASKS = [pm.SlidingWindow(1), pm.SlidingWindow(90), pm.SinksWindow(4, 30), pm.SinksWindow(70, 16), pm.Dilated(8),
         pm.LocalStrided(20, 16), pm.TwoBand(16, 100), pm.PrefixLM(90), MaskSpec(((7, 0, 0, 0),)),
         MaskSpec(((0, 0, 0, 0),), ((1, 40, 0, 0),)), MaskSpec(((1, 9, 0, 0), (6, 33, 0, 0)), ((2, 3, 0, 0),)),
         MaskSpec(((0, 0, 0, 0),), ((7, 0, 0, 0),)), MaskSpec(((1, 0, 0, 0),))]


@pytest.mark.parametrize("mask", MASKS, ids=lambda m: getattr(m, "name", str(getattr(m, "include", m))))
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64)])
def test_masks(gpu, dtype, D, mask):
    """Evaluated at each row's own position, over a prefix whose rows are at many."""
    groups = [(160, _tokens(7, 1, 90, 3) + [(4, 9), (40, 77)]), (32, [(1, 1), (2, 30)])]
    Shared(gpu, dtype, D, 16, 8, 2, groups, [(1, 120), (20, 33)], seed=5).check(mask)


def test_the_holder_goes_on(gpu):
    """The request that holds the prefix has tokens of its own, and others share less of it than some."""
    b = Shared(gpu, torch.bfloat16, 128, 16, 8, 2, [(160, _tokens(5, 1, 60, 3)), (48, _tokens(2, 2, 9, 4, 2))], [(1, 30)],
               holder_goes_on=True)
    b.check(pm.Causal())
    members = np.flatnonzero((b.holders == 0) & (np.arange(len(b.holders)) != 0))
    b.shared[members[0]] = 64       # (whose other pages happen to be the same)
    b.check(pm.Causal())


def test_many_requests_and_heads(gpu):
    rng = np.random.default_rng(0)
    for R, Hq, Hkv in ((200, 4, 2), (64, 64, 1), (30, 40, 40)):
        groups = [(16 * int(rng.integers(1, 9)), _tokens(R // 5, 1, 40, i)) for i in range(4)]
        Shared(gpu, torch.float16, 64, 16, Hq, Hkv, groups, _tokens(R // 5, 1, 90, 9), seed=R).check(pm.Causal())


def test_more_requests_than_a_work_group_has_threads(gpu):
    rng = np.random.default_rng(1)
    groups = [(16 * int(rng.integers(1, 4)), _tokens(int(rng.integers(1, 40)), 1, 20, i)) for i in range(60)]
    Shared(gpu, torch.float16, 64, 16, 2, 1, groups, _tokens(300, 1, 30, 9), seed=1).check(pm.Causal())


def test_offsets_past_32_bits(gpu):
    """Pages whose bytes lie past 4 GiB, for prefix and own keys."""
    b = Shared(gpu, torch.bfloat16, 128, 256, 8, 8, [(2048, _tokens(8, 1, 600, 1)), (256, [(200, 300), (1, 9)])], [(1, 700)])
    far = 8400                                  # pages of 512 KiB: 4.1 GiB
    k, v = (torch.empty(far + b.pages, 8, 256, 128, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    k[far:], v[far:] = b.k, b.v
    want, wl = b.run(pm.Causal())
    b.k, b.v, b.tables = k, v, np.where(b.tables >= 0, b.tables + far, b.tables)
    o, lse = b.run(pm.Causal())
    assert torch.equal(o, want) and torch.equal(lse, wl)


@pytest.mark.parametrize("dtype,D", TYPES)
def test_steps_of_many_rows(gpu, dtype, D):
    """More rows times heads than have a work-group each to merge them: tokens, drafts and chunks."""
    groups = [(320, [(300, 300), (33, 40), (1, 7), (64, 300)]), (64, [(257, 260), (1, 1), (5, 5)]), (160, _tokens(20, 1, 90, 3))]
    b = Shared(gpu, dtype, D, 32, 16, 4, groups, [(70, 90), (1, 400), (3, 3)])
    assert b.T * b.Hq > 8192
    o, lse = b.check(pm.Causal())
    again = b.run(pm.Causal())
    assert torch.equal(again[0], o) and torch.equal(again[1], lse)
    b.check(pm.SinksWindow(20, 100))
    b = Shared(gpu, dtype, D, 16, 16, 16, [(96, _tokens(700, 1, 30, 5)), (32, _tokens(3, 1, 9, 2))], seed=2)
    assert b.T * b.Hq > 8192
    b.check(pm.Causal())


@pytest.mark.parametrize("dtype,D,fresh", [(torch.bfloat16, 128, 1), (torch.float16, 64, 40), (torch.float32, 64, 3)])
@pytest.mark.parametrize("members", [9, 80, 1200])
def test_starts_that_fall_back(gpu, dtype, D, fresh, members):
    """Taken alike by the plan, both parts of the attention and the merge: as the starts that they stand for."""
    if members == 1200 and fresh > 3:
        fresh = 3
    rng = np.random.default_rng(members)
    rows = [(int(n), int(n) + int(x)) for n, x in zip(rng.integers(0, fresh + 1, members), rng.integers(1, 60, members))]
    b = Shared(gpu, dtype, D, 16, 4, 2, [(96, rows[::2]), (32, rows[1::2])], [(fresh, 50), (0, 20), (1, 3)], seed=members)
    want, wl = b.check(pm.Causal())
    starts, b.q_start = b.q_start, falling(b.q_start, b.n, rng)
    args = b.args()
    sharing = paged.sharing(args[1], args[2], dev(b.holders, gpu), dev(b.shared, gpu), 16, b.T)
    for g, w in zip(sharing, so.sharing(b.lengths, starts, b.holders, b.shared, 16, b.T)):
        assert np.array_equal(host(g), w)
    o, lse = torch.full_like(want, 7.0), torch.full_like(wl, 7.0)
    paged.shared_attention(b.q, b.k, b.v, *args, sharing, pm.Causal(), out=o, lse=lse)
    assert torch.equal(o, want) and torch.equal(lse, wl)


@pytest.mark.parametrize("most", [0, 1, 40, 10000])
def test_any_hint_gives_right_results(gpu, most):
    Shared(gpu, torch.bfloat16, 128, 32, 8, 2, [(320, [(1, 5), (90, 100), (3, 40)])], [(1, 90), (33, 33)]).check(pm.Causal(), max_fresh=most)


def test_equal_to_attention_without_sharing(gpu):
    """Requests that share nothing: the plain call's result, bit for bit."""
    b = Shared(gpu, torch.bfloat16, 128, 16, 8, 2, [], [(1, 300), (40, 200), (3, 77), (0, 9)])
    o, lse = b.run(pm.Causal())
    lse2 = torch.empty_like(lse)
    o2 = paged.attention(b.q, b.k, b.v, *b.args(), pm.Causal(), lse=lse2)
    n = int(b.n.sum())
    assert torch.equal(o[:n], o2[:n]) and torch.equal(lse[:n], lse2[:n])


@pytest.mark.parametrize("what", [NAN, INF])
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64)])
@pytest.mark.parametrize("fresh", [1, 30])
def test_masked_places_may_hold_anything(gpu, dtype, D, fresh, what):
    """A key of the prefix that some rows do not see: those stay as they were."""
    mask = pm.SinksWindow(2, 40)
    groups = [(160, [(fresh, x) for x in (fresh, 35, 36, 90, 200)])]
    make = lambda: Shared(gpu, dtype, D, 16, 8, 4, groups, [(1, 50)], seed=1)  # noqa: E731
    clean, lse0 = make().run(mask)
    b = make()
    t = 155
    page = int(b.tables[0, t // 16])
    b.v[page, :, t % 16, ::3] = what
    b.k[page, :, t % 16, 0] = what
    o, lse = b.run(mask)
    seen = np.concatenate([np.repeat(b.holders >= 0, b.n) & mask.live(
        np.concatenate([np.arange(L - n, L) for L, n in zip(b.lengths, b.n)]), t), np.zeros(b.T - int(b.n.sum()), dtype=bool)])
    assert seen.any() and not seen.all()
    d = torch.as_tensor(~seen, device=gpu)
    # (sums of some may be taken in another order, of at most 400 terms of |v| p; both round to the type)
    most = 800 * 2.0 ** -24 * 6
    assert torch.equal(lse[d], lse0[d])
    assert ((o[d].float() - clean[d].float()).abs() <= most + 2 * po.HALF_STEP[dtype] * clean[d].float().abs()).all()
    assert not torch.isfinite(o[~d].float()).all()


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 128)])
@pytest.mark.parametrize("n", [1, 50])
@pytest.mark.parametrize("sign", [1, -1])
def test_huge_scores_on_both_sides(gpu, dtype, D, n, sign):
    """Scores at 1e9 (f16) or 1e31, the same for all keys: prefix and own keys share the row equally."""
    big = (6e4, 1.6e4) if dtype == torch.float16 else (2.0 ** 60, 2.0 ** 44)
    b = Shared(gpu, dtype, D, 16, 4, 2, [(320, [(n, n), (n, 200)])], poison=0.0, pad=0)
    b.q.zero_()
    b.q[..., 0] = big[0]
    b.k.zero_()
    b.k[..., 0] = sign * big[1]
    o, lse = b.run(pm.Causal())
    for r in (1, 2):
        t = np.arange(b.lengths[r])
        v = f64(b.v)[b.tables[r, t // 16], :, t % 16].repeat(2, axis=1)
        for i in range(n):
            m = b.lengths[r] - n + i + 1
            got = f64(o)[b.q_start[r] + i]
            want, mass = v[:m].mean(0), np.abs(v[:m]).mean(0)
            assert (np.abs(got - want) <= 1.01 * po.HALF_STEP[dtype] * (np.abs(want) + mass) + 2.0 ** -18 * mass).all()
            wl = sign * big[0] * big[1] * D ** -0.5 + np.log(m)
            assert np.abs(f64(lse)[b.q_start[r] + i] - wl).max() <= 2.0 ** -18 + 2.0 ** -22 * abs(wl)


def test_prefixes_without_pages(gpu):
    """Entries that name no page: their keys are dead."""
    b = Shared(gpu, torch.bfloat16, 128, 16, 8, 2, [(96, _tokens(6, 1, 40, 1))], [(1, 5)])
    b.tables[:, 2] = -1
    b.tables[b.holders == 0, 4] = b.tables[0, 4] = 1 << 30
    b.check(pm.Causal())


def test_a_sharing_of_another_step_stays_in_bounds(gpu):
    """Entries out of range give other results and nothing worse: rows of no request stay."""
    b = Shared(gpu, torch.float16, 64, 16, 4, 2, [(96, _tokens(6, 1, 40, 1)), (32, _tokens(3, 1, 9, 2))], [(50, 60)])
    rng = np.random.default_rng(0)
    R = len(b.lengths)
    for _ in range(4):
        odd = lambda n: dev(rng.choice([-(1 << 31), -5, 0, 1, 7, 30, 97, 1 << 20, (1 << 31) - 1], n), gpu)  # noqa: E731
        s = paged.Sharing(odd(R + 1), odd(b.T), odd(b.T), odd(R), odd(R), odd(R), odd(R))
        for mask in (pm.Causal(), pm.SlidingWindow(20)):
            o = torch.full((b.T, b.Hq, b.D), 7.0, dtype=b.dtype, device=gpu)
            paged.shared_attention(b.q, b.k, b.v, *b.args(), s, mask, out=o)
            torch.cuda.synchronize()
            assert (o[int(b.n.sum()):] == 7).all()


def test_runs_of_a_launch_and_replays(gpu):
    b = Shared(gpu, torch.bfloat16, 128, 16, 8, 2, [(4000, _tokens(20, 1, 300, 5))], [(60, 900)])
    want, wl = b.run(pm.Causal())
    launch, o, lse = b.launch(pm.Causal())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        launch()
    for i in range(5):
        o.fill_(7.0)
        lse.fill_(7.0)
        graph.replay() if i % 2 == 0 else launch()
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(lse, wl), i


def test_two_calls_at_once(gpu):
    a = Shared(gpu, torch.bfloat16, 128, 16, 8, 2, [(4000, _tokens(20, 1, 300, 5))], seed=1)
    c = Shared(gpu, torch.float16, 64, 64, 4, 4, [(1024, _tokens(5, 40, 300, 5, 40))], seed=2)
    want = [x.run(pm.Causal()) for x in (a, c)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    made = [x.launch(pm.Causal()) for x in (a, c)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (launch, _, _) in zip(streams, made):
            with torch.cuda.stream(s):
                launch()
                launch()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w[0]) and torch.equal(lse, w[1]) for (_, o, lse), w in zip(made, want))


def test_refusals(gpu):
    b = Shared(gpu, torch.bfloat16, 128, 16, 8, 2, [(96, _tokens(6, 1, 40, 1))])
    t, n, s = b.args()
    w = paged.sharing(n, s, dev(b.holders, gpu), dev(b.shared, gpu), 16, b.T)
    call = lambda **kw: paged.shared_attention(**{**dict(q=b.q, k=b.k, v=b.v, tables=t, lengths=n, q_start=s, sharing=w,  # noqa: E731
                                                         mask=pm.Causal()), **kw})
    call()
    for i, bad in enumerate(w):
        with pytest.raises(ValueError):
            call(sharing=w._replace(**{w._fields[i]: bad[:-1]}))
        with pytest.raises(TypeError):
            call(sharing=w._replace(**{w._fields[i]: bad.long()}))
        with pytest.raises(RuntimeError):
            call(sharing=w._replace(**{w._fields[i]: bad.cpu()}))
    with pytest.raises(ValueError):
        call(scale=0.0)
    with pytest.raises(ValueError):
        call(q=b.q[:, :3])
    with pytest.raises(RuntimeError, match="overlap"):
        call(out=b.q)
    with pytest.raises(ValueError):
        paged.sharing(n, s, dev(b.holders, gpu), dev(b.shared, gpu), 20, b.T)
    with pytest.raises(ValueError):
        paged.sharing(n, s[:-1], dev(b.holders, gpu), dev(b.shared, gpu), 16, b.T)
    with pytest.raises(RuntimeError, match="overlap"):
        paged.sharing(n, s, dev(b.holders, gpu), dev(b.shared, gpu), 16, b.T, out=w._replace(first=w.high))


# ---- the cache ----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,D,P,G", [(torch.bfloat16, 128, 16, 4), (torch.float32, 64, 32, 1)])
def test_serving_requests_that_share(gpu, dtype, D, P, G):
    """A prompt is shared, by requests that come and go while its holder goes on, one of which shares it
    further; every step against float64 over what each request holds, and no page twice or lost."""
    R, H = 7, 2
    spec = paged._paged_mask(pm.Causal()).spec
    cache = paged.PagedKVCache(R, 400, 4 * 400 // P + 4, H, D, dtype, P, 1, gpu)
    g = torch.Generator().manual_seed(P)
    kept = [np.zeros((2, 0, H, D)) for _ in range(R)]
    n = 3 * P
    plan = [[n + 5, 0, 0, 9, 0, 0, 0], ("share", 0, [1, 2, 5], n), [1, 1, 20, 1, 0, 1, 0], [1, 1, 1, 1, 0, 0, 0],
            ("share", 1, [4], 2 * P), [0, 40, 1, 1, 1, 1, 0], ("finish", [2]), [1, 1, 0, 1, 1, 1, 0], ("share", 0, [2, 6], P),
            [1, 1, 3, 1, 1, 1, 30], ("finish", [1, 2, 4, 5, 6]), [1, 9, 0, 1, 0, 0, 0], ("finish", [0, 3]),
            [2, 1, 0, 0, 0, 50, 0]]
    for what in plan:
        if what[0] == "share":
            cache.share(what[1], what[2], what[3])
            for m in what[2]:
                kept[m] = kept[what[1]][:, :what[3]]
            continue
        if what[0] == "finish":
            cache.finish([r in what[1] for r in range(R)])
            for m in what[1]:
                kept[m] = np.zeros((2, 0, H, D))
        else:
            T = sum(what) + 2
            step = cache.begin(what, T)
            starts = np.concatenate([[0], np.cumsum(what)])
            kn, vn, q = (torch.randn(T, x, D, generator=g).to(dtype).to(gpu) for x in (H, H, H * G))
            cache.append(kn, vn, step)
            o = cache.attend(q, pm.Causal(), step, out=torch.zeros_like(q))
            for r in range(R):
                mine = slice(starts[r], starts[r + 1])
                kept[r] = np.concatenate([kept[r], np.stack([f64(kn), f64(vn)])[:, mine]], axis=1)
                if what[r]:
                    kv = kept[r].transpose(0, 2, 1, 3)[:, None]
                    want, _, eo, _ = po.attention(f64(q)[mine], kv[0], kv[1], np.zeros((1, 1), dtype=int), [kept[r].shape[1]],
                                                  [0, what[r]], spec.live, D ** -0.5, dtype)
                    assert (np.abs(f64(o)[mine] - want) <= eo).all(), (what, r)
        assert host(cache.lengths).tolist() == [x.shape[1] for x in kept]
        used = np.unique(host(cache.tables)[host(cache.tables) >= 0])
        free = host(cache.free_list)[:int(cache.free_count)]
        assert sorted(np.concatenate([used, free]).tolist()) == list(range(cache.pages))
    cache.check()


def test_prefixes_that_cannot_be_shared_or_finished(gpu):
    make = lambda: paged.PagedKVCache(5, 200, 60, 2, 64, torch.float16, 16, device=gpu)  # noqa: E731
    for bad in ((0, [0], 16), (0, [9], 16), (5, [1], 16), (0, [1], 17), (0, [1], 0), (0, [1], 416)):
        with pytest.raises(ValueError):
            make().share(*bad)
    for holder, members, tokens in ((0, [2], 48), (1, [2], 16), (0, [1, 2], 32), (0, [4], 16)):
        c = make()
        c.begin([40, 3, 0, 0, 0])
        c.share(0, [3], 32)
        if 4 in members:
            c.share(3, [4], 32)                 # (a second share of the same row)
        before = [host(x).tolist() for x in (c.tables, c.lengths, c.holders, c.shared)]
        c.check()
        c.share(holder, members, tokens)
        after = [host(x).tolist() for x in (c.tables, c.lengths, c.holders, c.shared)]
        ok = [m for m in members if (holder, m, tokens) == (0, 2, 32)]
        for r in range(5):
            if r not in ok:
                assert [x[r] for x in before] == [x[r] for x in after], r
        with pytest.raises(RuntimeError, match="shared"):
            c.check()
    c = make()
    c.begin([40, 3, 0, 0, 0])
    c.share(0, [3], 32)
    c.finish([True, True, False, False, False])
    assert host(c.lengths).tolist() == [40, 0, 0, 32, 0] and int(c.free_count) == 57
    with pytest.raises(RuntimeError, match="finished before"):
        c.check()
    c.finish([False, False, False, True, False])
    assert int(c.free_count) == 57
    c.finish([True] * 5)
    assert int(c.free_count) == 60 and (c.tables == -1).all() and (c.holders == -1).all() and (c.shared == 0).all()


def test_a_prefix_with_pages_given_back_is_not_shared(gpu):
    c = paged.PagedKVCache(3, 200, 30, 2, 64, torch.float16, 16, device=gpu)
    c.begin([100, 0, 0])
    c.trim(window=20)
    c.check()
    c.share(0, [1], 32)
    assert host(c.lengths).tolist() == [100, 0, 0] and host(c.holders).tolist() == [-1] * 3 and (c.tables[1] == -1).all()
    with pytest.raises(RuntimeError, match="shared"):
        c.check()


def test_a_captured_finish_keeps_what_is_shared_later(gpu):
    """finish and trim captured before the first prefix is shared, replayed after."""
    c = paged.PagedKVCache(4, 200, 40, 2, 64, torch.float16, 16, device=gpu)
    done = torch.zeros(4, dtype=torch.bool, device=gpu)
    c.begin([100, 0, 0, 20])
    end, cut = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(end):
        c.finish(done)
    with torch.cuda.graph(cut):
        c.trim(window=20)
    c.share(0, [1, 2], 64)
    c.begin([0, 5, 9, 1])
    prefix = host(c.tables)[0, :4]
    for ended, free in (((), 30), ((1,), 31), ((0, 3), 33), ((2,), 34), ((0,), 40)):
        done.zero_()
        done[list(ended)] = True
        end.replay()
        cut.replay()
        torch.cuda.synchronize()
        tables = host(c.tables)
        ids = np.concatenate([np.unique(tables[tables >= 0]), host(c.free_list)[:int(c.free_count)]])
        assert sorted(ids.tolist()) == list(range(40)) and int(c.free_count) == free, ended
        if ended != (0,):
            assert np.array_equal(tables[0, :4], prefix)
    with pytest.raises(RuntimeError, match="finished before"):   # (0, while 2 went on)
        c.check()


class _Count(TorchDispatchMode):
    """Counts torch's operations but those that only make or view a tensor."""

    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        name = func.overloadpacket.__name__
        if name not in ("empty", "view", "detach", "slice", "select", "alias", "unsqueeze", "expand"):
            self.names.append(name)
        return func(*args, **(kwargs or {}))


def test_a_cache_that_never_shares_gives_pages_back_in_few_launches(gpu):
    """Captured or not, as many as before requests could share."""
    c = paged.PagedKVCache(3, 200, 40, 2, 64, torch.float16, 16, device=gpu)
    c.begin([100, 40, 90])
    done = torch.zeros(3, dtype=torch.bool, device=gpu)
    torch.cuda.synchronize()
    for what, most in ((lambda: c.finish(done), 7), (lambda: c.trim(50), 8)):
        for captured in (False, True):
            count = _Count()
            if captured:
                with torch.cuda.graph(torch.cuda.CUDAGraph()), count:
                    what()
            else:
                with count:
                    what()
            assert len(count.names) <= most, count.names


@pytest.mark.parametrize("R,cols", [(1, 3), (7, 20), (64, 5), (1500, 70)])
def test_finish_against_numpy(gpu, R, cols):
    """Random members, holders and requests of their own, any of them done: twice, the second time captured."""
    P, rng = 16, np.random.default_rng(R)
    c = paged.PagedKVCache(R, cols * P, R * cols + 5, 1, 64, torch.float16, P, device=gpu)
    for captured in (False, True):
        held = rng.integers(0, cols + 1, R)
        lengths, holders, shared = held * P - rng.integers(0, P, R) * (held > 0), np.full(R, -1), np.zeros(R, dtype=np.int64)
        tables, next_page = np.full((R, cols), -1), 0
        for r in range(R):
            g = int(rng.integers(0, R))
            n = int(rng.integers(1, cols + 1))
            if g < r and holders[g] in (-1, g) and lengths[g] >= n * P and held[r] >= n and rng.random() < 0.7:
                holders[r], holders[g], shared[r], shared[g] = g, g, n * P, max(shared[g], n * P)
                tables[r, :n] = tables[g, :n]
            else:
                n = 0
            tables[r, n:held[r]] = next_page + np.arange(held[r] - n)
            next_page += held[r] - n
        pages = rng.permutation(c.pages)
        tables = np.where(tables < 0, -1, pages[tables])
        for x, y in ((c.lengths, lengths), (c.holders, holders), (c.shared, shared), (c.tables, tables)):
            x.copy_(dev(y, gpu))
        c.free_list[:c.pages - next_page] = dev(pages[next_page:], gpu)
        c.free_count.fill_(c.pages - next_page)
        c.failed.zero_()
        done = rng.random(R) < 0.6
        self_ = np.arange(R)
        member = (holders >= 0) & (holders != self_)
        busy = np.zeros(R, dtype=bool)
        busy[holders[member & ~done]] = True
        go = done & ~busy
        d = torch.as_tensor(done, device=gpu)
        if captured:
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                c.finish(d)
            graph.replay()
        else:
            c.finish(done.tolist())
        torch.cuda.synchronize()
        assert np.array_equal(host(c.lengths), np.where(go, 0, lengths)) and np.array_equal(host(c.shared), np.where(go, 0, shared))
        assert np.array_equal(host(c.holders), np.where(go, -1, holders))
        assert np.array_equal(host(c.tables), np.where(go[:, None], -1, tables))
        assert int(c.failed) == (paged.SHARED if (done & busy).any() else 0)
        used = np.unique(host(c.tables)[host(c.tables) >= 0])
        free = host(c.free_list)[:int(c.free_count)]
        assert sorted(np.concatenate([used, free]).tolist()) == list(range(c.pages))
