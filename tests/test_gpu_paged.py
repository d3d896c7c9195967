"""Serving from a paged cache (polyhedral_amd.paged) on the device: tables, free list, append and
attention against tests/paged_oracle.py, alone and together."""
import numpy as np
import pytest
import torch

from polyhedral_amd import _lib, paged
from polyhedral_amd.polyattn import masks as pm
from polyhedral_amd.spec import MaskSpec
from tests import paged_oracle as po

pytestmark = pytest.mark.gpu

I32 = torch.int32
NAN, INF = float("nan"), float("inf")


def dev(x, gpu):
    return torch.as_tensor(np.ascontiguousarray(x), dtype=I32).to(gpu)


def host(t):
    return t.detach().cpu().numpy().astype(np.int64)


# ---- tables -----------------------------------------------------------------------------
def _pool(rng, before, P, cols, spare, n_dead=0):
    """Tables that hold `before` tokens per request in random pages, and a free list of the rest."""
    n = int((-(-before // P)).sum())
    ids = rng.permutation(n + spare)
    tables = np.full((len(before), cols), -1, dtype=np.int64)
    tables[np.arange(cols)[None, :] < (-(-before // P))[:, None]] = ids[:n]
    free = np.concatenate([ids[n:], np.full(n, -7)])   # entries past the count are never read
    return tables, free, spare


def _check_step(gpu, before, fresh, tables, free, count, P, tokens, pitch_pad=0):
    R, cols = tables.shape
    wide = np.full((R, cols + pitch_pad), -99)
    wide[:, :cols] = tables
    t = dev(wide, gpu)[:, :cols]
    step = paged.build_tables(dev(before, gpu), dev(fresh, gpu), t, dev(free, gpu), dev([count], gpu), P, tokens)
    want = po.tables_step(before, fresh, tables, free, count, P, tokens)
    for got, w, name in zip(step, want, paged.TableStep._fields):
        assert np.array_equal(host(got), np.atleast_1d(w)), name
    assert np.array_equal(host(t), want[6])
    return step, want


@pytest.mark.parametrize("R,top,fresh_hi,pad,P", [
    (1, 1, 1, 0, 16), (1, 100, 400, 3, 32), (3, 40, 1, 0, 16), (63, 300, 9, 1, 64), (64, 300, 9, 0, 64), (65, 5, 70, 60, 16),
    (257, 1000, 1, 0, 128), (1025, 200, 4, 5, 256), (2048, 50, 2, 0, 16), (2049, 50, 2, 7, 16), (3001, 90, 3, 0, 32),
    (40, 2000, 900, 11, 16), (2, 0, 9000, 100, 64)])
def test_tables_against_numpy(gpu, R, top, fresh_hi, pad, P):
    rng = np.random.default_rng(R + P)
    before = rng.integers(0, top + 1, R)
    before[rng.random(R) < 0.2] = 0
    on_edge = rng.random(R) < 0.2
    before[on_edge] = before[on_edge] // P * P   # whole pages held
    fresh = rng.integers(0, fresh_hi + 1, R)
    cols = int(-(-(before + fresh).max() // P)) + 2
    need = int((-(-(before + fresh) // P) - -(-before // P)).sum())
    tables, free, count = _pool(rng, before, P, cols, need + int(rng.integers(0, 3)))
    _check_step(gpu, before, fresh, tables, free, count, P, int(fresh.sum()) + pad, pitch_pad=int(rng.integers(0, 4)))


def test_tables_with_nothing_to_do(gpu):
    z = np.zeros(0, dtype=np.int64)
    step, _ = _check_step(gpu, z, z, np.zeros((0, 4), dtype=np.int64), np.arange(3), 3, 16, 5)
    assert host(step.q_start).tolist() == [0]
    _check_step(gpu, np.array([5, 0]), np.array([0, 0]), np.array([[2, -1], [-1, -1]]), np.array([0, 1, -1]), 2, 16, 0)


@pytest.mark.parametrize("case", ["pages", "one page", "count", "count < 0", "length", "negative before", "negative fresh",
                                  "rows", "rows and pages", "huge"])
@pytest.mark.parametrize("R", [5, 3000])
def test_a_step_that_does_not_fit_takes_nothing(gpu, R, case):
    P, cols = 16, 8
    rng = np.random.default_rng(R)
    before, fresh = rng.integers(0, 60, R), rng.integers(0, 30, R)
    need = int((-(-(before + fresh) // P) - -(-before // P)).sum())
    tables, free, count = _pool(rng, before, P, cols, need)
    tokens = int(fresh.sum())
    bits = {"pages": 1, "one page": 1, "count": 1, "count < 0": 1, "rows": 4, "rows and pages": 5}.get(case, 2)
    if case == "pages":
        count = 0
    elif case == "one page":
        count -= 1
    elif case == "count":
        count = len(free) + 1
    elif case == "count < 0":
        count = -1
    elif case == "length":
        fresh[3] = cols * P + 1 - before[3]
        tokens = int(fresh.sum())
    elif case == "negative before":
        before[2] = -1
    elif case == "negative fresh":
        fresh[2] = -3
    elif case == "rows":
        tokens -= 1
    elif case == "rows and pages":
        tokens, count = tokens - 1, need - 1
    else:
        before[0] = fresh[0] = (1 << 31) - 1
    step, _ = _check_step(gpu, before, fresh, tables, free, count, P, max(tokens, 0))
    assert int(step.status) & bits == bits


def test_pages_that_are_none_of_the_cache_give_no_slot(gpu):
    """A half-filled page's entry that is out of range, and a free list that names one."""
    P, before, fresh = 16, np.array([5, 20, 0]), np.array([3, 20, 30])
    tables = np.array([[-1, -1, -1], [1, 1 << 30, -1], [-1, -1, -1]])
    free = np.array([9, 7, -2, 0])
    _check_step(gpu, before, fresh, tables, free, 4, P, 60)


def test_tables_advance_in_place(gpu):
    """lengths = before and free_left = free_count: every run is a step; against numpy, both kernels."""
    for R, tokens in ((7, 40), (2500, 3000), (9, 9000)):
        rng = np.random.default_rng(R)
        P, cols = 16, 12
        lengths, free = np.zeros(R, dtype=np.int64), np.arange(R * 4)
        tables, count = np.full((R, cols), -1, dtype=np.int64), R * 4
        fresh = rng.integers(0, 2, R)   # (rows past the few tokens of a step are padding)
        t, ln, fl, fc = dev(tables, gpu), dev(lengths, gpu), dev(free, gpu), dev([count], gpu)
        new = lambda n: torch.empty(n, dtype=I32, device=gpu)  # noqa: E731
        out = paged.TableStep(ln, new(R + 1), new(tokens), new(tokens), fc, new(1))
        launch = paged.prepare_tables(ln, dev(fresh, gpu), t, fl, fc, P, tokens, out)
        for _ in range(40):
            step = launch()
            lengths, q_start, slots, pos, count, status, tables = po.tables_step(lengths, fresh, tables, free, count, P, tokens)
            for got, w in zip(step, (lengths, q_start, slots, pos, [count], [status])):
                assert np.array_equal(host(got), w)
            assert np.array_equal(host(t), tables)


@pytest.mark.parametrize("R,cols", [(1, 1), (5, 7), (64, 130), (1500, 9), (3, 2000)])
def test_release_against_numpy(gpu, R, cols):
    rng = np.random.default_rng(R * cols)
    n = R * cols + 5
    tables = rng.permutation(n)[:R * cols].reshape(R, cols).astype(np.int64)
    tables[rng.random((R, cols)) < 0.3] = -1
    tables[rng.random((R, cols)) < 0.05] = n + 3     # none of the cache: skipped, left as it is
    first, last = rng.integers(-3, cols + 3, R), rng.integers(-3, cols + 3, R)
    first[0], last[0] = -(1 << 31), (1 << 31) - 1
    held = int(((tables >= 0) & (tables < n)).sum())
    free = np.full(n, -5)
    count = n - held
    free[:count] = np.arange(count) * 3
    for start in (count, count + 1 if held else count):
        t, fl = dev(tables, gpu), dev(free, gpu)
        fc, status = paged.release(dev(first, gpu), dev(last, gpu), t, fl, dev([start], gpu))
        want = po.release(first, last, tables, free, start)
        assert int(status) == want[3] and int(fc) == want[2]
        assert np.array_equal(host(fl), want[1])
        assert np.array_equal(host(t), tables if want[0] is None else want[0])
    # in place, and a second time: nothing is left to give back in these ranges
    t, fl, fc = dev(tables, gpu), dev(free, gpu), dev([count], gpu)
    launch = paged.prepare_release(dev(first, gpu), dev(last, gpu), t, fl, fc, (fc, torch.empty(1, dtype=I32, device=gpu)))
    for _ in range(2):
        launch()
        assert int(fc) == po.release(first, last, tables, free, count)[2]


def test_release_refuses_a_list_that_would_pass_its_length(gpu):
    t, fl, fc = dev([[0, 1]], gpu), dev([2, 3, 9, 9], gpu), dev([3], gpu)
    left, status = paged.release(dev([0], gpu), dev([2], gpu), t, fl, fc)
    assert int(status) == 1 and int(left) == 3 and host(t).tolist() == [[0, 1]] and host(fl).tolist() == [2, 3, 9, 9]


# ---- append -----------------------------------------------------------------------------
@pytest.mark.parametrize("rows_first", [False, True])
@pytest.mark.parametrize("dtype,H,D,P,T", [(torch.bfloat16, 8, 128, 64, 1), (torch.float16, 3, 64, 16, 77),
                                           (torch.float32, 5, 128, 32, 130), (torch.float32, 1, 64, 256, 1000),
                                           (torch.bfloat16, 2, 64, 128, 5000)])
def test_append_writes_the_slots_and_nothing_else(gpu, dtype, H, D, P, T, rows_first):
    rng = np.random.default_rng(T)
    pages = T // P + 3
    shape = (pages, P, H, D) if rows_first else (pages, H, P, D)
    k, v = (torch.randn(shape, device=gpu).to(dtype) for _ in range(2))
    if rows_first:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    slots = rng.permutation(pages * P)[:T]
    slots[rng.random(T) < 0.2] = -1
    slots[-1] = pages * P                       # just past the cache
    # rows of a fused projection: q, k and v of a token side by side
    qkv = torch.randn(T, 3 * H, D, device=gpu).to(dtype)
    kn, vn = qkv[:, H:2 * H], qkv[:, 2 * H:]
    want = [k.clone(), v.clone()]
    rows = np.flatnonzero((slots >= 0) & (slots < pages * P))
    at = torch.as_tensor(slots[rows], device=gpu)
    for w, n in zip(want, (kn, vn)):
        w[at // P, :, at % P] = n[torch.as_tensor(rows, device=gpu)]
    paged.append(kn, vn, dev(slots, gpu), k, v)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


# ---- attention --------------------------------------------------------------------------
class Batch:
    """Requests with new tokens in a cache whose every other row, page and pad row holds NaN."""

    def __init__(self, gpu, dtype, D, P, Hq, Hkv, sizes, seed=0, pad=3, spread=1.0, rows_first=False, poison=NAN):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.gpu, self.dtype, self.D, self.P, self.Hq, self.Hkv = gpu, dtype, D, P, Hq, Hkv
        self.n = np.array([n for n, _ in sizes])
        self.lengths = np.array([L for _, L in sizes])
        held = -(-self.lengths // P)
        self.pages = int(held.sum()) + 3
        cols = int(held.max(initial=0)) + 1
        self.tables = np.full((len(sizes), cols), -1, dtype=np.int64)
        self.tables[np.arange(cols)[None, :] < held[:, None]] = rng.permutation(self.pages)[:int(held.sum())]
        self.q_start = np.concatenate([[0], np.cumsum(self.n)])
        self.T = int(self.n.sum()) + pad
        # fused projection rows: q is a strided view
        self.q = torch.randn(self.T, Hq + 2, D, generator=g).mul_(spread).to(dtype).to(gpu)[:, 1:-1]
        k = torch.randn(self.pages, Hkv, P, D, generator=g).to(dtype)
        v = torch.randn(self.pages, Hkv, P, D, generator=g).to(dtype)
        used = torch.zeros(self.pages, P, dtype=torch.bool)
        for r, L in enumerate(self.lengths):
            t = np.arange(L)
            used[self.tables[r, t // P], t % P] = True
        for x in (k, v):
            x.masked_fill_(~used[:, None, :, None], poison)
        if rows_first:
            k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
            self.k, self.v = (torch.empty_strided(x.shape, x.stride(), dtype=dtype, device=gpu).copy_(x) for x in (k, v))
        else:
            self.k, self.v = k.to(gpu), v.to(gpu)

    def dev(self):
        return dev(self.tables, self.gpu), dev(self.lengths, self.gpu), dev(self.q_start, self.gpu)

    def run(self, mask, scale=None, max_fresh=None, launches=1):
        o = torch.full((self.T, self.Hq, self.D), 7.0, dtype=self.dtype, device=self.gpu)
        lse = torch.full((self.Hq, self.T), 7.0, device=self.gpu).t()
        launch = paged.prepare_attention(self.q, self.k, self.v, *self.dev(), mask, scale, max_fresh, o, lse)
        for _ in range(launches):
            assert launch() is o
        torch.cuda.synchronize()
        return o, lse

    def check(self, mask, spec=None, scale=None, max_fresh=None):
        spec = spec if spec is not None else paged._paged_mask(mask).spec
        o, lse = self.run(mask, scale, max_fresh)
        f = lambda t: t.float().cpu().numpy().astype(np.float64)  # noqa: E731
        want, wl, eo, el = po.attention(f(self.q), f(self.k), f(self.v), self.tables, self.lengths, self.q_start, spec.live,
                                        self.D ** -0.5 if scale is None else scale, self.dtype)
        n = int(self.n.sum())
        assert (f(o[n:]) == 7).all() and (f(lse[n:]) == 7).all(), "rows of no request were written"
        off = np.abs(f(o[:n]) - want[:n])
        over = off > eo[:n]
        assert not over.any(), (f"o: {int(over.sum())} of {over.size} over the bound, first at {np.argwhere(over)[0]}, "
                                f"{off[over][0]:.3e} > {eo[:n][over][0]:.3e}")
        assert np.isfinite(f(o[:n])).all()
        dead = np.isinf(wl[:n])
        gl = f(lse[:n])
        assert np.array_equal(np.isinf(gl), dead) and (gl[dead] < 0).all()
        offl = np.abs(gl[~dead] - wl[:n][~dead])
        assert (offl <= el[:n][~dead]).all(), f"lse off by {offl.max():.3e}"
        assert (f(o[:n])[dead] == 0).all()
        return o, lse


TYPES = [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 64),
         (torch.float32, 128)]
RAGGED = [(1, 1), (1, 2), (0, 40), (1, 15), (2, 16), (1, 17), (3, 33), (1, 64), (5, 65), (0, 0), (16, 16), (1, 129), (7, 250)]


@pytest.mark.parametrize("P", [16, 64, 256])
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 2), (3, 1), (16, 1)])
@pytest.mark.parametrize("dtype,D", TYPES)
def test_ragged_batch(gpu, dtype, D, Hq, Hkv, P):
    Batch(gpu, dtype, D, P, Hq, Hkv, RAGGED, seed=P + Hq).check(pm.Causal())


MASKS = [pm.SlidingWindow(1), pm.SlidingWindow(20), pm.SinksWindow(4, 30), pm.SinksWindow(70, 16), pm.Dilated(8),
         pm.LocalStrided(20, 16), pm.TwoBand(16, 100), pm.PrefixLM(90), MaskSpec(((7, 0, 0, 0),)),
         MaskSpec(((2, 16, 0, 0),), ((1, 40, 0, 0),)), MaskSpec(((1, 9, 0, 0), (6, 33, 0, 0)), ((2, 3, 0, 0),)),
         MaskSpec(((0, 0, 0, 0),), ((7, 0, 0, 0),)), MaskSpec(((1, 0, 0, 0),))]


@pytest.mark.parametrize("mask", MASKS, ids=lambda m: getattr(m, "name", str(getattr(m, "include", m))))
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64)])
def test_masks(gpu, dtype, D, mask):
    sizes = [(1, 200), (4, 131), (9, 9), (1, 1), (20, 300), (150, 410), (3, 33), (1, 500)]
    Batch(gpu, dtype, D, 32, 8, 2, sizes, seed=5).check(mask)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 64), (torch.float32, 128)])
@pytest.mark.parametrize("Hq,Hkv", [(2, 2), (8, 2), (5, 1)])
def test_chunks(gpu, dtype, D, Hq, Hkv):
    sizes = [(100, 100), (33, 400), (1, 700), (257, 513), (64, 64), (0, 10), (128, 1000), (31, 95), (2, 2)]
    b = Batch(gpu, dtype, D, 16, Hq, Hkv, sizes, seed=Hq)
    b.check(pm.Causal())
    b.check(pm.SinksWindow(5, 100))
    b.check(pm.LocalStrided(60, 16))


LATTICES = [pm.Dilated(2), pm.Dilated(16), pm.Dilated(33), pm.Dilated(5000), pm.LocalStrided(40, 16), pm.LocalStrided(0, 64),
            MaskSpec(((2, 16, 0, 0),), ((1, 40, 0, 0),)), MaskSpec(((2, 32, 0, 0), (5, 10, 3, 0))),
            MaskSpec(((2, 8, 0, 0), (2, 12, 0, 0))), MaskSpec(((3, 30, 24, 0),), ((2, 48, 0, 0), (1, 2, 0, 0)))]


@pytest.mark.parametrize("mask", LATTICES, ids=lambda m: getattr(m, "name", str(getattr(m, "include", m))))
@pytest.mark.parametrize("dtype,D,Hq,Hkv", [(torch.bfloat16, 128, 8, 1), (torch.float16, 64, 4, 4), (torch.float32, 64, 4, 2),
                                            (torch.float32, 128, 2, 2)])
def test_lattices_of_few_tokens(gpu, dtype, D, Hq, Hkv, mask):
    """Lists of live keys: none, one, exactly a step's and one more, a band inside the lattice, pages that
    end inside, more keys than a list, several shares, tokens of one tile with lists of their own."""
    sizes = [(1, 1), (1, 16), (1, 17), (2, 40), (3, 512), (1, 513), (5, 700), (1, 2049), (8, 2500), (16, 900), (0, 7), (1, 6000)]
    b = Batch(gpu, dtype, D, 16, Hq, Hkv, sizes, seed=D + Hq)
    b.tables[7, 40:44] = -1
    b.check(mask)


@pytest.mark.parametrize("mask", [pm.Causal(), pm.SinksWindow(64, 1024), pm.LocalStrided(256, 16)], ids=lambda m: m.name)
@pytest.mark.parametrize("dtype,D,sizes", [
    (torch.bfloat16, 128, [(1, 20001)]), (torch.float16, 64, [(1, 9000), (3, 16384), (1, 31), (2, 5000)]),
    (torch.float32, 64, [(1, 6001), (1, 100)]), (torch.bfloat16, 128, [(70, 6001), (1, 3001)])])
def test_long_axis_is_split(gpu, dtype, D, sizes, mask):
    Batch(gpu, dtype, D, 64, 4, 2, sizes, seed=len(sizes)).check(mask)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("tokens", [5, 70])
def test_tokens_beside_a_chunk(gpu, dtype, D, tokens):
    """Few and many long requests of a token beside chunks, whose shares depend on that."""
    sizes = [(1, 2500 + 7 * i) for i in range(tokens)]
    sizes[tokens // 2:tokens // 2] = [(60, 1200), (41, 41)]
    Batch(gpu, dtype, D, 64, 4, 2, sizes, seed=tokens).check(pm.Causal())


@pytest.mark.parametrize("R", [63, 64, 65, 200])
def test_many_requests(gpu, R):
    rng = np.random.default_rng(R)
    sizes = [(int(rng.integers(0, 3)), int(rng.integers(2, 300))) for _ in range(R)]
    sizes[R // 2] = (1, 4000)
    Batch(gpu, torch.bfloat16, 64, 16, 4, 2, sizes, seed=R).check(pm.Causal())


@pytest.mark.parametrize("max_fresh", [0, 1, 40, 10000])
def test_any_hint_gives_right_results(gpu, max_fresh):
    sizes = [(1, 300), (40, 200), (3, 90), (300, 301), (12, 600)]
    Batch(gpu, torch.float16, 128, 32, 8, 2, sizes).check(pm.Causal(), max_fresh=max_fresh)


def test_rows_first_layout_scale_and_large_scores(gpu):
    sizes = [(1, 300), (40, 200), (5, 77)]
    b = Batch(gpu, torch.bfloat16, 128, 32, 8, 2, sizes, rows_first=True)
    b.check(pm.Causal(), scale=0.3)
    # scores of hundreds: one key takes nearly all of a row
    Batch(gpu, torch.float16, 64, 16, 4, 2, sizes, spread=60.0).check(pm.Causal())
    Batch(gpu, torch.float32, 64, 16, 4, 2, sizes, spread=60.0).check(pm.Causal())


def test_scores_far_below_zero_still_sum_to_one(gpu):
    """Every live score at -1e32: softmax does not depend on a shift."""
    b = Batch(gpu, torch.float32, 64, 16, 2, 1, [(1, 40), (3, 20)], poison=0.0)
    b.q.zero_()
    b.q[..., 0] = 1e18
    b.k[..., 0] = -8e14
    o, lse = b.run(pm.Causal())
    for r in range(2):
        for i in range(int(b.n[r])):
            t = np.arange(b.lengths[r] - b.n[r] + i + 1)
            want = b.v[torch.as_tensor(b.tables[r, t // 16], device=gpu), 0, torch.as_tensor(t % 16, device=gpu)].double().mean(0)
            got = o[int(b.q_start[r]) + i].double()
            assert (got - want).abs().max() < 1e-5


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 64), (torch.float32, 128)])
@pytest.mark.parametrize("n", [2, 150])
def test_huge_scores(gpu, dtype, D, n):
    """Scores at 1e9 (f16) or 1e31, of either sign, the same for all keys of a row, or far apart: equal
    ones share the row (their mean, each term rounded to the type at most), and a lower one by an ulp
    is nothing; rows that see such keys first and others later are as if they had not."""
    big = (6e4, 1.6e4) if dtype == torch.float16 else (2.0 ** 60, 2.0 ** 44)
    L, P = 700, 16
    for sign, some in ((-1, False), (1, False), (1, True), (-1, True)):
        b = Batch(gpu, dtype, D, P, 4, 2, [(n, L), (n, n)], poison=0.0)
        b.q.zero_()
        b.q[..., 0] = big[0]
        t = np.arange(L)
        page, off = (torch.as_tensor(x, device=gpu) for x in (b.tables[0, t // P], t % P))
        b.k.zero_()
        b.k[page[:333] if some else page, :, off[:333] if some else off, 0] = sign * big[1]
        o, lse = b.run(pm.Causal())
        assert torch.isfinite(o).all() and torch.isfinite(lse).all()
        v = b.v[page, :, off].double().repeat_interleave(2, dim=1)          # [L, Hq, D]
        top = sign * big[0] * float(b.k.abs().max()) * D ** -0.5 if not some or sign > 0 else 0.0
        for i in (0, n // 2, n - 1):
            m = L - n + i + 1
            keys = v[:m] if not some else (v[:333] if sign > 0 else v[333:m])
            want, mass = keys.mean(0), keys.abs().mean(0)
            u = po.HALF_STEP[dtype]
            assert ((o[i].double() - want).abs() <= 1.01 * u * (want.abs() + mass) + 2.0 ** -18 * mass).all()
            wl = top + np.log(len(keys))
            assert (lse[i].double() - wl).abs().max() <= 2.0 ** -18 + 2.0 ** -22 * abs(wl)


# ---- what is dead contributes nothing -----------------------------------------------------------
@pytest.mark.parametrize("what", [NAN, INF, -INF])
@pytest.mark.parametrize("dtype,D", TYPES)
@pytest.mark.parametrize("n", [1, 6, 90])
def test_masked_places_may_hold_anything(gpu, dtype, D, n, what):
    """One cached key's K and V replaced: the rows it is live for change, the others stay.  Their
    sums may be taken in another order, whose L additions of parts of sum p |v| <= max |v| (sum p =
    1) round by 2^-24 of it each, in either order; then both round to the type, half a step each."""
    L, w = 200, 50
    for t in (L - 1, L - n // 2 - 1, L - n - 3, L - w - n // 2, 3):
        for mask in (pm.SlidingWindow(w), pm.SinksWindow(2, w), pm.LocalStrided(10, 24)):
            b = Batch(gpu, dtype, D, 32, 8, 4, [(n, L), (2, 33)], seed=n)
            clean, lse0 = b.run(mask)
            page, off = int(b.tables[0, t // 32]), t % 32
            live = mask.live(np.arange(L - n, L), t)
            most = 2 * L * 2.0 ** -24 * float(b.v.float().nan_to_num(0).abs().max())
            for k_too in (False, True):
                b.v[page, :, off, ::3] = what
                if k_too:
                    b.k[page, :, off] = NAN
                o, lse = b.run(mask)
                dead_rows = np.concatenate([~live, np.ones(b.T - n, dtype=bool)])
                d = torch.as_tensor(dead_rows, device=gpu)
                assert torch.equal(lse[d], lse0[d])
                assert ((o[d].float() - clean[d].float()).abs() <= most + 2 * po.HALF_STEP[dtype] * clean[d].float().abs()).all()
                hit = o[~d].float()
                if k_too:
                    assert torch.isnan(hit).all()
                elif what != what:
                    assert torch.isnan(hit[..., ::3]).all()
                else:
                    assert (hit[..., ::3] == what).all()
                if not k_too:
                    keep = torch.ones(D, dtype=torch.bool, device=gpu)
                    keep[::3] = False
                    assert torch.equal(lse[~d], lse0[~d])
                    assert (hit[..., keep] - clean[~d][..., keep].float()).abs().max() <= 0.05 if hit.numel() else True


@pytest.mark.parametrize("dtype,D,Hq,Hkv,sizes", [
    (torch.bfloat16, 128, 128, 1, [(1, 300), (3, 77), (0, 5)]), (torch.float32, 64, 96, 1, [(1, 200), (2, 40)]),
    (torch.float16, 64, 40, 40, [(1, 60), (9, 130)]), (torch.bfloat16, 64, 37 * 3, 37, [(2, 50), (50, 90)]),
    (torch.bfloat16, 128, 48, 2, [(1, 3000), (40, 41)])])
def test_many_heads(gpu, dtype, D, Hq, Hkv, sizes):
    b = Batch(gpu, dtype, D, 16, Hq, Hkv, sizes, seed=Hq)
    b.check(pm.Causal())
    b.check(pm.Dilated(16))


def test_nothing_to_attend_to(gpu):
    """No pages, no columns, no requests, no rows."""
    q = torch.ones(3, 4, 64, dtype=torch.float16, device=gpu)
    k = torch.zeros(0, 2, 16, 64, dtype=torch.float16, device=gpu)
    i32 = lambda *x: torch.tensor(x, dtype=I32, device=gpu)  # noqa: E731
    one = torch.zeros(5, 2, 16, 64, dtype=torch.float16, device=gpu)
    for kv, tables in ((k, torch.zeros(1, 4, dtype=I32, device=gpu)), (one, torch.zeros(1, 0, dtype=I32, device=gpu)),
                       (one, torch.full((1, 4), -1, dtype=I32, device=gpu))):
        for most in (0, 100):
            o, lse = torch.full_like(q, 7.0), torch.full((3, 4), 7.0, device=gpu)
            paged.attention(q, kv, kv, tables, i32(50), i32(0, 2), pm.Causal(), max_fresh=most, out=o, lse=lse)
            assert (o[:2] == 0).all() and (lse[:2] == -INF).all() and (o[2] == 7).all() and (lse[2] == 7).all()
    o = torch.full_like(q, 7.0)
    paged.attention(q, one, one, torch.zeros(0, 4, dtype=I32, device=gpu), i32(), i32(0), pm.Causal(), out=o)
    assert (o == 7).all()
    assert paged.attention(q[:0], one, one, torch.zeros(1, 4, dtype=I32, device=gpu), i32(50), i32(0, 0), pm.Causal()).shape == (0, 4, 64)
    paged.append(one[:0, :, 0], one[:0, :, 0], i32(), one, one)
    paged.append(one[:2, :, 0], one[:2, :, 0], i32(0, 5), k, k)


def test_thousands_of_requests_and_pages_in_two_tables(gpu):
    """More requests than a work-group has lanes many times over, some of which read the same pages (a
    prompt that they share)."""
    rng = np.random.default_rng(3)
    sizes = [(int(rng.integers(0, 2)), int(rng.integers(1, 40))) for _ in range(3000)]
    b = Batch(gpu, torch.float16, 64, 16, 2, 1, sizes, seed=3)
    shared = np.flatnonzero(b.lengths > 16)
    b.tables[shared[1:], 0] = b.tables[shared[0], 0]
    b.check(pm.Causal())


def test_entries_that_name_no_page_are_dead(gpu):
    """Table entries out of the cache's range hide their keys, wherever they are; so does a table
    that ends before the length."""
    b = Batch(gpu, torch.bfloat16, 128, 16, 8, 2, [(1, 300), (20, 200), (150, 400), (2, 40)])
    b.tables[0, 3], b.tables[0, 18], b.tables[1, 0], b.tables[1, 12] = -1, b.pages, 1 << 30, -(1 << 31)
    b.tables[2, 5:9], b.tables[3, :] = -1, b.pages + 7
    b.check(pm.Causal())
    for x in (torch.float16, torch.float32):
        c = Batch(gpu, x, 64, 16, 4, 2, [(1, 300), (20, 200), (70, 90)])
        c.tables[0, ::2] = -1
        c.tables[2, 1] = -1
        c.check(pm.Causal())


def test_lengths_and_starts_out_of_range_stay_inside(gpu):
    """Lengths past the table, starts past the rows: clamped (every access stays in the tensors)."""
    b = Batch(gpu, torch.bfloat16, 128, 16, 4, 2, [(2, 50), (1, 30), (3, 10)], pad=0)
    tables, _, _ = b.dev()
    for lengths, starts in (([1 << 30, -5, 10], [0, 2, 3, 6]), ([50, 30, 10], [0, 100, 3, 1 << 30]), ([1, 0, 1], [0, 2, 3, 6]),
                            ([50, 30, 10], [-9, 2, 1, 6])):
        o = torch.zeros(b.T, 4, 128, dtype=torch.bfloat16, device=gpu)
        paged.attention(b.q, b.k, b.v, tables, dev(lengths, gpu), dev(starts, gpu), pm.Causal(), out=o)
    torch.cuda.synchronize()


def test_offsets_past_32_bits(gpu):
    """A cache whose K and V are 6 GiB each, with pages at its very end."""
    P, H, D = 64, 8, 128
    pages = (6 << 30) // (P * H * D * 2)
    b = Batch(gpu, torch.bfloat16, D, P, 2 * H, H, [(1, 500), (130, 300), (3, 70)])
    k, v = (torch.empty(pages, H, P, D, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    at = pages - 1 - 3 * np.arange(b.pages)
    k[torch.as_tensor(at, device=gpu)], v[torch.as_tensor(at, device=gpu)] = b.k, b.v
    want, wl = b.run(pm.Causal())
    b.tables = np.where(b.tables >= 0, at[b.tables], -1)
    b.k, b.v = k, v
    got, gl = b.run(pm.Causal())
    assert torch.equal(got, want) and torch.equal(gl, wl)
    kn = torch.randn(2, H, D, device=gpu).to(torch.bfloat16)
    paged.append(kn, kn, dev([pages * P - 1, (pages - 1) * P], gpu), k, v)
    assert torch.equal(k[-1, :, -1], kn[0]) and torch.equal(v[-1, :, 0], kn[1])


# ---- streams, graphs, devices ----------------------------------------------------------------
def test_same_bits_every_time_and_on_another_stream(gpu):
    b = Batch(gpu, torch.bfloat16, 128, 64, 8, 2, [(1, 9000), (200, 3000), (1, 40)])
    first = b.run(pm.Causal())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        o, lse = b.run(pm.Causal(), launches=3)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(o, first[0]) and torch.equal(lse, first[1])


def test_a_captured_step_replays_for_other_lengths(gpu):
    """Tables, append and attention of one generated token in a graph: each replay is a step of its
    own (lengths advance on the device), against an eager cache stepped beside it."""
    R, H, G, D, P = 5, 2, 4, 128, 16
    g = torch.Generator().manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(gpu)  # noqa: E731
    new = lambda n: torch.empty(n, dtype=I32, device=gpu)  # noqa: E731
    prompt = [40, 1, 15, 16, 70]
    caches = [paged.PagedKVCache(R, 256, 60, H, D, torch.bfloat16, P, device=gpu) for _ in range(2)]
    kp, vp = rnd(sum(prompt), H, D), rnd(sum(prompt), H, D)
    for c in caches:
        step = c.begin(prompt)
        c.append(kp, vp, step)
    a, e = caches
    q, kn, vn = rnd(R, H * G, D), rnd(R, H, D), rnd(R, H, D)
    ones = torch.ones(R, dtype=I32, device=gpu)
    o, lse = torch.zeros(R, H * G, D, dtype=torch.bfloat16, device=gpu), torch.zeros(R, H * G, device=gpu)
    out = paged.TableStep(a.lengths, new(R + 1), new(R), new(R), a.free_count, new(1))
    tables = paged.prepare_tables(a.lengths, ones, a.tables, a.free_list, a.free_count, P, R, out)
    put = paged.prepare_append(kn, vn, out.slots, a.k[0], a.v[0])
    att = paged.prepare_attention(q, a.k[0], a.v[0], a.tables, a.lengths, out.q_start, pm.Causal(), max_fresh=1, out=o, lse=lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tables()
        put()
        att()
    for i in range(30):
        q.copy_(rnd(R, H * G, D))
        kn.copy_(rnd(R, H, D))
        vn.copy_(rnd(R, H, D))
        graph.replay()
        torch.cuda.synchronize()
        step = e.begin([1] * R)
        e.append(kn, vn, step)
        lse_e = torch.empty_like(lse)
        o_e = e.attend(q, pm.Causal(), step, max_fresh=1, lse=lse_e)
        assert torch.equal(a.tables, e.tables) and torch.equal(a.lengths, e.lengths) and torch.equal(a.free_count, e.free_count)
        assert torch.equal(o, o_e) and torch.equal(lse, lse_e), f"replay {i}"
    assert int(out.status) == 0
    e.check()


def test_a_launch_captured_before_its_first_run(gpu):
    """The workspace is cleared by the first run that happens, whether a replay or an eager one; two
    graphs with launches of their own run on two streams at once."""
    b = Batch(gpu, torch.bfloat16, 128, 32, 8, 2, [(1, 6000), (70, 900), (1, 40)])
    want, wl = b.run(pm.Causal())
    outs, graphs, launches = [], [], []
    for _ in range(2):
        o, lse = torch.full_like(want, 7.0), torch.full_like(wl, 7.0)
        junk = torch.full((1 << 26,), 0x5a, dtype=torch.uint8, device=gpu)   # memory that the workspace may get
        del junk
        launch = paged.prepare_attention(b.q, b.k, b.v, *b.dev(), pm.Causal(), out=o, lse=lse)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            launch()
        outs.append((o, lse))
        graphs.append(graph)
        launches.append(launch)
    launches[0]()                                  # eager before any replay
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for i in range(6):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, lse in outs:
            assert torch.equal(o, want) and torch.equal(lse, wl), i
            o.fill_(7.0)
            lse.fill_(7.0)
        torch.cuda.synchronize()


def test_two_calls_at_once(gpu):
    """Calls of different batches on two streams, each with its own workspace."""
    a = Batch(gpu, torch.bfloat16, 128, 16, 8, 2, [(1, 9000), (1, 3000)], seed=1)
    c = Batch(gpu, torch.float16, 64, 64, 4, 4, [(300, 2000), (2, 5000)], seed=2)
    want = [x.run(pm.Causal()) for x in (a, c)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for s, x in zip(streams, (a, c)):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                o = torch.full((x.T, x.Hq, x.D), 7.0, dtype=x.dtype, device=gpu)
                args = x.dev()
                for _ in range(4):
                    paged.attention(x.q, x.k, x.v, *args, pm.Causal(), out=o)
                got.append(o)
        torch.cuda.synchronize()
        assert all(torch.equal(g, w[0]) for g, w in zip(got, want))


# ---- all of it together ----------------------------------------------------------------------
@pytest.mark.parametrize("dtype,D,P,G", [(torch.bfloat16, 128, 16, 4), (torch.float32, 64, 32, 1), (torch.float16, 64, 64, 3)])
@pytest.mark.parametrize("sinks", [False, True])
def test_serving_a_batch(gpu, dtype, D, P, G, sinks):
    """Prompts in chunks, tokens, requests that finish and start again, with a window's pages given
    back: every step's attention against float64 over the tokens kept on the host."""
    R, H, layers = 4, 2, 2
    mask = pm.SinksWindow(10, 40) if sinks else pm.Causal()
    spec = paged._paged_mask(mask).spec
    cache = paged.PagedKVCache(R, 400, 4 * 400 // P + 4, H, D, dtype, P, layers, gpu)
    rng = np.random.default_rng(P)
    g = torch.Generator().manual_seed(P)
    kept = [[np.zeros((2, 0, H, D)) for _ in range(R)] for _ in range(layers)]
    plan = [[50, 3, 0, 17], [1, 60, 33, 0], [1, 1, 1, 1], [70, 0, 1, 200], "finish", [5, 9, 1, 1], [1, 1, 40, 1], [1, 1, 1, 1]]
    for fresh in plan:
        if fresh == "finish":
            cache.finish([False, True, False, True])
            for layer in kept:
                layer[1] = layer[3] = np.zeros((2, 0, H, D))
            continue
        pad = int(rng.integers(0, 4))
        T = sum(fresh) + pad
        step = cache.begin(fresh, T)
        starts = np.concatenate([[0], np.cumsum(fresh)])
        for layer in range(layers):
            kn, vn, q = (torch.randn(T, n, D, generator=g).to(dtype).to(gpu) for n in (H, H, H * G))
            cache.append(kn, vn, step, layer)
            o = cache.attend(q, mask, step, layer, out=torch.zeros_like(q))
            f = lambda t: t.float().cpu().numpy().astype(np.float64)  # noqa: E731
            for r in range(R):
                new = np.stack([f(kn), f(vn)])[:, starts[r]:starts[r + 1]]
                kept[layer][r] = np.concatenate([kept[layer][r], new], axis=1)
                n, L = fresh[r], kept[layer][r].shape[1]
                if not n:
                    continue
                kv = kept[layer][r].transpose(0, 2, 1, 3)[:, None]     # one "page" of the whole request
                want, _, eo, _ = po.attention(f(q)[starts[r]:starts[r + 1]], kv[0], kv[1], np.zeros((1, 1), dtype=int), [L],
                                              [0, n], spec.live, D ** -0.5, dtype)
                assert (np.abs(f(o)[starts[r]:starts[r + 1]] - want) <= eo).all()
        if sinks:
            cache.trim(40, 10)
            held = host(cache.tables) >= 0
            for r, L in enumerate(host(cache.lengths)):
                t = np.arange(held.shape[1] * P)
                need = (t < L) & ((t > L - 40) | (t < 10))     # keys that the next token may see
                assert held[r][np.unique(t[need] // P)].all()
                assert held[r].sum() <= 40 // P + 2 + -(-10 // P)
        used = host(cache.tables)
        used = used[used >= 0]
        free = host(cache.free_list)[:int(cache.free_count)]
        assert sorted(np.concatenate([used, free]).tolist()) == list(range(cache.pages))
    cache.check()


@pytest.mark.parametrize("T", [40, 5000])
def test_a_captured_step_of_a_cache(gpu, T):
    """begin, append and attend of a cache in a graph, replayed for other counts, with requests that
    finish and a window's pages given back eagerly in between: as a second cache without a graph."""
    R, H, G, D, P, layers = 6, 2, 2, 64, 16, 2
    mask = pm.SinksWindow(5, 60)
    a, e = (paged.PagedKVCache(R, 600, 200, H, D, torch.float16, P, layers, gpu) for _ in range(2))
    gen = torch.Generator().manual_seed(T)
    rng = np.random.default_rng(T)
    fresh = torch.zeros(R, dtype=I32, device=gpu)
    kn, vn, q = (torch.zeros(T, n, D, dtype=torch.float16, device=gpu) for n in (H, H, H * G))

    def a_step(cache, out):
        step = cache.begin(fresh, T)
        for layer in range(layers):
            cache.append(kn, vn, step, layer)
            cache.attend(q, mask, step, layer, out=out[layer])
    oa, oe = (torch.zeros(layers, T, H * G, D, dtype=torch.float16, device=gpu) for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a_step(a, oa)
    for i in range(12):
        n = rng.integers(0, 6, R)
        if i % 4 == 0:
            n[int(rng.integers(R))] = 12
        fresh.copy_(torch.as_tensor(n, dtype=I32))
        for x in (kn, vn, q):
            x.copy_(torch.randn(x.shape, generator=gen))
        graph.replay()
        a_step(e, oe)
        for x, y in ((a.tables, e.tables), (a.lengths, e.lengths), (a.free_count, e.free_count), (oa, oe)):
            assert torch.equal(x, y), i
        done = rng.random(R) < 0.1
        for c in (a, e):
            c.finish(done.tolist())
            if i % 3 == 2:
                c.trim(60, 5)
    a.check()
    fresh.fill_(T)   # (does not fit)
    graph.replay()
    with pytest.raises(RuntimeError, match="did not fit"):
        a.check()


def test_a_cache_that_is_full_says_so(gpu):
    cache = paged.PagedKVCache(2, 100, 3, 1, 64, torch.float16, 16, device=gpu)
    cache.begin([20, 10])
    before = cache.tables.clone(), cache.lengths.clone(), int(cache.free_count)
    step = cache.begin([1, 7])
    assert int(step.status) == paged.SHORT_OF_PAGES and (step.slots == -1).all()
    assert torch.equal(cache.tables, before[0]) and torch.equal(cache.lengths, before[1]) and int(cache.free_count) == before[2]
    # a step that was not taken attends nothing and writes nothing
    q = torch.ones(8, 1, 64, dtype=torch.float16, device=gpu)
    o = cache.attend(q, pm.Causal(), step, out=torch.full_like(q, 3.0))
    assert (o == 3).all()
    with pytest.raises(RuntimeError, match="free pages"):
        cache.check()
    big = paged.PagedKVCache(1, 100, 30, 1, 64, torch.float16, 16, device=gpu)
    big.begin([113])
    with pytest.raises(RuntimeError, match="past 112"):
        big.check()


def test_refusals(gpu):
    b = Batch(gpu, torch.bfloat16, 128, 16, 4, 2, [(1, 20), (2, 30)])
    t, ln, qs = b.dev()
    good = dict(q=b.q, k=b.k, v=b.v, tables=t, lengths=ln, q_start=qs, mask=pm.Causal())

    def refused(match, err=ValueError, **change):
        with pytest.raises(err, match=match):
            paged.attention(**{**good, **change})
    refused("head", q=b.q[:, :3])
    refused("must be", q=b.q.float())
    refused("must be", q=b.q[..., :64])
    refused("one of", k=b.k[:, :, :8], v=b.v[:, :, :8])
    refused("one shape", v=b.v[:, :1])
    refused("unit stride", q=torch.zeros(b.T, 128, 4, dtype=torch.bfloat16, device=gpu).transpose(1, 2))
    refused("shape", q_start=qs[:-1])
    refused("int32", lengths=ln.long(), err=TypeError)
    refused("tables must be", tables=t[:1])
    refused("overlap", tables=t[:1].expand(2, -1))
    refused("scale", scale=-1.0)
    refused("max_fresh", max_fresh=-1)
    refused("lse", lse=torch.zeros(4, b.T, device=gpu))
    refused("out must be", out=torch.zeros(1, 4, 128, dtype=torch.bfloat16, device=gpu))
    refused("different lengths", mask=pm.DenseMask(np.ones((4, 4), dtype=bool)))
    refused("GPU only", err=RuntimeError, lengths=ln.cpu())
    refused("aligned", err=_lib.PolyattnError, q=torch.zeros(b.T * 4 * 128 + 8, dtype=torch.bfloat16, device=gpu)[1:b.T * 512 + 1].view(b.T, 4, 128))
    with pytest.raises(ValueError, match="one of"):
        paged.build_tables(ln, ln, t, ln, ln[:1], 20, 4)
    with pytest.raises(ValueError, match="free_count"):
        paged.build_tables(ln, ln, t, ln, ln, 16, 4)
    with pytest.raises(ValueError, match="tokens"):
        paged.build_tables(ln, ln, t, ln, ln[:1], 16, -1)
    with pytest.raises(ValueError, match="share strides"):
        paged.append(b.k[0, :, 0][None], b.v[0, :, 0][None].contiguous().expand(1, 2, 128).clone(), ln[:1], b.k, b.v)
    with pytest.raises(ValueError, match="tokens"):
        paged.PagedKVCache(2, 64, 8, 1, 64, page_size=16, device=gpu).begin(ln)
    with pytest.raises(ValueError, match="one of"):
        paged.PagedKVCache(2, 64, 8, 1, 64, page_size=17, device=gpu)
    with pytest.raises(ValueError, match="D=80"):
        paged.PagedKVCache(2, 64, 8, 1, 80, device=gpu)
    with pytest.raises(TypeError, match="dtype"):
        paged.PagedKVCache(2, 64, 8, 1, 64, dtype=torch.int8, device=gpu)
