"""Chunks of new tokens over a paged cache (polyhedral_amd.paged) where steps of 64 keys are dead
for some of a tile's waves between live ones: every place of a window in a step, gaps of two
bands, wide lattices, pages that are missing; against tests/paged_oracle.py."""
import numpy as np
import pytest
import torch

from polyhedral_amd.polyattn import masks as pm
from polyhedral_amd.spec import MaskSpec
from tests.test_gpu_paged import Batch

pytestmark = pytest.mark.gpu

KINDS = [(torch.bfloat16, 128), (torch.float16, 64)]


@pytest.mark.parametrize("dtype,D", KINDS)
@pytest.mark.parametrize("mask", [pm.SinksWindow(4, 100), pm.SinksWindow(70, 300), pm.SlidingWindow(100), pm.SlidingWindow(20),
                                  pm.SinksWindow(64, 1024)], ids=lambda m: m.name)
def test_windows_at_every_place_in_a_step(gpu, dtype, D, mask):
    """Heads that share no KV head: a tile is 128 tokens, so its last wave's window starts 96 keys
    after the tile's, one or two steps on."""
    first = 1290
    Batch(gpu, dtype, D, 64, 1, 1, [(128, first + 128 + i) for i in range(64)], seed=7).check(mask)


@pytest.mark.parametrize("dtype,D", KINDS)
@pytest.mark.parametrize("Hq,Hkv", [(2, 2), (4, 1)])
@pytest.mark.parametrize("gap", [1, 2, 3, 4, 5, 6])
def test_gaps_between_two_bands(gpu, dtype, D, Hq, Hkv, gap):
    """The near band is 64 wide, the far one starts ``gap`` steps behind it."""
    sizes = [(150, 900 + 21 * i) for i in range(7)] + [(40, 1500), (260, 260)]
    Batch(gpu, dtype, D, 32, Hq, Hkv, sizes, seed=gap).check(pm.TwoBand(64, 64 * (gap + 1), 64))


@pytest.mark.parametrize("dtype,D", KINDS)
@pytest.mark.parametrize("Hq,Hkv,n", [(2, 2, 200), (8, 1, 40)])
@pytest.mark.parametrize("stride", [192, 256, 320])
def test_wide_lattices(gpu, dtype, D, Hq, Hkv, n, stride):
    """Strides of three steps and more, and more rows than the lists of live keys take."""
    b = Batch(gpu, dtype, D, 64, Hq, Hkv, [(n, 2000 + 17 * i) for i in range(5)] + [(1, 900)], seed=stride)
    b.check(pm.Dilated(stride))
    b.check(pm.LocalStrided(32, stride))


@pytest.mark.parametrize("dtype,D", KINDS)
@pytest.mark.parametrize("mask", [pm.Causal(), pm.SlidingWindow(700)], ids=lambda m: m.name)
@pytest.mark.parametrize("steps", [1, 2, 3, 4])
def test_missing_pages_of_whole_steps(gpu, dtype, D, mask, steps):
    """Table entries that name no page over whole steps, first, in the middle and twice."""
    b = Batch(gpu, dtype, D, 64, 4, 2, [(150, 1100), (64, 1000), (200, 1111), (70, 700)], seed=steps)
    b.tables[0, 9:9 + steps] = -1
    b.tables[1, 0:steps] = b.pages + 3
    b.tables[2, 7:7 + steps] = -1
    b.tables[2, 8 + steps:8 + 2 * steps] = -1
    b.tables[3, 2:2 + steps] = -1
    b.check(mask)


@pytest.mark.parametrize("dtype,D", KINDS)
@pytest.mark.parametrize("spec", [MaskSpec(((1, 40, 0, 0),), ((1, 40, 0, 0),)), MaskSpec(((1, 40, 0, 0),), ((1, 39, 0, 0),)),
                                  MaskSpec(((5, 40, 3, 0),), ((1, 40, 0, 0),))], ids=lambda s: str(s.exclude))
def test_rows_whose_steps_are_dead_from_the_first(gpu, dtype, D, spec):
    """A wave's first steps lie before its window, and the terms left out take all of it, or all but
    a key: rows with no live key give 0 and -inf."""
    Batch(gpu, dtype, D, 16, 1, 1, [(128, 1028 + i) for i in range(64)], seed=9).check(spec, spec)


@pytest.mark.parametrize("dtype,D", KINDS)
@pytest.mark.parametrize("products,extra,step", [([(2.0 ** 13, 2.0 ** 12)], (2.0, 0.0, 2.0), 4.0),
                                                 ([(256.0, 45312.0), (16.0, 1824.0)], (1.0, 23.0, 25.0), 2.0)])
def test_huge_scores_in_several_shares(gpu, dtype, D, products, extra, step):
    """Maxima at or past 2^24 in log2 units that differ by a few units from one share of the keys to
    another (2^25 and the next float32; 11629079 and 11629081 on either side of 2^24 ln 2): the weights are
    those of that difference, exp(-4) and exp(-2), whatever the maximum's size.  All sums are exact."""
    n, L, P = 150, 4000, 16
    b = Batch(gpu, dtype, D, P, 2, 1, [(n, L)], poison=0.0)
    t = np.arange(L)
    page, off = (torch.as_tensor(x, device=gpu) for x in (b.tables[0, t // P], t % P))
    for high in (0, 1):                  # the half of the keys with the larger scores
        b.q.zero_()
        b.k.zero_()
        b.v.zero_()
        for d, (x, y) in zip((0, 32), products):
            b.q[..., d] = x
            b.k[page, :, off, d] = y
        b.q[..., 48] = extra[0]
        b.k[page, :, off, 48] = extra[1]
        half = slice(0, L // 2) if high == 0 else slice(L // 2, L)
        b.k[page[half], :, off[half], 48] = extra[2]
        b.v[page[:L // 2], :, off[:L // 2]] = 1.0
        o, lse = b.run(pm.Causal(), scale=1.0)
        for i in (0, n // 2, n - 1):
            m = L - n + i + 1
            lo, hi = float(L // 2), float(m - L // 2)    # keys of either half
            lo, hi = (lo, hi * np.exp(-step)) if high == 0 else (lo * np.exp(-step), hi)
            want = lo / (lo + hi)
            u = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
            # P and o round to the type; the exponentials and their sums by less than 2^-18
            assert (o[i].double() - want).abs().max() <= 1.01 * 2 * u * want + 2.0 ** -17, (high, i, float(o[i, 0, 0]), want)
            # (its maximum and sum in log2 units round by 2 each, the products with the scale's log2 e and
            # with ln 2 by 2^-24 of it and twice that; log of the sum is below 9)
            wl = sum(x * y for x, y in products) + extra[0] * extra[2]
            assert (lse[i].double() - wl).abs().max() <= 9 + 4 + 3 * 2.0 ** -24 * wl
