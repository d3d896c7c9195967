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
