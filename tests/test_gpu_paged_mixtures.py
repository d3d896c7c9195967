"""Attention over a paged cache (polyhedral_amd.paged) in calls drawn at random: masks of several terms,
pages that are missing, groups, page sizes, layouts and hints, against tests/paged_oracle.py."""
import random

import numpy as np
import pytest
import torch

from polyhedral_amd.spec import CAUSAL, DILATED, FULL, LOCAL_STRIDED, PREFIX_LM, SINKS, TWOBAND, WINDOW, MaskSpec
from tests.test_gpu_paged import Batch

pytestmark = pytest.mark.gpu


def _log(rng, lo, hi):
    return int(round(np.exp(rng.uniform(np.log(lo), np.log(hi)))))


def _term(rng, far):
    return rng.choice([(CAUSAL, 0, 0, 0), (WINDOW, rng.choice([0, _log(rng, 1, far)]), 0, 0), (DILATED, _log(rng, 1, 400), 0, 0),
                       (LOCAL_STRIDED, _log(rng, 1, far), _log(rng, 1, 400), 0),
                       (TWOBAND, _log(rng, 1, 300), _log(rng, 1, far), _log(rng, 1, 300)),
                       (SINKS, _log(rng, 1, far), rng.choice([0, _log(rng, 1, 200)]), 0), (PREFIX_LM, _log(rng, 1, far), 0, 0),
                       (FULL, 0, 0, 0)])


@pytest.mark.parametrize("seed", range(40))
def test_calls_drawn_at_random(gpu, seed):
    """Six calls a seed, most with a chunk among the requests."""
    rng = random.Random(seed)
    for i in range(6):
        dtype = rng.choice([torch.bfloat16, torch.float16, torch.bfloat16, torch.float16, torch.float32])
        D, P, Hkv, G = rng.choice([64, 128]), rng.choice([16, 32, 64, 128, 256]), rng.choice([1, 1, 2, 3]), rng.choice([1, 1, 2, 4, 5, 20])
        R = rng.choice([1, 2, 3, 5, 9, 70])
        top, most = _log(rng, 40, 2500 if R < 20 else 300), _log(rng, 1, 400 if R < 20 else 20)
        sizes = []
        for _ in range(R):
            n = rng.choice([0, 1, rng.randint(0, most), most])
            sizes.append((n, max(n, _log(rng, 1, top))))
        far = rng.choice([50, 300, 2000])
        spec = MaskSpec(tuple(_term(rng, far) for _ in range(rng.choice([1, 1, 2, 3]))),
                        tuple(_term(rng, far) for _ in range(rng.choice([0, 0, 1, 2]))))
        b = Batch(gpu, dtype, D, P, Hkv * G, Hkv, sizes, seed=7 * seed + i, rows_first=rng.random() < 0.3, pad=rng.randint(0, 5))
        for _ in range(rng.choice([0, 0, 1, 3])):
            r, c = rng.randrange(R), rng.randrange(b.tables.shape[1])
            b.tables[r, c:c + rng.randint(1, max(1, 600 // P))] = rng.choice([-1, b.pages, 1 << 30])
        b.check(spec, spec, max_fresh=rng.choice([None, None, 0, 1, 10 ** 6]), scale=rng.choice([None, 0.5]))
