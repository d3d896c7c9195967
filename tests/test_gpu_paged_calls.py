"""Calls that the paged cache's documentation allows (polyhedral_amd.paged), beside those of
tests/test_gpu_paged.py."""
import numpy as np
import pytest
import torch

from polyhedral_amd import paged
from polyhedral_amd.polyattn import masks as pm

pytestmark = pytest.mark.gpu

I32 = torch.int32


@pytest.mark.parametrize("device", [None, "cuda", "cuda:0", torch.device("cuda"), torch.device("cuda", 0)], ids=str)
def test_a_cache_on_any_name_of_its_device(gpu, device):
    cache = paged.PagedKVCache(2, 64, 8, 2, 64, torch.float16, 16, device=device)
    assert cache.device == cache.k.device == gpu
    new = torch.ones(5, 2, 64, dtype=torch.float16, device=gpu)
    step = cache.begin([3, 2])
    cache.append(new, new, step)
    assert torch.equal(cache.attend(new, pm.Causal(), step), new)
    cache.begin(torch.ones(2, dtype=I32, device="cuda"), 2)
    cache.trim(4)
    cache.finish([True, False])
    assert cache.lengths.tolist() == [0, 3]
    cache.check()
