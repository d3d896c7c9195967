"""Ranges of queries and of listed keys (csrc/page_math.hpp) compiled for the host, against the masks'
pairwise definition."""
import ctypes

import numpy as np
import pytest

from polyhedral_amd.spec import CAUSAL, FULL, PREFIX_LM, SINKS, TWOBAND, WINDOW, MaskSpec, _term_struct
from tests import test_paged_math as tpm

HARNESS = tpm.HARNESS.replace('extern "C" {', r"""extern "C" {
void queries(const pa_mask* m, int k0, int k1, int* out) {
  const QueryRange r = query_range(of(m), k0, k1);
  out[0] = r.lo; out[1] = r.hi;
}
void entries(int low, int first, int high, int b, int* out) {
  const KeyList l{low, first, high};
  out[0] = l.before(b);
}
""", 1)


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    held, tpm.HARNESS = tpm.HARNESS, HARNESS
    try:
        yield tpm.host.__wrapped__(tmp_path_factory) if hasattr(tpm.host, "__wrapped__") else tpm.host.__pytest_wrapped__.obj(tmp_path_factory)
    finally:
        tpm.HARNESS = held


@pytest.mark.parametrize("spec", tpm.MASKS, ids=str)
def test_queries_that_may_see_keys(host, spec):
    m = ctypes.byref(_term_struct(spec.include, spec.exclude))
    N = 220
    live = spec.live(np.arange(N)[:, None], np.arange(N)[None, :])
    out, rng = (ctypes.c_int * 2)(), np.random.default_rng(1)
    for _ in range(400):
        k0 = int(rng.integers(N))
        k1 = min(N - 1, k0 + int(rng.integers(80)))
        host.queries(m, k0, k1, out)
        seen = np.flatnonzero(live[:, k0:k1 + 1].any(axis=1))
        assert not len(seen) or (out[0] <= seen[0] and seen[-1] <= out[1]), (k0, k1, out[0], out[1])


def test_ranges_are_tight_and_do_not_overflow(host):
    big = tpm.MAX
    out = (ctypes.c_int * 2)()
    for spec, keys, want in ((((CAUSAL, 0, 0, 0),), (64, 127), (64, big)), (((WINDOW, 10, 0, 0),), (64, 127), (64, 136)),
                             (((SINKS, 10, 64, 0),), (64, 127), (64, 136)), (((SINKS, 10, 65, 0),), (64, 127), (64, big)),
                             (((TWOBAND, 5, 100, 7),), (64, 127), (64, 233)), (((PREFIX_LM, 64, 0, 0),), (64, 127), (64, big)),
                             (((PREFIX_LM, 65, 0, 0),), (64, 127), (0, big)), (((FULL, 0, 0, 0),), (64, 127), (0, big)),
                             (((WINDOW, big, 0, 0),), (big - 3, big), (big - 3, big - 1)),
                             (((TWOBAND, big, big, big),), (5, big), (5, big - 1))):
        host.queries(ctypes.byref(_term_struct(MaskSpec(spec).include, ())), *keys, out)
        assert tuple(out) == want, (spec, keys, tuple(out))


def test_entries_before_a_block(host):
    out = (ctypes.c_int * 1)()
    for low in (0, 1, 4):
        for first in range(low, 9):
            for high in (0, 1, 5):
                blocks = list(range(low)) + list(range(first, first + high))
                for b in range(-2, 18):
                    host.entries(low, first, high, b, out)
                    assert out[0] == sum(x < b for x in blocks)
