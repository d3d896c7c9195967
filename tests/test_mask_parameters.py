"""Mask parameters past 32 bits in the structure that the kernels take."""
import sys

import numpy as np
import pytest

from polyhedral_amd import paged
from polyhedral_amd.polyattn import masks as pm
from polyhedral_amd.spec import DeviceMask, MaskSpec, _term_struct

FAR = (1 << 30) - 1


def _params(spec):
    m = DeviceMask(spec).struct()
    return [(t.p0, t.p1, t.p2) for t in m.terms[:m.n_include + m.n_exclude]]


@pytest.mark.parametrize("p", [1 << 31, 1 << 32, (1 << 32) + 5, (1 << 40) - 1, sys.maxsize, 10 ** 30])
def test_a_parameter_past_32_bits_is_as_far_as_any_distance(p):
    for mask, want in ((pm.SlidingWindow(p), (FAR, 0, 0)), (pm.SinksWindow(4, p), (FAR, 4, 0)), (pm.SinksWindow(p, 4), (4, FAR, 0)),
                       (pm.Dilated(p), (FAR, 0, 0)), (pm.PrefixLM(p), (FAR, 0, 0)), (pm.LocalStrided(3, p), (3, FAR, 0)),
                       (pm.TwoBand(2, p, 5), (2, FAR, 5)), (pm.TwoBand(2, 9, p), (2, 9, FAR))):
        assert _params(paged._paged_mask(mask).spec) == [want]
        # the same pairs as the parameter's own, near and far
        q, k = np.arange(0, FAR, 12345677)[:, None], np.arange(0, FAR, 7654321)[None, :]
        spec = paged._paged_mask(mask).spec
        t = spec.include[0]
        if p < 1 << 62:
            assert np.array_equal(spec.live(q, k), MaskSpec(((t[0], *want),)).live(q, k))


@pytest.mark.parametrize("p", [-1, -5, -(1 << 31), -(1 << 32) + 7, -sys.maxsize])
def test_a_parameter_below_0_stays_below_0(p):
    assert _params(MaskSpec(((1, p, 0, 0),)))[0][0] < 0


def test_parameters_of_32_bits_are_as_they_were():
    for p in (0, 1, 77, FAR, FAR + 1, (1 << 31) - 1):
        m = _term_struct(((4, p, p, p),), ((1, p, 0, 0),))
        assert (m.terms[0].kind, m.terms[0].p0, m.terms[0].p1, m.terms[0].p2, m.terms[1].p0) == (4, p, p, p, p)
