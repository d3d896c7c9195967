"""The largest sizes that the paged cache's C entry points take or refuse (no device work is reached)."""
import ctypes

import pytest

from polyhedral_amd import _lib


def _refused(rc, text):
    assert rc == _lib.PA_E_INVALID
    assert text in _lib.lib().pa_last_error().decode(), _lib.lib().pa_last_error()


def _workspace(**change):
    """(status, bytes) of a call of R = 2 requests, T = 300 rows of 8 heads on 2 of 128 bf16."""
    a = _lib.PaPagedArgs()
    a.n_pages, a.page_size, a.pitch, a.cols, a.R, a.T, a.max_fresh = 40, 16, 20, 20, 2, 300, 200
    a.Hq, a.Hkv, a.D, a.dtype, a.scale = 8, 2, 128, _lib.PA_BF16, 0.1
    a.mask.n_include = 1
    for f, x in change.items():
        setattr(a, f, x)
    need, zero = ctypes.c_int64(-1), ctypes.c_int64(-1)
    return _lib.lib().pa_paged_workspace(ctypes.byref(a), ctypes.byref(need), ctypes.byref(zero)), need.value


def test_sizes_whose_products_pass_64_bits_are_refused():
    for T in (1 << 30, 1 << 60, 1 << 61, 1 << 62, (1 << 61) + 1):
        _refused(_workspace(T=T)[0], "T Hq")
    for pages in (1 << 31, 1 << 55, 1 << 60, (1 << 60) + 3):
        _refused(_workspace(n_pages=pages)[0], "below 2^31")
        a = _lib.PaTablesArgs()
        a.n_pages, a.page_size = pages, 16
        _refused(_lib.lib().pa_page_tables(ctypes.byref(a), None), "below 2^31")
        _refused(_lib.lib().pa_paged_append(None, None, 0, 0, None, 0, None, None, 0, 0, 0, pages, 16, 1, 64, _lib.PA_F16, None),
                 "below 2^31")


@pytest.mark.parametrize("most", [300, 301, 1 << 31, 1 << 61, 1 << 62, (1 << 63) - 1])
def test_a_hint_past_the_rows_is_the_rows(most):
    assert _workspace(max_fresh=most) == _workspace(max_fresh=300)
    assert _workspace(max_fresh=300) != _workspace(max_fresh=1)


def test_more_work_groups_than_a_grid_has_are_refused():
    """A launch has less than 2^32 threads, 256 of them a work-group: tokens of 2^21 requests, 8 KV heads."""
    for dtype in (_lib.PA_F32, _lib.PA_BF16):
        for most in (1, 1 << 20):
            for n in (1 << 21, 1 << 24, (1 << 27) - 1):
                _refused(_workspace(T=n, R=n, Hq=8, Hkv=8, max_fresh=most, dtype=dtype)[0], "grid limit")
        assert _workspace(T=1 << 20, R=1 << 20, Hq=8, Hkv=8, max_fresh=1, dtype=dtype)[0] == 0
    # each part within it, both together not
    assert _workspace(T=1 << 20, R=1 << 20, Hq=11, Hkv=11, max_fresh=1)[0] == 0
    _refused(_workspace(T=1 << 20, R=1 << 20, Hq=11, Hkv=11, max_fresh=100)[0], "grid limit")
