"""What the C entry points of a shared cache that forgets refuse, before any device work: no address here
is read."""
import ctypes

import pytest

from polyhedral_amd import _lib

AT = 1 << 40
STEP = 1 << 20


def _call(entry, a, *more):
    rc = getattr(_lib.lib(), entry)(ctypes.byref(a), *more, None)
    return rc, _lib.lib().pa_last_error().decode()


def _refused(entry, a, text, *more):
    rc, message = _call(entry, a, *more)
    assert rc == _lib.PA_E_INVALID and text in message, (rc, message)


def _set(a, change):
    for f, x in change.items():
        setattr(a, f, x)
    return a


# bytes of each tensor, in order of address
SHARE = {"lengths": 8, "q_start": 12, "holders": 8, "shared": 8, "start": 12, "rows": 40, "positions": 40, "prefix": 8, "low": 8,
         "high": 8, "first": 8, "workspace": 64}
WEIGHTS = {"q": 5120, "k": 32768, "tables": 32, "lengths": 8, "q_start": 12, "first": 8, "lse": 80, "scores": 512}
CHOOSE = {"scores": 1536, "tables": 32, "lengths": 8, "first": 8, "kept": 384, "after": 8}
EVICT = {"kept": 384, "k": 98304, "v": 98304, "scores": 1536, "tables": 32, "lengths": 8, "first": 8}


def _place(a, sizes):
    for i, f in enumerate(sizes):
        setattr(a, f, AT + i * STEP)
    return a


def share(**change):
    a = _place(_lib.PaShareArgs(), SHARE)
    a.R, a.page_size, a.T = 2, 16, 10
    return _set(a, change)


def weights(**change):
    """T = 5 rows of 4 heads of 128 bf16, 2 KV heads, 4 pages of 16."""
    a = _place(_lib.PaWeightsArgs(), WEIGHTS)
    a.q_st, a.q_sh, a.c_sp, a.c_sh, a.c_sn, a.lse_st, a.lse_sh, a.s_sp, a.s_sh = 512, 128, 4096, 2048, 128, 4, 1, 32, 16
    a.n_pages, a.page_size, a.pitch, a.cols, a.R, a.T, a.max_fresh = 4, 16, 4, 4, 2, 5, 2
    a.Hq, a.Hkv, a.D, a.dtype, a.scale = 4, 2, 128, _lib.PA_BF16, 0.1
    a.mask.n_include = 1
    return _set(a, change)


def choose(**change):
    """3 layers of 4 pages of 16, 2 heads, 2 requests that keep 8."""
    a = _place(_lib.PaChooseArgs(), CHOOSE)
    a.s_sl, a.s_sp, a.s_sh, a.n_pages, a.page_size, a.pitch, a.cols = 128, 32, 16, 4, 16, 4, 4
    a.layers, a.R, a.Hkv, a.keep, a.recent, a.limit = 3, 2, 2, 8, 2, 9
    return _set(a, change)


def evict(**change):
    a = _place(_lib.PaEvictArgs(), EVICT)
    a.c_sl, a.c_sp, a.c_sh, a.c_sn, a.s_sl, a.s_sp, a.s_sh = 16384, 4096, 2048, 128, 128, 32, 16
    a.n_pages, a.page_size, a.pitch, a.cols, a.layers, a.R, a.Hkv, a.keep, a.D, a.dtype = 4, 16, 4, 4, 3, 2, 2, 8, 128, _lib.PA_BF16
    return _set(a, change)


@pytest.mark.parametrize("entry,make,sizes,outs", [
    ("pa_share_rows", share, SHARE, ["start", "rows", "positions", "prefix", "low", "high", "first", "workspace"]),
    ("pa_paged_weights", weights, WEIGHTS, ["scores"]), ("pa_choose_keys", choose, CHOOSE, ["kept", "after"]),
    ("pa_evict_rows", evict, EVICT, ["k", "v", "scores"])])
def test_outputs_that_share_memory_are_refused(entry, make, sizes, outs):
    place = {f: AT + i * STEP for i, f in enumerate(sizes)}
    for o in outs:
        unit = 16 if o in ("k", "v") else 4
        for f, n in sizes.items():
            if f == o:
                continue
            for p in {place[f], place[f] + (n - 1) // unit * unit, place[f] - (sizes[o] - 1) // unit * unit}:
                _refused(entry, make(**{o: p}), "overlap")


def test_rows_that_overlap_are_refused():
    for change in (dict(s_sp=16), dict(s_sh=0), dict(s_sh=15), dict(s_sp=0), dict(s_sp=31)):
        _refused("pa_paged_weights", weights(**change), "rows of scores overlap")
        _refused("pa_evict_rows", evict(**change), "rows of k, v or scores overlap")
    for change in (dict(c_sl=0), dict(c_sl=4096), dict(c_sp=2048), dict(c_sh=128), dict(s_sl=64)):
        _refused("pa_evict_rows", evict(**change), "overlap")
    for v in (0, 256, 4096, 8192, 32768):           # the values on the keys of other rows, heads, pages, layers
        _refused("pa_evict_rows", evict(v=AT + STEP + v), "k and v overlap")


@pytest.mark.parametrize("entry,make,bad", [
    ("pa_share_rows", share, [dict(page_size=20), dict(R=-1), dict(T=-1), dict(T=1 << 30), dict(start=None), dict(rows=None), dict(first=None),
                              dict(holders=None), dict(workspace=None), dict(R=1 << 24)]),
    ("pa_paged_weights", weights, [dict(page_size=8), dict(n_pages=-1), dict(n_pages=1 << 28), dict(D=96), dict(dtype=3), dict(Hq=3), dict(Hkv=0),
                                   dict(T=-1), dict(T=1 << 29), dict(cols=-1), dict(pitch=3), dict(scale=0.0), dict(scale=float("inf")),
                                   dict(scale=float("nan")), dict(max_fresh=-1), dict(q=None), dict(lse=None), dict(scores=None),
                                   dict(q=AT + 8), dict(k=AT + STEP + 4), dict(q_st=509), dict(c_sn=120), dict(c_sn=1 << 22), dict(c_sp=-4096),
                                   dict(s_sp=-32), dict(s_sh=-16), dict(R=-1)]),
    ("pa_choose_keys", choose, [dict(page_size=0), dict(keep=0), dict(recent=-1), dict(recent=9), dict(limit=7), dict(keep=1 << 30, limit=1 << 30),
                                dict(layers=-1), dict(R=-1), dict(Hkv=0), dict(Hkv=65536), dict(layers=1 << 20, R=4), dict(scores=None),
                                dict(kept=None), dict(after=None), dict(lengths=None), dict(tables=None), dict(pitch=3), dict(s_sl=-1)]),
    ("pa_evict_rows", evict, [dict(page_size=17), dict(keep=0), dict(D=32), dict(dtype=7), dict(k=None), dict(v=None), dict(kept=None),
                              dict(tables=None), dict(k=AT + STEP + 8), dict(c_sn=64), dict(c_sp=4100), dict(c_sl=-1), dict(s_sp=-1),
                              dict(layers=1 << 20, R=4), dict(cols=1 << 27, pitch=1 << 27)])])
def test_arguments_out_of_range_are_refused(entry, make, bad):
    for change in bad:
        rc, message = _call(entry, make(**change))
        assert rc == _lib.PA_E_INVALID and message.startswith(entry), (change, rc, message)
    assert getattr(_lib.lib(), entry)(None, None) == _lib.PA_E_INVALID


def test_nothing_to_do_needs_no_device():
    none = dict(R=0)
    for entry, a in (("pa_paged_weights", weights(**none)), ("pa_paged_weights", weights(T=0)), ("pa_paged_weights", weights(cols=0)),
                     ("pa_choose_keys", choose(**none)), ("pa_choose_keys", choose(layers=0)), ("pa_evict_rows", evict(**none)),
                     ("pa_evict_rows", evict(n_pages=0))):
        assert _call(entry, a)[0] == 0, entry


def test_masks_that_have_no_positions_are_refused():
    a = weights()
    a.mask.terms[0].kind = 8
    _refused("pa_paged_weights", a, "PA_DENSE")
    a = weights()
    a.mask.perm_q = AT
    _refused("pa_paged_weights", a, "permutation")


def test_a_null_sharing_is_refused():
    a = _lib.PaPagedArgs()
    assert _lib.lib().pa_shared_attn(ctypes.byref(a), None, None) == _lib.PA_E_INVALID
    assert "sharing" in _lib.lib().pa_last_error().decode()


def test_a_flag_of_missing_pages_that_shares_memory_is_refused():
    for i, (f, n) in enumerate(CHOOSE.items()):
        for p in (AT + i * STEP, AT + i * STEP + (n - 1) // 4 * 4):
            _refused("pa_choose_keys", choose(missing=p), "overlap")


def test_more_units_than_can_be_counted_are_refused():
    """Requests of many rows are taken by 256 keys and head, in numbers of 32 bits."""
    many = dict(T=1 << 13, max_fresh=1 << 13, R=1 << 20, Hq=1 << 15, Hkv=1 << 15)
    _refused("pa_paged_weights", weights(cols=1 << 25, pitch=1 << 25, **many), "units")
    _refused("pa_paged_weights", weights(cols=1 << 24, pitch=1 << 24, T=100, max_fresh=40, R=4, Hq=4096, Hkv=4096), "units")
    # (a token a request is taken by blocks; and so little of a table is no matter)
    for some in (dict(max_fresh=1), dict(cols=64, pitch=64), dict(dtype=_lib.PA_F32)):
        rc, message = _call("pa_paged_weights", weights(**{**many, "cols": 1 << 25, "pitch": 1 << 25, "q": None, **some}))
        assert rc == _lib.PA_E_INVALID and "null pointer" in message, (some, message)


FINISH = {"done": 2, "holders": 8, "shared": 8, "lengths": 8, "tables": 32, "refused": 4, "first": 8, "last": 8, "workspace": 8}


def finish(**change):
    a = _place(_lib.PaFinishArgs(), FINISH)
    a.R, a.page_size, a.pitch, a.cols, a.refused_bits = 2, 16, 4, 4, 16
    return _set(a, change)


def test_finishing_refuses_what_it_cannot_take():
    for o, (p, n) in {f: (AT + i * STEP, n) for i, (f, n) in enumerate(FINISH.items())}.items():
        for f, m in FINISH.items():
            if f != o:
                _refused("pa_page_finish", finish(**{f: p}), "overlap")
                _refused("pa_page_finish", finish(**{f: p - (m - 1) // 4 * 4 if f != "done" else p}), "overlap")
    for bad in (dict(R=-1), dict(R=1 << 24), dict(page_size=0), dict(cols=-1), dict(pitch=3), dict(cols=1 << 27, pitch=1 << 27),
                *(dict([(f, None)]) for f in FINISH)):
        rc, message = _call("pa_page_finish", finish(**bad))
        assert rc == _lib.PA_E_INVALID and message.startswith("pa_page_finish"), (bad, message)
    assert _call("pa_page_finish", finish(R=0))[0] == 0
