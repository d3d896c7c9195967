"""Which tensors of a call share memory (csrc/page_spans.hpp), compiled for the host, against sets of
bytes; and the C entry points' refusals of outputs that share it, which come before any device work."""
import ctypes
import itertools
import pathlib
import shutil
import subprocess

import numpy as np
import pytest

from polyhedral_amd import _lib

ROOT = pathlib.Path(__file__).resolve().parents[1]

HARNESS = r"""
#include "page_spans.hpp"
using namespace pa;
static Strided<2> of(const long long* x) {
  return strided<2>(reinterpret_cast<const void*>(x[0]), x[1], {x[2], x[3]}, {x[4], x[5]});
}
extern "C" {
int self2(const long long* x) { return overlaps_itself(of(x)); }
int both2(const long long* x, const long long* y) { return overlap(of(x), of(y)); }
int nested3(long long w, const long long* n, const long long* s) {
  return nested(strided<3>(nullptr, w, {n[0], n[1], n[2]}, {s[0], s[1], s[2]}));
}
int flat_rows(long long at, long long bytes, const long long* x) {
  return overlap(flat(reinterpret_cast<const void*>(at), bytes), of(x));
}
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    d = tmp_path_factory.mktemp("page_spans")
    (d / "h.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover",
                    f"-I{ROOT / 'polyhedral_amd' / 'csrc'}", "-o", str(d / "h.so"), str(d / "h.cpp")], check=True,
                   capture_output=True)
    lib = ctypes.CDLL(str(d / "h.so"))
    lib.nested3.argtypes = [ctypes.c_longlong, ctypes.c_void_p, ctypes.c_void_p]
    lib.flat_rows.argtypes = [ctypes.c_longlong, ctypes.c_longlong, ctypes.c_void_p]
    return lib


def _ll(*x):
    return (ctypes.c_longlong * len(x))(*x)


def _bytes(at, w, n, m, s, t):
    """The bytes of each row."""
    return [set(range(at + i * s + j * t, at + i * s + j * t + w)) for i in range(n) for j in range(m)]


def test_rows_on_top_of_each_other(host):
    for w, n, m in itertools.product((1, 3, 4), (0, 1, 2, 3), (0, 1, 2, 4)):
        for s, t in itertools.product((-7, -4, 0, 1, 2, 3, 4, 5, 6, 8, 9, 12, 13), repeat=2):
            rows = _bytes(1000, w, n, m, s, t)
            want = sum(map(len, rows)) > len(set().union(*rows))
            assert host.self2(_ll(1000, w, n, m, s, t)) == want, (w, n, m, s, t)


def test_parts_of_one_buffer(host):
    """The same sizes and strides: exact."""
    rng = np.random.default_rng(0)
    for _ in range(6000):
        n, m = (int(x) for x in rng.integers(1, 5, 2))
        w, u = (int(x) for x in rng.integers(1, 6, 2))
        s, t = (int(x) for x in rng.integers(-14, 15, 2))
        d = int(rng.integers(-60, 61))
        a, b = set().union(*_bytes(1000, w, n, m, s, t)), set().union(*_bytes(1000 + d, u, n, m, s, t))
        assert host.both2(_ll(1000, w, n, m, s, t), _ll(1000 + d, u, n, m, s, t)) == bool(a & b), (n, m, w, u, s, t, d)


def test_other_tensors_by_their_spans(host):
    rng = np.random.default_rng(1)
    for _ in range(3000):
        x, y = ([1000 + int(rng.integers(-80, 81)), int(rng.integers(1, 6)), *(int(v) for v in rng.integers(0, 4, 2)),
                 *(int(v) for v in rng.integers(-9, 20, 2))] for _ in range(2))
        a, b = (set().union(*_bytes(*v)) for v in (x, y))
        meet = bool(a and b and min(a) <= max(b) and min(b) <= max(a))
        got = host.both2(_ll(*x), _ll(*y))
        assert got <= meet and (got or not a & b), (x, y)
        assert host.flat_rows(x[0], x[1], _ll(*y)) == bool(b and x[0] <= max(b) and min(b) < x[0] + x[1])


def test_nested_strides_are_apart(host):
    rng = np.random.default_rng(2)
    some = 0
    for _ in range(4000):
        w, n, s = int(rng.integers(1, 4)), [int(x) for x in rng.integers(1, 4, 3)], [int(x) for x in rng.integers(0, 30, 3)]
        cells = [sum(i * t for i, t in zip(at, s)) + b for at in np.ndindex(*n) for b in range(w)]
        if host.nested3(w, _ll(*n), _ll(*s)):
            some += 1
            assert len(set(cells)) == len(cells), (w, n, s)
    assert some > 100
    # the layouts of a dense cache in any order of its dimensions are nested
    for order in itertools.permutations(range(3)):
        n, s, size = [5, 3, 16], [0, 0, 0], 256
        for i in order:
            s[i], size = size, size * n[i]
        assert host.nested3(256, _ll(*n), _ll(*s))


def test_the_largest_sizes_and_strides(host):
    big = (1 << 63) - 1
    assert host.self2(_ll(1 << 40, big, 1 << 30, 65535, big, big)) == 1
    assert host.self2(_ll(1 << 40, 256, 1 << 30, 4, 1024, 256)) == 0
    assert host.self2(_ll(1 << 40, 256, 1 << 30, 4, 1023, 256)) == 1
    assert host.both2(_ll(1 << 40, 256, 1 << 30, 32, big, 256), _ll((1 << 40) + 32 * 256, 256, 1 << 30, 32, big, 256)) == 0


# ---- refusals of the C entry points ---------------------------------------------------------
def _refused(rc, text):
    assert rc == _lib.PA_E_INVALID
    assert text in _lib.lib().pa_last_error().decode(), _lib.lib().pa_last_error()


ATTENTION = ("q", "k", "v", "tables", "lengths", "q_start", "o", "lse", "workspace")


def _attention(at, **change):
    """T = 5 rows of 4 heads of 128 bf16, 2 KV heads, 4 pages of 16, each tensor 64 KiB from the next."""
    a = _lib.PaPagedArgs()
    for i, f in enumerate(ATTENTION):
        setattr(a, f, at + i * 65536)
    a.q_st, a.q_sh, a.o_st, a.o_sh, a.c_sp, a.c_sh, a.c_sn, a.lse_st, a.lse_sh = 512, 128, 512, 128, 4096, 2048, 128, 4, 1
    a.n_pages, a.page_size, a.pitch, a.cols, a.R, a.T, a.max_fresh = 4, 16, 4, 4, 2, 5, 2
    a.Hq, a.Hkv, a.D, a.dtype, a.scale = 4, 2, 128, _lib.PA_BF16, 0.1
    a.mask.n_include = 1
    a.workspace_bytes = 1 << 40
    for f, x in change.items():
        setattr(a, f, x)
    return _lib.lib().pa_paged_attn(ctypes.byref(a), None)


def test_attention_refuses_outputs_whose_rows_overlap():
    at = 1 << 40   # (no address is read)
    for change in (dict(o_st=0), dict(o_sh=0), dict(o_sh=64), dict(o_st=256), dict(o_st=504), dict(o_st=128)):
        _refused(_attention(at, **change), "rows of o overlap")
    for change in (dict(lse_st=0), dict(lse_sh=0), dict(lse_st=1), dict(lse_st=3), dict(lse_st=-1)):
        _refused(_attention(at, **change), "rows of lse overlap")


@pytest.mark.parametrize("out", ["o", "lse", "workspace"])
def test_attention_refuses_outputs_that_overlap_others(out):
    at = 1 << 40
    size = {"q": 5120, "k": 32768, "v": 32768, "tables": 32, "lengths": 8, "q_start": 12, "o": 5120, "lse": 80}
    for f, n in size.items():
        if f == out:
            continue
        base = at + ATTENTION.index(f) * 65536
        if out == "workspace":
            places = [base - 256, base]
        else:
            places = [base, base + (n - 1) // 16 * 16, base - (size[out] - 1) // 16 * 16]
        for p in places:
            _refused(_attention(at, **{out: p}), "overlap")


RELEASE_IN, RELEASE_OUT = {"first": 8, "last": 8, "free_count": 4}, {"tables": 32, "free_list": 32, "free_left": 4, "status": 4,
                                                                     "workspace": 8}


def test_release_refuses_tensors_that_overlap():
    at = 1 << 40   # (no address is read)
    size = {**RELEASE_IN, **RELEASE_OUT}
    place = {f: at + 4096 * i for i, f in enumerate(size)}
    for o in RELEASE_OUT:
        for i, n in size.items():
            for p in {place[i], place[i] + n - 4, place[i] - size[o] + 4}:
                if i == o or (p == place[i] and {o, i} == {"free_left", "free_count"}):
                    continue
                w = {**place, o: p}
                rc = _lib.lib().pa_page_release(w["first"], w["last"], 2, w["tables"], 4, 4, w["free_list"], w["free_count"], 8,
                                                w["free_left"], w["status"], w["workspace"], None)
                _refused(rc, "overlap")


TABLES_IN = {"before": 8, "fresh": 8, "free_list": 32, "free_count": 4}
TABLES_OUT = {"lengths": 8, "q_start": 12, "slots": 40, "positions": 40, "free_left": 4, "status": 4, "workspace": 32, "tables": 32}


def test_tables_refuse_tensors_that_overlap():
    """Outputs and the tables, against each other and against the inputs."""
    at = 1 << 40   # (no address is read)
    size = {**TABLES_IN, **TABLES_OUT}
    for o in TABLES_OUT:
        for i, n in size.items():
            for shift in {0, n - 4, 4 - size[o]}:
                if i == o or (shift == 0 and {o, i} in ({"free_left", "free_count"}, {"lengths", "before"})):
                    continue
                a = _lib.PaTablesArgs()
                for x, f in enumerate(size):
                    setattr(a, f, at + 4096 * x)
                a.R, a.n_pages, a.page_size, a.pitch, a.cols, a.tokens = 2, 8, 16, 4, 4, 10
                setattr(a, o, getattr(a, i) + shift)
                _refused(_lib.lib().pa_page_tables(ctypes.byref(a), None), "overlap")


def test_append_refuses_a_cache_whose_rows_overlap():
    at = 1 << 40   # (no address is read)

    def append(sp, sh, sn, v, pages=4, P=16, H=2, same=False):
        return _lib.lib().pa_paged_append(at, at if same else at + 4096, 256, 128, at + 8192, 3, at + 65536, at + 65536 + v, sp, sh,
                                          sn, pages, P, H, 128, _lib.PA_BF16, None)
    for args in ((4096, 128, 128, 1 << 20), (2048, 2048, 128, 1 << 20), (4096, 2048, 136, 1 << 20), (4096, 2048, 256, 1 << 20),
                 (512, 256, 128, 1 << 20)):                     # (rows of a head on top of the next head's, and so on)
        _refused(append(*args), "rows of k and v overlap")
    for v in (0, 128, 256, 4096, -4096, 8192, 3 * 8192):        # k and v in one place, or some pages apart
        _refused(append(4096, 2048, 128, v), "rows of k and v overlap")
    _refused(append(4096, 128, 128, 0, same=True), "rows of k and v overlap")


def test_append_refuses_values_on_the_next_heads_keys():
    """Heads outermost, a page's pitch of two pages: v a page and a half on lies between the pages of its own
    head, but on the keys of the next head, which start at an odd half."""
    at, page = 1 << 40, 16 * 256
    pages, sp = 5, 2 * page

    def append(v, sh):
        return _lib.lib().pa_paged_append(at, at + 4096, 256, 128, at + 8192, 3, at + (1 << 20), at + (1 << 20) + v, sp // 2, sh // 2,
                                          128, pages, 16, 2, 128, _lib.PA_BF16, None)
    _refused(append(page + pages * sp, pages * sp + page), "rows of k and v overlap")
    _refused(append(-page - pages * sp, pages * sp + page), "rows of k and v overlap")


def test_strides_past_64_bits_are_not_taken_for_short_ones():
    """A pitch or stride whose bytes pass 64 bits: all above the first row is its span."""
    at = 1 << 40
    a = _lib.PaTablesArgs()
    for x, f in enumerate(["tables", *TABLES_IN, *(f for f in TABLES_OUT if f != "tables")]):
        setattr(a, f, at + 4096 * x)
    a.R, a.n_pages, a.page_size, a.pitch, a.cols, a.tokens = 2, 8, 16, 1 << 62, 4, 10
    _refused(_lib.lib().pa_page_tables(ctypes.byref(a), None), "and tables overlap")
    for change in (dict(c_sp=1 << 61), dict(q_st=1 << 60), dict(pitch=1 << 62)):
        _refused(_attention(at, **change), "overlap")
