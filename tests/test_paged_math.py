"""The paged cache's integer arithmetic (csrc/page_math.hpp) compiled for the host: verdicts, hulls
and words of a mask against its pairwise definition, slots of bad pages, rows of bad starts; and
the C entry points' refusals, which come before any device work."""
import ctypes
import pathlib
import shutil
import subprocess

import numpy as np
import pytest

from polyhedral_amd import _lib
from polyhedral_amd.spec import (CAUSAL, DILATED, FULL, LOCAL_STRIDED, PREFIX_LM, SINKS, TWOBAND, WINDOW, MaskSpec,
                                 _term_struct)

ROOT = pathlib.Path(__file__).resolve().parents[1]
MAX = (1 << 30) - 1

HARNESS = r"""
#include "page_math.hpp"
using namespace pa;
static PageMask<const pa_term*> of(const pa_mask* m) { return {m->n_include, m->n_exclude, m->terms[0], m->terms}; }
extern "C" {
int verdict(const pa_mask* m, int q0, int q1, int k0, int k1) { return mask_verdict(of(m), q0, q1, k0, k1); }
unsigned word(const pa_mask* m, int q, int k0, int len) { return mask_word(of(m), q, k0, len); }
void list(const pa_mask* m, int q0, int q1, int len, int lg, int* out) {
  const KeyList l = key_list(of(m), q0, q1, len, lg);
  out[0] = l.low; out[1] = l.first; out[2] = l.high;
}
int divided(int x, unsigned d) { return divide(x, divisor_of(d)); }
int slot(int page, int pos, int lg, long long n) { return slot_of(page, pos, lg, n); }
void request(int s0, int s1, int len, int T, int max_len, int* out) {
  const Request r = request_of(s0, s1, len, T, max_len);
  out[0] = r.start; out[1] = r.n; out[2] = r.len;
}
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    d = tmp_path_factory.mktemp("page_math")
    (d / "h.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-Wno-unknown-pragmas", "-fsanitize=undefined",
                    "-fno-sanitize-recover", f"-I{ROOT / 'include'}", f"-I{ROOT / 'polyhedral_amd' / 'csrc'}", "-o",
                    str(d / "h.so"), str(d / "h.cpp")], check=True, capture_output=True)
    lib = ctypes.CDLL(str(d / "h.so"))
    lib.word.restype = ctypes.c_uint
    lib.slot.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_longlong]
    return lib


MASKS = [MaskSpec(((CAUSAL, 0, 0, 0),)), MaskSpec(((WINDOW, 0, 0, 0),)), MaskSpec(((WINDOW, 1, 0, 0),)),
         MaskSpec(((WINDOW, 37, 0, 0),)), MaskSpec(((DILATED, 1, 0, 0),)), MaskSpec(((DILATED, 5, 0, 0),)),
         MaskSpec(((DILATED, 48, 0, 0),)), MaskSpec(((LOCAL_STRIDED, 20, 16, 0),)), MaskSpec(((LOCAL_STRIDED, 0, 70, 0),)),
         MaskSpec(((TWOBAND, 10, 50, 20),)), MaskSpec(((TWOBAND, 30, 10, 5),)), MaskSpec(((TWOBAND, 12, 90, 0),)),
         MaskSpec(((SINKS, 24, 4, 0),)), MaskSpec(((SINKS, 0, 65, 0),)), MaskSpec(((PREFIX_LM, 80, 0, 0),)),
         MaskSpec(((FULL, 0, 0, 0),)), MaskSpec(((DILATED, 16, 0, 0),), ((WINDOW, 40, 0, 0),)),
         MaskSpec(((WINDOW, 9, 0, 0), (PREFIX_LM, 33, 0, 0)), ((DILATED, 3, 0, 0), (TWOBAND, 2, 60, 9))),
         MaskSpec(((FULL, 0, 0, 0),), ((FULL, 0, 0, 0),)), MaskSpec(((CAUSAL, 0, 0, 0),), ((SINKS, 0, 20, 0),))]


@pytest.mark.parametrize("spec", MASKS, ids=str)
def test_words_verdicts_and_hulls_against_the_pairs(host, spec):
    m = ctypes.byref(_term_struct(spec.include, spec.exclude))
    N = 200
    q, k = np.arange(N)[:, None], np.arange(N + 64)[None, :]
    live = spec.live(q, k)
    rng = np.random.default_rng(3)
    for _ in range(400):
        qq, k0, ln = int(rng.integers(N)), 32 * int(rng.integers(7)), int(rng.integers(N + 1))
        want = sum(1 << b for b in range(32) if k0 + b < ln and live[qq, k0 + b])
        assert host.word(m, qq, k0, ln) == want, (qq, k0, ln)
    out = (ctypes.c_int * 3)()
    for _ in range(400):
        q0 = int(rng.integers(N))
        q1 = min(N - 1, q0 + int(rng.integers(40)))
        k0 = int(rng.integers(N))
        k1 = k0 + int(rng.choice([0, 15, 31, 63]))
        pairs = live[q0:q1 + 1, k0:k1 + 1]
        v = host.verdict(m, q0, q1, k0, k1)
        assert not (v == 0 and pairs.any()) and not (v == 2 and not pairs.all()), (q0, q1, k0, k1, v)
        ln, lg = int(rng.integers(q1 + 1, N + 1)), int(rng.integers(4, 7))
        host.list(m, q0, q1, ln, lg, out)
        low, first, high = out
        blocks = list(range(low)) + list(range(first, first + high))
        assert first >= low >= 0 and high >= 0 and len(set(blocks)) == len(blocks)
        assert all(b << lg < ln for b in blocks)
        need = {int(x) >> lg for x in np.flatnonzero(live[q0:q1 + 1, :ln].any(axis=0))}
        assert need <= set(blocks), (q0, q1, ln, lg)


def test_verdicts_decide_what_ranges_decide(host):
    """A window's hull and verdicts leave no block that is dead as a whole."""
    m = ctypes.byref(_term_struct(((SINKS, 100, 7, 0),), ()))
    out = (ctypes.c_int * 3)()
    host.list(m, 5000, 5031, 5032, 5, out)
    assert list(out) == [1, (5000 - 99) // 32, 5032 // 32 + 1 - (5000 - 99) // 32]
    assert host.verdict(m, 5000, 5031, 32, 63) == 0 and host.verdict(m, 5000, 5031, 4950, 4990) == 2
    assert host.verdict(m, 5000, 5031, 0, 6) == 2


@pytest.mark.parametrize("kind,p", [(WINDOW, (MAX, 0, 0)), (SINKS, (MAX, MAX, 0)), (TWOBAND, (MAX, MAX, MAX)),
                                    (PREFIX_LM, (MAX, 0, 0)), (DILATED, (MAX, 0, 0)), (LOCAL_STRIDED, (MAX, MAX, 0)),
                                    (CAUSAL, (0, 0, 0)), (FULL, (0, 0, 0))])
def test_the_largest_positions_and_parameters(host, kind, p):
    """No sum overflows (the host build traps on one), at either end of the positions, and for
    queries before the first token (a request with more rows than tokens)."""
    spec = MaskSpec(((kind, *p),))
    m = ctypes.byref(_term_struct(spec.include, ()))
    out = (ctypes.c_int * 3)()
    for q in (-MAX, -1, 0, MAX - 1):
        for k0 in (0, (MAX - 31) // 32 * 32):
            got = host.word(m, q, k0, MAX)
            want = sum(1 << b for b in range(32) if k0 + b < MAX and bool(spec.live(np.int64(q), np.int64(k0 + b))))
            assert got == want, (q, k0)
            host.verdict(m, q, q, k0, k0 + 31)
        host.list(m, q, q, MAX, 5, out)
        assert out[0] >= 0 and out[2] >= 0


def test_division_by_a_product(host):
    rng = np.random.default_rng(1)
    for d in [*range(1, 70), 127, 128, 129, 255, 1000, 4095, 4097, 32768, 32769, 65534, 65535]:
        top = (1 << 30) - 1
        xs = [0, 1, d - 1, d, d + 1, top, top // d * d, top // d * d - 1, *(int(x) for x in rng.integers(0, 1 << 30, 60))]
        xs += [int(q) * d + e for q in rng.integers(0, top // d, 40) for e in (-1, 0, 1)]
        for x in xs:
            if 0 <= x <= top:
                assert host.divided(x, d) == x // d, (x, d)


def test_bad_pages_and_starts(host):
    assert host.slot(0, 0, 4, 1) == 0 and host.slot(3, 37, 4, 4) == 3 * 16 + 5
    for page in (-1, 4, 1 << 30, -(1 << 31), (1 << 31) - 1):
        assert host.slot(page, 37, 4, 4) == -1
    assert host.slot(0, 0, 4, 0) == -1
    n = (1 << 31) // 256 - 1
    assert host.slot(n - 1, 255, 8, n) == n * 256 - 1
    out = (ctypes.c_int * 3)()
    rng = np.random.default_rng(0)
    for _ in range(2000):
        s0, s1, ln = (int(x) for x in rng.choice([-(1 << 31), -5, 0, 1, 7, 10, 11, (1 << 31) - 1], 3))
        host.request(s0, s1, ln, 10, 64, out)
        start, rows, length = out
        assert 0 <= start <= 10 and 0 <= rows <= 10 - start and 0 <= length <= 64
    host.request(2, 7, 9, 10, 64, out)
    assert list(out) == [2, 5, 9]


# ---- refusals of the C entry points (no device work is reached) -----------------------------
def _buf():
    b = (ctypes.c_char * 4096)()
    at = (ctypes.addressof(b) + 255) // 256 * 256
    return b, at


def _refused(rc, text):
    assert rc == _lib.PA_E_INVALID
    assert text in _lib.lib().pa_last_error().decode(), _lib.lib().pa_last_error()


def test_tables_refusals():
    keep, p = _buf()
    lib = _lib.lib()
    assert lib.pa_page_tables(None, None) == _lib.PA_E_INVALID

    def call(**change):
        a = _lib.PaTablesArgs()
        for f, t in _lib.PaTablesArgs._fields_:
            if t is ctypes.c_void_p:
                setattr(a, f, p)
        a.R, a.n_pages, a.page_size, a.pitch, a.cols, a.tokens = 2, 8, 16, 4, 4, 10
        for f, x in change.items():
            setattr(a, f, x)
        return lib.pa_page_tables(ctypes.byref(a), None)
    _refused(call(page_size=48), "page_size=48")
    _refused(call(page_size=8), "page_size=8")
    _refused(call(n_pages=-1), "n_pages")
    _refused(call(n_pages=1 << 27), "below 2^31")
    _refused(call(R=-1), "R=-1")
    _refused(call(cols=-1), "columns")
    _refused(call(cols=1 << 26, pitch=1 << 26), "columns")
    _refused(call(pitch=3), "pitch")
    _refused(call(tokens=-1), "tokens")
    _refused(call(lengths=p + 4), "overlap")
    for f in ("before", "fresh", "free_list", "free_count", "tables", "lengths", "q_start", "slots", "free_left", "status",
              "workspace"):
        _refused(call(**{f: None}), "null")


def test_tables_outputs_may_not_overlap_inputs():
    keep, p = _buf()
    inputs = {"before": 2, "fresh": 2, "free_list": 8, "free_count": 1, "tables": 8}
    outputs = {"lengths": 2, "q_start": 3, "slots": 10, "positions": 10, "free_left": 1, "status": 1, "workspace": 8}
    for o, n in outputs.items():
        for i, m in inputs.items():
            for shift in (0, 4 * (m - 1), -4 * (n - 1)):
                if shift == 0 and (o, i) in (("lengths", "before"), ("free_left", "free_count")):
                    continue   # (the state that advances in place)
                a = _lib.PaTablesArgs()
                for x, f in enumerate(list(inputs) + list(outputs)):
                    setattr(a, f, p + 256 * (x + 1))
                a.R, a.n_pages, a.page_size, a.pitch, a.cols, a.tokens = 2, 8, 16, 4, 4, 10
                setattr(a, o, getattr(a, i) + shift)
                _refused(_lib.lib().pa_page_tables(ctypes.byref(a), None), f"{o} and {i} overlap")


def test_append_refuses_pages_that_overlap():
    keep, p = _buf()
    for sp, sh, pages, H in ((0, 2048, 4, 2), (4096, 0, 4, 2), (120, 2048, 2, 1), (4096, 64, 1, 2)):
        _refused(_lib.lib().pa_paged_append(p, p, 256, 128, p, 3, p, p, sp, sh, 128, pages, 16, H, 128, _lib.PA_BF16, None),
                 "pages or heads closer than D")


def test_struct_layouts(tmp_path):
    """gcc's offsets of every field against the ctypes structures."""
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    lines, want = [], []
    for cname, cls in (("pa_tables_args", _lib.PaTablesArgs), ("pa_paged_args", _lib.PaPagedArgs)):
        for fname, _ in cls._fields_:
            lines.append(f'  printf("%zu %zu\\n", offsetof({cname}, {fname}), sizeof((({cname}*)0)->{fname}));')
            want.append((getattr(cls, fname).offset, getattr(cls, fname).size))
        lines.append(f'  printf("%zu 0\\n", sizeof({cname}));')
        want.append((ctypes.sizeof(cls), 0))
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "polyattn_amd.h"\nint main(void) {\n' + "\n".join(lines) +
                   "\n  return 0;\n}\n")
    subprocess.run([cc, "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    assert [tuple(map(int, line.split())) for line in out.splitlines()] == want


def test_release_and_append_refusals():
    keep, p = _buf()
    lib = _lib.lib()

    def release(R=2, pitch=4, cols=4, n_pages=8, **null):
        g = lambda n: None if n in null else p  # noqa: E731
        return lib.pa_page_release(g("first"), g("last"), R, g("tables"), pitch, cols, g("free_list"), g("free_count"),
                                   n_pages, g("free_left"), g("status"), g("ws"), None)
    _refused(release(R=-1), "R=-1")
    _refused(release(pitch=3), "pitch")
    _refused(release(n_pages=-1), "n_pages")
    for f in ("first", "last", "tables", "free_list", "free_count", "free_left", "status", "ws"):
        _refused(release(**{f: 1}), "null")

    def append(k_new=p, st=256, sh=128, T=3, k=p, sp=4096, ch=2048, cn=128, pages=4, ps=16, H=2, D=128, dt=_lib.PA_BF16):
        return lib.pa_paged_append(k_new, p, st, sh, p, T, k, p, sp, ch, cn, pages, ps, H, D, dt, None)
    assert append(T=0) == 0 and append(pages=0) == 0
    _refused(append(T=-1), "T=-1")
    _refused(append(D=96), "D=96")
    _refused(append(dt=7), "dtype")
    _refused(append(ps=24), "page_size")
    _refused(append(H=0), "Hkv")
    _refused(append(k_new=None), "null")
    _refused(append(k=p + 8), "aligned")
    _refused(append(st=260), "aligned")
    _refused(append(cn=64), "closer than D")
    _refused(append(sh=-128), "negative")


def test_attention_refusals():
    keep, p = _buf()
    lib = _lib.lib()
    need, zero = ctypes.c_int64(0), ctypes.c_int64(0)

    def args(**change):
        a = _lib.PaPagedArgs()
        for f in ("q", "k", "v", "tables", "lengths", "q_start", "o", "lse", "workspace"):
            setattr(a, f, p)
        a.q_st, a.q_sh, a.o_st, a.o_sh, a.c_sp, a.c_sh, a.c_sn = 1024, 128, 1024, 128, 4096, 2048, 128
        a.n_pages, a.page_size, a.pitch, a.cols, a.R, a.T, a.max_fresh = 4, 16, 4, 4, 2, 3, 2
        a.Hq, a.Hkv, a.D, a.dtype, a.scale = 8, 2, 128, _lib.PA_BF16, 0.1
        a.mask.n_include = 1
        a.workspace_bytes = 1 << 40
        for f, x in change.items():
            setattr(a, f, x)
        return a

    def call(**change):
        return lib.pa_paged_attn(ctypes.byref(args(**change)), None)
    assert lib.pa_paged_attn(None, None) == _lib.PA_E_INVALID
    assert lib.pa_paged_workspace(ctypes.byref(args()), ctypes.byref(need), ctypes.byref(zero)) == 0
    assert 0 < zero.value < need.value
    _refused(lib.pa_paged_workspace(ctypes.byref(args()), ctypes.byref(need), None), "null")
    assert call(R=0) == 0 and call(T=0) == 0
    _refused(call(workspace_bytes=need.value - 1), "workspace")
    _refused(call(workspace=p + 16), "workspace")
    _refused(call(workspace=None), "workspace")
    _refused(call(D=80), "D=80")
    _refused(call(dtype=9), "dtype")
    _refused(call(Hq=9), "multiple")
    _refused(call(Hkv=0), "heads")
    _refused(call(T=1 << 28), "T Hq")
    _refused(call(max_fresh=-1), "max_fresh")
    _refused(call(scale=0.0), "scale")
    _refused(call(scale=-1.0), "scale")
    _refused(call(scale=float("inf")), "scale")
    _refused(call(scale=float("nan")), "scale")
    _refused(call(page_size=0), "page_size")
    _refused(call(cols=5), "pitch")
    _refused(call(q=p + 2), "aligned")
    _refused(call(c_sn=100), "aligned")
    _refused(call(c_sn=64), "closer than D")
    _refused(call(o_st=-1024), "negative")
    for f in ("q", "k", "v", "o", "lengths", "q_start", "tables"):
        _refused(call(**{f: None}), "null")
    m = _lib.PaMask()
    _refused(call(mask=m), "n_include")
    m.n_include, m.perm_q = 1, p
    _refused(call(mask=m), "permutation")
    m.perm_q = None
    m.terms[0].kind = 8
    _refused(call(mask=m), "DENSE")
    m.terms[0].kind, m.terms[0].p0 = 2, 0
    _refused(call(mask=m), "stride")


def test_python_refuses_host_tensors_and_matrices():
    import torch

    from polyhedral_amd import paged
    from polyhedral_amd.polyattn import masks as pm
    z = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU only"):
        paged.build_tables(z, z, z[None], z, z[:1], 16, 4)
    with pytest.raises(RuntimeError, match="GPU only"):
        paged.release(z, z, z[None], z, z[:1])
    k = torch.zeros(2, 1, 16, 64)
    with pytest.raises(RuntimeError, match="GPU only"):
        paged.append(k[0, :1], k[0, :1], z, k, k)
    with pytest.raises(RuntimeError, match="GPU only"):
        paged.attention(k[0, :1], k, k, z[None], z[:1], z, pm.Causal())
    for bad in (pm.DenseMask(np.ones((4, 4), dtype=bool)), MaskSpec(((8, 0, 0, 0),)), pm.Permuted(pm.Causal(), np.arange(4))):
        with pytest.raises(ValueError, match="different lengths"):
            paged._paged_mask(bad)
    assert paged._paged_mask(pm.SinksWindow(4, 32)).spec.include == ((SINKS, 32, 4, 0),)
