"""The order of a chunk's steps (csrc/page_steps.hpp) compiled for the host: for every pattern of live
and dead steps, whose scores each step's sums are taken from."""
import ctypes
import pathlib
import shutil
import subprocess

import pytest

ROOT = pathlib.Path(__file__).resolve().parents[1]

HARNESS = r"""
#include "page_steps.hpp"
// Scores that know which step they are of (-1: never written).
struct Scores {
  int step = -1;
};
// Walks n steps of which those in the bits of `live` have a live key.  Returns 0, or 1 + the step whose
// sums were taken from another one's scores; -1 - j where live step j was summed not once.
extern "C" int walk(int n, unsigned live) {
  Scores a, b;
  a.step = 0;
  int bad = 0, at = 0, sums[32] = {};
  auto is_live = [&](int j) { return ((live >> j) & 1u) != 0u; };
  auto take = [&](int j, const Scores& x) {
    if (x.step != j && !bad) bad = 1 + j;
    ++sums[j];
  };
  auto next = [&](int j) {
    if (j != at && !bad) bad = 1 + j;
    return pa::LiveSteps{is_live(j), is_live(j + 1)};
  };
  auto body = [&](int j, bool now, const Scores& x, Scores& y) {
    if (now) take(j, x);
    y.step = j + 1;
  };
  auto turn = [&]() { ++at; };
  pa::walk_steps(n, a, b, next, body, turn);
  if (at != n - 1 && !bad) bad = n;
  if (is_live(n - 1)) take(n - 1, a);
  if (bad) return bad;
  for (int j = 0; j < n; ++j)
    if (is_live(j) && sums[j] != 1) return -1 - j;
  return 0;
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    d = tmp_path_factory.mktemp("page_steps")
    (d / "h.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-Wno-unknown-pragmas", "-Wno-attributes",
                    f"-I{ROOT / 'include'}", f"-I{ROOT / 'polyhedral_amd' / 'csrc'}", "-o", str(d / "h.so"), str(d / "h.cpp")],
                   check=True, capture_output=True)
    return ctypes.CDLL(str(d / "h.so"))


@pytest.mark.parametrize("n", range(1, 13))
def test_sums_are_of_a_steps_own_scores(host, n):
    for live in range(1 << n):
        assert host.walk(n, live) == 0, "".join("L" if (live >> j) & 1 else "." for j in range(n))


def test_long_lists(host):
    for live in (0xffffffff, 0x7ffffffe, 0x80000001, 0xcccccccc, 0x33333333, 0x99999999, 0x0ff00ff1, 0x40000002):
        for n in (29, 30, 31, 32):
            assert host.walk(n, live) == 0, (n, hex(live))
