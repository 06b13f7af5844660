"""How the warps of the expert layer's kernel share a phase's units, compiled for the host.

Every chunk of every unit is some warp's exactly once, and the warps that share a
unit meet: their barrier waits without a limit, so a warp whose copy did not come,
in whichever unit, must still join the others of its shared one."""
import ctypes
import itertools
import os
import subprocess

import pytest

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))

SOURCE = r"""
#include "qz_moe_walk.cuh"
using namespace qz;
// One warp's way through a phase, as the kernel's run_phase goes: units it takes
// (unit index, first and last chunk), then the barrier it joins, if any.  fails: the
// unit at which its copy does not come, -1: none, -2: the phase's operand does not.
extern "C" int walk(int begin, int end, int units, int chunks, int warp, int fails, int* taken, int* joins, int* partners) {
  const int bound[2] = {begin, end};
  MoeWalk w(bound, units, chunks, warp);
  bool ok = fails != -2;
  int n = 0;
  *joins = 0;
  *partners = 0;
  while (ok && !w.done()) {
    const int share = w.whole ? 1 : w.share;
    taken[3 * n] = w.group * units + w.unit;
    taken[3 * n + 1] = w.c0;
    taken[3 * n + 2] = w.c1;
    for (bool more = true; more;) {
      if (n == fails) { ok = false; break; }
      more = !w.advance();
    }
    ++n;
    if (share > 1) {
      w.met = true;
      *joins += 1 + warp / share;
      *partners = share;
    }
  }
  if (!ok && w.owes_meeting()) {
    *joins += 1 + warp / w.share;
    *partners = w.share;
  }
  return n;
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    d = tmp_path_factory.mktemp("walk")
    (d / "walk.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "qwantize_b200", "csrc"), str(d / "walk.cpp"), "-o", str(d / "walk.so")],
                   check=True)
    L = ctypes.CDLL(str(d / "walk.so"))

    def run(begin, end, units, chunks, warp, fails=-1):
        taken, joins, partners = (ctypes.c_int * 3000)(), ctypes.c_int(0), ctypes.c_int(0)
        n = L.walk(begin, end, units, chunks, warp, fails, taken, ctypes.byref(joins), ctypes.byref(partners))
        return [tuple(taken[3 * i: 3 * i + 3]) for i in range(n)], joins.value, partners.value

    return run


CASES = list(itertools.product([0, 5, 37], [0, 1, 2, 3, 5, 7, 8, 15, 16, 17, 19, 31, 32, 45, 64], [1, 2, 3, 9, 40]))


def test_every_chunk_once(walk):
    for begin, count, chunks in CASES:
        seen = []
        for warp in range(16):
            for unit, c0, c1 in walk(begin, begin + count, 6, chunks, warp)[0]:
                seen += [(unit, c) for c in range(c0, c1)]
        assert sorted(seen) == sorted(itertools.product(range(begin, begin + count), range(chunks)))


def test_a_warp_that_gives_up_still_meets_its_partners(walk):
    for begin, count, chunks in CASES:
        whole = [walk(begin, begin + count, 6, chunks, w) for w in range(16)]
        for warp in range(16):
            for fails in (-2, *range(len(whole[warp][0]))):
                ways = list(whole)
                ways[warp] = walk(begin, begin + count, 6, chunks, warp, fails)
                waiting = {}
                for _, bar, partners in ways:
                    if bar:
                        waiting.setdefault((bar, partners), []).append(bar)
                assert all(len(v) == partners for (_, partners), v in waiting.items()), (begin, count, chunks, warp, fails)
                assert ways[warp][1:] == whole[warp][1:]
