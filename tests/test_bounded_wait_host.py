"""The bounded wait of the tensor-core kernels (csrc/bounded_wait.h), compiled for the host."""
import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hybridagent_b200", "csrc")
PROGRAM = r"""
#include <cstdio>
#include "bounded_wait.h"
// A clock that moves by `tick` at every look, an arrival that comes at try `arrives` (never if 0), and a flag that another
// thread sets before try `stopped` (never if 0; -1: before the wait).  Prints result, tries and the flag.
template <bool EARLY>
static void run(uint64_t tick, long arrives, long stopped, uint64_t limit) {
  uint64_t t = 0;
  long tries = 0;
  volatile uint32_t stop = stopped < 0;
  const bool ok = ha::bounded_wait<EARLY>(
      [&] {
        ++tries;
        if (stopped > 0 && tries >= stopped) stop = 1;
        return arrives > 0 && tries >= arrives;
      },
      [&] { return t += tick; }, &stop, limit);
  std::printf("%d %ld %u\n", int(ok), tries, unsigned(stop));
}
template <bool EARLY>
static void all() {
  run<EARLY>(1, 1, 0, 100);
  run<EARLY>(1, 1000, 0, 100);
  run<EARLY>(0, 100000, 0, 100);
  run<EARLY>(1, 0, 0, 100);
  run<EARLY>(50, 0, 0, 100);
  run<EARLY>(0, 0, -1, 100);
  run<EARLY>(0, 0, 1, 100);
  run<EARLY>(0, 0, 700, 100);
  run<EARLY>(0, 1, -1, 100);
}
int main() {
  all<false>();
  all<true>();
}
"""


@pytest.fixture(scope="module")
def lines(tmp_path_factory):
    path = tmp_path_factory.mktemp("wait")
    (path / "wait.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", CSRC, str(path / "wait.cpp"), "-o", str(path / "wait")],
                   check=True)
    out = subprocess.run([str(path / "wait")], check=True, capture_output=True, text=True, timeout=60).stdout
    lines = [tuple(map(int, line.split())) for line in out.splitlines()]
    return {"late": lines[:9], "early": lines[9:]}


@pytest.mark.parametrize("kind", ["late", "early"])
def test_an_arrival_ends_the_wait(lines, kind):
    assert lines[kind][0] == (1, 1, 0)
    assert lines[kind][1] == (1, 1000, 0)
    assert lines[kind][2] == (1, 100000, 0)
    assert lines[kind][8] == (1, 1, 1)  # the flag is set, but it has arrived


@pytest.mark.parametrize("kind", ["late", "early"])
def test_a_lost_arrival_ends_it_at_the_limit_and_sets_the_flag(lines, kind):
    ok, tries, stop = lines[kind][3]
    assert not ok and stop and 100 * 256 <= tries <= 103 * 256
    ok, tries, stop = lines[kind][4]
    assert not ok and stop and tries <= 4 * 256


def test_the_flag_ends_it_at_the_next_look(lines):
    assert lines["late"][5] == lines["late"][6] == (0, 257, 1)
    assert lines["early"][5] == lines["early"][6] == (0, 1, 1)  # set before the first look
    assert lines["late"][7] == lines["early"][7] == (0, 1 + 3 * 256, 1)  # set before try 700


def test_warps_read_behind_a_barrier_what_one_lane_has_acquired():
    """The epilogue warps read diagonals that other CTAs stored after lane 0 alone has acquired the word that says so."""
    umma = open(os.path.join(CSRC, "umma.cuh")).read()
    for name in ("granted_to_warp(", "granted_wait_warp("):
        at = umma.index(name)
        body = umma[at:umma.index("\n}\n", at)]
        assert body.index("__all_sync(") < body.index("__syncwarp();") < body.index("return yes;")
    wide = open(os.path.join(CSRC, "newton_schulz.cu")).read()
    assert "granted_now(" not in wide
    for at in (m.start() for m in re.finditer("granted_wait\\(", wide)):  # by single threads, for what they copy
        assert "Warp" not in wide[wide.rindex("\ntemplate", 0, at):at].split("{")[0]


def test_every_wait_of_the_kernels_is_this_one():
    """No kernel polls a barrier by itself.  The narrow one, whose barriers keep all of its threads to the end, takes each
    wait's result and leaves the loops over a matrix's pieces, of which there may be thousands."""
    for name in os.listdir(CSRC):
        text = open(os.path.join(CSRC, name)).read()
        assert name == "umma.cuh" or ("mbar_try(" not in text and "try_wait" not in text), name
    narrow = open(os.path.join(CSRC, "newton_schulz_narrow.cu")).read()
    body = narrow[narrow.index("narrow_kernel("):narrow.index("}  // namespace\n")]
    assert body.count("mbar_wait") == body.count("ok &= mbar_wait<true>(") == 3
    loops = [body[m.start():] for m in re.finditer(r"for \(int i = (from; i < to|0; i < todo); \+\+i\)", body)]
    assert len(loops) == 2 and len(re.findall(r"< pieces\b", body)) == 0
    assert "to = min(from + kPartPieces, gram_pieces);" in body and "gram_pieces = dead ? 0 : pieces;" in body
    assert "if (!__all_sync(0xffffffffu, ok)) break;" in loops[0][:300]
    assert "__syncthreads_or(int(stop))) break;" in loops[1][:150]
