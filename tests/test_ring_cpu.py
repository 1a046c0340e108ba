"""The book-keeping of a warp's ring of copies (csrc/ring.cuh), compiled for the host.

A warp of the streaming product reads its blocks in order, refills a slot when it has read it, and stops at the
first block whose wait gives up.  Before it leaves it has to wait for each copy that is still in flight, and the
parity of each wait has to be that copy's: a phase that has completed already would be no wait at all.
"""

import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lastkv_b200", "csrc")

PROGRAM = """
#include <cstdio>
#include "ring.cuh"

template <int D>
void run(int blocks, int stop) {
  lkv::Ring<D> ring;
  int issued = 0;
  auto load = [&] {
    if (issued == blocks) return;
    std::printf(" c%d", ring.fill());
    ++issued;
  };
  std::printf("%d %d %d:", D, blocks, stop);
  for (int d = 0; d < D; ++d) load();
  for (int i = 0; i < blocks; ++i) {
    std::printf(" w%d,%u", ring.slot, ring.phase);
    if (i == stop) break;
    ring.next();
    load();
  }
  std::printf(" |");
  for (; ring.flying > 0; ring.next()) std::printf(" w%d,%u", ring.slot, ring.phase);
  std::printf("\\n");
}

int main() {
  for (int blocks = 0; blocks <= 13; ++blocks)
    for (int stop = 0; stop <= blocks; ++stop) {
      run<1>(blocks, stop);
      run<2>(blocks, stop);
      run<3>(blocks, stop);
      run<4>(blocks, stop);
    }
}
"""


@pytest.fixture(scope="module")
def lines(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("ring")
    (d / "ring.cpp").write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-I", CSRC, str(d / "ring.cpp"), "-o", str(d / "ring")], check=True)
    return subprocess.run([str(d / "ring")], check=True, capture_output=True, text=True).stdout.splitlines()


def test_waits_are_those_of_the_copies_in_flight(lines):
    assert len(lines) == 4 * sum(b + 1 for b in range(14))
    for line in lines:
        head, rest = line.split(":")
        depth, blocks, stop = map(int, head.split())
        steps, leave = (part.split() for part in rest.split("|"))
        copies = [int(s[1:]) for s in steps if s[0] == "c"]
        waits = [tuple(map(int, s[1:].split(","))) for s in steps if s[0] == "w"]
        left = [tuple(map(int, s[1:].split(","))) for s in leave]
        read = min(stop, blocks)  # blocks that were read before the wait that gave up
        assert copies == [j % depth for j in range(min(blocks, read + depth))]
        assert waits == [(j % depth, j // depth % 2) for j in range(min(blocks, stop + 1))]
        assert left == [(j % depth, j // depth % 2) for j in range(read, len(copies))]
