"""The product inside the decoder reads only the elements of x that it multiplies: its column arithmetic
(csrc/zn_dot_cols.h, as compiled into the kernel) replayed on the host for every chunk, segment, round
and lane of many weights."""

import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuzipnn_b200", "csrc")

REPLAY = r"""
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include "zn_dot_cols.h"
using namespace zn;

// rows cols chunk log2(sub-chunks): the loops of decode_chunk and dot_round, without the data.
int main(int argc, char** argv) {
  for (int a = 1; a + 3 < argc; a += 4) {
    const int64_t rows = atoll(argv[a]), cols = atoll(argv[a + 1]), chunk = atoll(argv[a + 2]);
    const int t = atoi(argv[a + 3]);
    const int64_t n = rows * cols;
    int64_t loads = 0;
    for (int64_t j = 0; j * chunk < n; ++j) {
      const int64_t m = std::min(chunk, n - j * chunk);
      const int64_t sc = ((((m + (1ll << t) - 1) >> t) + kDotRound - 1) / kDotRound) * kDotRound;
      const int64_t nu = (m + sc - 1) / sc, rounds = sc / kDotRound;
      for (int64_t gi = 0; gi < (nu + 3) / 4 * 4; ++gi) {  // whole warps: segments past nu hold nothing
        const int64_t base = gi * sc, len = gi < nu ? std::min(sc, m - base) : 0, e0 = j * chunk + base;
        DotCols seg;
        seg.start(int(e0 % cols));
        for (int64_t r = 0; r < rounds; ++r) {
          bool active[8], over = false;
          for (int l = 0; l < 8; ++l) {
            const int64_t off = r * kDotRound + l * kDotSteps;
            active[l] = off < len;
            const int c = seg.next(l, active[l], int(cols));
            if (active[l] ? c != (e0 + off) % cols || c + kDotSteps > cols : c != -1) {
              printf("%ld x %ld, chunk %ld, %d sub-chunks: chunk %ld segment %ld round %ld lane %d reads %d\n", rows, cols,
                     chunk, 1 << t, j, gi, r, l, c);
              return 1;
            }
            loads += active[l];
          }
          seg.advance();
          for (int l = 0; l < 8; ++l) over |= seg.wrapped(l, active[l], int(cols));
          if (over) seg.wrap(int(cols));
        }
      }
    }
    if (loads != n / kDotSteps) return printf("%ld loads for %ld elements\n", loads, n), 1;
  }
}
"""


@pytest.fixture(scope="module")
def replay(tmp_path_factory):
    folder = tmp_path_factory.mktemp("dot_cols")
    src, exe = folder / "replay.cpp", folder / "replay"
    src.write_text(REPLAY)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wno-format", "-I", CSRC, str(src), "-o", str(exe)], check=True)

    def run(cases):
        done = subprocess.run([str(exe), *(str(v) for c in cases for v in c)], capture_output=True, text=True)
        assert done.returncode == 0, done.stdout

    return run


def test_short_last_sub_chunks(replay):
    """The last sub-chunk holds a few rounds of many, or whole segments hold nothing."""
    replay([(65, 512, 131072, 4), (100, 640, 65536, 4), (100, 640, 65536, 6), (1, 128, 1024, 2), (3, 144, 4096, 6),
            (97, 3584, 8192, 4), (5, 20000, 1024, 4), (31, 4096, 131072, 6), (257, 272, 16000, 2)])


def test_random_weights(replay):
    rng = random.Random(0)
    cases = []
    for _ in range(400):
        cols = 16 * rng.randint(8, rng.choice([12, 64, 640]))
        cases.append((rng.randint(1, max(1, min(400, 2_000_000 // cols))), cols, 16 * rng.choice([1, 7, 64, 250, 1024, 8192]),
                      rng.randint(2, 6)))
    replay(cases)
