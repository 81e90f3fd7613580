// Which elements of x a lane of the product inside the decoder multiplies (DotSink of zn_decode.cuh).
// Plain C++ without CUDA headers, so that the column arithmetic can be replayed on the host for every
// size and lane, where a read out of range costs nothing (tests/test_dot_cols_cpu.py).
#pragma once

#ifdef __CUDACC__
#define ZN_HD __host__ __device__ __forceinline__
#else
#define ZN_HD inline
#endif

namespace zn {

constexpr int kDotSteps = 16;           // elements per lane and round
constexpr int kDotRound = 8 * kDotSteps;  // and per segment (8 lanes)

// A segment's place in its row of W: `col` is the column of its first element of the round before (below
// 0 when the row ended inside that round).  Only lanes that hold elements move it on into the next row,
// so past a sub-chunk's end (a short last one, or a segment without a sub-chunk) it only grows: lanes
// without elements have no column.
struct DotCols {
  int col;

  ZN_HD void start(int c0) { col = c0 - kDotRound; }
  // Lane l's first column in the next round, or -1 when it holds no elements then.  The lane's elements
  // lie in one row (cols is a multiple of 16 and at least a round), in this one or the next.
  ZN_HD int next(int l, bool active, int cols) const {
    if (!active) return -1;
    const int c = col + kDotRound + l * kDotSteps;
    return c >= cols ? c - cols : c;
  }
  ZN_HD void advance() { col += kDotRound; }
  // After advance(): whether lane l's elements lie in the next row.
  ZN_HD bool wrapped(int l, bool active, int cols) const { return active && col + l * kDotSteps >= cols; }
  // Some lane's did.
  ZN_HD void wrap(int cols) { col -= cols; }
};

}  // namespace zn
