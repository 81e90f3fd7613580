// A compressed weight as the operand of a product: a rows x cols matrix of 16-bit floats held as a
// blob (the non-stored layout), decoded a range of chunks at a time into a caller's buffer, or
// multiplied with a vector inside the decoder.  Implemented in zn_weight.cu (weight_scan in zn_decode.cu).
#pragma once

#include "zn_common.cuh"

namespace zn {

struct WeightBlob {
  const uint8_t* blob;
  int64_t blob_bytes;
  int64_t rows, cols;
  int64_t chunk;  // elements per chunk
  bool bf16;      // else fp16
  bool direct;    // every chunk finds its units itself, without weight_scan (weight_direct)
};

// Whether a product runs inside the decoder (see DotSink): that of one token.  Measured over 152064 x 3584
// (128 Ki chunks) with a form for several, 1, 2 and 4 tokens took 689, 1016 and 1141 us there (a second
// token's registers cost a fifth of the decoder's occupancy), against 1000 us for decoding and a product
// of any number up to 128; over 3584 x 3584 (16 Ki) 51, 52 and 57 us against 54.
inline bool dot_shape(int64_t tokens, int64_t cols, int64_t chunk) {
  return tokens == 1 && cols % 16 == 0 && cols >= kRound && cols < (int64_t(1) << 30) && chunk % 16 == 0;
}

inline int64_t weight_chunks(const WeightBlob& w) { return cdiv(w.rows * w.cols, w.chunk); }
// Scratch of one weight (unit offsets, the chunks' flags, a counter).
size_t weight_temp_bytes(const WeightBlob& w);
// Whether a weight decoded by one call is better off without the scan of its tables: up to 2048
// chunks, where the 24 KB of tables that a chunk's CTA then reads cost it about 2 us, against 6 us
// or more of a kernel before all others.
inline bool weight_direct(const WeightBlob& w, int64_t pieces) { return pieces == 1 && weight_chunks(w) <= 2048; }
// First step of a call unless w.direct: the offsets of the blob's units; sets the status word.
int weight_scan(const WeightBlob& w, void* temp, int32_t* status, cudaStream_t s);
// A copy of `rows` rows of `cols` 16-bit elements to another pitch, a multiple of 8 (rows = 0: none).
struct PitchCopy {
  const uint16_t* src;
  uint16_t* dst;
  int64_t lds, ldd, rows, cols;
};
#ifdef __CUDACC__
// Its share of warp `w` of `n`: 256 columns of a row at a time, 8 per lane.  A row of the source may
// start at any element, and does so alike for all its groups of 8: a lane loads the one or two
// 16-byte blocks that hold its elements (never one without any of them) and shifts them into place;
// the shift is the warp's.
__device__ __forceinline__ void pitch_rows(const PitchCopy& p, int64_t w, int64_t n) {
  const int64_t per_row = cdiv(p.cols, 256), total = p.rows * per_row;
  const int lane = threadIdx.x & 31;
  for (int64_t i = w; i < total; i += n) {
    const int64_t r = i / per_row, c = (i - r * per_row) * 256 + 8 * lane;
    if (c >= p.cols) continue;
    const int held = int(min(int64_t(8), p.cols - c));
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.src + r * p.lds + c);
    const int shift = int(at & 15) / 2;  // elements before the first in its block
    const uint4* block = reinterpret_cast<const uint4*>(at & ~uintptr_t(15));
    const uint4 v0 = block[0], v1 = held > 8 - shift ? block[1] : make_uint4(0, 0, 0, 0);
    const uint32_t q[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
    uint32_t o[5];
#pragma unroll
    for (int k = 0; k < 5; ++k) {
      const int word = shift >> 1;
      o[k] = word == 0 ? q[k] : word == 1 ? q[(k + 1) & 7] : word == 2 ? q[(k + 2) & 7] : q[(k + 3) & 7];
    }
    if (shift & 1) {
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = __byte_perm(o[k], o[k + 1], 0x5432);
    }
    // The pitch covers the last group of 8 (its padding gets whatever the block held).
    *reinterpret_cast<uint4*>(p.dst + r * p.ldd + c) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}
#endif

// Copies up to this size are made by the kernel that checks the chunks, so that odd sizes cost no
// launches; that kernel has a few CTAs per SM only and moves a larger one at a third of the rate.
constexpr int64_t kTailCopy = 1 << 20;  // elements
// Decode chunks [c0, c1) to `out` (the address of chunk c0's first element, 16-byte aligned), then make
// the two copies (of the decoded rows, and of another operand; each at most kTailCopy elements or
// empty).  Sets the status word (w.direct) or adds to it.
int weight_decode(const WeightBlob& w, void* temp, int64_t c0, int64_t c1, void* out, const PitchCopy& copy0,
                  const PitchCopy& copy1, int32_t* status, cudaStream_t s);
// Chunks that the decoder works on at once on this device (its resident blocks).
int weight_wave(const WeightBlob& w, int64_t* chunks);

// Product inside the decoder: z[r] = sum_c x[c] * W[r, c] (x 16-bit, 16-byte aligned).  Rows that lie in one
// chunk go to z; the parts of rows that span chunks go to `part` ([chunk][2], dot_part_bytes): slot 1
// holds the part of a row that starts in the chunk, slot 0 of one that started before it.
size_t dot_part_bytes(const WeightBlob& w);
// Without w.direct, weight_scan comes first.
int weight_dot(const WeightBlob& w, void* temp, const void* x, float* z, float* part, int32_t* status, cudaStream_t s);

}  // namespace zn
