// The chunk decoder: one CTA decodes one chunk of a blob (or one payload of the batched seam) and
// hands its elements to a sink, which stores them or multiplies them.  Included by the two files
// whose kernels run it; everything but the types is local to each.
#pragma once

#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "zn_common.cuh"
#include "zn_dot_cols.h"
#include "zn_weight.cuh"

namespace zn {
namespace {

constexpr int kDecThreads = 128;  // 4 warps per chunk
constexpr int kChains = 1;        // rANS states per lane (sub-chunks per lane)
static_assert(kDotSteps == kSteps && kDotRound == kRound, "a round of the decoder");
constexpr int64_t kCodedBit = int64_t(1) << 62;
constexpr int64_t kOffMask = kCodedBit - 1;

// One decompression job (a blob, or the payload list of the batched seam).  Jobs live in device
// memory; a decode CTA finds its job by global chunk index (find_job).
struct DecArgs {
  // whole-blob mode
  const uint8_t* blob;
  int64_t blob_bytes;
  int64_t* src;           // per unit: blob offset | kCodedBit, or -1 if invalid
  int64_t sizes_off, idx_off, data_off, n_comp;
  int64_t n, C, nch, units, chunk0;
  uint8_t* out;
  int32_t* status;
  // batched mode (K == 1): payload i at in_ptrs[i] (in_bytes[i]) decodes into out_ptrs[i]
  const int64_t* in_ptrs;
  const int64_t* in_bytes;
  const int64_t* out_ptrs;
  const int64_t* out_cap;
  int32_t* statuses;
  uint8_t* overflow;      // per chunk: more coded planes than the main pass holds (weights: its flags)
  int mode;               // kJob, or for a weight kDirect / kScanned
};

// A weight's chunks report through one byte each (kChunkOver | error bits) instead of the status
// word.  kScanned: dscan_kernel has filled `src`.  kDirect: every chunk finds its units itself.
constexpr int kJob = 0, kScanned = 1, kDirect = 2;
constexpr uint8_t kChunkOver = 128;

struct PlaneInfo {
  const uint8_t* pl;  // payload (coded) or raw bytes of this unit's chunk
  const uint8_t* lo;  // stream block loads may touch [lo, hi)
  const uint8_t* hi;
  int64_t size;
  int coded;
  int t;
  int single;              // the symbol of a plane with one symbol (f = M: no words, no state change), else -1
  int64_t states_off;
  int64_t lens_off;        // per-state stream lengths
  int lw;                  // bytes per length field
  int32_t stream_off[64];  // halfword index of each sub-chunk's first (lane 0) stream
};

struct DecSmem {
  uint32_t hi[256];            // per present symbol, ascending: f << 20 | symbol << 12
  uint32_t cum[256];           // and its first slot
  uint32_t start[kM / 32];     // bit z: a symbol's slots start at z
  uint32_t sub[64];            // words of each sub-chunk's streams
  uint32_t count[kDecThreads / 32], freq[kDecThreads / 32], starts[kDecThreads / 32];
  int err;
  int64_t sums[2][kDecThreads / 32];
  int coded[2];
  PlaneInfo p[8];
};

// Inclusive sum over the lanes of a warp.
__device__ __forceinline__ uint32_t warp_scan(uint32_t v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xFFFFFFFFu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// Parse a ZNR2 payload header and build its decode table.  Entry of slot z (symbol s, cum c, freq
// f < M): f << 20 | s << 12 | (z - c), so the state update f * (x >> 12) + (z - c) is one IMAD
// after the lookup.  A plane with a single symbol (f = M) needs no table: its state never changes
// and it has no words; P.single holds that symbol.  Returns false (uniformly) if the payload is
// malformed.
//
// A chunk's start is all latency, so the steps are few and wide: thread i owns symbols 2i and 2i + 1
// (ballots number the present ones, one scan gives their first slots) and loads a stream length;
// the table is filled 32 slots per warp step, a slot's symbol being the count of symbol starts up
// to it (a bit mask of starts, popc and a scan over its words).
__device__ bool build_plane(PlaneInfo& P, int64_t m, uint32_t* tab, DecSmem& S) {
  static_assert(kDecThreads == 128 && kM / 32 == kDecThreads, "two symbols and one start word per thread");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint8_t* pl = P.pl;
  const int64_t size = P.size;
  if (size < 34) return false;
  const int t = pl[0], flag = pl[1];
  const uint32_t bits = (pl[2 + (tid >> 2)] >> (2 * (tid & 3))) & 3;  // presence of symbols 2 tid, 2 tid + 1
  if (t < kMinSubLog2 || t > kMaxSubLog2 || flag != 0) return false;
  S.start[tid] = 0;
  const uint32_t b0 = __ballot_sync(0xFFFFFFFFu, bits & 1), b1 = __ballot_sync(0xFFFFFFFFu, bits >> 1);
  if (lane == 0) S.count[warp] = __popc(b0) + __popc(b1);
  __syncthreads();
  const uint32_t below = (1u << lane) - 1;
  uint32_t np = 0, k = __popc(b0 & below) + __popc(b1 & below);
#pragma unroll
  for (int w = 0; w < kDecThreads / 32; ++w) {
    if (w < warp) k += S.count[w];
    np += S.count[w];
  }
  const int64_t tb = table_bytes(int(np));
  const Geom g = geom_of(m, t);
  const int64_t mb = meta_bytes(int(np), g);
  if (np == 0 || mb > size) return false;
  uint32_t f[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    f[h] = 0;
    if ((bits >> h) & 1) {
      const uint32_t bit = 12 * (k + (h ? bits & 1 : 0));
      const uint8_t* q = pl + 34 + (bit >> 3);
      const uint32_t v = (uint32_t(q[0]) | (uint32_t(q[1]) << 8) | (uint32_t(q[2]) << 16)) >> (bit & 7);
      f[h] = (v & 0xFFF) + 1;
    }
  }
  // Stream lengths, a field per thread; a sub-chunk's are 8 neighbouring lanes.
  bool good = true;
  const int fields = g.nu * kLanes;
  for (int f0 = 0; f0 < fields; f0 += kDecThreads) {
    const int fi = f0 + tid;
    uint32_t nw = 0;
    if (fi < fields)
      nw = g.lw == 2 ? *reinterpret_cast<const uint16_t*>(pl + tb + 2 * fi)
                     : *reinterpret_cast<const uint32_t*>(pl + tb + 4 * int64_t(fi));
    good &= nw <= g.sc / kLanes;
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) nw += __shfl_xor_sync(0xFFFFFFFFu, nw, o);
    if (fi < fields && (lane & (kLanes - 1)) == 0) S.sub[fi / kLanes] = nw;
  }
  const uint32_t incl = warp_scan(f[0] + f[1]);
  if (lane == 31) S.freq[warp] = incl;
  __syncthreads();
  uint32_t c = incl - f[0] - f[1], total = 0;
#pragma unroll
  for (int w = 0; w < kDecThreads / 32; ++w) {
    if (w < warp) c += S.freq[w];
    total += S.freq[w];
  }
  if (total != kM) return false;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (f[h]) {
      const uint32_t s = 2 * tid + h;
      S.hi[k] = (f[h] << 20) | (s << 12);  // f = M (one symbol) wraps: the table is unused
      S.cum[k] = c;
      atomicOr(&S.start[c >> 5], 1u << (c & 31));
      if (np == 1) P.single = int(s);
      ++k;
      c += f[h];
    }
  if (warp == 0) {  // where each sub-chunk's streams start
    int64_t pos = mb / 2;
    for (int g0 = 0; g0 < g.nu; g0 += 32) {
      const int gi = g0 + lane;
      const int64_t sub = gi < g.nu ? S.sub[gi] : 0;
      int64_t in = sub;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xFFFFFFFFu, in, o);
        if (lane >= o) in += v;
      }
      if (gi < g.nu) P.stream_off[gi] = int32_t(pos + in - sub);
      pos += __shfl_sync(0xFFFFFFFFu, in, 31);
    }
    good &= 2 * pos == size;
    if (tid == 0) {
      P.t = t;
      P.lens_off = tb;
      P.lw = g.lw;
      P.states_off = tb + lengths_bytes(g);
    }
  }
  if (!__syncthreads_and(good)) return false;
  // Warp w fills slots [1024 w, 1024 w + 1024): lane i holds start word 32 w + i.
  const uint32_t word = S.start[tid];
  const uint32_t in = warp_scan(__popc(word));
  if (lane == 31) S.starts[warp] = in;
  __syncthreads();
  uint32_t before = in - __popc(word);
#pragma unroll
  for (int w = 0; w < kDecThreads / 32; ++w)
    if (w < warp) before += S.starts[w];
  const uint32_t upto = 0xFFFFFFFFu >> (31 - lane);
#pragma unroll 8
  for (int i = 0; i < 32; ++i) {
    const uint32_t wi = __shfl_sync(0xFFFFFFFFu, word, i), bi = __shfl_sync(0xFFFFFFFFu, before, i);
    const uint32_t q = bi + __popc(wi & upto) - 1, z = 1024 * warp + 32 * i + lane;
    tab[z] = S.hi[q] | (z - S.cum[q]);
  }
  __syncthreads();
  return true;
}

// One 16-byte block of a word stream.  Blocks wholly inside [lo, hi) are one 16-byte load; a block
// that straddles the edge is read halfword by halfword (outside halfwords read as 0).
__device__ __forceinline__ uint4 load_block(const uint8_t* gb, uint32_t q, const uint8_t* lo, const uint8_t* hi) {
  const uint8_t* p = gb + 16 * uint64_t(q);
  if (p >= lo && p + 16 <= hi) return __ldg(reinterpret_cast<const uint4*>(p));
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int h = 0; h < 8; ++h) {
    const uint8_t* q2 = p + 2 * h;
    if (q2 >= lo && q2 + 2 <= hi) w[h >> 1] |= uint32_t(*reinterpret_cast<const uint16_t*>(q2)) << (16 * (h & 1));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Decoder state of one rANS state (a lane of a sub-chunk) of one coded plane.  Stream positions
// are halfword indices relative to the 16-byte aligned base gb of the payload.  Each state keeps
// a ring of kRing words of its stream in shared memory: at every round start [ptr, ptr + 16) is
// present (a round consumes at most 16 words) and 16-byte blocks ahead are loaded, to be stored
// at the round's end.
struct Cursor {
  uint32_t x, ptr, end, fill, nload;
  uint4 r0, r1;
};

// Ring layout: slot p of the state of thread t sits at rings[(p % kRing) * kDecThreads + t] (rows
// of kDecThreads slots), so the 32 states of a warp read their next words from 32 different banks
// when a slot is 32 bits wide (one stream halfword in its low half; the decoder ignores the upper
// half).  With more than 4 coded planes in shared memory the slots are halfwords (at most two
// lanes per bank).
constexpr int kRing = 32;
template <int KC>
using RingSlot = std::conditional_t<(KC > 4), uint16_t, uint32_t>;

// Store the 16-byte stream block that starts at halfword `fill` (a multiple of 8) into a ring.
template <typename Slot>
__device__ __forceinline__ void ring_put(Slot* ring, uint32_t fill, const uint4& v) {
  Slot* r = ring + (fill & (kRing - 1)) * kDecThreads;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[(2 * i) * kDecThreads] = Slot(w[i]);
    r[(2 * i + 1) * kDecThreads] = Slot(w[i] >> 16);
  }
}

// One decode step of one state (symbol into byte (i & 3) of acc, next word read one step ahead).
template <bool FULL, int I, typename Slot>
__device__ __forceinline__ void decode_step(uint32_t& xv, uint32_t& pv, uint32_t& wn, uint32_t& acc, bool act,
                                            const uint32_t* __restrict__ tab, const Slot* ring) {
  const uint32_t e = tab[xv & (kM - 1)];
  const uint32_t q = xv >> kScaleBits;
  uint32_t xn = (e >> 20) * q + (e & 0xFFFu);
  if (!FULL) xn = act ? xn : xv;
  acc = __byte_perm(acc, e >> 12, (0x3210 & ~(0xF << (4 * (I & 3)))) | (4 << (4 * (I & 3))));
  const bool need = (FULL || act) && xn < kL;
  const uint32_t w = wn;
  pv += need;
  wn = ring[(pv & (kRing - 1)) * kDecThreads];
  xv = need ? __byte_perm(w, xn, 0x5410) : xn;  // (xn << 16) | (w & 0xFFFF)
}

// 16 steps of the lane's kChains states, interleaved so the independent chains overlap.  A stream
// over-read is not tested per step: it leaves the final state or position wrong, which the caller
// checks (ring reads are always in bounds).
template <bool FULL, typename Slot>
__device__ __forceinline__ void decode_round(Cursor* cb, const uint32_t* __restrict__ tab, Slot* const* ring,
                                             const int* nact, uint32_t (*acc)[4]) {
  uint32_t xv[kChains], pv[kChains], wn[kChains];
#pragma unroll
  for (int c = 0; c < kChains; ++c) {
    xv[c] = cb[c].x;
    pv[c] = cb[c].ptr;
    wn[c] = ring[c][(pv[c] & (kRing - 1)) * kDecThreads];
  }
#define ZN_STEP(I)                                                                                    \
  _Pragma("unroll") for (int c = 0; c < kChains; ++c)                                                 \
      decode_step<FULL, I>(xv[c], pv[c], wn[c], acc[c][(I) >> 2], (I) < nact[c], tab, ring[c]);
  ZN_STEP(0) ZN_STEP(1) ZN_STEP(2) ZN_STEP(3) ZN_STEP(4) ZN_STEP(5) ZN_STEP(6) ZN_STEP(7)
  ZN_STEP(8) ZN_STEP(9) ZN_STEP(10) ZN_STEP(11) ZN_STEP(12) ZN_STEP(13) ZN_STEP(14) ZN_STEP(15)
#undef ZN_STEP
#pragma unroll
  for (int c = 0; c < kChains; ++c) {
    cb[c].x = xv[c];
    cb[c].ptr = pv[c];
  }
}

// The fast path's 16 steps of the lane's kChains states.  A state's ring position is kept as the
// byte offset tid * 4 + (ptr % kRing) * kDecThreads * 4 from its ring's first row, so the word
// read after a renormalisation costs one masked add; the position advance is recovered at the end
// (a round consumes at most 16 < kRing words).
__device__ __forceinline__ void decode_round_fast(Cursor* cb, const uint32_t* __restrict__ tab, const uint8_t* rows,
                                                  int tid, uint32_t (*acc)[4]) {
  constexpr uint32_t kRowBytes = kDecThreads * 4, kRingBytes = kRing * kRowBytes;
  uint32_t xv[kChains], ro[kChains], ro0[kChains], wn[kChains], pair[kChains];
#pragma unroll
  for (int c = 0; c < kChains; ++c) {
    xv[c] = cb[c].x;
    ro0[c] = uint32_t(tid) * 4 + (cb[c].ptr & (kRing - 1)) * kRowBytes;
    ro[c] = ro0[c];
    wn[c] = *reinterpret_cast<const uint32_t*>(rows + c * kRingBytes + ro[c]);
  }
#define ZN_FSTEP(I)                                                                                   \
  _Pragma("unroll") for (int c = 0; c < kChains; ++c) {                                               \
    const uint32_t e = tab[xv[c] & (kM - 1)];                                                         \
    const uint32_t xn = (e >> 20) * (xv[c] >> kScaleBits) + (e & 0xFFFu);                             \
    const bool need = xn < kL;                                                                        \
    const uint32_t w = wn[c];                                                                         \
    ro[c] = need ? ((ro[c] + kRowBytes) & (kRingBytes - 1)) : ro[c];                                  \
    wn[c] = *reinterpret_cast<const uint32_t*>(rows + c * kRingBytes + ro[c]);                        \
    xv[c] = need ? __byte_perm(w, xn, 0x5410) : xn;                                                   \
    /* Symbols (bits 12-19 of the entries) four at a time: two entries' middle bytes side by side,  \
       shifted to the byte boundary, then one byte of each. */                                        \
    if (((I) & 1) == 0) pair[c] = e;                                                                  \
    else if (((I) & 3) == 1) acc[c][(I) >> 2] = __byte_perm(pair[c], e, 0x6521) >> 4;                 \
    else acc[c][(I) >> 2] = __byte_perm(acc[c][(I) >> 2], __byte_perm(pair[c], e, 0x6521) >> 4, 0x6420); \
  }
  ZN_FSTEP(0) ZN_FSTEP(1) ZN_FSTEP(2) ZN_FSTEP(3) ZN_FSTEP(4) ZN_FSTEP(5) ZN_FSTEP(6) ZN_FSTEP(7)
  ZN_FSTEP(8) ZN_FSTEP(9) ZN_FSTEP(10) ZN_FSTEP(11) ZN_FSTEP(12) ZN_FSTEP(13) ZN_FSTEP(14) ZN_FSTEP(15)
#undef ZN_FSTEP
#pragma unroll
  for (int c = 0; c < kChains; ++c) {
    cb[c].x = xv[c];
    cb[c].ptr += (ro[c] / kRowBytes - ro0[c] / kRowBytes) & (kRing - 1);
  }
}

// The 16 symbols of a round of a one-symbol plane, for every chain.
__device__ __forceinline__ void fill_single(uint32_t (*acc)[4], int s) {
#pragma unroll
  for (int c = 0; c < kChains; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[c][i] = uint32_t(s) * 0x01010101u;
}

// Raw (stored) plane bytes of round r for each chain: 16 bytes per plane from the lane's 16
// symbols, byte by byte in a partial last round.  Coded planes are left untouched.
template <int K, int NC>
__device__ __forceinline__ void load_raw_round(const uint8_t* const* src, const bool* coded, const int64_t* base,
                                               const int64_t* len, int r, int l, uint32_t (*p)[K][4]) {
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int64_t off = int64_t(r) * kRound + l * kSteps;
    const int nact = int(max(int64_t(0), min(int64_t(kSteps), len[c] - off)));
#pragma unroll
    for (int b = 0; b < K; ++b) {
      if (coded[b]) continue;
      const uint8_t* sp = src[b] + base[c] + off;
      if (nact == 16) {
        const uint2 v0 = reinterpret_cast<const uint2*>(sp)[0], v1 = reinterpret_cast<const uint2*>(sp)[1];
        p[c][b][0] = v0.x; p[c][b][1] = v0.y; p[c][b][2] = v1.x; p[c][b][3] = v1.y;
      } else {
        uint64_t vlo = 0, vhi = 0;
        for (int i = 0; i < nact; ++i) {
          const uint64_t byte = sp[i];
          if (i < 8) vlo |= byte << (8 * i);
          else vhi |= byte << (8 * (i - 8));
        }
        p[c][b][0] = uint32_t(vlo); p[c][b][1] = uint32_t(vlo >> 32);
        p[c][b][2] = uint32_t(vhi); p[c][b][3] = uint32_t(vhi >> 32);
      }
    }
  }
}

// 16 elements (4 * K little-endian words) from their K byte planes (4 words each), with the
// exponent reorder undone.  bf16 has a direct form: with E the exponent plane (high bytes after
// the reorder, e8) and B the sign / mantissa plane (s m7), the element's high byte is
// s | e8 >> 1 and its low byte (e8 & 1) << 7 | m7, four elements per 32-bit operation.
template <int K, bool REORDER>
__device__ __forceinline__ void assemble_elements(const uint32_t (*p)[4], uint32_t* e) {
  if constexpr (K == 2 && REORDER) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t E = p[1][i], B = p[0][i];
      const uint32_t hi = (B & 0x80808080u) | ((E >> 1) & 0x7F7F7F7Fu);
      const uint32_t lo = ((E << 7) & 0x80808080u) | (B & 0x7F7F7F7Fu);
      e[2 * i] = __byte_perm(lo, hi, 0x5140);
      e[2 * i + 1] = __byte_perm(lo, hi, 0x7362);
    }
  } else {
    planes_to_elements<K>(p, e);
    reorder_words<K, REORDER, false>(e, 4 * K);
  }
}

// Where a chunk's elements go.  StoreSink: to the job's output, as they lie in the tensor.
struct StoreSink {
  static constexpr bool kDot = false;
};

// DotSink: the elements are rows of a weight W[rows, cols] and are multiplied with the matching
// elements of a vector x as they leave the decoder; W itself is never written.
//
// A lane's 16 elements of a round lie in one row (cols and the chunk size are multiples of 16), and
// a row is at least one round (128 elements) long, so a segment (8 lanes, one sub-chunk) crosses at
// most one row end per round.  The products are taken by mma.m16n8k16 with 32-bit sums, although
// every lane has its own place in W and x: with a lane's words of W as its part of A's rows 0-7 and
// the matching words of x as its part of B, the diagonal element D[r, r] is the sum of the own
// products of lanes 4r .. 4r + 3, whatever these are (the other elements mean nothing and are
// dropped).  4 such steps take the lane's 16 elements as they are packed; with scalar arithmetic
// their 32 conversions and 16 dependent additions made one token's product 30 % slower than the
// decoding alone.  At a row end the segment's two diagonal elements are added, and lanes beyond it
// start the next row.
//
// A row inside one sub-chunk is complete then and goes to z.  Parts of rows that span sub-chunks go
// to shared slots (per sub-chunk: 0 = the row started before it, 1 = it starts here and goes on),
// which the CTA adds in order at the end; rows that span chunks leave their parts in `part` with the
// same rule per chunk.  No atomics: the result does not depend on the order in which chunks are
// decoded.
template <typename T>
struct DotSink {
  static constexpr bool kDot = true;
  using Elem = T;
  const T* x;
  int cols;
  float* z;     // [rows]
  float* part;  // [chunk][2]
};

struct DotState {
  float c[2];      // row lane / 4, columns 2 (lane % 4) and + 1 of the accumulator
  DotCols cols;    // the segment's place in its current row
  int row;         // the segment's current row
  bool first;      // no row end met in this sub-chunk yet
  bool mid;        // the sub-chunk starts inside a row
  uint4 x[2];      // the round's elements of x, loaded before it is decoded
};

// Loads the next round's elements of x.  Lanes without elements load nothing: dot_products masks what
// they hold.
template <class Sink>
__device__ __forceinline__ void dot_load(const Sink& k, DotState& st, int l, bool active) {
  const int col = st.cols.next(l, active, k.cols);
  if (col < 0) return;
  const uint4* xp = reinterpret_cast<const uint4*>(k.x + col);
  st.x[0] = __ldg(xp);
  st.x[1] = __ldg(xp + 1);
}

// One step of the products: rows 0-7 of A from a0, a2, rows 8-15 zero.
__device__ __forceinline__ void dot_mma(float* c, uint32_t a0, uint32_t a2, uint32_t b0, uint32_t b1, __nv_bfloat16) {
  [[maybe_unused]] float d2, d3;
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %5}, {%7, %8}, {%9, %10, %11, %11};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(d2), "=f"(d3)
      : "r"(a0), "r"(0u), "r"(a2), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(0.0f));
}
__device__ __forceinline__ void dot_mma(float* c, uint32_t a0, uint32_t a2, uint32_t b0, uint32_t b1, __half) {
  [[maybe_unused]] float d2, d3;
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %5}, {%7, %8}, {%9, %10, %11, %11};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(d2), "=f"(d3)
      : "r"(a0), "r"(0u), "r"(a2), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(0.0f));
}
// Lanes with `use` add their products, the others nothing (both factors are zeroed: 0 * inf is NaN).
template <class Sink, bool MASKED>
__device__ __forceinline__ void dot_products(DotState& st, const uint32_t* e, bool use) {
  const uint4 a = st.x[0], b = st.x[1];
  uint32_t w[8], x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    w[i] = !MASKED || use ? e[i] : 0u;
    if (MASKED && !use) x[i] = 0u;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) dot_mma(st.c, w[2 * i], w[2 * i + 1], x[2 * i], x[2 * i + 1], typename Sink::Elem());
}

// The segment's sum (on all its lanes): its two quads' diagonal elements.
__device__ __forceinline__ float segment_sum(const DotState& st) {
  const int lane = threadIdx.x & 31, quad = lane >> 2;
  float v = (lane & 3) == (quad >> 1) ? ((quad & 1) ? st.c[1] : st.c[0]) : 0.0f;
#pragma unroll
  for (int o = 4; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// One round of a warp's segments: 16 elements per lane (8 words), none for inactive lanes.  Called
// by whole warps.
template <class Sink, bool ALL>
__device__ __forceinline__ void dot_round(const Sink& k, DotState& st, const uint32_t* e, bool active, int l, int seg,
                                          float* slot0) {
  st.cols.advance();
  const bool wrapped = st.cols.wrapped(l, active, k.cols);  // the lane's elements lie in the next row
  const uint32_t over = __ballot_sync(0xFFFFFFFFu, wrapped);
  if (!over) {
    dot_products<Sink, !ALL>(st, e, active);
    return;
  }
  dot_products<Sink, true>(st, e, active && !wrapped);
  const float v = segment_sum(st);
  if ((over >> (8 * seg)) & 0xFF) {
    if (l == 0) {
      if (st.first && st.mid) *slot0 = v;
      else k.z[st.row] = v;
    }
    st.c[0] = st.c[1] = 0.0f;
    st.first = false;
    ++st.row;
    st.cols.wrap(k.cols);
  }
  dot_products<Sink, true>(st, e, wrapped);
}

// The rows of chunk j (elements [g0, g1)) that no single sub-chunk completed: the sums of their
// slots, in order, to z (rows inside the chunk) or `part`.  With `bad`, zeros for every row.
template <class Sink>
__device__ __forceinline__ void dot_finish_chunk(const Sink& k, int64_t j, int64_t g0, int64_t g1, int64_t sc,
                                                 const float* slots, bool bad) {
  const int64_t r0 = g0 / k.cols, r1 = (g1 - 1) / k.cols;
  for (int64_t row = r0 + threadIdx.x; row <= r1; row += kDecThreads) {
    const int64_t lo = row * k.cols, hi = lo + k.cols;
    const bool starts = lo >= g0, complete = starts && hi <= g1;
    const int sa = int((max(lo, g0) - g0) / sc), sb = int((min(hi, g1) - 1 - g0) / sc);
    if (sa == sb && complete && !bad) continue;
    float v = 0.0f;
    if (!bad)
      for (int s = sa; s <= sb; ++s) {
        const int64_t s0 = g0 + s * sc, s1 = min(s0 + sc, g1);
        v += slots[2 * s + (lo >= s0 && hi > s1 ? 1 : 0)];
      }
    if (complete) k.z[row] = v;
    else k.part[2 * j + starts] = v;
  }
}

// Offset (with kCodedBit, or -1) of the units of chunk j of a weight, by the whole CTA from the blob's
// tables: what dscan_kernel computes for all units at once, with the same checks.  It reads the
// tables up to the chunk's second unit (12 bytes per chunk of the blob, from L2 but for the first
// CTA), so it pays for small weights (weight_direct), whose launch it saves.
__device__ __forceinline__ void find_units(const DecArgs& a, int64_t j, DecSmem& S, int64_t* unit, bool* bad) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < 2) S.coded[tid] = 0;
  __syncthreads();
  const int64_t n_comp = *reinterpret_cast<const uint32_t*>(a.blob + 12);
  const int64_t data_off = align8(a.idx_off + 4 * n_comp);
  bool wrong = false;
  *bad = false;
  if (n_comp > a.units || data_off > a.blob_bytes) {  // uniform
    unit[0] = unit[1] = -1;
    *bad = true;
    return;
  }
  const int32_t* stored = reinterpret_cast<const int32_t*>(a.blob + a.sizes_off);
  const int32_t* idx = reinterpret_cast<const int32_t*>(a.blob + a.idx_off);
  const int nch = int(a.nch), end = nch + int(j);
  int64_t s0 = 0, s1 = 0;
#pragma unroll 4
  for (int i = tid; i < end; i += kDecThreads) {
    const int32_t s = stored[i];
    wrong |= s < 0;
    const int64_t v = s < 0 ? 0 : align8(s);
    s1 += v;
    if (i < j) s0 += v;
  }
#pragma unroll 4
  for (int i = tid; i < int(n_comp); i += kDecThreads) {
    const int32_t u = idx[i];
    wrong |= u < 0 || u >= a.units;
    if (u == j) S.coded[0] = 1;
    if (u == end) S.coded[1] = 1;
  }
  for (int o = 16; o; o >>= 1) {
    s0 += __shfl_xor_sync(0xFFFFFFFFu, s0, o);
    s1 += __shfl_xor_sync(0xFFFFFFFFu, s1, o);
  }
  if (lane == 0) {
    S.sums[0][warp] = s0;
    S.sums[1][warp] = s1;
  }
  wrong = __syncthreads_or(wrong);
  const int64_t raw = j == a.nch - 1 ? a.n - j * a.C : a.C;
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    int64_t off = data_off;
#pragma unroll
    for (int w = 0; w < kDecThreads / 32; ++w) off += S.sums[b][w];
    const int64_t st = stored[b * a.nch + j];
    const bool coded = S.coded[b] != 0;
    unit[b] = st < 0 || off + st > a.blob_bytes || (!coded && st != raw) ? -1 : off | (coded ? kCodedBit : 0);
  }
  *bad = wrong;
}

// Decode chunk j of a job with the whole CTA.  KC: coded planes per chunk held in shared memory.
// The main pass (KC = 1 for K > 1) flags chunks with more coded planes; a second pass with KC = K
// decodes only those.  Every return is taken by all threads of the CTA together.
// Work split: a warp item is 8 sub-chunks; lane l of 8-lane segment g runs chain c on sub-chunk
// 8 * item + 4 * c + g.
// WEIGHT: a chunk of a weight (DecArgs::mode).
template <int K, bool REORDER, int KC, bool WEIGHT = false, class Sink>
__device__ __forceinline__ void decode_chunk(const DecArgs& a, int64_t j, bool overflow_pass, const Sink& sink) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  using Slot = RingSlot<KC>;
  uint32_t* tabs = reinterpret_cast<uint32_t*>(smem_raw);                      // [KC][4096]
  Slot* rings = reinterpret_cast<Slot*>(smem_raw + KC * kM * 4);                // [KC][kChains][kRing][threads]
  DecSmem& S = *reinterpret_cast<DecSmem*>(smem_raw + KC * kM * 4 + KC * kChains * kRing * kDecThreads * sizeof(Slot));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  static_assert(!Sink::kDot || (K == 2 && kChains == 1), "products take 16-bit elements, one chain per lane");
  [[maybe_unused]] float* slots = reinterpret_cast<float*>(&S + 1);  // DotSink: [64 sub-chunks][2]
  if (overflow_pass && !a.overflow[j]) return;
  const bool batched = a.in_ptrs != nullptr;
  int64_t m;
  uint8_t* outc;
  if (batched) {
    m = a.out_cap[j];
    outc = reinterpret_cast<uint8_t*>(a.out_ptrs[j]);
  } else {
    m = min(a.C, a.n - j * a.C);
    outc = a.out + j * a.C * K;
  }
  if constexpr (Sink::kDot)
    for (int i = tid; i < 64 * 2; i += kDecThreads) slots[i] = 0.0f;
  int flags = 0;  // weights: error bits of this chunk
  [[maybe_unused]] int64_t unit[2] = {-1, -1};
  if constexpr (WEIGHT)
    if (a.mode == kDirect) {
      bool wrong;
      find_units(a, j, S, unit, &wrong);
      if (wrong) flags |= kErrTable;
    }
  if (tid == 0) S.err = 0;
  if constexpr (WEIGHT) __syncthreads();
  if (tid < K) {
    PlaneInfo& P = S.p[tid];
    if (batched) {
      P.pl = reinterpret_cast<const uint8_t*>(a.in_ptrs[j]);
      P.size = a.in_bytes[j];
      P.coded = 1;
      P.lo = P.pl;
      P.hi = P.pl + P.size;
    } else {
      const int64_t u = int64_t(tid) * a.nch + j;
      int64_t s;
      if constexpr (WEIGHT) s = a.mode != kDirect ? a.src[u] : tid == 0 ? unit[0] : unit[1];
      else s = a.src[u];
      // dscan_kernel has checked that the tables lie inside the blob for every unit with s >= 0.
      const int64_t stored = s >= 0 ? *reinterpret_cast<const int32_t*>(a.blob + a.sizes_off + 4 * u) : 0;
      P.coded = s >= 0 && (s & kCodedBit);
      P.pl = a.blob + (s & kOffMask);
      P.size = stored;
      P.lo = a.blob;
      P.hi = a.blob + a.blob_bytes;
      if (s < 0) atomicOr(&S.err, 1);
    }
    P.t = -1;
    P.single = -1;
  }
  __syncthreads();
  int ncoded = 0;
  int pslot[KC];  // plane of each coded slot
#pragma unroll
  for (int q = 0; q < KC; ++q) pslot[q] = 0;
  for (int b = 0; b < K; ++b)
    if (S.p[b].coded) {
      if (ncoded < KC) pslot[ncoded] = b;
      ++ncoded;
    }
  if (KC < K && !overflow_pass) {
    const bool over = ncoded > KC;
    if constexpr (WEIGHT) {
      if (over) {
        if (tid == 0) a.overflow[j] = uint8_t(kChunkOver | flags);
        return;
      }
    } else {
      if (tid == 0) a.overflow[j] = over;
      if (over) return;
    }
  }
  bool bad = S.err != 0 || m <= 0;
  for (int q = 0; q < KC && q < ncoded && !bad; ++q)
    if (!build_plane(S.p[pslot[q]], m, tabs + q * kM, S)) bad = true;
  int t = 4;
  if (!bad && ncoded) {
    t = S.p[pslot[0]].t;
    // All coded planes of a chunk must share one sub-chunk geometry.
    for (int q = 0; q < KC && q < ncoded; ++q)
      if (S.p[pslot[q]].t != t) bad = true;
  }
  if (bad) {
    if (tid == 0) {
      if (WEIGHT) a.overflow[j] = uint8_t((overflow_pass ? kChunkOver : 0) | flags | kErrPayload);
      else if (batched) a.statuses[j] = kErrPayload;
      else atomicOr(a.status, kErrPayload);
    }
    if constexpr (Sink::kDot) {
      if (m > 0) dot_finish_chunk(sink, j, j * a.C, j * a.C + m, m, slots, true);
    } else {
      if (m > 0)
        for (int64_t i = tid; i < m * K; i += kDecThreads) outc[i] = 0;
    }
    return;
  }

  const Geom g = geom_of(m, t);
  const int seg = lane >> 3, l = lane & 7;
  const int rounds = int(g.sc / kRound);
  const bool out16 = (reinterpret_cast<uintptr_t>(outc) & 15) == 0;
  // A lane's 16 elements as whole 32-byte sectors per store instruction (two 16-byte stores at a
  // 32-byte stride use half of every sector they touch).
  [[maybe_unused]] const bool out32 = (reinterpret_cast<uintptr_t>(outc) & 31) == 0;
  bool coded[K];
  const uint8_t* src[K];
#pragma unroll
  for (int b = 0; b < K; ++b) {
    coded[b] = S.p[b].coded;
    src[b] = S.p[b].pl;
  }
  bool raw16 = true;  // every raw plane starts on a 16-byte boundary (units are aligned to 8)
#pragma unroll
  for (int b = 0; b < K; ++b)
    if (!coded[b]) raw16 &= (reinterpret_cast<uintptr_t>(src[b]) & 15) == 0;
  const uint8_t* gb[KC];
  const uint8_t* lo[KC];
  const uint8_t* hi[KC];
#pragma unroll
  for (int q = 0; q < KC; ++q) {
    gb[q] = reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(S.p[pslot[q]].pl) & ~uintptr_t(15));
    lo[q] = S.p[pslot[q]].lo;
    hi[q] = S.p[pslot[q]].hi;
  }
  bool err = false;
  const int items = int(cdiv(g.nu, 4 * kChains));
  for (int item = warp; item < items; item += kDecThreads / 32) {
    int gi[kChains];
    int64_t base[kChains], len[kChains];
    bool valid[kChains];
#pragma unroll
    for (int c = 0; c < kChains; ++c) {
      gi[c] = 4 * kChains * item + 4 * c + seg;
      valid[c] = gi[c] < g.nu;
      base[c] = int64_t(gi[c]) * g.sc;
      len[c] = valid[c] ? min(g.sc, m - base[c]) : 0;
    }
    Cursor cur[KC][kChains];
    Slot* ring[KC][kChains];
    int single[KC];  // symbol of a one-symbol coded plane, else -1
#pragma unroll
    for (int q = 0; q < KC; ++q) single[q] = q < ncoded ? S.p[pslot[q]].single : -1;
#pragma unroll
    for (int q = 0; q < KC; ++q)
#pragma unroll
      for (int c = 0; c < kChains; ++c) {
        Cursor& cb = cur[q][c];
        ring[q][c] = rings + (q * kChains + c) * kRing * kDecThreads + tid;
        cb.x = kL;
        cb.ptr = cb.end = cb.fill = cb.nload = 0;
        if (q >= ncoded) continue;
        const PlaneInfo& P = S.p[pslot[q]];
        const int64_t fbase = int64_t(gi[c]) * kLanes;
        uint32_t mine = 0;
        if (valid[c])
          mine = P.lw == 2 ? *reinterpret_cast<const uint16_t*>(P.pl + P.lens_off + 2 * (fbase + l))
                           : *reinterpret_cast<const uint32_t*>(P.pl + P.lens_off + 4 * (fbase + l));
        uint32_t before = mine;  // words of the sub-chunk's lanes before this one
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) {
          const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, before, o, kLanes);
          if (l >= o) before += v;
        }
        before -= mine;
        if (valid[c]) {
          const uint32_t h0 = uint32_t((P.pl - gb[q]) >> 1) + uint32_t(P.stream_off[gi[c]]) + before;
          cb.x = *reinterpret_cast<const uint32_t*>(P.pl + P.states_off + 4 * (fbase + l));
          cb.ptr = h0;
          cb.end = h0 + mine;
          cb.fill = h0 & ~7u;
          err |= cb.x < kL || cb.x >= 0x80000000u;
        }
      }
    uint32_t pn[kChains][K][4];
    load_raw_round<K, kChains>(src, coded, base, len, 0, l, pn);
    int r = 0;
    [[maybe_unused]] auto dot = [&] {
      if constexpr (Sink::kDot) {
        DotState st{};
        const int64_t e0 = j * a.C + base[0];
        st.row = int(e0 / sink.cols);
        const int c0 = int(e0 - int64_t(st.row) * sink.cols);
        st.cols.start(c0);
        st.first = true;
        st.mid = c0 != 0;
        return st;
      } else {
        return 0;
      }
    }();
    [[maybe_unused]] float* slot0 = nullptr;
    if constexpr (Sink::kDot) slot0 = slots + 2 * min(gi[0], 63);
    if constexpr (KC == 1) {
      // Full rounds (all 16 steps of every chain's state valid): no per-step predication, 32-bit
      // bookkeeping and running element offsets; the partial rounds at the end of a sub-chunk
      // take the general loop below.
      const int64_t l16 = int64_t(l) * kSteps;
      int rfull = rounds;
      uint32_t end8[kChains], off[kChains];  // off: element offset of the lane's round r in the chunk
#pragma unroll
      for (int c = 0; c < kChains; ++c) {
        // Products are taken by whole warps: rounds that are full for all lanes of all segments.
        if constexpr (Sink::kDot) rfull = int(__reduce_min_sync(0xFFFFFFFFu, uint32_t(len[c] / kRound)));
        else rfull = min(rfull, len[c] >= l16 + kSteps ? int((len[c] - l16 - kSteps) / kRound) + 1 : 0);
        end8[c] = (cur[0][c].end + 7) & ~7u;
        off[c] = uint32_t(base[c] + l16);
      }
      // Stream blocks [qbeg, qend) from gb lie wholly inside [lo, hi): one 16-byte load each.
      const uint4* gb4 = reinterpret_cast<const uint4*>(gb[0]);
      const uint32_t qbeg = gb[0] < lo[0] ? 1u : 0u;
      const uint64_t span = hi[0] > gb[0] ? uint64_t(hi[0] - gb[0]) / 16 : 0;
      const uint32_t qend = span > 0xFFFFFFFFull ? 0xFFFFFFFFu : uint32_t(span);
      auto block = [&](uint32_t q) {
        return q >= qbeg && q < qend ? __ldg(gb4 + q) : load_block(gb[0], q, lo[0], hi[0]);
      };
      const uint8_t* rows = reinterpret_cast<const uint8_t*>(rings);
      // LAST: the one coded plane is plane K - 1 (the exponent plane of every float type) and has more
      // than one symbol, so the raw planes and the decoded symbols have fixed places (no per-round
      // plane selection).
      auto full_rounds = [&](auto last) {
        constexpr bool LAST = decltype(last)::value;
        for (; r < rfull; ++r) {
          if (LAST || ncoded > 0) {
            // [ptr, ptr + 16) must be present (synchronous loads only when the ring ran low), then
            // at most one block is fetched ahead per round, stored at the round's end.
#pragma unroll
            for (int c = 0; c < kChains; ++c) {
              Cursor& cb = cur[0][c];
              const uint32_t need = min((cb.ptr + 16 + 7) & ~7u, end8[c]);
              while (cb.fill < need) {
                ring_put(ring[0][c], cb.fill, block(cb.fill / 8));
                cb.fill += 8;
              }
              cb.nload = cb.fill < end8[c] && cb.fill + 8 <= cb.ptr + kRing ? 1u : 0u;
              if (cb.nload) cb.r0 = block(cb.fill / 8);
            }
          }
          if constexpr (Sink::kDot) dot_load(sink, dot, l, true);
          uint32_t p[kChains][K][4];
#pragma unroll
          for (int c = 0; c < kChains; ++c)
#pragma unroll
            for (int b = 0; b < K; ++b)
#pragma unroll
              for (int i = 0; i < 4; ++i) p[c][b][i] = pn[c][b][i];
          if (r + 1 < rfull) {
#pragma unroll
            for (int c = 0; c < kChains; ++c)
#pragma unroll
              for (int b = 0; b < K; ++b) {
                if (LAST ? b == K - 1 : coded[b]) continue;
                const uint8_t* sp = src[b] + off[c] + kRound;
                if (raw16) {
                  const uint4 v = load_once16(sp);
                  pn[c][b][0] = v.x; pn[c][b][1] = v.y; pn[c][b][2] = v.z; pn[c][b][3] = v.w;
                } else {
                  const uint2 v0 = load_once8(sp), v1 = load_once8(sp + 8);
                  pn[c][b][0] = v0.x; pn[c][b][1] = v0.y; pn[c][b][2] = v1.x; pn[c][b][3] = v1.y;
                }
              }
          } else if (r + 1 < rounds) {
            load_raw_round<K, kChains>(src, coded, base, len, r + 1, l, pn);
          }
          if (LAST || ncoded > 0) {
            uint32_t acc[kChains][4] = {};
            if (LAST || single[0] < 0) decode_round_fast(cur[0], tabs, rows, tid, acc);
            else fill_single(acc, single[0]);
#pragma unroll
            for (int c = 0; c < kChains; ++c)
#pragma unroll
              for (int b = 0; b < K; ++b)
                if (LAST ? b == K - 1 : b == pslot[0]) {
#pragma unroll
                  for (int i = 0; i < 4; ++i) p[c][b][i] = acc[c][i];
                }
          }
          // (No branch lies between the 16 steps and this: four elements can be put together while
          // the next four symbols wait for their lookups.)
          uint32_t e[kChains][4 * K];
#pragma unroll
          for (int c = 0; c < kChains; ++c) assemble_elements<K, REORDER>(p[c], e[c]);
          if (LAST || ncoded > 0) {
#pragma unroll
            for (int c = 0; c < kChains; ++c) {
              Cursor& cb = cur[0][c];
              if (cb.nload) ring_put(ring[0][c], cb.fill, cb.r0);
              cb.fill += 8 * cb.nload;
            }
          }
#pragma unroll
          for (int c = 0; c < kChains; ++c) {
            if constexpr (Sink::kDot) dot_round<Sink, true>(sink, dot, e[c], true, l, seg, slot0);
            else if (K >= 2 && out32) store_sectors<4 * K>(outc + size_t(off[c]) * K, e[c]);
            else store_words(outc + size_t(off[c]) * K, e[c], 4 * K, out16);  // 16-byte aligned when outc is
            off[c] += kRound;
          }
        }
      };
      if (ncoded == 1 && pslot[0] == K - 1 && single[0] < 0) full_rounds(std::true_type{});
      else full_rounds(std::false_type{});
    }
    for (; r < rounds; ++r) {
      int nact[kChains];
      int64_t off[kChains];
#pragma unroll
      for (int c = 0; c < kChains; ++c) {
        off[c] = int64_t(r) * kRound + l * kSteps;
        nact[c] = int(max(int64_t(0), min(int64_t(kSteps), len[c] - off[c])));
      }
      // Ring upkeep: make [ptr, ptr + 16) present, start up to two block loads ahead.
#pragma unroll
      for (int q = 0; q < KC; ++q) {
        if (q >= ncoded) break;
#pragma unroll
        for (int c = 0; c < kChains; ++c) {
          Cursor& cb = cur[q][c];
          const uint32_t end8 = (cb.end + 7) & ~7u;
          const uint32_t need = min((cb.ptr + 16 + 7) & ~7u, end8);
          while (cb.fill < need) {
            ring_put(ring[q][c], cb.fill, load_block(gb[q], cb.fill / 8, lo[q], hi[q]));
            cb.fill += 8;
          }
          const uint32_t limit = min((cb.ptr + kRing) & ~7u, end8);
          cb.nload = limit > cb.fill ? min((limit - cb.fill) / 8, 2u) : 0u;
          if (cb.nload > 0) cb.r0 = load_block(gb[q], cb.fill / 8, lo[q], hi[q]);
          if (cb.nload > 1) cb.r1 = load_block(gb[q], cb.fill / 8 + 1, lo[q], hi[q]);
        }
      }
      // This round's raw-plane bytes were loaded during the previous round; start the next
      // round's loads now, so that they overlap this round's decoding.
      uint32_t p[kChains][K][4];
#pragma unroll
      for (int c = 0; c < kChains; ++c)
#pragma unroll
        for (int b = 0; b < K; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i) p[c][b][i] = pn[c][b][i];
      if (r + 1 < rounds) load_raw_round<K, kChains>(src, coded, base, len, r + 1, l, pn);
      if constexpr (Sink::kDot) dot_load(sink, dot, l, nact[0] == kSteps);
      const bool full = nact[0] == kSteps && nact[kChains - 1] == kSteps;
#pragma unroll
      for (int q = 0; q < KC; ++q) {
        if (q >= ncoded) break;
        uint32_t acc[kChains][4] = {};
        if (single[q] >= 0) fill_single(acc, single[q]);
        else if (full) decode_round<true>(cur[q], tabs + q * kM, ring[q], nact, acc);
        else decode_round<false>(cur[q], tabs + q * kM, ring[q], nact, acc);
#pragma unroll
        for (int c = 0; c < kChains; ++c)
#pragma unroll
          for (int b = 0; b < K; ++b)
            if (b == pslot[q]) {
#pragma unroll
              for (int i = 0; i < 4; ++i) p[c][b][i] = acc[c][i];
            }
      }
      // Store the blocks loaded at the round's start (this round's reads are done).
#pragma unroll
      for (int q = 0; q < KC; ++q) {
        if (q >= ncoded) break;
#pragma unroll
        for (int c = 0; c < kChains; ++c) {
          Cursor& cb = cur[q][c];
          if (cb.nload > 0) ring_put(ring[q][c], cb.fill, cb.r0);
          if (cb.nload > 1) ring_put(ring[q][c], cb.fill + 8, cb.r1);
          cb.fill += 8 * cb.nload;
        }
      }
#pragma unroll
      for (int c = 0; c < kChains; ++c) {
        if (!Sink::kDot && nact[c] <= 0) continue;
        uint32_t e[4 * K];
        assemble_elements<K, REORDER>(p[c], e);
        if constexpr (Sink::kDot) {
          dot_round<Sink, false>(sink, dot, e, nact[c] == kSteps, l, seg, slot0);
          continue;
        }
        uint8_t* dst = outc + (base[c] + off[c]) * K;
        if (nact[c] == 16) {
          store_words(dst, e, 4 * K, out16 && ((((base[c] + off[c]) * K) & 15) == 0));
        } else {
#pragma unroll
          for (int w = 0; w < 4 * K; ++w)
#pragma unroll
            for (int qq = 0; qq < 4; ++qq)
              if (4 * w + qq < nact[c] * K) dst[4 * w + qq] = uint8_t(e[w] >> (8 * qq));
        }
      }
    }
#pragma unroll
    for (int q = 0; q < KC; ++q)
#pragma unroll
      for (int c = 0; c < kChains; ++c)
        if (q < ncoded && valid[c]) err |= (cur[q][c].x != kL) || (cur[q][c].ptr != cur[q][c].end);
    if constexpr (Sink::kDot) {
      const float sum = segment_sum(dot);
      if (valid[0]) {  // the row that the sub-chunk ends in
        const int64_t e1 = j * a.C + base[0] + len[0];
        const bool ended = e1 % sink.cols == 0, here = !(dot.first && dot.mid);
        if (l == 0) {
          if (ended && here) sink.z[dot.row] = sum;
          else slot0[here ? 1 : 0] = sum;
        }
      }
    }
  }
  const bool any_err = __syncthreads_or(err);
  if constexpr (Sink::kDot) dot_finish_chunk(sink, j, j * a.C, j * a.C + m, g.sc, slots, any_err);
  if constexpr (WEIGHT) {
    // A broken stream shows at its end only: what was stored is replaced by zeros.
    if constexpr (!Sink::kDot)
      if (any_err)
        for (int64_t i = tid; i < m * K; i += kDecThreads) outc[i] = 0;
    if (tid == 0) a.overflow[j] = uint8_t((overflow_pass ? kChunkOver : 0) | flags | (any_err ? kErrStream : 0));
    return;
  }
  if (any_err && tid == 0) {
    if (batched) a.statuses[j] = kErrStream;
    else atomicOr(a.status, kErrStream);
  } else if (batched && tid == 0) {
    a.statuses[j] = 0;
  }
}

inline size_t dec_smem(int KC) {
  return size_t(KC) * kM * 4 + size_t(KC) * kChains * kRing * kDecThreads * (KC > 4 ? 2 : 4) + sizeof(DecSmem);
}

inline size_t dec_job_bytes(int64_t n, int k, int64_t chunk_bytes) {
  const int64_t nch = cdiv(n, chunk_bytes);
  return (size_t(int64_t(k) * nch) * 8 + size_t(nch) + 255) & ~size_t(255);  // unit offsets, overflow flags
}

// The decoder's job for a weight, with its scratch in `temp`.
inline DecArgs weight_args(const WeightBlob& w, void* temp, int32_t* status, int mode) {
  DecArgs a{};
  a.mode = mode;
  a.blob = w.blob;
  a.blob_bytes = w.blob_bytes;
  a.n = w.rows * w.cols;
  a.C = w.chunk;
  a.nch = weight_chunks(w);
  a.units = 2 * a.nch;
  a.sizes_off = 24 + 8 * 2;
  a.idx_off = a.sizes_off + 4 * a.units;
  a.n_comp = -1;  // dscan_kernel reads it from the blob
  a.data_off = -1;
  a.status = status;
  uint8_t* t = static_cast<uint8_t*>(temp);
  a.src = reinterpret_cast<int64_t*>(t + job_structs_bytes<DecArgs>(1));
  a.overflow = reinterpret_cast<uint8_t*>(a.src + a.units);
  return a;
}

}  // namespace
}  // namespace zn
