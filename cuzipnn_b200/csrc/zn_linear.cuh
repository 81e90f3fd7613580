// The linear layer's epilogue, on a tile of a product (EpiLinear) or element by element (Finish).
#pragma once

#include "zn_gemm.cuh"
#include "zn_weight.cuh"

namespace zn {

constexpr int kNone = 0, kRelu = 1, kGelu = 2, kGeluTanh = 3, kSilu = 4;

// The normal distribution's upper tail at t >= 0 over exp(-t^2 / 2): a polynomial of degree 7 in
// u = 1 / (1 + 0.2375 t), times u (fitted here to erfcx(t / sqrt(2)) / 2 for the least relative error on
// [0, 16]: 2^-21 in 32-bit arithmetic; beyond, both go to 0 as 1 / t).  gelu's value and derivative are
// differences of near numbers below zero if taken from 1 + erf, which has no digits left at -5; from the
// tail itself they keep theirs.  4096 rows of 5120 x 1280 take 143 us (158 with the derivative); erfcf in
// its place takes 176 (217), 1 + erff 148 (174).
__device__ __forceinline__ float mills(float t) {
  const float u = __fdividef(1.0f, fmaf(0.2375f, t, 1.0f));
  float p = -0.05875275f;
  p = fmaf(p, u, 0.18125452f);
  p = fmaf(p, u, -0.10428442f);
  p = fmaf(p, u, 0.14710677f);
  p = fmaf(p, u, 0.05084207f);
  p = fmaf(p, u, 0.09489430f);
  p = fmaf(p, u, 0.09416503f);
  p = fmaf(p, u, 0.09477440f);
  return p * u;
}

// act(z) and its derivative (where asked for), in 32 bits.
template <int ACT, bool SLOPE>
__device__ __forceinline__ float activate(float z, float& slope) {
  if constexpr (ACT == kRelu) {
    if (SLOPE) slope = z > 0.0f ? 1.0f : 0.0f;
    return z < 0.0f ? 0.0f : z;  // keeps NaN
  } else if constexpr (ACT == kGelu) {
    const float bell = __expf(-0.5f * z * z), tail = bell * mills(fabsf(z)), cdf = z > 0.0f ? 1.0f - tail : tail;
    if (SLOPE) slope = cdf + z * 0.3989422804014327f * bell;
    return z * cdf;
  } else if constexpr (ACT == kGeluTanh) {  // 0.5 z (1 + tanh u) = z sigmoid(2u)
    const float c = 0.7978845608028654f, z2 = z * z;
    const float sig = __fdividef(1.0f, 1.0f + __expf(-2.0f * c * z * (1.0f + 0.044715f * z2)));
    if (SLOPE) slope = sig + z * sig * (1.0f - sig) * 2.0f * c * (1.0f + 3.0f * 0.044715f * z2);
    return z * sig;
  } else if constexpr (ACT == kSilu) {
    const float sig = __fdividef(1.0f, 1.0f + __expf(-z));
    if (SLOPE) slope = sig * (1.0f + z * (1.0f - sig));
    return z * sig;
  } else {
    if (SLOPE) slope = 1.0f;
    return z;
  }
}
template <bool SLOPE>
__device__ __forceinline__ float activate(int act, float z, float& slope) {
  switch (act) {
    case kRelu: return activate<kRelu, SLOPE>(z, slope);
    case kGelu: return activate<kGelu, SLOPE>(z, slope);
    case kGeluTanh: return activate<kGeluTanh, SLOPE>(z, slope);
    case kSilu: return activate<kSilu, SLOPE>(z, slope);
    default: return activate<kNone, SLOPE>(z, slope);
  }
}

// The derivative act'(z) is kept for the backward pass as float16 of 2^15 act'(z), whatever the weight's
// type: every activation's derivative lies in [-0.13, 1.13], so the scaled one stays below 37100, and the
// 15 exponents that a float16 would leave unused above 1 extend it downwards.  Off by 2^-11 of itself at
// most (an eighth of a bf16 rounding, one of fp16) as far as |act'(z)| >= 2^-29, and by 2^-40 below:
// silu' keeps its digits to z = -23, gelu' to -6.
constexpr float kSlopeScale = 32768.0f;
__device__ __forceinline__ uint32_t slope_codes(float s0, float s1) {
  return Num<__half>::pack(s0 * kSlopeScale, s1 * kSlopeScale);
}
__device__ __forceinline__ float slope_lo(uint32_t w) { return Num<__half>::lo(w) * (1.0f / kSlopeScale); }
__device__ __forceinline__ float slope_hi(uint32_t w) { return Num<__half>::hi(w) * (1.0f / kSlopeScale); }

// Per-warp staging: a thread holds 64 bytes (32 16-bit columns) of its own row; through shared
// memory the warp writes them as 8 rows x 64 contiguous bytes per store.  The 16-byte chunks of a
// row are permuted by the row, so that both sides touch every bank once.
__device__ __forceinline__ uint4* stage_at(uint8_t* buf, int row, int chunk) {
  return reinterpret_cast<uint4*>(buf + row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4));
}
// Rows m0 + r < M, columns n0 .. n0 + 31 < N of a 16-bit matrix from the warp's 16 words per thread.
template <typename T>
__device__ __forceinline__ void stage_rows(uint8_t* buf, const uint32_t* w, T* out, int64_t ld, int64_t m0, int64_t M,
                                           int64_t n0, int64_t N, bool vec) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i) *stage_at(buf, lane, i) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  __syncwarp();
  if (vec) {  // 16-byte aligned rows, N a multiple of 8
    const int64_t n = n0 + 8 * (lane & 3);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 8 * i + (lane >> 2);
      if (m0 + r < M && n < N) *reinterpret_cast<uint4*>(out + (m0 + r) * ld + n) = *stage_at(buf, r, lane & 3);
    }
  } else if (n0 + lane < N) {
    const int rows = int(min(int64_t(32), M - m0));
    for (int r = 0; r < rows; ++r)
      out[(m0 + r) * ld + n0 + lane] = reinterpret_cast<const T*>(stage_at(buf, r, lane >> 3))[lane & 7];
  }
  __syncwarp();
}

// The reverse, for the residual: a warp's rows m0 .. m0 + 31 (those below M) of columns n0 .. n0 + 31
// (those below N), loaded as whole sectors into registers and handed to the threads that own the
// rows.  The aligned form is split, so that the next columns' loads run during this columns' work.
template <typename T>
__device__ __forceinline__ void fetch_rows(const T* in, int64_t ld, int64_t m0, int64_t M, int64_t n0, int64_t N,
                                           uint4* q) {
  const int lane = threadIdx.x & 31;
  const int64_t n = n0 + 8 * (lane & 3);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 8 * i + (lane >> 2);
    if (m0 + r < M && n < N) q[i] = *reinterpret_cast<const uint4*>(in + (m0 + r) * ld + n);
  }
}
__device__ __forceinline__ void hand_rows(uint8_t* buf, const uint4* q) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i) *stage_at(buf, 8 * i + (lane >> 2), lane & 3) = q[i];
  __syncwarp();
}
template <typename T>
__device__ __forceinline__ void fetch_rows_plain(uint8_t* buf, const T* in, int64_t ld, int64_t m0, int64_t M,
                                                 int64_t n0, int64_t N) {
  const int lane = threadIdx.x & 31;
  const int rows = int(min(int64_t(32), M - m0));
  if (n0 + lane < N) {
#pragma unroll 8
    for (int r = 0; r < rows; ++r)
      reinterpret_cast<T*>(stage_at(buf, r, lane >> 3))[lane & 7] = in[(m0 + r) * ld + n0 + lane];
  }
  __syncwarp();
}

// y = act(acc + bias) + residual, rounded once to 16 bits, and (where asked for) the slopes.
template <typename T>
struct EpiLinear {
  static constexpr bool kParts = true;
  const T* bias;  // or null
  const T* res;   // or null
  T* y;
  __half* slope;  // or null
  int64_t ldr, ldy, M, N;
  int act;
  bool vec;  // 16-byte accesses: every pointer and pitch allows them, and N is a multiple of 8

  struct Row {
    int64_t m, n0;
    int width;
    uint8_t* buf;
    uint4 ahead[4];  // the residual of the next 32 columns
    __device__ __forceinline__ Row(const EpiLinear& e, int64_t m_, int64_t n0_, int width_, uint8_t* b)
        : m(m_), n0(n0_), width(width_), buf(b) {
      if (e.res && e.vec) fetch_rows(e.res, e.ldr, m - (threadIdx.x & 31), e.M, n0, e.N, ahead);
    }

    template <int ACT, bool SLOPE>
    __device__ __forceinline__ void run(const EpiLinear& e, int64_t n, float* v) {
      uint32_t sw[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float s0, s1;
        v[2 * i] = activate<ACT, SLOPE>(v[2 * i], s0);
        v[2 * i + 1] = activate<ACT, SLOPE>(v[2 * i + 1], s1);
        if (SLOPE) sw[i] = slope_codes(s0, s1);
      }
      if (SLOPE) stage_rows(buf, sw, e.slope, e.ldy, m - (threadIdx.x & 31), e.M, n, e.N, e.vec);
    }

    __device__ __forceinline__ void cols(const EpiLinear& e, int c, float* v) {
      const int64_t n = n0 + c;
      if (n >= e.N) return;
      if (e.bias) add_bias(e.bias, n, e, v);
      if (e.slope) {
        switch (e.act) {
          case kRelu: run<kRelu, true>(e, n, v); break;
          case kGelu: run<kGelu, true>(e, n, v); break;
          case kGeluTanh: run<kGeluTanh, true>(e, n, v); break;
          case kSilu: run<kSilu, true>(e, n, v); break;
          default: run<kNone, true>(e, n, v);
        }
      } else {
        switch (e.act) {
          case kRelu: run<kRelu, false>(e, n, v); break;
          case kGelu: run<kGelu, false>(e, n, v); break;
          case kGeluTanh: run<kGeluTanh, false>(e, n, v); break;
          case kSilu: run<kSilu, false>(e, n, v); break;
          default: break;
        }
      }
      uint32_t w[16];
      if (e.res) {
        const int64_t m0 = m - (threadIdx.x & 31);
        if (e.vec) {
          hand_rows(buf, ahead);
          if (c + 32 < width) fetch_rows(e.res, e.ldr, m0, e.M, n + 32, e.N, ahead);
        } else {
          fetch_rows_plain(buf, e.res, e.ldr, m0, e.M, n, e.N);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 q = *stage_at(buf, threadIdx.x & 31, i);
          w[4 * i] = q.x; w[4 * i + 1] = q.y; w[4 * i + 2] = q.z; w[4 * i + 3] = q.w;
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          v[2 * i] += Num<T>::lo(w[i]);
          v[2 * i + 1] += Num<T>::hi(w[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = Num<T>::pack(v[2 * i], v[2 * i + 1]);
      stage_rows(buf, w, e.y, e.ldy, m - (threadIdx.x & 31), e.M, n, e.N, e.vec);
    }
    __device__ __forceinline__ void end(const EpiLinear&) {}

    // v += row[n .. n + 31], as far as the columns go: the same for all rows, one broadcast load each.
    static __device__ __forceinline__ void add_bias(const T* row, int64_t n, const EpiLinear& e, float* v) {
      if (e.vec) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          if (n + 8 * g >= e.N) break;
          const uint4 q = *reinterpret_cast<const uint4*>(row + n + 8 * g);
          const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v[8 * g + 2 * i] += Num<T>::lo(w[i]);
            v[8 * g + 2 * i + 1] += Num<T>::hi(w[i]);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (n + i < e.N) v[i] += Num<T>::to(row[n + i]);
      }
    }
  };
};

// z[r] of weight_dot: from z, or the parts of a row that spans chunks, in order.
struct DotValue {
  const float* z;
  const float* part;
  int64_t rows, cols, chunk;
  __device__ __forceinline__ float get(int64_t r) const {
    // The chunk of the row's first element, and how many more the row reaches into (32 bits: a chunk has
    // 2^24 elements at most, dot_shape's rows fewer than 2^30).
    const int64_t c0 = r * cols / chunk;
    const uint32_t more = (uint32_t(r * cols - c0 * chunk) + uint32_t(cols) - 1) / uint32_t(chunk);
    if (more == 0) return z[r];
    float v = part[2 * c0 + 1];
    for (int64_t c = c0 + 1; c <= c0 + more; ++c) v += part[2 * c];
    return v;
  }
};

// One element of the epilogue.
template <typename T>
__device__ __forceinline__ void finish_value(const EpiLinear<T>& e, int64_t m, int64_t n, float z) {
  if (e.bias) z += Num<T>::to(e.bias[n]);
  float sl;
  z = e.slope ? activate<true>(e.act, z, sl) : activate<false>(e.act, z, sl);
  if (e.res) z += Num<T>::to(e.res[m * e.ldr + n]);
  e.y[m * e.ldy + n] = Num<T>::from(z);
  if (e.slope) e.slope[m * e.ldy + n] = Num<__half>::from(sl * kSlopeScale);
}

// y = act(z + bias) + residual from z = acc, or from weight_dot.
template <typename T>
struct Finish {
  const float* acc;  // [M][ld], or null: dot (M = 1)
  int64_t M, N, ld;
  DotValue dot;
  EpiLinear<T> lin;
};

template <typename T>
__device__ __forceinline__ void finish_element(const Finish<T>& f, int64_t i) {
  const int64_t m = i / f.N, n = i - m * f.N;
  finish_value(f.lin, m, n, f.acc ? f.acc[m * f.ld + n] : f.dot.get(n));
}

// weight_dot, then f (whose dot it fills in) on every element.
template <typename T>
int weight_linear(const WeightBlob& w, void* temp, const void* x, float* z, float* part, const Finish<T>& f,
                  int32_t* status, cudaStream_t s);

}  // namespace zn
