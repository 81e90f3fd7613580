// Operators on compressed weights (the zn_linear_* and zn_loss_* entry points).
//
// The weight W [rows, cols] stays a blob.  A call decodes it a piece of rows at a time into its
// scratch (a few waves of the decoder, so that a weight of any size needs a bounded buffer) and
// multiplies each piece on the tensor cores (zn_gemm.cuh), with the rest of the operator in the
// product's epilogue:
//   linear              y = act(x W^T + b) + r                   EpiLinear
//   loss                running maximum and sum of exp           EpiStats (per row and half tile)
//   loss and gradient   P = exp(s - r), one piece wide           EpiSoft, then acc += P W by EpiAccum
// A product with one row is bound by decoding; it runs inside the decoder instead
// (weight_dot) and W is never written at all.
//
// Losses.  With s = h W^T / T, lse = log sum_v exp s_v and a sparse distribution q over the ids of
// a row (sum q = 1):  L = T^2 (sum_k q_k (log q_k - s_{id_k}) + lse),  dL/dh = T (softmax(s) - q) W.
// A cross entropy is the case of one id with q = 1 and T = 1.  The logits are never kept.
//
// The gradient comes with the loss, in one pass over the vocabulary, like attention with W as keys
// and values:  softmax(s) W = (sum_v exp(s_v - r) W_v) / (sum_v exp(s_v - r)) for any reference r of
// the row.  Each piece is decoded once and multiplied twice (4 tokens rows cols operations in all,
// against 6 and two decodings for computing the logits again in a backward pass).
//
// P = exp(s - r) is rounded to 16 bits.  At the row's own ids that would be wrong where it matters most
// (a confident softmax less q is a small difference), so the ids' columns take no part in P nor in r:
// P is zero there, and the ids' terms are added in 32 bits (gather_kernel, soft_end_kernel).  With a
// single id p - q is -S / (S + e), from the sum S over the other columns and the id's own e: no
// difference is taken at all, and a confident row's gradient is as exact as any other's.
// r is the maximum of the other columns of the first kSample rows of W, less kBelow powers of two in
// fp16, whose P would else lose the tail of the softmax: it spans 2^kBelow at the largest column down to
// 2^-25, so that of V columns those below lose V 2^(-25 - kBelow) of the sum at most (2^-15.8 for
// 152064, under fp16's rounding of 2^-11).  Up to a bound (2^60 for bf16, 2^15 for fp16) P may exceed
// that.  Where a group of 32 logits passes the bound, its P is zero, the row's r is raised for its
// maximum, what was summed is scaled down, and the piece is multiplied again with the groups that were
// left out alone (kernels that end at once when there are none).
#include <algorithm>

#include "zn_linear.cuh"

namespace zn {

int make_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t pitch, int box_rows, bool bf16) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q{};
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
    return e == cudaSuccess && q == cudaDriverEntryPointSuccess ? reinterpret_cast<Encode>(fn) : nullptr;
  }();
  if (!encode) return set_error(ZN_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[2] = {cuuint64_t(cols), cuuint64_t(rows)};
  const cuuint64_t strides[1] = {cuuint64_t(pitch) * 2};
  const cuuint32_t box[2] = {kBK, cuuint32_t(box_rows)};
  const cuuint32_t step[2] = {1, 1};
  const CUresult r = encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                            const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(ZN_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", int(r));
  return ZN_OK;
}

int sm_count(int* sms) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
  return e == cudaSuccess ? ZN_OK : set_error(ZN_ERR_CUDA, "SM count: %s", cudaGetErrorString(e));
}

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kMean = 0, kRows = 2;  // reductions (1: sum)
constexpr int kMaxTop = 256;

// ---- epilogues ------------------------------------------------------------------------------

// Per-row state of a loss (state buffer of a call, kept for the backward pass).
struct LossRows {
  float* q0;       // sum_k q_k log q_k
  int32_t* count;  // ids of the row (0: the row does not count; -1: an id is out of range)
  int32_t* ids;    // [tokens][top], ascending
  float* q;        // [tokens][top], in the order of ids
  float* rows;     // [1] rows that count
  int top;
};

// Position of the first id >= n.
__device__ __forceinline__ int first_id(const int32_t* ids, int count, int64_t n) {
  int lo = 0, hi = count;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ids[mid] < n) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// 2^x, as the unit computes it (2 units of the last place; subnormal results are 0).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// One pass over the logits of a row: running maximum and sum of 2^(s' - max) with s' = s log2(e),
// and sum_k q_k s'_{id_k} over the row's ids among the columns seen.
struct RowStats {
  float mx, sum, hit;
};
__device__ __forceinline__ void stats_join(RowStats& a, float mx, float sum, float hit) {
  const float m = fmaxf(a.mx, mx);
  const float base = m == -INFINITY ? 0.0f : m;
  a.sum = a.sum * ex2(a.mx - base) + sum * ex2(mx - base);
  a.mx = m;
  a.hit += hit;
}

struct EpiStats {
  static constexpr bool kParts = false;
  LossRows rows;
  float* part;    // [half tile][3][M]: max, sum, hit
  int64_t M, N;   // N: columns of this piece
  int64_t v0;     // first vocabulary row of this piece
  int64_t tile0;  // its first half tile
  int tile_cols;  // columns of a half tile
  float scale;    // log2(e) / T
  struct Row {
    int64_t m, n0;
    RowStats st;
    const int32_t* ids;
    const float* q;
    int at, count;
    int64_t next;  // column (of the piece) of the next id
    __device__ __forceinline__ Row(const EpiStats& e, int64_t m_, int64_t n0_, int, uint8_t*) : m(m_), n0(n0_) {
      st = {-INFINITY, 0.0f, 0.0f};
      at = count = 0;
      next = INT64_MAX;
      ids = nullptr;
      q = nullptr;
      if (m < e.M) {
        count = e.rows.count[m];
        ids = e.rows.ids + m * e.rows.top;
        q = e.rows.q + m * e.rows.top;
        at = first_id(ids, count, e.v0 + n0);
        if (at < count) next = ids[at] - e.v0;
      }
    }
    __device__ __forceinline__ void cols(const EpiStats& e, int c, const float* v) {
      if (m >= e.M) return;
      const int left = int(min(int64_t(32), e.N - n0 - c));
      if (left <= 0) return;
      float s[32], mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        s[i] = i < left ? v[i] * e.scale : -INFINITY;
        mx = fmaxf(mx, s[i]);
      }
      const float m2 = fmaxf(st.mx, mx), base = m2 == -INFINITY ? 0.0f : m2;
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 32; ++i) sum += ex2(s[i] - base);
      st.sum = st.sum * ex2(st.mx - base) + sum;
      st.mx = m2;
      if (next < n0 + c + 32) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          while (next == n0 + c + i) {
            if (q[at] != 0.0f) st.hit += q[at] * s[i];
            ++at;
            next = at < count ? ids[at] - e.v0 : INT64_MAX;
          }
      }
    }
    __device__ __forceinline__ void end(const EpiStats& e) {
      if (m >= e.M || n0 >= e.N) return;  // (the last tile's second half may hold no column)
      float* p = e.part + (e.tile0 + n0 / e.tile_cols) * 3 * e.M + m;
      p[0] = st.mx;
      p[e.M] = st.sum;
      p[2 * e.M] = st.hit;
    }
  };
};

// The ids of a row among the columns that a thread reads from n0 on, in their order.
struct IdWalk {
  const int32_t* ids = nullptr;
  int at = 0, count = 0;
  int64_t next = INT64_MAX;  // column (of the piece) of the next id
  int64_t v0 = 0;
  __device__ __forceinline__ IdWalk() {}
  __device__ __forceinline__ IdWalk(const LossRows& rows, int64_t m, int64_t v0_, int64_t n0) : v0(v0_) {
    count = max(0, rows.count[m]);
    ids = rows.ids + m * rows.top;
    at = first_id(ids, count, v0 + n0);
    if (at < count) next = ids[at] - v0;
  }
  __device__ __forceinline__ void step() {
    ++at;
    next = at < count ? ids[at] - v0 : INT64_MAX;
  }
};

// The maximum of a row's logits but for its ids' (for the first reference).
struct EpiMax {
  static constexpr bool kParts = false;
  LossRows rows;
  float* part;    // [half tile][M]
  int64_t M, N;   // columns 0 .. N - 1 of the vocabulary
  int tile_cols;  // columns of a half tile
  float scale;    // log2(e) / T
  struct Row {
    int64_t m, n0;
    float mx;
    IdWalk walk;
    __device__ __forceinline__ Row(const EpiMax& e, int64_t m_, int64_t n0_, int, uint8_t*)
        : m(m_), n0(n0_), mx(-INFINITY) {
      if (m < e.M) walk = IdWalk(e.rows, m, 0, n0);
    }
    __device__ __forceinline__ void cols(const EpiMax& e, int c, float* v) {
      if (m >= e.M) return;
      const int left = int(min(int64_t(32), e.N - n0 - c));
      if (walk.next < n0 + c + 32) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          while (walk.next == n0 + c + i) {
            v[i] = -INFINITY;
            walk.step();
          }
      }
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i < left) mx = fmaxf(mx, v[i] * e.scale);
    }
    __device__ __forceinline__ void end(const EpiMax& e) {
      if (m < e.M && n0 < e.N) e.part[n0 / e.tile_cols * e.M + m] = mx;
    }
  };
};

// State of a loss with its gradient, per row, in units of log2(e) (s' = s log2(e)).
struct SoftRows {
  float* ref;      // r
  float* before;   // r before this piece
  float* scale;    // 2^(before - r)
  float* sum;      // sum of 2^(s' - r) over the columns so far, without the ids'
  float* hit;      // [tokens][top] s' at the row's ids
  int32_t* again;  // of this piece: a group was left out, or an id lies far above r
};

// How far below the largest column r lies, in powers of two (see the head of this file).
template <typename T>
constexpr float kBelow = Num<T>::kCode == 1 ? 0.0f : 8.0f;
// Rows of several ids add 2^(s'_k - r) W to the others' sum: r is raised so that this stays in a float.
constexpr float kIdBound = 100.0f, kIdAbove = 64.0f;

// P = 2^(s' - r) of one piece, in 16 bits, as the operand of the product with the piece; zero at the
// row's ids, and in rows that do not count whatever their logits are.  AGAIN: the groups that the
// first pass left out, with the r that was raised for them.
template <typename T, bool AGAIN>
struct EpiSoft {
  static constexpr bool kParts = false;
  static constexpr float kBound = Num<T>::kCode == 1 ? 60.0f : 15.0f;
  LossRows rows;
  SoftRows soft;
  T* p;
  float* part;       // [half tile][2][M]: sum, and the reference that the groups left out ask for
  int64_t M, N, ld;  // N: columns of this piece; ld: a multiple of 8
  int64_t v0;        // first vocabulary row of this piece
  int tile_cols;     // columns of a half tile
  float scale;       // log2(e) / T
  struct Row {
    int64_t m, n0;
    uint8_t* buf;
    float ref, before, sum, out;
    IdWalk walk;
    __device__ __forceinline__ Row(const EpiSoft& e, int64_t m_, int64_t n0_, int, uint8_t* b) : m(m_), n0(n0_), buf(b) {
      ref = before = sum = 0.0f;
      out = -INFINITY;
      if (m < e.M) {
        ref = e.soft.ref[m];
        before = AGAIN ? e.soft.before[m] : ref;
        walk = IdWalk(e.rows, m, e.v0, n0);
      }
    }
    __device__ __forceinline__ void cols(const EpiSoft& e, int c, float* v) {
      if (n0 + c >= e.N) return;
      const int left = int(min(int64_t(32), e.N - n0 - c));
      if (walk.next < n0 + c + 32) {  // the ids' logits, and their columns out of P
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (walk.next == n0 + c + i) {
            const float s = v[i] * e.scale;
            if (!AGAIN && e.rows.top > 1 && (before == -INFINITY || s - before > kIdBound)) out = fmaxf(out, s - kIdAbove);
            while (walk.next == n0 + c + i) {
              if (!AGAIN) e.soft.hit[m * e.rows.top + walk.at] = s;
              walk.step();
            }
            v[i] = -INFINITY;
          }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i < left) mx = fmaxf(mx, v[i]);
      const bool over = before == -INFINITY ? mx > -INFINITY : fmaf(mx, e.scale, -before) > kBound;
      const bool take = walk.count > 0 && over == AGAIN;
      if (!AGAIN && over) out = fmaxf(out, fmaf(mx, e.scale, -kBelow<T>));
      const float base = ref == -INFINITY ? 0.0f : ref;
      float add = 0.0f;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float t = ex2(fmaf(v[i], e.scale, -base));
        v[i] = take && i < left ? t : 0.0f;
        add += v[i];
      }
      sum += add;
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = Num<T>::pack(v[2 * i], v[2 * i + 1]);
      // The pitch covers the last group of 8 columns.
      stage_rows(buf, w, e.p, e.ld, m - (threadIdx.x & 31), e.M, n0 + c, e.ld, true);
    }
    __device__ __forceinline__ void end(const EpiSoft& e) {
      if (m >= e.M || n0 >= e.N) return;
      float* p = e.part + (n0 / e.tile_cols) * 2 * e.M + m;
      p[0] = sum;
      p[e.M] = walk.count > 0 ? out : -INFINITY;
    }
  };
};

// ---- small kernels --------------------------------------------------------------------------

__global__ void __launch_bounds__(256) pitch_kernel(const __grid_constant__ PitchCopy p) {
  pdl_wait();
  pdl_trigger();
  pitch_rows(p, int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5), int64_t(gridDim.x) * 8);
}

__device__ __forceinline__ void parts_end(const EpiAccum& e, int64_t m, int64_t n, const float* v) {
  for (int i = 0; i < 4; ++i)
    if (n + i < e.N) {
      float* p = e.acc + m * e.ld + n + i;
      *p = e.add ? fmaf(*p, e.scale ? e.scale[m] : 1.0f, v[i]) : v[i];
    }
}
template <typename T>
__device__ __forceinline__ void parts_end(const EpiLinear<T>& e, int64_t m, int64_t n, const float* v) {
  for (int i = 0; i < 4; ++i)
    if (n + i < e.N) finish_value(e, m, n + i, v[i]);
}

// The tiles that a product computed in parts: four columns per thread, the parts added in order (13 us
// for 34 tiles of 256 x 256 with silu and its slopes).
template <class Epi>
__global__ void __launch_bounds__(256) parts_kernel(const __grid_constant__ GemmShape g,
                                                    const __grid_constant__ Epi epi, int tile) {
  pdl_wait();
  pdl_trigger();
  const int quads = tile / 4, blocks = tile * quads / 256, which = blockIdx.x / blocks;
  const int i = (blockIdx.x - which * blocks) * 256 + threadIdx.x, r = i / quads, c = 4 * (i - r * quads);
  int tm, tn;
  tile_place(g, g.full + which, tm, tn);
  const int64_t m = int64_t(tm) * tile + r, n = int64_t(tn) * tile + c;
  if (m >= g.M || n >= g.N) return;
  const float4* p = reinterpret_cast<const float4*>(g.parts + int64_t(which) * g.splits * tile * tile + r * tile + c);
  float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int k = 0; k < g.splits; ++k) {
    const float4 v = p[int64_t(k) * tile * tile / 4];
    s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
  }
  const float v[4] = {s.x, s.y, s.z, s.w};
  parts_end(epi, m, n, v);
}

template <typename T>
__global__ void __launch_bounds__(256) finish_kernel(const __grid_constant__ Finish<T> f) {
  pdl_wait();
  pdl_trigger();
  const int64_t total = f.M * f.N, step = int64_t(gridDim.x) * blockDim.x;
  for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += step) finish_element(f, i);
}

// dz = dy * slope in 16 bits (the operand of dx = dz W, as the gradient between two layers would be: the
// tensor cores take no 32-bit one at this rate; dz null: not wanted) and the column sums of the unrounded
// products over `per` rows per block: to dbias when that is all rows (one launch less for a few tokens),
// else to part[row block][n] (32 bits), which column_sum_kernel adds in order.
// V columns per thread: 8 in 16-byte accesses, four rows in flight, where the matrices allow it (70 us
// for 4096 x 18944, the bandwidth of its 465 MB), else 1.
constexpr int kSumRows = 64, kSumAll = 512;
template <typename T, int V>
__global__ void __launch_bounds__(256) slope_kernel(const T* __restrict__ dy, int64_t ldy,
                                                    const __half* __restrict__ slope, T* __restrict__ dz, int64_t ldz,
                                                    float* __restrict__ part, T* __restrict__ dbias, int64_t M,
                                                    int64_t N, int64_t per) {
  pdl_wait();
  pdl_trigger();
  const int64_t col_blocks = cdiv(N, 32 * V), mb = blockIdx.x / col_blocks;
  const int lane = threadIdx.x & 31, sub = threadIdx.x >> 5;
  const int64_t n = (blockIdx.x - mb * col_blocks) * 32 * V + V * lane;
  const int64_t m1 = min(M, (mb + 1) * per);
  float s[V];
#pragma unroll
  for (int i = 0; i < V; ++i) s[i] = 0.0f;
  if (n < N) {
    if constexpr (V == 8) {
      constexpr int kDeep = 4;
      for (int64_t m = mb * per + sub; m < m1; m += 8 * kDeep) {
        uint4 g[kDeep], w[kDeep];
#pragma unroll
        for (int q = 0; q < kDeep; ++q)
          if (m + 8 * q < m1) {
            g[q] = *reinterpret_cast<const uint4*>(dy + (m + 8 * q) * ldy + n);
            if (slope) w[q] = *reinterpret_cast<const uint4*>(slope + (m + 8 * q) * N + n);
          }
#pragma unroll
        for (int q = 0; q < kDeep; ++q)
          if (m + 8 * q < m1) {
            const uint32_t gw[4] = {g[q].x, g[q].y, g[q].z, g[q].w}, ww[4] = {w[q].x, w[q].y, w[q].z, w[q].w};
            uint32_t z[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float a = Num<T>::lo(gw[i]), b = Num<T>::hi(gw[i]);
              if (slope) {
                a *= slope_lo(ww[i]);
                b *= slope_hi(ww[i]);
              }
              z[i] = Num<T>::pack(a, b);
              s[2 * i] += a;
              s[2 * i + 1] += b;
            }
            if (dz) *reinterpret_cast<uint4*>(dz + (m + 8 * q) * ldz + n) = make_uint4(z[0], z[1], z[2], z[3]);
          }
      }
    } else {
      for (int64_t m = mb * per + sub; m < m1; m += 8) {
        float d = Num<T>::to(dy[m * ldy + n]);
        if (slope) d *= slope_lo(__half_as_ushort(slope[m * N + n]));
        if (dz) dz[m * ldz + n] = Num<T>::from(d);
        s[0] += d;
      }
    }
  }
  if (!part && !dbias) return;
  __shared__ float sm[8][32 * V];
#pragma unroll
  for (int i = 0; i < V; ++i) sm[sub][V * lane + i] = s[i];
  __syncthreads();
  const int64_t c0 = n - V * lane;
  for (int c = threadIdx.x; c < 32 * V; c += 256) {
    if (c0 + c >= N) continue;
    float v = 0.0f;
    for (int i = 0; i < 8; ++i) v += sm[i][c];
    if (dbias) dbias[c0 + c] = Num<T>::from(v);
    else part[mb * N + c0 + c] = v;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) column_sum_kernel(const float* part, int64_t blocks, int64_t N, T* out) {
  pdl_wait();
  pdl_trigger();
  const int64_t n = int64_t(blockIdx.x) * 32 + (threadIdx.x & 31);
  const int sub = threadIdx.x >> 5;
  float s = 0.0f;
  if (n < N)
    for (int64_t b = sub; b < blocks; b += 8) s += part[b * N + n];
  __shared__ float sm[8][32];
  sm[sub][threadIdx.x & 31] = s;
  __syncthreads();
  if (sub == 0 && n < N) {
    for (int i = 1; i < 8; ++i) s += sm[i][threadIdx.x];
    out[n] = Num<T>::from(s);
  }
}

// One warp per row: the row's ids in ascending order with their q.  Without logits the row has one
// id (a target, left out when it equals `ignore`) and q = 1; with them, q = softmax(logits / T)
// over the ids >= 0.  A row without ids, or whose logits are all -inf, does not count.  The rank of
// an entry is counted against all others (top <= 256), so no sort network is needed.
__global__ void __launch_bounds__(128) loss_prep_kernel(const int64_t* ids, const float* logits, int64_t tokens,
                                                        int64_t vocab, int64_t ignore, float inv_t, LossRows out) {
  pdl_wait();
  pdl_trigger();
  const int64_t m = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (m >= tokens) return;
  const int top = out.top;
  int32_t* oid = out.ids + m * top;
  float* oq = out.q + m * top;
  if (!logits) {
    if (lane == 0) {
      const int64_t id = ids[m];
      const bool in = id >= 0 && id < vocab;
      out.count[m] = id == ignore ? 0 : in ? 1 : -1;
      out.q0[m] = 0.0f;
      oid[0] = in ? int32_t(id) : 0;
      oq[0] = 1.0f;
    }
    return;
  }
  const int64_t* rid = ids + m * top;
  const float* rl = logits + m * top;
  float mx = -INFINITY;
  bool nan = false, bad = false;
  int held = 0;
  for (int k = lane; k < top; k += 32) {
    const int64_t id = rid[k];
    if (id < 0) continue;
    ++held;
    bad |= id >= vocab;
    nan |= rl[k] != rl[k];
    mx = fmaxf(mx, rl[k]);
  }
  for (int o = 16; o; o >>= 1) {
    mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
    held += __shfl_xor_sync(0xFFFFFFFFu, held, o);
  }
  nan = __any_sync(0xFFFFFFFFu, nan);
  bad = __any_sync(0xFFFFFFFFu, bad);
  if (held == 0 || bad || (mx == -INFINITY && !nan)) {
    if (lane == 0) {
      out.count[m] = bad ? -1 : 0;
      out.q0[m] = 0.0f;
    }
    return;
  }
  float sum = 0.0f, zq = 0.0f;  // sum of e^z, and of z e^z
  for (int k = lane; k < top; k += 32)
    if (rid[k] >= 0) {
      const float z = (rl[k] - mx) * inv_t, e = expf(z);
      sum += e;
      if (e > 0.0f) zq += z * e;
    }
  for (int o = 16; o; o >>= 1) {
    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    zq += __shfl_xor_sync(0xFFFFFFFFu, zq, o);
  }
  for (int k = lane; k < top; k += 32) {
    const int64_t id = rid[k];
    if (id < 0) continue;
    int rank = 0;
    for (int i = 0; i < top; ++i) {
      const int64_t o = rid[i];
      rank += o >= 0 && (o < id || (o == id && i < k));
    }
    oid[rank] = int32_t(id);
    oq[rank] = expf((rl[k] - mx) * inv_t) / sum;
  }
  if (lane == 0) {
    out.count[m] = held;
    out.q0[m] = nan ? NAN : zq / sum - logf(sum);
  }
}

// Statistics of the logits of weight_dot: a block per column tile of kStatCols.  A thread's columns are a
// chain of divisions and loads each, so the tiles are small: 27000 columns take 4.8 us in tiles of 512 and
// 12.3 in tiles of 2048.
constexpr int kStatCols = 512;
__global__ void __launch_bounds__(256) dot_stats_kernel(DotValue v, LossRows rows, float* part, float scale) {
  pdl_wait();
  pdl_trigger();
  const int64_t n0 = int64_t(blockIdx.x) * kStatCols, n1 = min(v.rows, n0 + kStatCols);
  const int count = rows.count[0];
  const int32_t* ids = rows.ids;
  const float* q = rows.q;
  constexpr int kPer = kStatCols / 256;
  float s[kPer], mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int64_t n = n0 + threadIdx.x + 256 * i;
    s[i] = n < n1 ? v.get(n) * scale : -INFINITY;
    mx = fmaxf(mx, s[i]);
  }
  const float base = mx == -INFINITY ? 0.0f : mx;
  float sum = 0.0f, hit = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    sum += ex2(s[i] - base);
    const int64_t n = n0 + threadIdx.x + 256 * i;
    if (n < n1)
      for (int k = first_id(ids, count, n); k < count && ids[k] == n; ++k)
        if (q[k] != 0.0f) hit += q[k] * s[i];
  }
  __shared__ RowStats sm[8];
  RowStats st{mx, sum, hit};
  for (int o = 16; o; o >>= 1) {
    const float a = __shfl_xor_sync(0xFFFFFFFFu, st.mx, o), b = __shfl_xor_sync(0xFFFFFFFFu, st.sum, o),
                c = __shfl_xor_sync(0xFFFFFFFFu, st.hit, o);
    stats_join(st, a, b, c);
  }
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = st;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) stats_join(st, sm[i].mx, sm[i].sum, sm[i].hit);
    float* p = part + int64_t(blockIdx.x) * 3;
    p[0] = st.mx;
    p[1] = st.sum;
    p[2] = st.hit;
  }
}

// Joins the tiles' statistics of 32 rows per block (in a fixed order) into lse and the rows' losses.
__global__ void __launch_bounds__(1024) loss_rows_kernel(const float* part, int64_t tiles, int64_t tokens,
                                                         float temperature, LossRows rows, float* loss) {
  pdl_wait();
  pdl_trigger();
  const int64_t m = int64_t(blockIdx.x) * 32 + (threadIdx.x & 31);
  const int sub = threadIdx.x >> 5;
  RowStats st{-INFINITY, 0.0f, 0.0f};
  if (m < tokens)
    for (int64_t t = sub; t < tiles; t += 32) {
      const float* p = part + t * 3 * tokens + m;
      stats_join(st, p[0], p[tokens], p[2 * tokens]);
    }
  __shared__ RowStats sm[32][33];
  sm[sub][threadIdx.x & 31] = st;
  __syncthreads();
  if (sub != 0 || m >= tokens) return;
  for (int i = 1; i < 32; ++i) stats_join(st, sm[i][threadIdx.x].mx, sm[i][threadIdx.x].sum, sm[i][threadIdx.x].hit);
  const int count = rows.count[m];
  // (mx - hit first: a confident row's loss is small beside both.)
  const float nats = count < 0 ? NAN : ((st.mx - st.hit) + log2f(st.sum)) * kLn2;
  loss[m] = count == 0 ? 0.0f : temperature * temperature * (rows.q0[m] + nats);
}

// The first reference of each row: its maximum over the columns of the sample, less `below`.
__global__ void __launch_bounds__(1024) sample_kernel(const float* part, int64_t tiles, int64_t tokens, float below,
                                                      SoftRows soft) {
  pdl_wait();
  pdl_trigger();
  const int64_t m = int64_t(blockIdx.x) * 32 + (threadIdx.x & 31);
  const int sub = threadIdx.x >> 5;
  float mx = -INFINITY;
  if (m < tokens)
    for (int64_t t = sub; t < tiles; t += 32) mx = fmaxf(mx, part[t * tokens + m]);
  __shared__ float sm[32][33];
  sm[sub][threadIdx.x & 31] = mx;
  __syncthreads();
  if (sub != 0 || m >= tokens) return;
  for (int i = 1; i < 32; ++i) mx = fmaxf(mx, sm[i][threadIdx.x]);
  soft.ref[m] = mx - below;
  soft.sum[m] = 0.0f;
}

// After a piece: its sums to the rows', and a new reference for the rows with groups left out (5 us for
// 2048 rows and 211 tiles).
__global__ void __launch_bounds__(1024) soft_rows_kernel(const float* part, int64_t tiles, int64_t tokens,
                                                         SoftRows soft) {
  pdl_wait();
  pdl_trigger();
  const int64_t m = int64_t(blockIdx.x) * 32 + (threadIdx.x & 31);
  const int sub = threadIdx.x >> 5;
  float sum = 0.0f, out = -INFINITY;
  if (m < tokens)
    for (int64_t t = sub; t < tiles; t += 32) {
      sum += part[t * 2 * tokens + m];
      out = fmaxf(out, part[t * 2 * tokens + tokens + m]);
    }
  __shared__ float2 sm[32][33];
  sm[sub][threadIdx.x & 31] = make_float2(sum, out);
  __syncthreads();
  if (sub != 0 || m >= tokens) return;
  for (int i = 1; i < 32; ++i) {
    sum += sm[i][threadIdx.x].x;
    out = fmaxf(out, sm[i][threadIdx.x].y);
  }
  const float ref = soft.ref[m];
  sum += soft.sum[m];
  soft.before[m] = ref;
  float scale = 1.0f;
  if (out > -INFINITY) {
    const float raised = fmaxf(ref, out);
    scale = ref == -INFINITY ? 0.0f : ex2(ref - raised);
    soft.ref[m] = raised;
    *soft.again = 1;
  }
  soft.scale[m] = scale;
  soft.sum[m] = sum * scale;
}

// The terms of a row's ids in this piece: acc += 2^(s'_k - r) W[id_k], acc_q += q_k W[id_k], in 32 bits,
// or for a row of a single id acc_q = W[id] (soft_end_kernel knows its factor); and the sums of the groups
// that were multiplied again.  One CTA per row.  4096 rows of 3584 with one id each take 10 us in each of
// three pieces, beside 2000 us of products; 2048 rows of 2560 with 32 ids 75 us in each of two, beside 860.
template <typename T>
__global__ void __launch_bounds__(128) gather_kernel(LossRows rows, SoftRows soft, const T* w, int64_t pitch,
                                                     int64_t v0, int64_t v1, int64_t cols, float* acc, float* acc_q,
                                                     int64_t ld, const float* part, int64_t tiles, int64_t tokens) {
  pdl_wait();
  pdl_trigger();
  __shared__ float s_p[kMaxTop], s_q[kMaxTop], s_sum[128];
  const int64_t m = blockIdx.x;
  const int count = max(0, rows.count[m]), tid = threadIdx.x;
  const int32_t* ids = rows.ids + m * rows.top;
  const int a = first_id(ids, count, v0), b = first_id(ids, count, v1);
  if (*soft.again) {
    float v = 0.0f;
    for (int64_t t = tid; t < tiles; t += 128) v += part[t * 2 * tokens + m];
    s_sum[tid] = v;
    __syncthreads();
    for (int o = 64; o; o >>= 1) {
      if (tid < o) s_sum[tid] += s_sum[tid + o];
      __syncthreads();
    }
    if (tid == 0) soft.sum[m] += s_sum[0];
  }
  if (a == b) return;
  if (rows.top == 1) {
    const T* src = w + (ids[0] - v0) * pitch;
    for (int64_t c = 8 * tid; c < cols; c += 8 * 128) {
      const uint4 q = *reinterpret_cast<const uint4*>(src + c);
      float4* out = reinterpret_cast<float4*>(acc_q + m * ld + c);
      out[0] = make_float4(Num<T>::lo(q.x), Num<T>::hi(q.x), Num<T>::lo(q.y), Num<T>::hi(q.y));
      if (c + 4 < cols) out[1] = make_float4(Num<T>::lo(q.z), Num<T>::hi(q.z), Num<T>::lo(q.w), Num<T>::hi(q.w));
    }
    return;
  }
  const float ref = soft.ref[m], base = ref == -INFINITY ? 0.0f : ref;
  for (int k = a + tid; k < b; k += 128) {
    // An id given twice is one column of the softmax: only its first entry carries it.
    s_p[k - a] = k > a && ids[k] == ids[k - 1] ? 0.0f : ex2(soft.hit[m * rows.top + k] - base);
    s_q[k - a] = rows.q[m * rows.top + k];
  }
  __syncthreads();
  for (int64_t c = 8 * tid; c < cols; c += 8 * 128) {
    float x[8] = {}, y[8] = {};
    for (int k = a; k < b; ++k) {
      const uint4 q = *reinterpret_cast<const uint4*>(w + (ids[k] - v0) * pitch + c);
      const uint32_t ww[4] = {q.x, q.y, q.z, q.w};
      const float fp = s_p[k - a], fq = s_q[k - a];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float lo = Num<T>::lo(ww[i]), hi = Num<T>::hi(ww[i]);
        if (fp != 0.0f) {
          x[2 * i] = fmaf(fp, lo, x[2 * i]);
          x[2 * i + 1] = fmaf(fp, hi, x[2 * i + 1]);
        }
        y[2 * i] = fmaf(fq, lo, y[2 * i]);
        y[2 * i + 1] = fmaf(fq, hi, y[2 * i + 1]);
      }
    }
#pragma unroll
    for (int h = 0; h < 8; h += 4)
      if (c + h < cols) {  // the pitch covers the last group of 4
        float4* pa = reinterpret_cast<float4*>(acc + m * ld + c + h);
        float4* pq = reinterpret_cast<float4*>(acc_q + m * ld + c + h);
        const float4 va = *pa, vq = *pq;
        *pa = make_float4(va.x + x[h], va.y + x[h + 1], va.z + x[h + 2], va.w + x[h + 3]);
        *pq = make_float4(vq.x + y[h], vq.y + y[h + 1], vq.z + y[h + 2], vq.w + y[h + 3]);
      }
  }
}

// V = 1 or 4 (16-byte accesses) floats.
template <int V>
__device__ __forceinline__ void load_floats(const float* p, float* v) {
  if constexpr (V == 4) {
    const float4 q = *reinterpret_cast<const float4*>(p);
    v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
  } else {
    v[0] = *p;
  }
}
template <int V>
__device__ __forceinline__ void store_floats(float* p, const float* v) {
  if constexpr (V == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  else *p = v[0];
}

// Sum or maximum over a block of 128 threads, on every thread.
template <bool MAX>
__device__ __forceinline__ float block_join(float v, float* sm) {
  for (int o = 16; o; o >>= 1) {
    const float u = __shfl_xor_sync(0xFFFFFFFFu, v, o);
    v = MAX ? fmaxf(v, u) : v + u;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  return MAX ? fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])) : (sm[0] + sm[1]) + (sm[2] + sm[3]);
}

// A row's loss and its gradient, V columns per thread.  With S = sum over the columns that are no ids, of
// 2^(s' - r), and E the same over the ids: lse' = r + log2(S + E), and the gradient is
//   T (acc / (S + E) - acc_q)                      for several ids, acc and acc_q holding their terms,
//   T (acc / (S + E) - S / (S + E) W[id])          for one (q = 1, acc_q = W[id]), whose loss is
//                                                  log(1 + S / E): no difference of near numbers.
// One CTA per row.  Bound by its bytes: 2048 x 3584 in 15 us (88 MB at 5.9 TB/s; one column at a time
// took 22 us).
template <int V>
__global__ void __launch_bounds__(128) soft_end_kernel(LossRows rows, SoftRows soft, const float* __restrict__ acc,
                                                       const float* __restrict__ acc_q, int64_t ld, int64_t cols,
                                                       float temperature, float* loss, float* __restrict__ unit) {
  pdl_wait();
  pdl_trigger();
  __shared__ float sm[4];
  const int64_t m = blockIdx.x;
  const int count = rows.count[m], tid = threadIdx.x;
  const float ref = soft.ref[m], sum = soft.sum[m];
  const int32_t* ids = rows.ids + m * rows.top;
  const float* q = rows.q + m * rows.top;
  const float* hit = soft.hit + m * rows.top;
  float nats = 0.0f, total = 1.0f, fq = 0.0f;  // the loss over T^2 less q0, S + E, the factor of acc_q
  if (rows.top == 1) {
    if (count > 0) {
      const float s = hit[0] < INFINITY ? hit[0] : NAN;  // an infinite target has no loss
      const float x = (ref - s) + log2f(sum), e = ref > -INFINITY ? ex2(s - ref) : s > -INFINITY ? 1.0f : NAN;
      nats = fmaxf(x, 0.0f) * kLn2 + log1pf(exp2f(-fabsf(x)));
      total = sum + e;
      fq = -q[0] * (sum / total);
    }
  } else {
    float mx = ref;
    for (int k = tid; k < count; k += 128) mx = fmaxf(mx, hit[k]);
    mx = block_join<true>(mx, sm);
    const float base = ref == -INFINITY ? 0.0f : ref;
    float e = 0.0f, z = 0.0f, d = 0.0f;
    for (int k = tid; k < count; k += 128) {
      if (k == 0 || ids[k] != ids[k - 1]) {  // an id given twice is one column of the softmax
        e += ex2(hit[k] - base);
        z += ex2(hit[k] - mx);
      }
      if (q[k] != 0.0f) d += q[k] * (mx - hit[k]);
    }
    e = block_join<false>(e, sm);
    z = block_join<false>(z, sm);
    d = block_join<false>(d, sm);
    nats = (d + log2f(sum * ex2(ref - mx) + z)) * kLn2;
    total = sum + e;
    fq = -1.0f;
  }
  if (tid == 0) loss[m] = count == 0 ? 0.0f : count < 0 ? NAN : temperature * temperature * (rows.q0[m] + nats);
  const float f = temperature / total;
  fq *= temperature;
#pragma unroll 4
  for (int64_t c = V * tid; c < cols; c += V * 128) {
    float a[V], g[V];
    load_floats<V>(acc + m * ld + c, a);
    load_floats<V>(acc_q + m * ld + c, g);
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] = count < 0 ? NAN : count == 0 ? 0.0f : fmaf(a[i], f, fq * g[i]);
    store_floats<V>(unit + m * cols + c, a);
  }
}

// dh = unit * (gradient of the row's loss) in 16 bits, V columns per lane; all of a step's loads come first.
// 2048 x 3584 in 8.5 us (44 MB at 5.2 TB/s; 21.6 us with 4-byte loads).
template <typename T, int V>
__global__ void __launch_bounds__(256) unit_kernel(const float* __restrict__ unit, int64_t tokens, int64_t cols,
                                                   LossRows rows, const float* grad, int64_t grad_step, bool mean,
                                                   T* __restrict__ dh) {
  pdl_wait();
  pdl_trigger();
  constexpr int kSteps = V == 4 ? 4 : 8;
  const int64_t per_row = cdiv(cols, 32 * V * kSteps), total = tokens * per_row;
  const int lane = threadIdx.x & 31;
  for (int64_t i = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5); i < total; i += int64_t(gridDim.x) * 8) {
    const int64_t m = i / per_row, c0 = (i - m * per_row) * (32 * V * kSteps) + V * lane;
    float v[kSteps][V];
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
      if (c0 + 32 * V * k < cols) load_floats<V>(unit + m * cols + c0 + 32 * V * k, v[k]);
    const bool counts = rows.count[m] != 0;
    const float f = counts ? grad[m * grad_step] / (mean ? *rows.rows : 1.0f) : 0.0f;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const int64_t c = c0 + 32 * V * k;
      if (c >= cols) break;
#pragma unroll
      for (int q = 0; q < V; ++q) v[k][q] = counts ? v[k][q] * f : 0.0f;
      if constexpr (V == 4) {
        *reinterpret_cast<uint2*>(dh + m * cols + c) = make_uint2(Num<T>::pack(v[k][0], v[k][1]), Num<T>::pack(v[k][2], v[k][3]));
      } else {
        dh[m * cols + c] = Num<T>::from(v[k][0]);
      }
    }
  }
}

// Sum or mean over the rows that count, added in 64 bits by one block in a fixed order.
__global__ void __launch_bounds__(1024) loss_reduce_kernel(const float* row_loss, LossRows rows, int64_t tokens,
                                                           bool mean, float* loss) {
  pdl_wait();
  double s = 0.0;
  int64_t n = 0;
  for (int64_t m = threadIdx.x; m < tokens; m += 1024) {
    s += row_loss[m];
    n += rows.count[m] != 0;
  }
  __shared__ double ss[1024];
  __shared__ int64_t sn[1024];
  ss[threadIdx.x] = s;
  sn[threadIdx.x] = n;
  __syncthreads();
  for (int o = 512; o; o >>= 1) {
    if (int(threadIdx.x) < o) {
      ss[threadIdx.x] += ss[threadIdx.x + o];
      sn[threadIdx.x] += sn[threadIdx.x + o];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const double count = sn[0] > 0 ? double(sn[0]) : 1.0;
    *loss = float(mean ? ss[0] / count : ss[0]);
    *rows.rows = float(count);
  }
}

// ---- host side ------------------------------------------------------------------------------

// Carves a scratch buffer into 256-byte aligned parts; with a null base it only counts.
struct Arena {
  uint8_t* base;
  size_t used = 0;
  template <typename T = void>
  T* take(size_t bytes) {
    const size_t at = used;
    used += (bytes + 255) & ~size_t(255);
    return base ? reinterpret_cast<T*>(base + at) : nullptr;
  }
};

int64_t round8(int64_t n) { return (n + 7) & ~int64_t(7); }
unsigned grid_1d(int64_t items, int per, int64_t most) {
  return unsigned(std::max<int64_t>(1, std::min(most, cdiv(items, per))));
}

// A 16-bit matrix that TMA can read.
struct Matrix {
  const void* p;
  int64_t rows, cols, pitch;
};
bool tma_ready(const void* p, int64_t pitch) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && pitch % 8 == 0; }

int copy_pitch(const PitchCopy& p, cudaStream_t s) {
  if (p.rows * p.cols == 0) return ZN_OK;
  return launch_after(pitch_kernel, dim3(grid_1d(p.rows * cdiv(p.cols, 256), 8, 148 * 8)), 256, 0, s, "pitch_kernel", p);
}

// A weight and the scratch that its pieces are decoded into.
struct Weight {
  WeightBlob b;
  bool stored;
  int64_t piece_rows, pieces;
  void* temp;
  uint8_t* flat;    // decoded chunks of a piece
  uint8_t* padded;  // its rows at a pitch that TMA can read, when cols is not a multiple of 8
  int64_t pitch;
  int32_t* status;
};

constexpr int64_t kStoredPiece = 4 * 5 * 148 * (int64_t(1) << 17);  // as four waves of default chunks: 0.78 GB

// rows_cap bounds the rows of a piece (0: no bound).
int plan_weight(const zn_weight* w, int64_t rows_cap, int32_t* status, Arena& ar, Weight* out) {
  *out = {};
  out->b = {static_cast<const uint8_t*>(w->blob), w->blob_bytes, w->rows, w->cols, w->chunk_bytes, w->dtype == 8};
  out->stored = w->chunk_bytes == 0;
  out->status = status;
  out->pitch = round8(w->cols);
  const int64_t n = w->rows * w->cols;
  int64_t rows = w->rows;
  if (!out->stored) {
    // A piece is at most four waves of the decoder (5 blocks per SM, 128 Ki elements each at the default
    // chunk size: 0.78 GB).  Every piece ends in a thinning wave, and the products of a piece in an
    // incomplete one: with pieces of half a wave, 1, 2 and 4 waves 64 rows over 152064 x 3584 take 1322,
    // 990, 909 and 875 us.
    int64_t wave = 0;
    if (int rc = weight_wave(out->b, &wave)) return rc;
    const int64_t wave_rows = std::max<int64_t>(1, wave * w->chunk_bytes / w->cols);
    rows = 4 * wave_rows;
    if (rows_cap > 0 && rows > rows_cap) rows = rows_cap >= wave_rows ? rows_cap / wave_rows * wave_rows : rows_cap;
  } else {  // copied to an address that TMA can read, as many elements at a time
    rows = std::min(rows, std::max<int64_t>(1, kStoredPiece / w->cols));
    if (rows_cap > 0) rows = std::min(rows, rows_cap);
  }
  if (rows < w->rows) rows = std::max<int64_t>(256, rows / 256 * 256);
  out->piece_rows = std::min(rows, w->rows);
  out->pieces = cdiv(w->rows, out->piece_rows);
  out->b.direct = !out->stored && weight_direct(out->b, out->pieces);
  if (!out->stored) {
    out->temp = ar.take(weight_temp_bytes(out->b));
    const int64_t chunks = std::min(cdiv(n, w->chunk_bytes), cdiv(out->piece_rows * w->cols, w->chunk_bytes) + 1);
    out->flat = ar.take<uint8_t>(size_t(chunks) * w->chunk_bytes * 2);
  }
  if (out->stored || w->cols % 8) out->padded = ar.take<uint8_t>(size_t(out->piece_rows) * out->pitch * 2);
  return ZN_OK;
}

int start_weight(const Weight& w, cudaStream_t s) {
  if (!w.stored) return w.b.direct ? ZN_OK : weight_scan(w.b, w.temp, w.status, s);
  const cudaError_t e = cudaMemsetAsync(w.status, 0, sizeof(int32_t), s);
  return e == cudaSuccess ? ZN_OK : set_error(ZN_ERR_CUDA, "status: %s", cudaGetErrorString(e));
}

// Rows [r0, r1) as a matrix in memory.  With the first rows goes the copy of the other operand.
int load_piece(const Weight& w, int64_t r0, int64_t r1, const PitchCopy& other, Matrix* out, cudaStream_t s) {
  const int64_t cols = w.b.cols, c0 = w.stored ? 0 : r0 * cols / w.b.chunk;
  const uint8_t* src = w.stored ? w.b.blob + 24 + 8 * 2 + r0 * cols * 2 : w.flat + (r0 * cols - c0 * w.b.chunk) * 2;
  const PitchCopy second = r0 == 0 ? other : PitchCopy{};
  PitchCopy first{};
  *out = {src, r1 - r0, cols, cols};
  if (w.padded) {  // else cols and the chunk size are multiples of 8: the rows are aligned
    first = {reinterpret_cast<const uint16_t*>(src), reinterpret_cast<uint16_t*>(w.padded), cols, w.pitch, r1 - r0, cols};
    *out = {w.padded, r1 - r0, cols, w.pitch};
  }
  const bool tail0 = first.rows * first.cols <= kTailCopy, tail1 = second.rows * second.cols <= kTailCopy;
  if (!w.stored)
    if (int rc = weight_decode(w.b, w.temp, c0, cdiv(r1 * cols, w.b.chunk), w.flat, tail0 ? first : PitchCopy{},
                               tail1 ? second : PitchCopy{}, w.status, s))
      return rc;
  if (w.stored || !tail0)
    if (int rc = copy_pitch(first, s)) return rc;
  if (w.stored || !tail1)
    if (int rc = copy_pitch(second, s)) return rc;
  return ZN_OK;
}

// A caller's matrix, copied to an aligned pitch when TMA cannot read it as it lies; the copy is left
// to the caller (PitchCopy).
void* plan_matrix(const void* p, int64_t rows, int64_t cols, int64_t pitch, Arena& ar) {
  return tma_ready(p, pitch) ? nullptr : ar.take(size_t(rows) * round8(cols) * 2);
}
Matrix load_matrix(const void* p, int64_t rows, int64_t cols, int64_t pitch, void* copy, PitchCopy* job) {
  *job = {};
  if (!copy) return {p, rows, cols, pitch};
  *job = {static_cast<const uint16_t*>(p), static_cast<uint16_t*>(copy), pitch, round8(cols), rows, cols};
  return {copy, rows, cols, round8(cols)};
}

template <typename T, bool BMN, class Epi>
int product(const Matrix& a, const Matrix& b, const Cut& cut, float* parts, const Epi& epi, int32_t* status,
            cudaStream_t s, const int32_t* go = nullptr) {
  const int64_t M = a.rows, K = a.cols, N = BMN ? b.cols : b.rows;
  constexpr bool bf16 = Num<T>::kCode == 1;
  CUtensorMap ma, mb;
  if (int rc = make_map(&ma, a.p, a.rows, a.cols, a.pitch, kBM, bf16)) return rc;
  if (int rc = make_map(&mb, b.p, b.rows, b.cols, b.pitch, BMN ? kBK : 128, bf16)) return rc;
  const GemmShape g = gemm_shape(M, N, K, cut, parts, status, go);
  if (int rc = cut.cg == 2 ? launch_gemm<T, 2, BMN>(ma, mb, g, epi, s) : launch_gemm<T, 1, BMN>(ma, mb, g, epi, s))
    return rc;
  if constexpr (Epi::kParts) {
    if (g.rest) {
      const int tile = kBM * cut.cg;
      TimedLaunch tl("finish", s);
      return launch_after(parts_kernel<Epi>, dim3(unsigned(int64_t(g.rest) * (tile * tile / 4 / 256))), 256, 0, s,
                          "parts_kernel", g, epi, tile);
    }
  }
  return ZN_OK;
}
// Products whose epilogue takes parts: cut by their own sizes.
template <typename T, bool BMN, class Epi>
int product(const Matrix& a, const Matrix& b, int sms, float* parts, const Epi& epi, int32_t* status, cudaStream_t s) {
  const Cut cut = cut_of(a.rows, BMN ? b.cols : b.rows, a.cols, sms, true);
  return product<T, BMN>(a, b, cut, parts, epi, status, s);
}

template <typename T>
int run_finish(const Finish<T>& f, cudaStream_t s) {
  TimedLaunch tl("finish", s);
  return launch_after(finish_kernel<T>, dim3(grid_1d(f.M * f.N, 256, 148 * 16)), 256, 0, s, "finish_kernel", f);
}

int bad(const char* what) { return set_error(ZN_ERR_INVALID, "%s: bad arguments", what); }

bool weight_ok(const zn_weight* w) {
  constexpr int64_t kMost = int64_t(1) << 31;
  if (!w || w->rows <= 0 || w->cols <= 0 || w->rows >= kMost || w->cols >= kMost) return false;
  if (w->rows > (int64_t(1) << 46) / w->cols || (w->dtype != 7 && w->dtype != 8)) return false;
  if (w->chunk_bytes < 0 || w->chunk_bytes % 8 || w->chunk_bytes > kMaxChunkBytes) return false;
  if (w->chunk_bytes == 0) return w->blob_bytes >= 24 + 16 + w->rows * w->cols * 2;
  return w->blob_bytes >= 40 && cdiv(w->rows * w->cols, w->chunk_bytes) <= 0x7FFFFFFF;
}
bool sizes_ok(int64_t tokens, int64_t pitch, int64_t cols) {
  return tokens > 0 && tokens < (int64_t(1) << 31) && pitch >= cols && pitch < (int64_t(1) << 39);
}

// ---- linear ---------------------------------------------------------------------------------

struct LinearPlan {
  Weight w;
  bool dot;
  void* x_copy;
  float* acc;   // parts of a product's last tiles, or z of the dot path
  float* part;  // dot path
  int sms;
};

int plan_linear(const zn_weight* w, const void* x, int64_t ldx, int64_t tokens, int32_t* status, Arena& ar,
                LinearPlan* p) {
  *p = {};
  if (int rc = sm_count(&p->sms)) return rc;
  p->dot = w->chunk_bytes > 0 && dot_shape(tokens, w->cols, w->chunk_bytes);
  p->x_copy = plan_matrix(x, tokens, w->cols, ldx, ar);
  if (p->dot) {
    p->w.b = {static_cast<const uint8_t*>(w->blob), w->blob_bytes, w->rows, w->cols, w->chunk_bytes, w->dtype == 8};
    p->w.b.direct = weight_direct(p->w.b, 1);
    p->w.status = status;
    p->w.temp = ar.take(weight_temp_bytes(p->w.b));
    p->acc = ar.take<float>(size_t(w->rows) * 4);
    p->part = ar.take<float>(dot_part_bytes(p->w.b));
    return ZN_OK;
  }
  if (int rc = plan_weight(w, 0, status, ar, &p->w)) return rc;
  p->acc = ar.take<float>(parts_bytes(p->sms));
  return ZN_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T>
EpiLinear<T> linear_epilogue(const void* bias, const void* res, int64_t ldr, void* y, void* slope, int64_t ldy,
                             int64_t M, int64_t r0, int64_t r1, int act) {
  EpiLinear<T> e{};
  e.bias = bias ? static_cast<const T*>(bias) + r0 : nullptr;
  e.res = res ? static_cast<const T*>(res) + r0 : nullptr;
  e.y = static_cast<T*>(y) + r0;
  e.slope = slope ? static_cast<__half*>(slope) + r0 : nullptr;
  e.ldr = ldr;
  e.ldy = ldy;
  e.M = M;
  e.N = r1 - r0;
  e.act = act;
  e.vec = aligned16(e.bias) && aligned16(e.res) && aligned16(e.y) && aligned16(e.slope) && ldy % 8 == 0 &&
          (!res || ldr % 8 == 0);
  return e;
}

template <typename T>
int run_linear(const LinearPlan& p, const void* x, int64_t ldx, int64_t tokens, const void* bias, int act,
               const void* res, int64_t ldr, void* y, void* slope, cudaStream_t s) {
  const int64_t rows = p.w.b.rows, cols = p.w.b.cols;
  if (int rc = start_weight(p.w, s)) return rc;
  PitchCopy x_job;
  const Matrix xm = load_matrix(x, tokens, cols, ldx, p.x_copy, &x_job);
  Finish<T> f{};
  f.M = tokens;
  if (p.dot) {
    if (int rc = copy_pitch(x_job, s)) return rc;
    f.N = rows;
    f.lin = linear_epilogue<T>(bias, res, ldr, y, slope, rows, tokens, 0, rows, act);
    return weight_linear<T>(p.w.b, p.w.temp, xm.p, p.acc, p.part, f, p.w.status, s);
  }
  for (int64_t r0 = 0; r0 < rows; r0 += p.w.piece_rows) {
    const int64_t r1 = std::min(rows, r0 + p.w.piece_rows);
    Matrix wm;
    if (int rc = load_piece(p.w, r0, r1, x_job, &wm, s)) return rc;
    const EpiLinear<T> e = linear_epilogue<T>(bias, res, ldr, y, slope, rows, tokens, r0, r1, act);
    if (int rc = product<T, false>(xm, wm, p.sms, p.acc, e, p.w.status, s)) return rc;
  }
  return ZN_OK;
}

struct LinearGradPlan {
  Weight w;
  int sms;
  void* dz;  // dy * slope, or an aligned copy of dy
  int64_t ldz;
  float* acc;  // dx in 32 bits over the pieces, when there are several
  float* parts;
  float* part;
  int64_t ld, sum_rows, sum_blocks;
};

int plan_linear_grad(const zn_weight* w, const void* dy, int64_t ldy, int64_t tokens, bool slope, bool dx, bool dbias,
                     int32_t* status, Arena& ar, LinearGradPlan* p) {
  *p = {};
  if (int rc = sm_count(&p->sms)) return rc;
  p->sum_rows = tokens <= kSumAll ? kSumAll : kSumRows;
  p->sum_blocks = cdiv(tokens, p->sum_rows);
  if (dbias && p->sum_blocks > 1) p->part = ar.take<float>(size_t(p->sum_blocks) * w->rows * 4);
  p->w.status = status;
  if (!dx) return ZN_OK;
  p->ldz = round8(w->rows);
  if (slope || !tma_ready(dy, ldy)) p->dz = ar.take(size_t(tokens) * p->ldz * 2);
  if (int rc = plan_weight(w, 0, status, ar, &p->w)) return rc;
  p->ld = (w->cols + 3) & ~int64_t(3);
  p->parts = ar.take<float>(parts_bytes(p->sms));
  if (p->w.pieces > 1) p->acc = ar.take<float>(size_t(tokens) * p->ld * 4);
  return ZN_OK;
}

template <typename T>
int run_linear_grad(const LinearGradPlan& p, const zn_weight* w, const void* dy, int64_t ldy, int64_t tokens,
                    const void* slope, void* dx, void* dbias, cudaStream_t s) {
  const int64_t rows = w->rows, cols = w->cols;
  const T* g = static_cast<const T*>(dy);
  if (slope || dbias) {
    T* dz = slope ? static_cast<T*>(p.dz) : nullptr;
    const bool vec = rows % 8 == 0 && tma_ready(g, ldy) && tma_ready(slope, 0) && tma_ready(dz, p.ldz);
    const int64_t grid = cdiv(rows, vec ? 256 : 32) * p.sum_blocks;
    if (grid > 0x7FFFFFFF) return bad("zn_linear_grad");
    auto fn = vec ? slope_kernel<T, 8> : slope_kernel<T, 1>;
    if (int rc = launch_after(fn, dim3(unsigned(grid)), 256, 0, s, "slope_kernel", g, ldy,
                              static_cast<const __half*>(slope), dz, p.ldz, p.part,
                              dbias && !p.part ? static_cast<T*>(dbias) : nullptr, tokens, rows, p.sum_rows))
      return rc;
  }
  if (p.part)
    if (int rc = launch_after(column_sum_kernel<T>, dim3(unsigned(cdiv(rows, 32))), 256, 0, s, "column_sum_kernel",
                              static_cast<const float*>(p.part), p.sum_blocks, rows, static_cast<T*>(dbias)))
      return rc;
  if (!dx) {
    const cudaError_t e = cudaMemsetAsync(p.w.status, 0, sizeof(int32_t), s);
    return e == cudaSuccess ? ZN_OK : set_error(ZN_ERR_CUDA, "status: %s", cudaGetErrorString(e));
  }
  if (int rc = start_weight(p.w, s)) return rc;
  PitchCopy dy_job{};
  Matrix dzm{p.dz, tokens, rows, p.ldz};
  if (!slope) dzm = load_matrix(dy, tokens, rows, ldy, p.dz, &dy_job);
  const EpiLinear<T> e = linear_epilogue<T>(nullptr, nullptr, 0, dx, nullptr, cols, tokens, 0, cols, kNone);
  for (int64_t r0 = 0; r0 < rows; r0 += p.w.piece_rows) {
    const int64_t r1 = std::min(rows, r0 + p.w.piece_rows);
    Matrix wm;
    if (int rc = load_piece(p.w, r0, r1, dy_job, &wm, s)) return rc;
    // Columns [r0, r1) of dz (r0 is a multiple of 256: the rows stay 16-byte aligned).
    const Matrix a{static_cast<const T*>(dzm.p) + r0, tokens, r1 - r0, dzm.pitch};
    const EpiAccum acc{p.acc, tokens, cols, p.ld, r0 > 0, nullptr};
    if (int rc = p.acc ? product<T, true>(a, wm, p.sms, p.parts, acc, p.w.status, s)
                       : product<T, true>(a, wm, p.sms, p.parts, e, p.w.status, s))
      return rc;
  }
  if (!p.acc) return ZN_OK;
  Finish<T> f{};
  f.acc = p.acc;
  f.M = tokens;
  f.N = cols;
  f.ld = p.ld;
  f.lin = e;
  return run_finish(f, s);
}

// ---- losses ---------------------------------------------------------------------------------

LossRows loss_state(void* state, int64_t tokens, int top, size_t* bytes) {
  Arena ar{static_cast<uint8_t*>(state)};
  LossRows r{};
  r.q0 = ar.take<float>(size_t(tokens) * 4);
  r.count = ar.take<int32_t>(size_t(tokens) * 4);
  r.ids = ar.take<int32_t>(size_t(tokens) * top * 4);
  r.q = ar.take<float>(size_t(tokens) * top * 4);
  r.rows = ar.take<float>(4);
  r.top = top;
  if (bytes) *bytes = ar.used;
  return r;
}

struct LossPlan {
  Weight w;
  bool dot;
  Cut cut;
  void* x_copy;
  float* part;      // tile statistics
  float* row_loss;  // when the call returns their sum or mean
  float* z;         // dot path
  float* z_part;
  int64_t tiles;
};

int plan_loss(const zn_weight* w, const void* x, int64_t ldx, int64_t tokens, int32_t* status, Arena& ar, LossPlan* p) {
  *p = {};
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  p->x_copy = plan_matrix(x, tokens, w->cols, ldx, ar);
  p->row_loss = ar.take<float>(size_t(tokens) * 4);
  p->dot = w->chunk_bytes > 0 && dot_shape(tokens, w->cols, w->chunk_bytes);
  if (p->dot) {
    p->w.b = {static_cast<const uint8_t*>(w->blob), w->blob_bytes, w->rows, w->cols, w->chunk_bytes, w->dtype == 8};
    p->w.b.direct = weight_direct(p->w.b, 1);
    p->w.status = status;
    p->w.temp = ar.take(weight_temp_bytes(p->w.b));
    p->z = ar.take<float>(size_t(w->rows) * 4);
    p->z_part = ar.take<float>(dot_part_bytes(p->w.b));
    p->tiles = cdiv(w->rows, kStatCols);
  } else {
    if (int rc = plan_weight(w, 0, status, ar, &p->w)) return rc;
    p->cut = cut_of(tokens, p->w.piece_rows, w->cols, sms, false);
    // Every piece but the last is a multiple of 256 rows.
    p->tiles = cdiv(w->rows, 64 * p->cut.cg);
  }
  p->part = ar.take<float>(size_t(p->tiles) * 3 * tokens * 4);
  return ZN_OK;
}

template <typename T>
int run_loss(const LossPlan& p, const void* x, int64_t ldx, int64_t tokens, const int64_t* ids, const float* logits,
             int64_t ignore, float temperature, int reduction, float* loss, const LossRows& rows, cudaStream_t s) {
  const int64_t vocab = p.w.b.rows, cols = p.w.b.cols;
  const float inv_t = 1.0f / temperature;
  if (int rc = launch_after(loss_prep_kernel, dim3(unsigned(cdiv(tokens, 4))), 128, 0, s, "loss_prep_kernel", ids,
                            logits, tokens, vocab, ignore, inv_t, rows))
    return rc;
  if (int rc = start_weight(p.w, s)) return rc;
  PitchCopy x_job;
  const Matrix xm = load_matrix(x, tokens, cols, ldx, p.x_copy, &x_job);
  if (p.dot) {
    if (int rc = copy_pitch(x_job, s)) return rc;
    if (int rc = weight_dot(p.w.b, p.w.temp, xm.p, p.z, p.z_part, p.w.status, s)) return rc;
    const DotValue v{p.z, p.z_part, vocab, cols, p.w.b.chunk};
    if (int rc = launch_after(dot_stats_kernel, dim3(unsigned(p.tiles)), 256, 0, s, "dot_stats_kernel", v, rows, p.part,
                              kLog2e * inv_t))
      return rc;
  } else {
    for (int64_t r0 = 0; r0 < vocab; r0 += p.w.piece_rows) {
      const int64_t r1 = std::min(vocab, r0 + p.w.piece_rows);
      Matrix wm;
      if (int rc = load_piece(p.w, r0, r1, x_job, &wm, s)) return rc;
      const EpiStats e{rows, p.part, tokens, r1 - r0, r0, r0 / (64 * p.cut.cg), 64 * p.cut.cg, kLog2e * inv_t};
      const Cut cut = whole_cut(p.cut.cg, tokens, r1 - r0);
      if (int rc = product<T, false>(xm, wm, cut, nullptr, e, p.w.status, s)) return rc;
    }
  }
  float* row_loss = reduction == kRows ? loss : p.row_loss;
  if (int rc = launch_after(loss_rows_kernel, dim3(unsigned(cdiv(tokens, 32))), 1024, 0, s, "loss_rows_kernel",
                            static_cast<const float*>(p.part), p.tiles, tokens, temperature, rows, row_loss))
    return rc;
  if (reduction == kRows) return ZN_OK;
  return launch_after(loss_reduce_kernel, dim3(1), 1024, 0, s, "loss_reduce_kernel", static_cast<const float*>(row_loss),
                      rows, tokens, reduction == kMean, loss);
}

// With the gradient, pieces are bounded so that P [tokens, piece] stays within 512 MB too.
constexpr int64_t kProbBytes = int64_t(1) << 29;
constexpr int64_t kSample = 512;

struct LossGradPlan {
  Weight w;
  Cut cut;
  int sms;
  void* x_copy;
  void* prob;
  int64_t ldp, ld;
  float* part;
  float* row_loss;
  float* acc;
  float* acc_q;  // followed by the pieces' `again` flags: zeroed together
  size_t zeroed;
  float* parts;
  SoftRows soft;
};

int plan_loss_grad(const zn_weight* w, const void* x, int64_t ldx, int64_t tokens, int top, int32_t* status, Arena& ar,
                   LossGradPlan* p) {
  *p = {};
  if (int rc = sm_count(&p->sms)) return rc;
  p->x_copy = plan_matrix(x, tokens, w->cols, ldx, ar);
  if (int rc = plan_weight(w, std::max<int64_t>(256, kProbBytes / 2 / tokens), status, ar, &p->w)) return rc;
  p->cut = cut_of(tokens, p->w.piece_rows, w->cols, p->sms, false);
  p->ldp = round8(p->w.piece_rows);
  p->prob = ar.take(size_t(tokens) * p->ldp * 2);
  p->ld = (w->cols + 3) & ~int64_t(3);
  const int64_t tiles = cdiv(std::max(p->w.piece_rows, std::min(kSample, w->rows)), 64);
  p->part = ar.take<float>(size_t(tiles) * 3 * tokens * 4);
  p->row_loss = ar.take<float>(size_t(tokens) * 4);
  p->acc = ar.take<float>(size_t(tokens) * p->ld * 4);
  const size_t acc_bytes = size_t(tokens) * p->ld * 4;
  p->zeroed = acc_bytes + size_t(p->w.pieces) * 4;
  p->acc_q = ar.take<float>(p->zeroed);
  p->soft.again = p->acc_q ? reinterpret_cast<int32_t*>(reinterpret_cast<uint8_t*>(p->acc_q) + acc_bytes) : nullptr;
  p->parts = ar.take<float>(parts_bytes(p->sms));
  for (float** f : {&p->soft.ref, &p->soft.before, &p->soft.scale, &p->soft.sum}) *f = ar.take<float>(size_t(tokens) * 4);
  p->soft.hit = ar.take<float>(size_t(tokens) * top * 4);
  return ZN_OK;
}

// One decoded piece: P and its sums, acc += P W, again for the groups left out, and the ids' terms.
template <typename T>
int soft_piece(const LossGradPlan& p, const Matrix& xm, const Matrix& wm, int64_t r0, const LossRows& rows,
               const SoftRows& soft, float scale, cudaStream_t s) {
  const int64_t tokens = xm.rows, cols = xm.cols, n = wm.rows;
  const int half = 64 * p.cut.cg;
  const int64_t tiles = cdiv(n, half);
  const unsigned row_blocks = unsigned(cdiv(tokens, 32));
  const Matrix pm{p.prob, tokens, n, p.ldp};
  const Cut cut = whole_cut(p.cut.cg, tokens, n);
  if (r0 == 0) {
    const Matrix first{wm.p, std::min(kSample, n), cols, wm.pitch};
    const Cut c = cut_of(tokens, first.rows, cols, p.sms, false);
    const EpiMax e{rows, p.part, tokens, first.rows, 64 * c.cg, scale};
    if (int rc = product<T, false>(xm, first, c, nullptr, e, p.w.status, s)) return rc;
    if (int rc = launch_after(sample_kernel, dim3(row_blocks), 1024, 0, s, "sample_kernel",
                              static_cast<const float*>(p.part), cdiv(first.rows, 64 * c.cg), tokens, kBelow<T>, soft))
      return rc;
  }
  const EpiSoft<T, false> e{rows, soft, static_cast<T*>(p.prob), p.part, tokens, n, p.ldp, r0, half, scale};
  if (int rc = product<T, false>(xm, wm, cut, nullptr, e, p.w.status, s)) return rc;
  const EpiAccum a{p.acc, tokens, cols, p.ld, r0 > 0, nullptr};
  if (int rc = product<T, true>(pm, wm, p.sms, p.parts, a, p.w.status, s)) return rc;
  if (int rc = launch_after(soft_rows_kernel, dim3(row_blocks), 1024, 0, s, "soft_rows_kernel",
                            static_cast<const float*>(p.part), tiles, tokens, soft))
    return rc;
  const EpiSoft<T, true> e2{rows, soft, static_cast<T*>(p.prob), p.part, tokens, n, p.ldp, r0, half, scale};
  if (int rc = product<T, false>(xm, wm, cut, nullptr, e2, p.w.status, s, soft.again)) return rc;
  const EpiAccum a2{p.acc, tokens, cols, p.ld, true, soft.scale};
  const Cut whole = cut_of(tokens, cols, n, p.sms, false);
  if (int rc = product<T, true>(pm, wm, whole, nullptr, a2, p.w.status, s, soft.again)) return rc;
  return launch_after(gather_kernel<T>, dim3(unsigned(tokens)), 128, 0, s, "gather_kernel", rows, soft,
                      static_cast<const T*>(wm.p), wm.pitch, r0, r0 + n, cols, p.acc, p.acc_q, p.ld,
                      static_cast<const float*>(p.part), tiles, tokens);
}

template <typename T>
int run_loss_grad(const LossGradPlan& p, const void* x, int64_t ldx, int64_t tokens, const int64_t* ids,
                  const float* logits, int64_t ignore, float temperature, int reduction, float* loss, float* unit,
                  const LossRows& rows, cudaStream_t s) {
  const int64_t vocab = p.w.b.rows, cols = p.w.b.cols;
  const float inv_t = 1.0f / temperature;
  const cudaError_t err = cudaMemsetAsync(p.acc_q, 0, p.zeroed, s);
  if (err != cudaSuccess) return set_error(ZN_ERR_CUDA, "zn_loss: %s", cudaGetErrorString(err));
  if (int rc = launch_after(loss_prep_kernel, dim3(unsigned(cdiv(tokens, 4))), 128, 0, s, "loss_prep_kernel", ids,
                            logits, tokens, vocab, ignore, inv_t, rows))
    return rc;
  if (int rc = start_weight(p.w, s)) return rc;
  PitchCopy x_job;
  const Matrix xm = load_matrix(x, tokens, cols, ldx, p.x_copy, &x_job);
  SoftRows soft = p.soft;
  for (int64_t r0 = 0; r0 < vocab; r0 += p.w.piece_rows, ++soft.again) {
    const int64_t r1 = std::min(vocab, r0 + p.w.piece_rows);
    Matrix wm;
    if (int rc = load_piece(p.w, r0, r1, x_job, &wm, s)) return rc;
    if (int rc = soft_piece<T>(p, xm, wm, r0, rows, soft, kLog2e * inv_t, s)) return rc;
  }
  float* row_loss = reduction == kRows ? loss : p.row_loss;
  auto end = cols % 4 == 0 && aligned16(unit) ? soft_end_kernel<4> : soft_end_kernel<1>;  // acc is aligned, its pitch too
  if (int rc = launch_after(end, dim3(unsigned(tokens)), 128, 0, s, "soft_end_kernel", rows, soft,
                            static_cast<const float*>(p.acc), static_cast<const float*>(p.acc_q), p.ld, cols,
                            temperature, row_loss, unit))
    return rc;
  if (reduction == kRows) return ZN_OK;
  return launch_after(loss_reduce_kernel, dim3(1), 1024, 0, s, "loss_reduce_kernel", static_cast<const float*>(row_loss),
                      rows, tokens, reduction == kMean, loss);
}

template <typename T>
int run_loss_grad_end(int64_t tokens, int64_t cols, const LossRows& rows, int reduction, const float* unit,
                      const float* grad, void* dh, cudaStream_t s) {
  const bool vec = cols % 4 == 0 && aligned16(unit) && (reinterpret_cast<uintptr_t>(dh) & 7) == 0;
  const dim3 grid(grid_1d(tokens * cdiv(cols, vec ? 512 : 256), 8, 148 * 16));
  return launch_after(vec ? unit_kernel<T, 4> : unit_kernel<T, 1>, grid, 256, 0, s, "unit_kernel", unit, tokens, cols,
                      rows, grad, int64_t(reduction == kRows), reduction == kMean, static_cast<T*>(dh));
}

bool loss_ok(const zn_weight* w, int64_t tokens, int64_t ldx, int top, float temperature, int reduction) {
  return weight_ok(w) && sizes_ok(tokens, ldx, w->cols) && top >= 1 && top <= kMaxTop && temperature > 0.0f &&
         temperature < INFINITY && reduction >= kMean && reduction <= kRows;
}

}  // namespace
}  // namespace zn

using namespace zn;

extern "C" {

size_t zn_linear_temp_bytes(const zn_weight* w, const void* x, int64_t ldx, int64_t tokens) {
  if (!weight_ok(w) || !sizes_ok(tokens, ldx, w->cols)) return 0;
  Arena ar{nullptr};
  LinearPlan p;
  return plan_linear(w, x, ldx, tokens, nullptr, ar, &p) ? 0 : ar.used;
}

int zn_linear(const zn_weight* w, const void* x, int64_t ldx, int64_t tokens, const void* bias, int activation,
              const void* residual, int64_t ldr, void* y, void* slope, int32_t* status, void* temp, size_t temp_bytes,
              void* stream) {
  if (!weight_ok(w) || !sizes_ok(tokens, ldx, w->cols) || (residual && !sizes_ok(tokens, ldr, w->rows)) ||
      activation < kNone || activation > kSilu || !w->blob || (reinterpret_cast<uintptr_t>(w->blob) & 7) || !x || !y ||
      !status)
    return bad("zn_linear");
  NvtxScope range("zn_linear");
  Arena ar{static_cast<uint8_t*>(temp)};
  LinearPlan p;
  if (int rc = plan_linear(w, x, ldx, tokens, status, ar, &p)) return rc;
  if (!temp || temp_bytes < ar.used) return set_error(ZN_ERR_SPACE, "zn_linear: temp buffer too small");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return w->dtype == 8
             ? run_linear<__nv_bfloat16>(p, x, ldx, tokens, bias, activation, residual, ldr, y, slope, s)
             : run_linear<__half>(p, x, ldx, tokens, bias, activation, residual, ldr, y, slope, s);
}

size_t zn_linear_grad_temp_bytes(const zn_weight* w, const void* dy, int64_t ldy, int64_t tokens, int slope, int dx,
                                 int dbias) {
  if (!weight_ok(w) || !sizes_ok(tokens, ldy, w->rows)) return 0;
  Arena ar{nullptr};
  LinearGradPlan p;
  return plan_linear_grad(w, dy, ldy, tokens, slope != 0, dx != 0, dbias != 0, nullptr, ar, &p) ? 0 : ar.used;
}

int zn_linear_grad(const zn_weight* w, const void* dy, int64_t ldy, int64_t tokens, const void* slope, void* dx,
                   void* dbias, int32_t* status, void* temp, size_t temp_bytes, void* stream) {
  if (!weight_ok(w) || !sizes_ok(tokens, ldy, w->rows) || !w->blob || (reinterpret_cast<uintptr_t>(w->blob) & 7) ||
      !dy || !status || (!dx && !dbias))
    return bad("zn_linear_grad");
  NvtxScope range("zn_linear_grad");
  Arena ar{static_cast<uint8_t*>(temp)};
  LinearGradPlan p;
  if (int rc = plan_linear_grad(w, dy, ldy, tokens, slope, dx, dbias, status, ar, &p)) return rc;
  if (!temp || temp_bytes < ar.used) return set_error(ZN_ERR_SPACE, "zn_linear_grad: temp buffer too small");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return w->dtype == 8 ? run_linear_grad<__nv_bfloat16>(p, w, dy, ldy, tokens, slope, dx, dbias, s)
                       : run_linear_grad<__half>(p, w, dy, ldy, tokens, slope, dx, dbias, s);
}

size_t zn_loss_state_bytes(int64_t tokens, int top) {
  if (tokens <= 0 || top < 1 || top > kMaxTop) return 0;
  size_t bytes = 0;
  loss_state(nullptr, tokens, top, &bytes);
  return bytes;
}

size_t zn_loss_temp_bytes(const zn_weight* w, const void* hidden, int64_t ldh, int64_t tokens, int top, int with_grad) {
  if (!loss_ok(w, tokens, ldh, top, 1.0f, 0)) return 0;
  Arena ar{nullptr};
  LossPlan p;
  LossGradPlan g;
  const int rc = with_grad ? plan_loss_grad(w, hidden, ldh, tokens, top, nullptr, ar, &g)
                           : plan_loss(w, hidden, ldh, tokens, nullptr, ar, &p);
  return rc ? 0 : ar.used;
}

int zn_loss(const zn_weight* w, const void* hidden, int64_t ldh, int64_t tokens, const int64_t* ids,
            const float* logits, int top, int64_t ignore_index, float temperature, int reduction, float* loss,
            float* unit_grad, void* state, int32_t* status, void* temp, size_t temp_bytes, void* stream) {
  if (!loss_ok(w, tokens, ldh, top, temperature, reduction) || (!logits && top != 1) || !w->blob ||
      (reinterpret_cast<uintptr_t>(w->blob) & 7) || !hidden || !ids || !loss || !state || !status)
    return bad("zn_loss");
  NvtxScope range("zn_loss");
  Arena ar{static_cast<uint8_t*>(temp)};
  const LossRows rows = loss_state(state, tokens, top, nullptr);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf16 = w->dtype == 8;
  if (unit_grad) {
    LossGradPlan p;
    if (int rc = plan_loss_grad(w, hidden, ldh, tokens, top, status, ar, &p)) return rc;
    if (!temp || temp_bytes < ar.used) return set_error(ZN_ERR_SPACE, "zn_loss: temp buffer too small");
    return bf16 ? run_loss_grad<__nv_bfloat16>(p, hidden, ldh, tokens, ids, logits, ignore_index, temperature,
                                               reduction, loss, unit_grad, rows, s)
                : run_loss_grad<__half>(p, hidden, ldh, tokens, ids, logits, ignore_index, temperature, reduction,
                                        loss, unit_grad, rows, s);
  }
  LossPlan p;
  if (int rc = plan_loss(w, hidden, ldh, tokens, status, ar, &p)) return rc;
  if (!temp || temp_bytes < ar.used) return set_error(ZN_ERR_SPACE, "zn_loss: temp buffer too small");
  return bf16 ? run_loss<__nv_bfloat16>(p, hidden, ldh, tokens, ids, logits, ignore_index, temperature, reduction,
                                        loss, rows, s)
              : run_loss<__half>(p, hidden, ldh, tokens, ids, logits, ignore_index, temperature, reduction, loss,
                                 rows, s);
}

int zn_loss_grad(int dtype, int64_t tokens, int64_t cols, int top, int reduction, const void* state,
                 const float* unit_grad, const float* grad_loss, void* dhidden, void* stream) {
  if ((dtype != 7 && dtype != 8) || tokens <= 0 || tokens >= (int64_t(1) << 31) || cols <= 0 ||
      cols >= (int64_t(1) << 31) || top < 1 || top > kMaxTop || reduction < kMean || reduction > kRows || !state ||
      !unit_grad || !grad_loss || !dhidden)
    return bad("zn_loss_grad");
  NvtxScope range("zn_loss_grad");
  const LossRows rows = loss_state(const_cast<void*>(state), tokens, top, nullptr);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == 8 ? run_loss_grad_end<__nv_bfloat16>(tokens, cols, rows, reduction, unit_grad, grad_loss, dhidden, s)
                    : run_loss_grad_end<__half>(tokens, cols, rows, reduction, unit_grad, grad_loss, dhidden, s);
}

}  // extern "C"
