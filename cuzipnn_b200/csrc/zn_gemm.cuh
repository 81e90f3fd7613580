// Matrix products of 16-bit matrices on the fifth-generation tensor cores (sm_100a), with the
// epilogue as a template argument: D[m, n] = sum_k A[m, k] * B(n, k), accumulated in 32 bits.
//
// A is row-major [M, K].  B is either row-major [N, K] (BMN = false: the contraction runs along its
// rows, as in x W^T) or row-major [K, N] (BMN = true: the contraction runs down its columns, as in
// dz W), so a decoded weight serves both directions as it lies in memory.
//
// Persistent CTAs (CG = 1) or pairs of CTAs on neighbouring SMs (CG = 2) take output tiles in turn:
// 128 x 128 for one CTA, 256 x 256 for a pair, where each CTA loads its half of both operands and
// holds its 128 rows of the result, so that a byte loaded is used twice as often.  Warp 0 loads
// 64-wide blocks with TMA (128-byte swizzle) into a ring of shared-memory stages, one thread of warp
// 1 (of the pair's first CTA) issues tcgen05.mma into one of two accumulators in tensor memory, and
// warps 4-11 read the other accumulator (a thread owns a row of one half of the tile's columns) and
// run the epilogue meanwhile.  Two warps per scheduler: an activation's dependent arithmetic leaves
// one warp idle most of the time.
//
// Bound by the tensor pipe and, in calls of a millisecond and more, by the power limit: 4096 x 18944 x
// 3584 takes 370 us (1500 TFLOP/s, 0.91 of a library product's burst on the same device), with the pipe
// active 75 to 79 % of the cycles.  With tiles of 128 x 128 alone, 2047 rows of it took 595 us where
// pairs took 324, decoding included in both.
//
// Every wait has an iteration limit.  A wait that gives up sets kErrWait in the status word and the
// abort flag, upon which all warps leave their loops, the loads in flight are waited for (again
// with a limit) and the tensor memory is freed; the other CTA of a pair runs into its own limits.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "zn_common.cuh"

namespace zn {

constexpr int32_t kErrWait = 16;  // a bounded wait inside a product kernel gave up

constexpr int kBM = 128;          // rows of a tile per CTA (tensor memory lanes)
constexpr int kBK = 64;           // contraction block: 128 bytes of a 16-bit type, one swizzle row
constexpr int kGemmThreads = 384;  // TMA, MMA, allocation, an idle warp, and 8 epilogue warps
constexpr int kEpiWarps = 8;
constexpr uint32_t kWaitLimit = 1u << 24;  // polls of up to kPollNs each (about 4 s at most)
constexpr uint32_t kPollNs = 256;

struct GemmShape {
  int64_t M, N, K;
  int tiles_m, tiles_n;  // output tiles
  int group_m;           // row tiles that share a column tile before the next one is taken
  int kblocks;           // 64-wide blocks of the contraction
  int64_t full;          // the first `full` tiles are computed whole,
  int rest, splits;      // the `rest` last ones in `splits` parts of the contraction each,
  float* parts;          // whose sums go to parts[rest][splits][tile rows][tile columns]
  int32_t* status;
  const int32_t* go;     // or null: the kernel does nothing where *go is 0
};

// Tile order: within a group of row tiles, the row tile runs fastest, then the column tile, so that
// the CTAs of one wave share a few column blocks of B and a group's rows of A in L2.
__host__ __device__ inline void tile_place(const GemmShape& g, int64_t t, int& tm, int& tn) {
  const int64_t per = int64_t(g.group_m) * g.tiles_n;
  const int grp = int(t / per);
  const int64_t r = t - grp * per;
  const int left = g.tiles_m - grp * g.group_m, gm = left < g.group_m ? left : g.group_m;
  tm = grp * g.group_m + int(r % gm);
  tn = int(r / gm);
}

// ---- PTX ------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok) : "r"(bar), "r"(parity), "r"(kPollNs) : "memory");
  return ok != 0;
}
// Wait for the barrier's phase; gives up when another role aborted or at the limit (and aborts).
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  for (uint32_t i = 0; i < kWaitLimit; ++i) {
    if (mbar_try(bar, parity)) return true;
    if ((i & 255) == 255 && *abort_flag) return false;
  }
  *abort_flag = 1;
  return false;
}
__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// The same shared address in the pair's first CTA.
__device__ __forceinline__ uint32_t in_leader(uint32_t addr) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
template <int CG>
__device__ __forceinline__ void group_sync() {
  if constexpr (CG == 2) {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
  } else {
    __syncthreads();
  }
}
// With CG = 2 the barrier may lie in the other CTA of the pair.
template <int CG>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if constexpr (CG == 2) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
  }
}
// Arrive on the barrier (of both CTAs of a pair) when the MMAs issued so far have ended.
template <int CG>
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  if constexpr (CG == 2) {
    asm volatile(
        "{\n .reg .b16 m;\n mov.b16 m, 3;\n"
        " tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n}\n"
        ::"r"(bar) : "memory");
  } else {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  }
}
template <int CG>
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 2) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  } else {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  }
}
template <int CG, int COLS>
__device__ __forceinline__ void tmem_alloc(uint32_t dst) {
  if constexpr (CG == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "n"(COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "n"(COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
}
template <int CG, int COLS>
__device__ __forceinline__ void tmem_free(uint32_t addr) {
  if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "n"(COLS));
  else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "n"(COLS));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 accumulator columns of the calling thread's row (its warp's quarter of the lanes).
__device__ __forceinline__ void tc_load32(uint32_t addr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tc_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Shared-memory matrix descriptors, 128-byte swizzle (layout code 2 in bits 61-63, version 1 in
// bits 46-47; addresses and offsets in units of 16 bytes).
// Contraction along the rows of the stage (K-major): 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_kmajor(uint32_t addr) {
  return uint64_t((addr & 0x3FFFF) >> 4) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
         (uint64_t(2) << 61);
}
// Contraction down the columns (MN-major): blocks of 64 columns lie kBK * 128 bytes apart (leading
// offset), groups of 8 contraction rows 1024 bytes apart (stride offset).
__device__ __forceinline__ uint64_t desc_mnmajor(uint32_t addr) {
  return uint64_t((addr & 0x3FFFF) >> 4) | (uint64_t((kBK * 128) >> 4) << 16) | (uint64_t(1024 >> 4) << 32) |
         (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

template <typename T>
struct Num;
template <>
struct Num<__nv_bfloat16> {
  static constexpr uint32_t kCode = 1;  // operand format of the instruction descriptor
  static __device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
  static __device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Num<__half> {
  static constexpr uint32_t kCode = 0;
  static __device__ __forceinline__ float lo(uint32_t w) { return __half2float(__ushort_as_half(uint16_t(w))); }
  static __device__ __forceinline__ float hi(uint32_t w) { return __half2float(__ushort_as_half(uint16_t(w >> 16))); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};

// A tile of CG CTAs: 128 CG x 128 CG.
template <int CG>
struct GemmCfg {
  static constexpr int kBN = 128 * CG;
  static constexpr int kOperand = 128 * kBK * 2;  // bytes of A, and of B, that a CTA holds per stage
  static constexpr int kStageBytes = 2 * kOperand;
  static constexpr int kStages = 6;
  static constexpr int kWarpBuf = 4096;  // per epilogue warp, to turn rows into whole sectors
  static constexpr int kSmem = kStages * kStageBytes + kEpiWarps * kWarpBuf + 1024;  // + alignment of the first stage
};

// Instruction descriptor: f32 accumulator, 16-bit operands of one type, B's major-ness, N and M.
template <typename T, int CG, bool BMN>
__device__ constexpr uint32_t instr_desc() {
  return (1u << 4) | (Num<T>::kCode << 7) | (Num<T>::kCode << 10) | (uint32_t(BMN) << 16) |
         (uint32_t(GemmCfg<CG>::kBN / 8) << 17) | (uint32_t(kBM * CG / 16) << 24);
}

// acc[m][n] (32 bits) = the tile, or acc[m][n] * scale[m] + the tile: what a product over one piece of a
// contraction adds to the pieces before, or a part of a tile's contraction.  A thread's 128 bytes per 32 columns go through
// the staging buffer, so that the warp reads and writes 4 rows of whole 128-byte lines at a time.
struct EpiAccum {
  static constexpr bool kParts = true;
  float* acc;
  int64_t M, N, ld;  // ld: a multiple of 4
  bool add;
  const float* scale;  // with add, or null: 1
  struct Row {
    int64_t m, n0;
    uint8_t* buf;
    __device__ __forceinline__ Row(const EpiAccum&, int64_t m_, int64_t n0_, int, uint8_t* b) : m(m_), n0(n0_), buf(b) {}
    __device__ __forceinline__ float4* at(int row, int chunk) const {
      return reinterpret_cast<float4*>(buf + row * 128 + ((chunk ^ (row & 7)) << 4));
    }
    __device__ __forceinline__ void cols(const EpiAccum& e, int c, const float* v) {
      const int lane = threadIdx.x & 31;
      if (n0 + c >= e.N) return;
#pragma unroll
      for (int g = 0; g < 8; ++g) *at(lane, g) = make_float4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
      __syncwarp();
      const int64_t n = n0 + c + 4 * (lane & 7), m0 = m - lane;
      float4 s[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + (lane >> 3);
        s[i] = *at(r, lane & 7);
        if (e.add && m0 + r < e.M && n < e.N) {
          const float4 o = *reinterpret_cast<const float4*>(e.acc + (m0 + r) * e.ld + n);
          const float f = e.scale ? e.scale[m0 + r] : 1.0f;
          s[i] = make_float4(fmaf(o.x, f, s[i].x), fmaf(o.y, f, s[i].y), fmaf(o.z, f, s[i].z), fmaf(o.w, f, s[i].w));
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + (lane >> 3);
        if (m0 + r < e.M && n < e.N) *reinterpret_cast<float4*>(e.acc + (m0 + r) * e.ld + n) = s[i];
      }
      __syncwarp();
    }
    __device__ __forceinline__ void end(const EpiAccum&) {}
  };
};

// Epilogue interface.  Epi::kParts: tiles may be computed in parts (else GemmShape::rest is 0), whose
// sums another kernel hands to the epilogue.  Epi::Row row(epi, m, n0, width, buf) at the start of a thread's half row (the
// warp holds rows m - lane .. m - lane + 31; m may be past the last row: nothing may be accessed
// then), row.cols(epi, c, v) for each 32 columns n0 + c .. n0 + c + 31, by whole warps, row.end(epi)
// after the last.  buf: kWarpBuf bytes of the warp's own shared memory.
template <typename T, int CG, bool BMN, class Epi>
__global__ void __launch_bounds__(kGemmThreads, 1)
gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
            const __grid_constant__ GemmShape g, const __grid_constant__ Epi epi) {
  using Cfg = GemmCfg<CG>;
  constexpr int kStages = Cfg::kStages, BN = Cfg::kBN;
  constexpr uint32_t kIdesc = instr_desc<T, CG, BMN>();
  extern __shared__ uint8_t smem_dyn[];
  __shared__ __align__(8) uint64_t bars[2 * kStages + 5];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  const uint32_t stage0 = (smem_addr(smem_dyn) + 1023) & ~1023u;
  const uint32_t full0 = smem_addr(bars), empty0 = full0 + 8 * kStages;
  const uint32_t accfull0 = empty0 + 8 * kStages, accempty0 = accfull0 + 16, drain = accempty0 + 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cta_rank() : 0;
  if (g.go) {  // the same value for every CTA: the kernel before wrote it
    pdl_wait();
    if (*reinterpret_cast<const volatile int32_t*>(g.go) == 0) return;
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full0 + 8 * i, 1);
      mbar_init(empty0 + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(accfull0 + 8 * i, 1);
      mbar_init(accempty0 + 8 * i, kEpiWarps * CG);  // one arrival per epilogue warp
    }
    mbar_init(drain, 1);
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 2) tmem_alloc<CG, 2 * BN>(smem_addr(&s_tmem));  // both accumulators
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) group_sync<2>();
  tc_fence_after();
  pdl_wait();
  const uint32_t tmem = s_tmem;
  volatile int* abort_flag = &s_abort;

  const int64_t first = blockIdx.x / CG, step = gridDim.x / CG;
  // The n-th tile (or part of a tile, its place in `parts` in `part`) of this CTA or pair.  With parts,
  // `full` is a multiple of the grid, and every CTA has at most one part, after its whole tiles.
  auto item = [&](int64_t n, int& tm, int& tn, int& kb0, int& kb1, int& part) {
    const int64_t t = first + n * step;
    if (t < g.full) {
      tile_place(g, t, tm, tn);
      kb0 = 0;
      kb1 = g.kblocks;
      part = -1;
      return true;
    }
    if (t - g.full >= int64_t(g.rest) * g.splits) return false;
    part = int(t - g.full);
    const int ks = part % g.splits;
    tile_place(g, g.full + part / g.splits, tm, tn);
    kb0 = int(int64_t(g.kblocks) * ks / g.splits);
    kb1 = int(int64_t(g.kblocks) * (ks + 1) / g.splits);
    return true;
  };

  if (warp == 0) {
    if (lane == 0) {
      int64_t it = 0;  // blocks loaded
      bool ok = true;
      int tm, tn, kb0, kb1, part;
      for (int64_t n = 0; ok && item(n, tm, tn, kb0, kb1, part); ++n) {
        const int ya = (tm * CG + int(rank)) * kBM, yb = tn * BN + int(rank) * 128;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = int(it % kStages);
          if (it >= kStages && !mbar_wait(empty0 + 8 * s, uint32_t((it / kStages - 1) & 1), abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t a = stage0 + s * Cfg::kStageBytes, b = a + Cfg::kOperand;
          // The first CTA's barrier counts the bytes of both.
          if (rank == 0) mbar_expect(full0 + 8 * s, CG * Cfg::kStageBytes);
          const uint32_t bar = CG == 2 ? in_leader(full0 + 8 * s) : full0 + 8 * s;
          tma_load<CG>(a, &map_a, kb * kBK, ya, bar);
          if constexpr (!BMN) {
            tma_load<CG>(b, &map_b, kb * kBK, yb, bar);
          } else {
            tma_load<CG>(b, &map_b, yb, kb * kBK, bar);
            tma_load<CG>(b + kBK * 128, &map_b, yb + 64, kb * kBK, bar);
          }
        }
      }
      // Leave only once every load has landed and every stage was released (no barrier of this
      // CTA is touched after it ends); after an abort only the loads are waited for.
      for (int64_t j = it > kStages ? it - kStages : 0; j < it; ++j) {
        const int s = int(j % kStages);
        if (ok) ok = mbar_wait(empty0 + 8 * s, uint32_t((j / kStages) & 1), abort_flag);
        if (!ok && rank == 0)
          for (uint32_t i = 0; i < kWaitLimit && !mbar_try(full0 + 8 * s, uint32_t((j / kStages) & 1)); ++i) {}
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      int64_t it = 0;  // blocks consumed
      bool ok = true;
      int tm, tn, kb0, kb1, part;
      for (int64_t n = 0; ok && item(n, tm, tn, kb0, kb1, part); ++n) {
        const int acc = int(n & 1);
        if (n >= 2 && !mbar_wait(accempty0 + 8 * acc, uint32_t((n / 2 - 1) & 1), abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + acc * BN;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = int(it % kStages);
          if (!mbar_wait(full0 + 8 * s, uint32_t((it / kStages) & 1), abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a = stage0 + s * Cfg::kStageBytes, b = a + Cfg::kOperand;
          const uint64_t da = desc_kmajor(a), db = BMN ? desc_mnmajor(b) : desc_kmajor(b);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k)
            tc_mma<CG>(d, da + uint64_t(k * 2), db + uint64_t(BMN ? k * (2048 >> 4) : k * 2), kIdesc,
                       uint32_t(kb > kb0 || k > 0));
          tc_commit<CG>(empty0 + 8 * s);
        }
        if (ok) tc_commit<CG>(accfull0 + 8 * acc);
      }
      if (!ok) {  // MMAs in flight end before the tensor memory is freed
        tc_commit<CG>(drain);
        for (uint32_t i = 0; i < kWaitLimit && !mbar_try(drain, 0); ++i) {}
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    constexpr int kHalf = BN / 2;
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    uint8_t* buf = smem_dyn + (stage0 - smem_addr(smem_dyn)) + kStages * Cfg::kStageBytes + (warp - 4) * Cfg::kWarpBuf;
    int tm, tn, kb0, kb1, part;
    for (int64_t n = 0; item(n, tm, tn, kb0, kb1, part); ++n) {
      const int acc = int(n & 1);
      const bool ok = mbar_wait(accfull0 + 8 * acc, uint32_t((n / 2) & 1), abort_flag);
      if (!__all_sync(0xFFFFFFFFu, ok)) break;
      tc_fence_after();
      const uint32_t src = tmem + (uint32_t(quarter * 32) << 16) + acc * BN + half * kHalf;
      // The accumulator's columns through `row`; it is handed back before the last ones' work.
      auto drain_tile = [&](auto& row, const auto& e) {
#pragma unroll 1
        for (int c = 0; c < kHalf; c += 32) {
          float v[32];
          tc_load32(src + c, v);
          tc_wait_load();
          if (c + 32 >= kHalf) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if constexpr (CG == 2) mbar_arrive_cluster(in_leader(accempty0 + 8 * acc));
              else mbar_arrive(accempty0 + 8 * acc);
            }
          }
          row.cols(e, c, v);
        }
        row.end(e);
      };
      const int64_t m = rank * kBM + quarter * 32 + lane, c0 = half * kHalf;  // in the tile
      if constexpr (Epi::kParts) {
        if (part >= 0) {
          const EpiAccum e{g.parts + int64_t(part) * (CG * kBM * BN), CG * kBM, BN, BN, false, nullptr};
          EpiAccum::Row row(e, m, c0, kHalf, buf);
          drain_tile(row, e);
          continue;
        }
      }
      typename Epi::Row row(epi, int64_t(tm) * CG * kBM + m, int64_t(tn) * BN + c0, kHalf, buf);
      drain_tile(row, epi);
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) group_sync<2>();
  tc_fence_after();
  if (warp == 2) tmem_free<CG, 2 * BN>(tmem);
  if (threadIdx.x == 0 && s_abort) atomicOr(g.status, kErrWait);
}

// ---- host side ------------------------------------------------------------------------------

// A tensor map over a row-major [rows, cols] matrix of 16-bit elements (pitch in elements, a
// multiple of 8; 16-byte aligned base), loaded in boxes of box_rows x 64 columns.
int make_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t pitch, int box_rows, bool bf16);
int sm_count(int* sms);

// How a product [M, K] x [N, K] is cut: tiles of 256 x 256 by pairs of CTAs or of 128 x 128 by single
// ones, and whether the tiles of the last, incomplete wave are computed in parts of the contraction.
struct Cut {
  int cg;
  int64_t full;
  int rest, splits;
};
// The cheaper of the possible cuts by these figures, measured on products of a thousand and more
// blocks: 0.43 us per 64-wide block of a pair's tile (4096 x 18944 x 3584: 1400 TFLOP/s), 0.29 us of a
// single CTA's (301 x 1280 x 51866), 6 us for the kernel that adds the parts.  Parts are at least 8
// blocks long.
inline Cut cut_of(int64_t M, int64_t N, int64_t K, int sms, bool parts) {
  Cut best{1, 0, 0, 1};
  double least = 0;
  const int64_t kb = cdiv(K, kBK);
  for (int cg = 1; cg <= 2; ++cg) {
    const int64_t workers = sms / cg, tiles = cdiv(M, 128 * cg) * cdiv(N, 128 * cg);
    const double block = cg == 1 ? 0.29 : 0.43;
    auto take = [&](const Cut& c, double us) {
      if (least == 0 || us < least) {
        best = c;
        least = us;
      }
    };
    take({cg, tiles, 0, 1}, double(cdiv(tiles, workers)) * double(kb) * block);
    const int64_t rest = tiles % workers;
    const int64_t splits = rest ? (workers / rest < kb / 8 ? workers / rest : kb / 8) : 0;
    if (parts && splits >= 2)
      take({cg, tiles - rest, int(rest), int(splits)},
           (double(tiles / workers) * double(kb) + double(cdiv(kb, splits))) * block + 6.0);
  }
  return best;
}
// Whole tiles only, of a given kind (every piece of a weight cut alike).
inline Cut whole_cut(int cg, int64_t M, int64_t N) { return {cg, cdiv(M, 128 * cg) * cdiv(N, 128 * cg), 0, 1}; }
// Bytes of GemmShape::parts that any cut needs: a tile per CTA or pair.
inline size_t parts_bytes(int sms) { return size_t(sms) * (2 * kBM * kBM) * sizeof(float); }

inline GemmShape gemm_shape(int64_t M, int64_t N, int64_t K, const Cut& cut, float* parts, int32_t* status,
                            const int32_t* go = nullptr) {
  GemmShape g{};
  g.M = M;
  g.N = N;
  g.K = K;
  g.tiles_m = int(cdiv(M, kBM * cut.cg));
  g.tiles_n = int(cdiv(N, 128 * cut.cg));
  g.kblocks = int(cdiv(K, kBK));
  g.group_m = 32 / cut.cg;
  g.full = cut.full;
  g.rest = cut.rest;
  g.splits = cut.splits;
  g.parts = parts;
  g.status = status;
  g.go = go;
  return g;
}

template <typename T, int CG, bool BMN, class Epi>
int launch_gemm(const CUtensorMap& a, const CUtensorMap& b, const GemmShape& g, const Epi& epi, cudaStream_t s) {
  auto fn = gemm_kernel<T, CG, BMN, Epi>;
  if (int rc = set_max_smem(reinterpret_cast<const void*>(fn), GemmCfg<CG>::kSmem)) return rc;
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  // With parts, the grid is all workers (`full` is a multiple of it, or 0).
  const int64_t total = g.rest && g.full ? sms / CG : g.full + int64_t(g.rest) * g.splits;
  if (total <= 0) return ZN_OK;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(CG * (total < sms / CG ? total : sms / CG)));
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = GemmCfg<CG>::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CG > 1 ? 2 : 1;
  TimedLaunch tl("gemm", s);
  cudaLaunchKernelEx(&cfg, fn, a, b, g, epi);
  count_launch();
  return check_launch("gemm_kernel");
}

}  // namespace zn
