// Matrix products of 16-bit matrices on the fifth-generation tensor cores (sm_100a), with the
// epilogue as a template argument: D[m, n] = sum_k A[m, k] * B(n, k), accumulated in 32 bits.
//
// A is row-major [M, K].  B is either row-major [N, K] (BMN = false: the contraction runs along its
// rows, as in x W^T) or row-major [K, N] (BMN = true: the contraction runs down its columns, as in
// dz W), so a decoded weight serves both directions as it lies in memory.
//
// One persistent CTA per SM takes output tiles of 128 x BN in turn.  Warp 0 loads 64-wide blocks of
// both operands with TMA (128-byte swizzle) into a ring of shared-memory stages, one thread of warp
// 1 issues tcgen05.mma into one of two accumulators in tensor memory, and warps 4-7 read the other
// accumulator (a thread owns a row of the tile) and run the epilogue meanwhile.
//
// Every wait has an iteration limit.  A wait that gives up sets kErrWait in the status word and the
// abort flag, upon which all warps leave their loops, the loads in flight are waited for (again
// with a limit) and the tensor memory is freed.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "zn_common.cuh"

namespace zn {

constexpr int32_t kErrWait = 16;  // a bounded wait inside a product kernel gave up

constexpr int kBM = 128;          // rows of a tile (tensor memory lanes)
constexpr int kBK = 64;           // contraction block: 128 bytes of a 16-bit type, one swizzle row
constexpr int kGemmThreads = 256;
constexpr uint32_t kWaitLimit = 1u << 24;  // polls of up to kPollNs each (about 4 s at most)
constexpr uint32_t kPollNs = 256;

struct GemmShape {
  int64_t M, N, K;
  int tiles_m, tiles_n;  // output tiles
  int splits;            // the contraction is cut into this many parts, one tile each
  int kblocks;           // 64-wide blocks of the whole contraction
  int group_m;           // row tiles that share a column tile before the next one is taken
  int32_t* status;
};

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
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
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

// Instruction descriptor: f32 accumulator, 16-bit operands of one type, B's major-ness, N and M.
template <typename T, int BN, bool BMN>
__device__ constexpr uint32_t instr_desc() {
  return (1u << 4) | (Num<T>::kCode << 7) | (Num<T>::kCode << 10) | (uint32_t(BMN) << 16) | (uint32_t(BN / 8) << 17) |
         (uint32_t(kBM / 16) << 24);
}

template <int BN>
struct GemmCfg {
  static constexpr int kStageBytes = (kBM + BN) * kBK * 2;
  static constexpr int kStages = 196608 / kStageBytes;
  static constexpr int kSmem = kStages * kStageBytes + 1024;  // + alignment of the first stage
};

// Epilogue interface: Epi::Row row(epi, m, n0, split) at the start of a thread's tile row (m may be
// past the last row: nothing may be accessed then), row.cols(epi, c, v) for each 32 columns
// n0 + c .. n0 + c + 31, row.end(epi) after the last.
template <typename T, int BN, bool BMN, class Epi>
__global__ void __launch_bounds__(kGemmThreads, 1)
gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
            const __grid_constant__ GemmShape g, const __grid_constant__ Epi epi) {
  using Cfg = GemmCfg<BN>;
  constexpr int kStages = Cfg::kStages;
  constexpr uint32_t kIdesc = instr_desc<T, BN, BMN>();
  extern __shared__ uint8_t smem_dyn[];
  __shared__ __align__(8) uint64_t bars[2 * kStages + 5];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  const uint32_t stage0 = (smem_addr(smem_dyn) + 1023) & ~1023u;
  const uint32_t full0 = smem_addr(bars), empty0 = full0 + 8 * kStages;
  const uint32_t accfull0 = empty0 + 8 * kStages, accempty0 = accfull0 + 16,
                 drain = accempty0 + 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full0 + 8 * i, 1);
      mbar_init(empty0 + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(accfull0 + 8 * i, 1);
      mbar_init(accempty0 + 8 * i, 128);
    }
    mbar_init(drain, 1);
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 2) {  // both accumulators: 2 * BN columns
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)),
                 "n"(2 * BN) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  volatile int* abort_flag = &s_abort;

  const int64_t total = int64_t(g.tiles_m) * g.tiles_n * g.splits;
  // Tile order: within a group of row tiles, the row tile runs fastest, then the column tile, so
  // that the CTAs of one wave share a few column blocks of B and a group's rows of A in L2.
  auto tile_of = [&](int64_t t, int& tm, int& tn, int& ks) {
    ks = int(t % g.splits);
    t /= g.splits;
    const int64_t per = int64_t(g.group_m) * g.tiles_n;
    const int grp = int(t / per);
    const int64_t r = t - grp * per;
    const int gm = min(g.group_m, g.tiles_m - grp * g.group_m);
    tm = grp * g.group_m + int(r % gm);
    tn = int(r / gm);
  };
  auto k_range = [&](int ks, int& kb0, int& kb1) {
    kb0 = int(int64_t(g.kblocks) * ks / g.splits);
    kb1 = int(int64_t(g.kblocks) * (ks + 1) / g.splits);
  };

  if (warp == 0) {
    if (lane == 0) {
      int64_t it = 0;  // blocks loaded
      bool ok = true;
      for (int64_t t = blockIdx.x; t < total && ok; t += gridDim.x) {
        int tm, tn, ks, kb0, kb1;
        tile_of(t, tm, tn, ks);
        k_range(ks, kb0, kb1);
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = int(it % kStages);
          if (it >= kStages && !mbar_wait(empty0 + 8 * s, uint32_t((it / kStages - 1) & 1), abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t a = stage0 + s * Cfg::kStageBytes, b = a + kBM * kBK * 2, bar = full0 + 8 * s;
          mbar_expect(bar, Cfg::kStageBytes);
          tma_load(a, &map_a, kb * kBK, tm * kBM, bar);
          if constexpr (!BMN) {
            tma_load(b, &map_b, kb * kBK, tn * BN, bar);
          } else {
#pragma unroll
            for (int i = 0; i < BN / 64; ++i)
              tma_load(b + i * (kBK * 128), &map_b, tn * BN + 64 * i, kb * kBK, bar);
          }
        }
      }
      // Leave only once every load has landed and every stage was released (no barrier of this
      // CTA is touched after it ends); after an abort only the loads are waited for.
      for (int64_t j = it > kStages ? it - kStages : 0; j < it; ++j) {
        const int s = int(j % kStages);
        if (ok) ok = mbar_wait(empty0 + 8 * s, uint32_t((j / kStages) & 1), abort_flag);
        if (!ok)
          for (uint32_t i = 0; i < kWaitLimit && !mbar_try(full0 + 8 * s, uint32_t((j / kStages) & 1)); ++i) {}
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      int64_t it = 0, n = 0;  // blocks consumed, tiles done
      bool ok = true;
      for (int64_t t = blockIdx.x; t < total && ok; t += gridDim.x, ++n) {
        int tm, tn, ks, kb0, kb1;
        tile_of(t, tm, tn, ks);
        k_range(ks, kb0, kb1);
        const int acc = int(n & 1);
        if (n >= 2 && !mbar_wait(accempty0 + 8 * acc, uint32_t((n / 2 - 1) & 1), abort_flag)) break;
        tc_fence_after();
        const uint32_t d = tmem + acc * BN;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = int(it % kStages);
          if (!mbar_wait(full0 + 8 * s, uint32_t((it / kStages) & 1), abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a = stage0 + s * Cfg::kStageBytes, b = a + kBM * kBK * 2;
          const uint64_t da = desc_kmajor(a), db = BMN ? desc_mnmajor(b) : desc_kmajor(b);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k)
            tc_mma(d, da + uint64_t(k * 2), db + uint64_t(BMN ? k * (2048 >> 4) : k * 2), kIdesc,
                   uint32_t(kb > kb0 || k > 0));
          tc_commit(empty0 + 8 * s);
        }
        if (ok) tc_commit(accfull0 + 8 * acc);
      }
      if (!ok || *abort_flag) {  // MMAs in flight end before the tensor memory is freed
        tc_commit(drain);
        for (uint32_t i = 0; i < kWaitLimit && !mbar_try(drain, 0); ++i) {}
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    const int quarter = warp & 3;
    int64_t n = 0;
    for (int64_t t = blockIdx.x; t < total; t += gridDim.x, ++n) {
      int tm, tn, ks;
      tile_of(t, tm, tn, ks);
      const int acc = int(n & 1);
      const bool ok = mbar_wait(accfull0 + 8 * acc, uint32_t((n / 2) & 1), abort_flag);
      if (!__all_sync(0xFFFFFFFFu, ok)) break;
      tc_fence_after();
      const uint32_t src = tmem + (uint32_t(quarter * 32) << 16) + acc * BN;
      typename Epi::Row row(epi, int64_t(tm) * kBM + quarter * 32 + lane, int64_t(tn) * BN, ks);
#pragma unroll 1
      for (int c = 0; c < BN; c += 32) {
        float v[32];
        tc_load32(src + c, v);
        tc_wait_load();
        if (c + 32 >= BN) {  // the accumulator is read: hand it back before the last columns' work
          tc_fence_before();
          mbar_arrive(accempty0 + 8 * acc);
        }
        row.cols(epi, c, v);
      }
      row.end(epi);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(2 * BN));
  if (threadIdx.x == 0 && s_abort) atomicOr(g.status, kErrWait);
}

// ---- host side ------------------------------------------------------------------------------

// A tensor map over a row-major [rows, cols] matrix of 16-bit elements (pitch in elements, a
// multiple of 8; 16-byte aligned base), loaded in boxes of box_rows x 64 columns.
int make_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t pitch, int box_rows, bool bf16);
int sm_count(int* sms);

inline GemmShape gemm_shape(int64_t M, int64_t N, int64_t K, int BN, int32_t* status) {
  GemmShape g{};
  g.M = M;
  g.N = N;
  g.K = K;
  g.tiles_m = int(cdiv(M, kBM));
  g.tiles_n = int(cdiv(N, BN));
  g.kblocks = int(cdiv(K, kBK));
  g.splits = 1;
  g.group_m = 32;
  g.status = status;
  return g;
}

template <typename T, int BN, bool BMN, class Epi>
int launch_gemm(const CUtensorMap& a, const CUtensorMap& b, const GemmShape& g, const Epi& epi, cudaStream_t s) {
  auto fn = gemm_kernel<T, BN, BMN, Epi>;
  if (int rc = set_max_smem(reinterpret_cast<const void*>(fn), GemmCfg<BN>::kSmem)) return rc;
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  const int64_t total = int64_t(g.tiles_m) * g.tiles_n * g.splits;
  if (total <= 0) return ZN_OK;
  TimedLaunch tl("gemm", s);
  fn<<<unsigned(total < sms ? total : sms), kGemmThreads, GemmCfg<BN>::kSmem, s>>>(a, b, g, epi);
  count_launch();
  return check_launch("gemm_kernel");
}

}  // namespace zn
