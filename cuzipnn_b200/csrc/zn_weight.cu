// Weights as operands (zn_weight.cuh): ranges of a blob's chunks decoded into a buffer, or multiplied
// with a vector inside the decoder.
#include "zn_decode.cuh"
#include "zn_linear.cuh"

namespace zn {
namespace {

// ---- a weight's chunks (zn_weight.cuh) -------------------------------------------------------

// CTAs per SM that the registers have to allow.  With 6 (80 registers, and less shared memory for L1's
// share of the streams) a single wave of chunks took 5 to 40 % longer.
constexpr int kWeightBlocks = 5;

// Chunks [c0, c0 + gridDim.x) of one weight.
template <bool REORDER, class Sink>
__global__ void __launch_bounds__(kDecThreads, kWeightBlocks) weight_kernel(const __grid_constant__ DecArgs a, int64_t c0,
                                                             const __grid_constant__ Sink sink, uint32_t* counter) {
  pdl_wait();
  pdl_trigger();
  if (blockIdx.x == 0 && threadIdx.x == 0) *counter = 0;
  decode_chunk<2, REORDER, 1, true>(a, c0 + blockIdx.x, false, sink);
}

// What the tail does once the weight's chunks are done (elements split over `n` threads).
struct NoFin {
  __device__ __forceinline__ void run(int64_t, int64_t) const {}
};
struct PitchFin {
  PitchCopy copy[2];
  __device__ __forceinline__ void run(int64_t i, int64_t n) const {
    pitch_rows(copy[0], i / 32, n / 32);
    pitch_rows(copy[1], i / 32, n / 32);
  }
};
template <typename T>
struct LinearFin {
  Finish<T> f;
  __device__ __forceinline__ void run(int64_t i, int64_t n) const {
    for (; i < f.M * f.N; i += n) finish_element(f, i);
  }
};

// After weight_kernel: the status from the chunks' flags, the chunks with both planes coded (whose
// flags weight_kernel set), and `fin`.  Usually no chunk is left: every CTA sees that from the flags
// and does its share of `fin` at once.  Otherwise the CTAs decode the flagged chunks, and the last
// one to finish does all of `fin`.
template <bool REORDER, class Sink, class Fin>
__global__ void __launch_bounds__(kDecThreads) weight_tail_kernel(const __grid_constant__ DecArgs a, int64_t c0,
                                                                  int64_t c1, const __grid_constant__ Sink sink,
                                                                  const __grid_constant__ Fin fin, uint32_t* counter) {
  __shared__ uint32_t s_any[kDecThreads / 32];
  __shared__ uint32_t s_last;
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x;
  auto all_flags = [&] {  // OR of the chunks' flags, on every thread
    uint32_t any = 0;
    // Whole words in the middle (the array starts on an 8-byte boundary), bytes at the ends.
    const int64_t w0 = (c0 + 3) / 4, w1 = c1 / 4;
    const volatile uint32_t* words = reinterpret_cast<const volatile uint32_t*>(a.overflow);
    const volatile uint8_t* bytes = a.overflow;
#pragma unroll 4
    for (int64_t i = w0 + tid; i < w1; i += kDecThreads) any |= words[i];
    any |= any >> 16;
    any |= any >> 8;
    if (w0 <= w1) {
      if (c0 + tid < 4 * w0) any |= bytes[c0 + tid];
      if (4 * w1 + tid < c1) any |= bytes[4 * w1 + tid];
    } else if (c0 + tid < c1) {
      any |= bytes[c0 + tid];
    }
    any = __reduce_or_sync(0xFFFFFFFFu, any & 0xFF);
    __syncthreads();
    if ((tid & 31) == 0) s_any[tid >> 5] = any;
    __syncthreads();
    any = 0;
#pragma unroll
    for (int w = 0; w < kDecThreads / 32; ++w) any |= s_any[w];
    return any;
  };
  const uint32_t any = all_flags();
  auto report = [&](uint32_t flags) {
    if (tid == 0) *a.status = (a.mode == kDirect ? 0 : *a.status) | int32_t(flags & ~uint32_t(kChunkOver));
  };
  if (!(any & kChunkOver)) {
    if (blockIdx.x == 0) report(any);
    fin.run(int64_t(blockIdx.x) * kDecThreads + tid, int64_t(gridDim.x) * kDecThreads);
    return;
  }
  for (int64_t c = c0 + blockIdx.x; c < c1; c += gridDim.x) {
    if (!(a.overflow[c] & kChunkOver)) continue;  // uniform: this CTA alone changes the flag's other bits
    __syncthreads();
    decode_chunk<2, REORDER, 2, true>(a, c, true, sink);
    __syncthreads();
  }
  __threadfence();
  __syncthreads();
  if (tid == 0) s_last = atomicAdd(counter, 1) == gridDim.x - 1;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  report(all_flags());
  fin.run(tid, kDecThreads);
}

template <class Sink>
constexpr size_t sink_smem() {
  if constexpr (Sink::kDot) return 64 * 2 * sizeof(float);
  else return 0;
}

// `work`: elements of `fin`.
template <bool REORDER, class Sink, class Fin>
int launch_weight(const DecArgs& a, int64_t c0, int64_t c1, const Sink& sink, const Fin& fin, int64_t work,
                  cudaStream_t s) {
  if (c1 <= c0) return ZN_OK;
  uint32_t* counter = reinterpret_cast<uint32_t*>(a.overflow + ((a.nch + 3) & ~int64_t(3)));
  {
    auto fn = weight_kernel<REORDER, Sink>;
    const size_t sm = dec_smem(1) + sink_smem<Sink>();
    if (int rc = set_max_smem(reinterpret_cast<const void*>(fn), int(sm))) return rc;
    TimedLaunch tl("decode", s);
    if (int rc = launch_after(fn, dim3(unsigned(c1 - c0)), kDecThreads, sm, s, "weight_kernel", a, c0, sink, counter))
      return rc;
  }
  auto fn = weight_tail_kernel<REORDER, Sink, Fin>;
  const size_t sm = dec_smem(2) + sink_smem<Sink>();
  if (int rc = set_max_smem(reinterpret_cast<const void*>(fn), int(sm))) return rc;
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  const int64_t grid = min(max(c1 - c0, cdiv(work, kDecThreads)), int64_t(2 * sms));
  TimedLaunch tl("decode_overflow", s);
  return launch_after(fn, dim3(unsigned(grid)), kDecThreads, sm, s, "weight_tail_kernel", a, c0, c1, sink, fin, counter);
}

template <typename T, bool REORDER, class Fin>
int launch_dot(const DecArgs& a, const WeightBlob& w, const void* x, float* z, float* part, const Fin& fin, int64_t work,
               cudaStream_t s) {
  const DotSink<T> k{static_cast<const T*>(x), int(w.cols), z, part};
  return launch_weight<REORDER>(a, 0, a.nch, k, fin, work, s);
}

}  // namespace

size_t weight_temp_bytes(const WeightBlob& w) {
  return job_structs_bytes<DecArgs>(1) + dec_job_bytes(w.rows * w.cols, 2, w.chunk) + 256;  // + the counter
}

int weight_decode(const WeightBlob& w, void* temp, int64_t c0, int64_t c1, void* out, const PitchCopy& copy0,
                  const PitchCopy& copy1, int32_t* status, cudaStream_t s) {
  DecArgs a = weight_args(w, temp, status, w.direct ? kDirect : kScanned);
  a.out = static_cast<uint8_t*>(out) - c0 * w.chunk * 2;
  const PitchFin fin{{copy0, copy1}};
  const int64_t work = (copy0.rows * copy0.cols + copy1.rows * copy1.cols) / 8;
  return w.bf16 ? launch_weight<true>(a, c0, c1, StoreSink(), fin, work, s)
                : launch_weight<false>(a, c0, c1, StoreSink(), fin, work, s);
}

int weight_wave(const WeightBlob& w, int64_t* chunks) {
  // The register bound of weight_kernel; a query of the occupancy costs a microsecond of every call.
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  *chunks = int64_t(sms) * kWeightBlocks;
  return ZN_OK;
}

size_t dot_part_bytes(const WeightBlob& w) { return size_t(weight_chunks(w)) * 2 * sizeof(float); }

int weight_dot(const WeightBlob& w, void* temp, const void* x, float* z, float* part, int32_t* status, cudaStream_t s) {
  const DecArgs a = weight_args(w, temp, status, w.direct ? kDirect : kScanned);
  return w.bf16 ? launch_dot<__nv_bfloat16, true>(a, w, x, z, part, NoFin(), 0, s)
                : launch_dot<__half, false>(a, w, x, z, part, NoFin(), 0, s);
}

template <typename T>
int weight_linear(const WeightBlob& w, void* temp, const void* x, float* z, float* part, const Finish<T>& f,
                  int32_t* status, cudaStream_t s) {
  const DecArgs a = weight_args(w, temp, status, w.direct ? kDirect : kScanned);
  LinearFin<T> fin{f};
  fin.f.dot = {z, part, w.rows, w.cols, w.chunk};
  return launch_dot<T, Num<T>::kCode == 1>(a, w, x, z, part, fin, f.N, s);
}
template int weight_linear<__nv_bfloat16>(const WeightBlob&, void*, const void*, float*, float*,
                                          const Finish<__nv_bfloat16>&, int32_t*, cudaStream_t);
template int weight_linear<__half>(const WeightBlob&, void*, const void*, float*, float*, const Finish<__half>&, int32_t*,
                                   cudaStream_t);

}  // namespace zn
