// Weights as operands (zn_weight.cuh): ranges of a blob's chunks decoded into a buffer, or multiplied
// with a few vectors inside the decoder.
#include "zn_decode.cuh"

namespace zn {
namespace {

// ---- a weight's chunks (zn_weight.cuh) -------------------------------------------------------

// Chunks [c0, c0 + gridDim.x) of one weight.
template <bool REORDER, class Sink>
__global__ void __launch_bounds__(kDecThreads) weight_kernel(const __grid_constant__ DecArgs a, int64_t c0,
                                                             const __grid_constant__ Sink sink) {
  decode_chunk<2, REORDER, 1>(a, c0 + blockIdx.x, false, sink);
}

// The chunks of [c0, c1) with both planes coded.  Their flags were set by weight_kernel.
template <bool REORDER, class Sink>
__global__ void __launch_bounds__(kDecThreads) weight_overflow_kernel(const __grid_constant__ DecArgs a, int64_t c0,
                                                                      int64_t c1, const __grid_constant__ Sink sink) {
  __shared__ int64_t flagged[kDecThreads];
  __shared__ int nflagged;
  const int64_t stride = gridDim.x;
  for (int64_t first = c0 + blockIdx.x; first < c1; first += stride * kDecThreads) {
    const int64_t c = first + stride * threadIdx.x;
    if (threadIdx.x == 0) nflagged = 0;
    __syncthreads();
    if (c < c1 && a.overflow[c]) flagged[atomicAdd(&nflagged, 1)] = c;
    __syncthreads();
    const int nf = nflagged;
    for (int q = 0; q < nf; ++q) {
      decode_chunk<2, REORDER, 2>(a, flagged[q], true, sink);
      __syncthreads();
    }
    __syncthreads();
  }
}

template <class Sink>
constexpr size_t sink_smem() {
  if constexpr (Sink::kDot) return 64 * 2 * Sink::kRows * sizeof(float);
  else return 0;
}

template <bool REORDER, class Sink>
int launch_weight(const DecArgs& a, int64_t c0, int64_t c1, const Sink& sink, cudaStream_t s) {
  if (c1 <= c0) return ZN_OK;
  {
    auto fn = weight_kernel<REORDER, Sink>;
    const size_t sm = dec_smem(1) + sink_smem<Sink>();
    if (int rc = set_max_smem(reinterpret_cast<const void*>(fn), int(sm))) return rc;
    TimedLaunch tl("decode", s);
    fn<<<unsigned(c1 - c0), kDecThreads, sm, s>>>(a, c0, sink);
  }
  count_launch();
  if (int rc = check_launch("weight_kernel")) return rc;
  auto fn = weight_overflow_kernel<REORDER, Sink>;
  const size_t sm = dec_smem(2) + sink_smem<Sink>();
  if (int rc = set_max_smem(reinterpret_cast<const void*>(fn), int(sm))) return rc;
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return set_error(ZN_ERR_CUDA, "weight_overflow_kernel: %s", cudaGetErrorString(e));
  TimedLaunch tl("decode_overflow", s);
  fn<<<unsigned(min(c1 - c0, int64_t(2 * sms))), kDecThreads, sm, s>>>(a, c0, c1, sink);
  count_launch();
  return check_launch("weight_overflow_kernel");
}

template <typename T, bool REORDER>
int launch_dot(const DecArgs& a, const WeightBlob& w, const void* x, int64_t ldx, int tokens, float* z, float* part,
               cudaStream_t s) {
  auto go = [&](auto mt) {
    constexpr int MT = decltype(mt)::value;
    DotSink<T, MT> k{static_cast<const T*>(x), ldx, w.cols, w.rows, tokens, z, part};
    return launch_weight<REORDER>(a, 0, a.nch, k, s);
  };
  if (tokens == 1) return go(std::integral_constant<int, 1>());
  if (tokens == 2) return go(std::integral_constant<int, 2>());
  if (tokens <= 4) return go(std::integral_constant<int, 4>());
  return go(std::integral_constant<int, kDotRows>());
}

}  // namespace

size_t weight_temp_bytes(const WeightBlob& w) {
  return job_structs_bytes<DecArgs>(1) + dec_job_bytes(w.rows * w.cols, 2, w.chunk);
}

int weight_decode(const WeightBlob& w, void* temp, int64_t c0, int64_t c1, void* out, int32_t* status, cudaStream_t s) {
  DecArgs a = weight_args(w, temp, status);
  a.out = static_cast<uint8_t*>(out) - c0 * w.chunk * 2;
  return w.bf16 ? launch_weight<true>(a, c0, c1, StoreSink(), s) : launch_weight<false>(a, c0, c1, StoreSink(), s);
}

int weight_wave(const WeightBlob& w, int64_t* chunks) {
  int dev = 0, sms = 0, per_sm = 0;
  const void* fn = w.bf16 ? reinterpret_cast<const void*>(weight_kernel<true, StoreSink>)
                          : reinterpret_cast<const void*>(weight_kernel<false, StoreSink>);
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, fn, kDecThreads, dec_smem(1));
  if (e != cudaSuccess) return set_error(ZN_ERR_CUDA, "weight_kernel occupancy: %s", cudaGetErrorString(e));
  *chunks = int64_t(sms) * max(1, per_sm);
  return ZN_OK;
}

size_t dot_part_bytes(const WeightBlob& w) { return size_t(weight_chunks(w)) * 2 * kDotRows * sizeof(float); }

int weight_dot(const WeightBlob& w, void* temp, const void* x, int64_t ldx, int tokens, float* z, float* part,
               int32_t* status, cudaStream_t s) {
  const DecArgs a = weight_args(w, temp, status);
  return w.bf16 ? launch_dot<__nv_bfloat16, true>(a, w, x, ldx, tokens, z, part, s)
                : launch_dot<__half, false>(a, w, x, ldx, tokens, z, part, s);
}

}  // namespace zn
