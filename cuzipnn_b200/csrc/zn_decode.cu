// Decompression: the fused whole-tensor path (zn_decompress) and the batched ANS seam
// (zn_ans_decompress).
//
// zn_decompress replaces src/cuzipnn/_codec.py:471-530 (table upload, cumsum, nvCOMP ANS decode
// into a planar buffer, then the Triton merge) with two kernels:
//   1. dscan_kernel: one CTA turns the blob's stored_bytes and comp_idx tables into the blob
//      offset of every (plane, chunk) unit, flags the rANS-coded ones and validates the tables.
//   2. decode_kernel: one CTA per chunk.  It builds a 4096-entry decode table in shared memory for
//      each coded plane, then each warp decodes 4 sub-chunks (8 lanes each, one shared word stream
//      per sub-chunk), reads the raw planes of the same elements straight from the blob, merges
//      the planes, reverts the exponent bit reorder and writes the elements.  There is no planar
//      intermediate buffer.
// Every blob access is bounds-checked; a malformed unit raises a bit in the status word and its
// elements are zeroed.  No wait in these kernels depends on another thread's progress except
// __syncthreads().
#include <vector>

#include "zn_decode.cuh"

namespace zn {
namespace {

// Main pass: one CTA per chunk.
template <int K, bool REORDER, int KC>
__global__ void __launch_bounds__(kDecThreads) decode_kernel(const DecArgs* __restrict__ jobs, int njobs) {
  const DecArgs& a = jobs[find_job(jobs, njobs, int64_t(blockIdx.x))];
  decode_chunk<K, REORDER, KC>(a, blockIdx.x - a.chunk0, false, StoreSink());
}

// Overflow pass: a grid of resident CTAs scans the per-chunk flags, kDecThreads chunks a round at a
// stride of the grid (flagged chunks that cluster in one tensor spread over the CTAs), and decodes
// the flagged ones one after another.
template <int K, bool REORDER, int KC>
__global__ void __launch_bounds__(kDecThreads) decode_overflow_kernel(const DecArgs* __restrict__ jobs, int njobs,
                                                                      int64_t total_chunks) {
  __shared__ int64_t flagged[kDecThreads];
  __shared__ int nflagged;
  const int64_t stride = gridDim.x;
  for (int64_t first = blockIdx.x; first < total_chunks; first += stride * kDecThreads) {
    const int64_t c = first + stride * threadIdx.x;
    bool f = false;
    if (c < total_chunks) {
      const DecArgs& a = jobs[find_job(jobs, njobs, c)];
      f = a.overflow[c - a.chunk0] != 0;
    }
    if (threadIdx.x == 0) nflagged = 0;
    __syncthreads();
    if (f) flagged[atomicAdd(&nflagged, 1)] = c;
    __syncthreads();
    const int nf = nflagged;
    for (int q = 0; q < nf; ++q) {
      const DecArgs& a = jobs[find_job(jobs, njobs, flagged[q])];
      decode_chunk<K, REORDER, KC>(a, flagged[q] - a.chunk0, true, StoreSink());
      __syncthreads();
    }
    __syncthreads();
  }
}

// ---- table scan (src/cuzipnn/_codec.py:492-496, 529) ----------------------------------------

constexpr int kScanThreads = 1024;

// One CTA per job.  It first zeroes the job's status word.  A job whose n_comp is negative reads
// it from the blob's header (u32 at byte 12) here; tables that do not fit the blob then mark every
// unit invalid (the decoder zero-fills them) and set kErrTable.
// The first kernel of a call: a single-job call passes its job by value (`one`), which CTA 0 also
// stores into the table at `table` for the kernels after this one.
__global__ void __launch_bounds__(kScanThreads) dscan_kernel(const DecArgs* __restrict__ jobs,
                                                             const __grid_constant__ FirstJob<DecArgs> one,
                                                             DecArgs* table) {
  __shared__ int64_t sm[64];
  __shared__ int64_t s_ncomp;
  if (one.valid && blockIdx.x == 0) store_job(one.job, table);
  const DecArgs& a = one.valid ? one.job : jobs[blockIdx.x];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  if (tid == 0) {
    *a.status = 0;
    int64_t nc = a.n_comp;
    if (nc < 0) nc = a.blob_bytes >= 16 ? int64_t(*reinterpret_cast<const uint32_t*>(a.blob + 12)) : -1;
    s_ncomp = nc;
  }
  __syncthreads();
  const int64_t n_comp = s_ncomp;
  const int64_t data_off = align8(a.idx_off + 4 * n_comp);
  if (n_comp < 0 || n_comp > a.units || data_off > a.blob_bytes) {
    for (int64_t i = tid; i < a.units; i += kScanThreads) a.src[i] = -1;
    if (tid == 0) atomicOr(a.status, kErrTable);
    return;
  }
  const int64_t last = a.n - (a.nch - 1) * a.C;
  const int32_t* stored = reinterpret_cast<const int32_t*>(a.blob + a.sizes_off);
  int64_t carry = data_off;
  bool bad = false;
  for (int64_t start = 0; start < a.units; start += kScanThreads) {
    const int64_t i = start + tid;
    int64_t v = 0;
    if (i < a.units) {
      const int64_t s = stored[i];
      bad |= s < 0;
      v = s < 0 ? 0 : align8(s);
    }
    int64_t incl = v;
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xFFFFFFFFu, incl, o);
      if (lane >= o) incl += u;
    }
    if (lane == 31) sm[w] = incl;
    __syncthreads();
    if (w == 0) {
      int64_t q = sm[lane];
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xFFFFFFFFu, q, o);
        if (lane >= o) q += u;
      }
      sm[32 + lane] = q;
    }
    __syncthreads();
    const int64_t excl = carry + (w ? sm[32 + w - 1] : 0) + incl - v;
    if (i < a.units) a.src[i] = excl;
    carry += sm[32 + 31];
    __syncthreads();
  }
  __syncthreads();
  const int32_t* idx = reinterpret_cast<const int32_t*>(a.blob + a.idx_off);
  for (int64_t q = tid; q < n_comp; q += kScanThreads) {
    const int64_t i = idx[q];
    if (i < 0 || i >= a.units) { bad = true; continue; }
    a.src[i] |= kCodedBit;
  }
  __syncthreads();
  for (int64_t i = tid; i < a.units; i += kScanThreads) {
    const int64_t s = a.src[i];
    const int64_t off = s & kOffMask, st = stored[i];
    const int64_t raw = (i % a.nch) == a.nch - 1 ? last : a.C;
    const bool coded = s & kCodedBit;
    // A raw unit holds exactly the chunk's bytes; a coded one must lie inside the blob.
    if (st < 0 || off + st > a.blob_bytes || (!coded && st != raw)) {
      a.src[i] = -1;
      bad = true;
    }
  }
  if (__syncthreads_or(bad) && tid == 0) atomicOr(a.status, kErrTable);
}


template <int K, bool REORDER, int KC, bool OVERFLOW>
int launch_decode_pass(const DecArgs* jobs, int njobs, int64_t total_chunks, cudaStream_t s) {
  const size_t sm = dec_smem(KC);
  if constexpr (!OVERFLOW) {
    auto fn = decode_kernel<K, REORDER, KC>;
    if (int rc = set_max_smem(reinterpret_cast<const void*>(fn), int(sm))) return rc;
    TimedLaunch tl("decode", s);
    fn<<<unsigned(total_chunks), kDecThreads, sm, s>>>(jobs, njobs);
  } else {
    auto fn = decode_overflow_kernel<K, REORDER, KC>;
    if (int rc = set_max_smem(reinterpret_cast<const void*>(fn), int(sm))) return rc;
    int dev = 0, sms = 0, per_sm = 0;  // the grid: the CTAs that fit on the device at once
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, fn, kDecThreads, sm);
    if (e != cudaSuccess) return set_error(ZN_ERR_CUDA, "decode_overflow_kernel occupancy: %s", cudaGetErrorString(e));
    const int64_t grid = min(total_chunks, int64_t(max(1, sms * per_sm)));
    TimedLaunch tl("decode_overflow", s);
    fn<<<unsigned(grid), kDecThreads, sm, s>>>(jobs, njobs, total_chunks);
  }
  count_launch();
  return check_launch("decode_kernel");
}

// Main pass with one coded plane per chunk in shared memory, then (K > 1) the overflow pass.
template <int K, bool REORDER>
int launch_decode(const DecArgs* jobs, int njobs, int64_t grid, cudaStream_t s) {
  if (grid <= 0) return ZN_OK;
  if (int rc = launch_decode_pass<K, REORDER, 1, false>(jobs, njobs, grid, s)) return rc;
  if constexpr (K > 1) return launch_decode_pass<K, REORDER, K, true>(jobs, njobs, grid, s);
  return ZN_OK;
}

}  // namespace

int weight_scan(const WeightBlob& w, void* temp, int32_t* status, cudaStream_t s) {
  const DecArgs a = weight_args(w, temp, status, kScanned);
  FirstJob<DecArgs> fj{};
  fj.job = a;
  fj.valid = 1;
  DecArgs* table = static_cast<DecArgs*>(temp);
  {
    TimedLaunch tl("dscan", s);
    dscan_kernel<<<1, kScanThreads, 0, s>>>(table, fj, table);
  }
  count_launch();
  return check_launch("dscan_kernel");
}

}  // namespace zn

using namespace zn;

extern "C" {

size_t zn_ans_decompress_temp_bytes(int64_t count) { return job_table_bytes<DecArgs>(1, count); }

int zn_ans_decompress(const int64_t* in_ptrs, const int64_t* in_bytes, const int64_t* out_capacity, int64_t count,
                      const int64_t* out_ptrs, int32_t* statuses, void* temp, size_t temp_bytes, void* stream) {
  if (count < 0 || count > 0x7FFFFFFF) return set_error(ZN_ERR_INVALID, "zn_ans_decompress: bad arguments");
  if (count == 0) return ZN_OK;
  if (!temp || temp_bytes < job_table_bytes<DecArgs>(1, count)) return set_error(ZN_ERR_SPACE, "zn_ans_decompress: temp buffer too small");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  DecArgs a{};
  a.in_ptrs = in_ptrs;
  a.in_bytes = in_bytes;
  a.out_ptrs = out_ptrs;
  a.out_cap = out_capacity;
  a.statuses = statuses;
  a.nch = count;
  DecArgs* dj = static_cast<DecArgs*>(temp);
  if (int rc = upload_jobs(&a, 1, dj, count, s)) return rc;
  return launch_decode<1, false>(dj, 1, count, s);
}

size_t zn_decompress_batch_temp_bytes(int njobs, const int64_t* n, int k, const int64_t* chunk_bytes) {
  if (njobs < 0 || k <= 0) return 0;
  size_t total = 0;
  int64_t chunks = 0;
  for (int i = 0; i < njobs; ++i) {
    if (n[i] < 0 || chunk_bytes[i] <= 0) return 0;
    chunks += cdiv(n[i], chunk_bytes[i]);
    total += dec_job_bytes(n[i], k, chunk_bytes[i]);
  }
  return total + job_table_bytes<DecArgs>(njobs, chunks);
}

size_t zn_decompress_temp_bytes(int64_t n, int k, int64_t chunk_bytes) {
  return zn_decompress_batch_temp_bytes(1, &n, k, &chunk_bytes);
}

int zn_decompress_batch(int njobs, const void* const* blobs, const int64_t* blob_bytes, const int64_t* n, int k,
                        int reorder, const int* ndim, const int64_t* chunk_bytes, const int64_t* n_comp,
                        void* const* out, int32_t* status, void* temp, size_t temp_bytes, void* stream) {
  if (njobs < 0 || (k != 1 && k != 2 && k != 4 && k != 8) || (reorder && k != 2 && k != 4))
    return set_error(ZN_ERR_INVALID, "zn_decompress: bad arguments");
  if (njobs == 0) return ZN_OK;
  NvtxScope range("zn_decompress_batch");
  if (!temp || temp_bytes < zn_decompress_batch_temp_bytes(njobs, n, k, chunk_bytes))
    return set_error(ZN_ERR_SPACE, "zn_decompress: temp buffer too small");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* tb = static_cast<uint8_t*>(temp);
  int64_t total_chunks = 0;
  for (int i = 0; i < njobs; ++i) total_chunks += n[i] > 0 && chunk_bytes[i] > 0 ? cdiv(n[i], chunk_bytes[i]) : 0;
  uint8_t* region = tb + job_table_bytes<DecArgs>(njobs, total_chunks);
  std::vector<DecArgs> jobs;
  jobs.reserve(static_cast<size_t>(njobs));
  int64_t chunk0 = 0;
  for (int i = 0; i < njobs; ++i) {
    if (n[i] < 0 || chunk_bytes[i] <= 0 || ndim[i] < 0 || ndim[i] > 64 || n_comp[i] < -1 ||
        (reinterpret_cast<uintptr_t>(blobs[i]) & 7))
      return set_error(ZN_ERR_INVALID, "zn_decompress: bad arguments (job %d)", i);
    if (n[i] == 0) continue;
    DecArgs a{};
    a.blob = static_cast<const uint8_t*>(blobs[i]);
    a.blob_bytes = blob_bytes[i];
    a.n = n[i];
    a.C = chunk_bytes[i];
    a.nch = cdiv(n[i], chunk_bytes[i]);
    a.units = int64_t(k) * a.nch;
    if (a.nch > 0x7FFFFFFF || n_comp[i] > a.units) return set_error(ZN_ERR_INVALID, "zn_decompress: bad tables (job %d)", i);
    a.sizes_off = 24 + 8 * int64_t(ndim[i]);
    a.idx_off = a.sizes_off + 4 * a.units;
    a.n_comp = n_comp[i];  // -1: dscan_kernel reads it from the blob
    a.data_off = n_comp[i] < 0 ? -1 : align8(a.idx_off + 4 * a.n_comp);
    if (n_comp[i] >= 0 && a.blob_bytes < a.data_off)
      return set_error(ZN_ERR_INVALID, "zn_decompress: blob is truncated (job %d)", i);
    a.chunk0 = chunk0;
    a.out = static_cast<uint8_t*>(out[i]);
    a.status = status + i;
    a.src = reinterpret_cast<int64_t*>(region);
    a.overflow = region + size_t(a.units) * 8;
    region += dec_job_bytes(n[i], k, chunk_bytes[i]);
    chunk0 += a.nch;
    jobs.push_back(a);
  }
  const int nj = int(jobs.size());
  if (nj == 0) return ZN_OK;
  if (chunk0 > 0x7FFFFFFF) return set_error(ZN_ERR_INVALID, "zn_decompress: too many chunks");
  DecArgs* dj = reinterpret_cast<DecArgs*>(tb);
  // A single job goes to the scan kernel by value (it stores the table itself).
  FirstJob<DecArgs> fj{};
  if (nj == 1) {
    fj.job = jobs[0];
    fj.valid = 1;
  } else if (int rc = upload_jobs(jobs.data(), nj, dj, chunk0, s)) {
    return rc;
  }
  {
    TimedLaunch tl("dscan", s);
    dscan_kernel<<<unsigned(nj), kScanThreads, 0, s>>>(dj, fj, dj);
  }
  count_launch();
  if (int rc = check_launch("dscan_kernel")) return rc;
  switch (k * 2 + (reorder ? 1 : 0)) {
    case 2: return launch_decode<1, false>(dj, nj, chunk0, s);
    case 4: return launch_decode<2, false>(dj, nj, chunk0, s);
    case 5: return launch_decode<2, true>(dj, nj, chunk0, s);
    case 8: return launch_decode<4, false>(dj, nj, chunk0, s);
    case 9: return launch_decode<4, true>(dj, nj, chunk0, s);
    default: return launch_decode<8, false>(dj, nj, chunk0, s);
  }
}

int zn_decompress(const void* blob, int64_t blob_bytes, int64_t n, int k, int reorder, int ndim, int64_t chunk_bytes,
                  int64_t n_comp, void* out, int32_t* status, void* temp, size_t temp_bytes, void* stream) {
  return zn_decompress_batch(1, &blob, &blob_bytes, &n, k, reorder, &ndim, &chunk_bytes, &n_comp, &out, status, temp,
                             temp_bytes, stream);
}

}  // extern "C"
