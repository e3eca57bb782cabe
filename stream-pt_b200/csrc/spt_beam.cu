// spt_beam.cu -- beam search's selection over beams and vocabulary.
//
//   score(j, t) = scores[j] + x_j[t] - log sum_u e^(x_j[u])
//
// and for each search the `keep` best (j, t): by score, then the lowest beam,
// then the lowest token.  A finished beam offers end_token alone, its score
// unchanged.  A NaN logit is no token (it is left out of the sum too), a score
// that is NaN or -inf no candidate.
//
// One pass over the logits, each CTA a chunk of one row in registers: its
// maximum, its sum, and its `keep` best tokens.  Within a row scores order as
// logits do, so these decide everything; a second, small launch joins the
// chunks' sums in 64 bits and picks the best of all beams.  Bound by memory:
// every logit is read once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "spt_device.cuh"
#include "spt_internal.cuh"
#include "spt_kv.cuh"

namespace spt {
namespace {

constexpr int kBeamThreads = 256, kBeamWarps = kBeamThreads / 32;
constexpr int kBeamEach = 32;                        // logits a thread holds
constexpr int kBeamChunk = kBeamThreads * kBeamEach;
constexpr int kBeamList = 1024;                      // candidates ranked at once

struct BeamChunk {  // one chunk's result, before its `keep` candidates
  float top, sum;
};

// Larger is better: the logit in an order-preserving form, then the lower token.
__device__ __forceinline__ uint64_t beam_key(float v, uint32_t token) {
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 and +0 are equal
  return (uint64_t)((b >> 31) ? ~b : b | 0x80000000u) << 32 | (0xffffffffu - token);
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return __uint_as_float((b >> 31) ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ uint32_t key_token(uint64_t k) { return 0xffffffffu - (uint32_t)k; }

__device__ __forceinline__ float load_logit(const float *p) { return *p; }
__device__ __forceinline__ float load_logit(const __half *p) { return __half2float(*p); }
__device__ __forceinline__ float load_logit(const __nv_bfloat16 *p) { return __bfloat162float(*p); }

// The n-th largest (n in 1..32) of a value held by each lane.
template <typename T>
__device__ __forceinline__ T warp_nth(T v, int n) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int step = size >> 1; step; step >>= 1) {
      const T o = __shfl_xor_sync(0xffffffffu, v, step);
      const bool down = (lane & size) == 0, low = (lane & step) == 0;  // descending
      v = (down == low) ? (v > o ? v : o) : (v > o ? o : v);
    }
  return __shfl_sync(0xffffffffu, v, n - 1);
}

template <typename T>
__device__ __forceinline__ T block_max(T v, T *scratch) {
#pragma unroll
  for (int m = 16; m; m >>= 1) {
    const T o = __shfl_xor_sync(0xffffffffu, v, m);
    v = v > o ? v : o;
  }
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = scratch[0];
#pragma unroll
  for (int w = 1; w < kBeamWarps; ++w) v = scratch[w] > v ? scratch[w] : v;
  __syncthreads();
  return v;
}

// Logits of chunk blockIdx.x of row blockIdx.y.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kBeamThreads) k_beam_chunk(const BeamArgs a, BeamChunk *chunks, uint64_t *keys) {
  __shared__ uint64_t list[kBeamList];
  __shared__ uint64_t scratch[kBeamWarps];
  __shared__ float fscratch[kBeamWarps];
  __shared__ int found;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.y;
  pdl_wait();
  pdl_trigger();
  if (a.finished && a.finished[row]) return;
  const T *x = static_cast<const T *>(a.logits) + row * a.row_stride;
  const int64_t base = (int64_t)blockIdx.x * kBeamChunk;
  const int64_t rest = a.vocab - base;
  constexpr int V = VEC ? 16 / (int)sizeof(T) : 1;  // logits a load
  float v[kBeamEach];
#pragma unroll
  for (int i = 0; i < kBeamEach / V; ++i) {
    const int64_t at = ((int64_t)i * kBeamThreads + tid) * V;
    if (VEC && at + V <= rest) {
      const uint4 w = __ldcs(reinterpret_cast<const uint4 *>(x + base + at));
      const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
      for (int j = 0; j < V; ++j) v[i * V + j] = load_logit(e + j);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v[i * V + j] = at + j < rest ? load_logit(x + base + at + j) : -INFINITY;
    }
  }
  auto token = [&](int i) { return (uint32_t)(base + ((int64_t)(i / V) * kBeamThreads + tid) * V + i % V); };
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kBeamEach; ++i) {
    if (isnan(v[i])) v[i] = -INFINITY;
    top = fmaxf(top, v[i]);
  }
  if (tid == 0) found = 0;
  const float all = block_max(top, fscratch);
  // keep distinct logits are at least `least`: the smallest of the warps'
  // n-th largest thread maxima, n = keep over the warps rounded up
  const float nth = warp_nth(top, (a.keep + kBeamWarps - 1) / kBeamWarps);
  const float least = -block_max(-nth, fscratch);
  float sum = 0.0f;
  const float shift = all == -INFINITY ? 0.0f : all;
#pragma unroll
  for (int i = 0; i < kBeamEach; ++i) {
    sum += exp2f((v[i] - shift) * 1.4426950408889634f);
    if (v[i] >= least && v[i] > -INFINITY) {
      const int at = atomicAdd(&found, 1);
      if (at < kBeamList) list[at] = beam_key(v[i], token(i));
    }
  }
#pragma unroll
  for (int m = 16; m; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  if ((tid & 31) == 0) fscratch[tid >> 5] = sum;
  __syncthreads();
  const int64_t chunk = row * gridDim.x + blockIdx.x;
  if (tid == 0) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kBeamWarps; ++w) s += fscratch[w];
    chunks[chunk] = {all, s};
  }
  uint64_t *out = keys + chunk * a.keep;
  const int n = found;
  if (n <= kBeamList) {  // a candidate's rank is its place
    for (int i = tid; i < n; i += kBeamThreads) {
      const uint64_t k = list[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += list[j] > k;
      if (rank < a.keep) out[rank] = k;
    }
    for (int i = n + tid; i < a.keep; i += kBeamThreads) out[i] = 0;
    return;
  }
  // more logits tie for a place than the list holds: one place after another
  uint64_t last = ~0ull;
  for (int r = 0; r < a.keep; ++r) {
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < kBeamEach; ++i) {
      const uint64_t k = v[i] > -INFINITY ? beam_key(v[i], token(i)) : 0;
      if (k < last && k > best) best = k;
    }
    last = block_max(best, scratch);
    if (tid == 0) out[r] = last;
    if (last == 0) last = 1;  // no more: nothing is below this but 0
  }
}

// One CTA per search: the chunks' sums joined, then the best of all beams.
__global__ void __launch_bounds__(kBeamThreads) k_beam_pick(const BeamArgs a, const BeamChunk *chunks,
                                                           const uint64_t *keys, int n_chunks) {
  __shared__ double norm[kBeamMaxBeams];
  __shared__ double score[kBeamList];
  __shared__ uint64_t place[kBeamList];  // beam and token: the lower wins among equals
  __shared__ double scratch[kBeamWarps];
  __shared__ uint64_t pscratch[kBeamWarps];
  __shared__ int found;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t search = blockIdx.x, row0 = search * a.beams;
  pdl_wait();
  pdl_trigger();
  if (tid == 0) found = 0;
  for (int j = warp; j < a.beams; j += kBeamWarps) {
    if (a.finished && a.finished[row0 + j]) continue;
    const BeamChunk *c = chunks + (row0 + j) * n_chunks;
    float top = -INFINITY;
    for (int i = lane; i < n_chunks; i += 32) top = fmaxf(top, c[i].top);
#pragma unroll
    for (int m = 16; m; m >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
    double sum = 0.0;
    for (int i = lane; i < n_chunks; i += 32)
      if (c[i].top > -INFINITY) sum += (double)c[i].sum * exp((double)c[i].top - (double)top);
#pragma unroll
    for (int m = 16; m; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    if (lane == 0) norm[j] = (double)top + log(sum);
  }
  __syncthreads();
  const int64_t per_beam = (int64_t)n_chunks * a.keep, total = per_beam * a.beams;
  // candidate i of beam i / per_beam; false where there is none
  auto candidate = [&](int64_t i, double *s, uint64_t *p) {
    const int j = (int)(i / per_beam);
    const int64_t at = i - j * per_beam;
    if (a.finished && a.finished[row0 + j]) {
      if (at != 0) return false;
      *s = (double)a.scores[row0 + j];
      *p = (uint64_t)j << 32 | (uint32_t)a.end_token;
    } else {
      const uint64_t k = keys[(row0 + j) * per_beam + at];
      if (k == 0) return false;
      *s = ((double)key_value(k) - norm[j]) + (double)a.scores[row0 + j];
      *p = (uint64_t)j << 32 | key_token(k);
    }
    return *s > -INFINITY;
  };
  double best = -INFINITY;
  for (int64_t i = tid; i < total; i += kBeamThreads) {
    double s;
    uint64_t p;
    if (candidate(i, &s, &p) && s > best) best = s;
  }
  const double nth = warp_nth(best, (a.keep + kBeamWarps - 1) / kBeamWarps);
  const double least = -block_max(-nth, scratch);
  for (int64_t i = tid; i < total; i += kBeamThreads) {
    double s;
    uint64_t p;
    if (!candidate(i, &s, &p) || !(s >= least)) continue;
    const int at = atomicAdd(&found, 1);
    if (at < kBeamList) score[at] = s, place[at] = p;
  }
  __syncthreads();
  const int n = found;
  auto put = [&](int r, double s, uint64_t p, bool any) {
    a.out_scores[search * a.keep + r] = any ? (float)s : -INFINITY;
    a.out_parents[search * a.keep + r] = any ? (int32_t)(p >> 32) : -1;
    a.out_tokens[search * a.keep + r] = any ? (int32_t)(uint32_t)p : -1;
  };
  if (n <= kBeamList) {
    for (int i = tid; i < n; i += kBeamThreads) {
      const double s = score[i];
      const uint64_t p = place[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += score[j] > s || (score[j] == s && place[j] < p);
      if (rank < a.keep) put(rank, s, p, true);
    }
    for (int i = n + tid; i < a.keep; i += kBeamThreads) put(i, 0.0, 0, false);
    return;
  }
  double last = INFINITY;
  uint64_t last_place = 0;
  for (int r = 0; r < a.keep; ++r) {  // the best behind the last one
    double top = -INFINITY;
    uint64_t at = ~0ull;
    for (int64_t i = tid; i < total; i += kBeamThreads) {
      double s;
      uint64_t p;
      if (!candidate(i, &s, &p)) continue;
      if (r > 0 && !(s < last || (s == last && p > last_place))) continue;
      if (s > top || (s == top && p < at)) top = s, at = p;
    }
    const double all = block_max(top, scratch);
    const uint64_t mine = top == all ? ~at : 0;  // the lowest place is the largest complement
    const uint64_t first = ~block_max(mine, pscratch);
    if (tid == 0) put(r, all, first, all > -INFINITY);
    last = all, last_place = first;
  }
}

int64_t beam_chunks(int64_t vocab) { return (vocab + kBeamChunk - 1) / kBeamChunk; }

template <typename T>
cudaError_t launch_rows(const BeamArgs &a, cudaStream_t stream) {
  const int64_t rows = a.batch * a.beams, chunks = beam_chunks(a.vocab);
  if (rows > 65535 || chunks > 0x7fffffffll) return cudaErrorInvalidValue;
  BeamChunk *c = static_cast<BeamChunk *>(a.work);
  uint64_t *keys = reinterpret_cast<uint64_t *>(c + rows * chunks);
  const bool vec = (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 && (a.row_stride * sizeof(T)) % 16 == 0;
  const dim3 grid((unsigned)chunks, (unsigned)rows);
  cudaError_t e = vec ? launch_pdl(k_beam_chunk<T, true>, grid, dim3(kBeamThreads), 0, stream, a, c, keys)
                      : launch_pdl(k_beam_chunk<T, false>, grid, dim3(kBeamThreads), 0, stream, a, c, keys);
  if (e != cudaSuccess) return e;
  return launch_pdl(k_beam_pick, dim3((unsigned)a.batch), dim3(kBeamThreads), 0, stream, a,
                    static_cast<const BeamChunk *>(c), static_cast<const uint64_t *>(keys), (int)chunks);
}

}  // namespace

size_t beam_workspace_bytes(int64_t batch, int64_t beams, int64_t vocab, int keep, int sm_count) {
  (void)sm_count;
  return (size_t)(batch * beams * beam_chunks(vocab)) * (sizeof(BeamChunk) + (size_t)keep * sizeof(uint64_t));
}

cudaError_t launch_beam_select(const BeamArgs &a, cudaStream_t stream) {
  switch (a.type) {
    case kKvF32: return launch_rows<float>(a, stream);
    case kKvF16: return launch_rows<__half>(a, stream);
    case kKvBF16: return launch_rows<__nv_bfloat16>(a, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace spt
