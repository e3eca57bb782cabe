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
constexpr int kPickThreads = 512;
constexpr int kPickEach = 8;                         // candidates a thread keeps in registers
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
  if (n == 1) {
#pragma unroll
    for (int m = 16; m; m >>= 1) {
      const T o = __shfl_xor_sync(0xffffffffu, v, m);
      v = v > o ? v : o;
    }
    return v;
  }
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

template <int WARPS, typename T>
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
  for (int w = 1; w < WARPS; ++w) v = scratch[w] > v ? scratch[w] : v;
  __syncthreads();
  return v;
}

// Logits of chunk blockIdx.x of row blockIdx.y.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kBeamThreads, 3) k_beam_chunk(const BeamArgs a, BeamChunk *chunks, uint64_t *keys) {
  __shared__ uint64_t list[kBeamList];
  __shared__ uint64_t scratch[kBeamWarps];
  __shared__ float fscratch[2 * kBeamWarps];
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
  float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // (fmaxf passes NaNs by)
#pragma unroll
  for (int i = 0; i < kBeamEach; ++i) tops[i & 3] = fmaxf(tops[i & 3], v[i]);
  const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  if (tid == 0) found = 0;
  // keep distinct logits are at least `least`: the smallest of the warps'
  // n-th largest thread maxima, n = keep over the warps rounded up
  const float nth = warp_nth(top, (a.keep + kBeamWarps - 1) / kBeamWarps);
  float most = top;
#pragma unroll
  for (int m = 16; m; m >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, m));
  if ((tid & 31) == 0) fscratch[tid >> 5] = most, fscratch[kBeamWarps + (tid >> 5)] = nth;
  __syncthreads();
  float all = fscratch[0], least = fscratch[kBeamWarps];
#pragma unroll
  for (int w = 1; w < kBeamWarps; ++w) all = fmaxf(all, fscratch[w]), least = fminf(least, fscratch[kBeamWarps + w]);
  __syncthreads();
  least = fmaxf(least, -3.402823466e38f);  // -inf is no candidate
  const float shift = all == -INFINITY ? 0.0f : all;
  constexpr float kLog2e = 1.4426950408889634f;
  const float off = -shift * kLog2e;
  float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < kBeamEach; ++i) {
    // (v - shift) log2 e: the product's rounding is of 2^-24 of it, and weights that count lie near 1
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(__fmaf_rn(v[i], kLog2e, off)));
    sums[i & 3] += e;
    if (v[i] >= least) {
      const int at = atomicAdd(&found, 1);
      if (at < kBeamList) list[at] = beam_key(v[i], token(i));
    }
  }
  float sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  if (isnan(sum) && all < INFINITY) {  // NaN logits are left out (an infinite one makes its row's sum a NaN)
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kBeamEach; ++i)
      if (!isnan(v[i])) sum += exp2f((v[i] - shift) * kLog2e);
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
    last = block_max<kBeamWarps>(best, scratch);
    if (tid == 0) out[r] = last;
    if (last == 0) last = 1;  // no more: nothing is below this but 0
  }
}

// One CTA per search: the chunks' sums joined, then the best of all beams.
// Bound by latency: a few thousand candidates, of which a thread keeps up to
// kPickEach in registers.
__global__ void __launch_bounds__(kPickThreads) k_beam_pick(const BeamArgs a, const BeamChunk *chunks,
                                                           const uint64_t *keys, int n_chunks) {
  constexpr int WARPS = kPickThreads / 32;
  __shared__ double norm[kBeamMaxBeams];
  __shared__ double score[kBeamList];
  __shared__ uint64_t place[kBeamList];  // beam and token: the lower wins among equals
  __shared__ double scratch[WARPS];
  __shared__ uint64_t pscratch[WARPS];
  __shared__ int found;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t search = blockIdx.x, row0 = search * a.beams;
  pdl_wait();
  pdl_trigger();
  if (tid == 0) found = 0;
  const uint32_t per_beam = (uint32_t)n_chunks * a.keep, total = per_beam * (uint32_t)a.beams;
  // key of candidate i of beam i / per_beam; 0: there is none
  auto key_of = [&](uint32_t i) -> uint64_t {
    if (i >= total) return 0;
    const uint32_t j = i / per_beam;
    if (a.finished && a.finished[row0 + j]) return i == j * per_beam ? 1 : 0;
    return __ldcg(keys + row0 * per_beam + i);
  };
  uint64_t mine[kPickEach];
#pragma unroll
  for (int x = 0; x < kPickEach; ++x) mine[x] = key_of(tid + x * kPickThreads);
  for (int j = warp; j < a.beams; j += WARPS) {
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
  // score and place of a candidate; false where it is none
  auto candidate = [&](uint32_t i, uint64_t k, double *s, uint64_t *p) {
    if (k == 0) return false;
    const uint32_t j = i / per_beam;
    if (a.finished && a.finished[row0 + j]) {
      *s = (double)a.scores[row0 + j];
      *p = (uint64_t)j << 32 | (uint32_t)a.end_token;
    } else {
      *s = ((double)key_value(k) - norm[j]) + (double)a.scores[row0 + j];
      *p = (uint64_t)j << 32 | key_token(k);
    }
    return *s > -INFINITY;
  };
  double best = -INFINITY, s;
  uint64_t p;
#pragma unroll
  for (int x = 0; x < kPickEach; ++x)
    if (candidate(tid + x * kPickThreads, mine[x], &s, &p) && s > best) best = s;
  for (uint32_t i = tid + kPickEach * kPickThreads; i < total; i += kPickThreads)
    if (candidate(i, key_of(i), &s, &p) && s > best) best = s;
  const double nth = warp_nth(best, (a.keep + WARPS - 1) / WARPS);
  const double least = -block_max<WARPS>(-nth, scratch);
  auto take = [&](uint32_t i, uint64_t k) {
    if (!candidate(i, k, &s, &p) || !(s >= least)) return;
    const int at = atomicAdd(&found, 1);
    if (at < kBeamList) score[at] = s, place[at] = p;
  };
#pragma unroll
  for (int x = 0; x < kPickEach; ++x) take(tid + x * kPickThreads, mine[x]);
  for (uint32_t i = tid + kPickEach * kPickThreads; i < total; i += kPickThreads) take(i, key_of(i));
  __syncthreads();
  const int n = found;
  auto put = [&](int r, double sc, uint64_t pl, bool any) {
    a.out_scores[search * a.keep + r] = any ? (float)sc : -INFINITY;
    a.out_parents[search * a.keep + r] = any ? (int32_t)(pl >> 32) : -1;
    a.out_tokens[search * a.keep + r] = any ? (int32_t)(uint32_t)pl : -1;
  };
  if (n <= kBeamList) {
    for (int i = tid; i < n; i += kPickThreads) {
      const double si = score[i];
      const uint64_t pi = place[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += score[j] > si || (score[j] == si && place[j] < pi);
      if (rank < a.keep) put(rank, si, pi, true);
    }
    for (int i = n + tid; i < a.keep; i += kPickThreads) put(i, 0.0, 0, false);
    return;
  }
  double last = INFINITY;
  uint64_t last_place = 0;
  for (int r = 0; r < a.keep; ++r) {  // the best behind the last one
    double top = -INFINITY;
    uint64_t at = ~0ull;
    for (uint32_t i = tid; i < total; i += kPickThreads) {
      if (!candidate(i, key_of(i), &s, &p)) continue;
      if (r > 0 && !(s < last || (s == last && p > last_place))) continue;
      if (s > top || (s == top && p < at)) top = s, at = p;
    }
    const double all = block_max<WARPS>(top, scratch);
    const uint64_t own = top == all ? ~at : 0;  // the lowest place is the largest complement
    const uint64_t first = ~block_max<WARPS>(own, pscratch);
    if (tid == 0) put(r, all, first, all > -INFINITY);
    last = all, last_place = first;
  }
}

int64_t beam_chunks(int64_t vocab) { return (vocab + kBeamChunk - 1) / kBeamChunk; }

template <typename T>
cudaError_t launch_rows(const BeamArgs &a, cudaStream_t stream) {
  const int64_t rows = a.batch * a.beams, chunks = beam_chunks(a.vocab);
  if (rows > 65535 || chunks * a.keep * a.beams > 0x7fffffffll) return cudaErrorInvalidValue;
  BeamChunk *c = static_cast<BeamChunk *>(a.work);
  uint64_t *keys = reinterpret_cast<uint64_t *>(c + rows * chunks);
  const bool vec = (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 && (a.row_stride * sizeof(T)) % 16 == 0;
  const dim3 grid((unsigned)chunks, (unsigned)rows);
  cudaError_t e = vec ? launch_pdl(k_beam_chunk<T, true>, grid, dim3(kBeamThreads), 0, stream, a, c, keys)
                      : launch_pdl(k_beam_chunk<T, false>, grid, dim3(kBeamThreads), 0, stream, a, c, keys);
  if (e != cudaSuccess) return e;
  return launch_pdl(k_beam_pick, dim3((unsigned)a.batch), dim3(kPickThreads), 0, stream, a,
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
