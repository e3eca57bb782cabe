// spt_beam.cu -- beam search's selection over beams and vocabulary.
//
//   score(j, t) = scores[j] + x_j[t] - log sum_u e^(x_j[u])
//
// and for each search the `keep` best (j, t): by score, then the lowest beam,
// then the lowest token.  A finished beam offers end_token alone, its score
// unchanged.  A NaN logit is no token (it is left out of the sum too), a score
// that is NaN or -inf no candidate.
//
// One pass over the logits.  A CTA takes a chunk of a row, a piece of 8,192
// logits at a time in registers with the next piece on its way: the running
// maximum and sum, and the tokens that can be among the chunk's `keep` best.
// Within a row scores order as logits do, so these decide everything; a second,
// small launch joins the chunks' sums in 64 bits and picks the best of all
// beams.  Bound by memory: every logit is read once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "spt_device.cuh"
#include "spt_internal.cuh"
#include "spt_kv.cuh"
#include "spt_ptx.cuh"

namespace spt {
namespace {

constexpr int kBeamThreads = 256, kBeamWarps = kBeamThreads / 32;
constexpr int kPickThreads = 512;
constexpr int kPickEach = 8;                         // candidates a thread keeps in registers
constexpr int kBeamEach = 32;                        // logits a thread holds
constexpr int kBeamPiece = kBeamThreads * kBeamEach; // logits a CTA holds
constexpr int kBeamStages = 2;
constexpr int kBeamCtas = 3;                         // CTAs an SM
constexpr int kBeamMaxChunks = 512;                  // a row's
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

template <typename T>
__device__ __forceinline__ T warp_max(T v) {
#pragma unroll
  for (int m = 16; m; m >>= 1) {
    const T o = __shfl_xor_sync(0xffffffffu, v, m);
    v = v > o ? v : o;
  }
  return v;
}
// A score that is no NaN in an order-preserving form, and back.
__device__ __forceinline__ uint64_t score_key(double s) {
  const uint64_t b = (uint64_t)__double_as_longlong(s + 0.0);  // -0 and +0 are equal
  return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double key_score(uint64_t k) {
  return __longlong_as_double((long long)(k >> 63 ? k & ~(1ull << 63) : ~k));
}

// The n-th largest (n in 1..32) of a value held by each lane.
template <typename T>
__device__ __forceinline__ T warp_nth(T v, int n) {
  const int lane = threadIdx.x & 31;
  if (n == 1) return warp_max(v);
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
  v = warp_max(v);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = scratch[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) v = scratch[w] > v ? scratch[w] : v;
  __syncthreads();
  return v;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float m;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}

// The next larger float; NaN, which nothing reaches, above infinity.
__device__ __forceinline__ float float_above(float v) {
  if (v == INFINITY) return __uint_as_float(0x7fffffffu);
  if (v == 0.0f) return __uint_as_float(1u);
  return __uint_as_float(__float_as_uint(v) + (v > 0.0f ? 1u : 0xffffffffu));
}

template <typename T>
__device__ __forceinline__ T lowest_logit() {
  if constexpr (std::is_same<T, float>::value) return -INFINITY;
  else if constexpr (std::is_same<T, __half>::value) return __ushort_as_half(0xfc00u);
  else return __ushort_as_bfloat16(0xff80u);
}

// Logits of chunk blockIdx.x of row blockIdx.y.  A thread fetches and reads its
// own logits alone, 16 bytes at a time, so shared memory needs no barrier;
// kBeamStages pieces are on their way while one is worked on.  Bound by
// instructions and their latency, at 6 warps a scheduler: 128 rows of 201,088
// f32 logits in 36 us (2.5 TB/s of the 88 MB that unfinished beams have), where
// a CTA a piece takes the same and leaves 25 lists a row to join instead of 3.
template <typename T>
__global__ void __launch_bounds__(kBeamThreads, kBeamCtas) k_beam_chunk(const BeamArgs a, BeamChunk *chunks,
                                                                      uint64_t *keys) {
  extern __shared__ __align__(16) uint8_t stages[];  // [kBeamStages][loads][kBeamThreads] of 16 bytes
  __shared__ uint64_t list[kBeamList];
  __shared__ uint64_t best_keys[kBeamMaxKeep];
  __shared__ uint64_t scratch[kBeamWarps];
  __shared__ float warp_top[kBeamWarps], warp_least[kBeamWarps];
  __shared__ double warp_sum[kBeamWarps];
  __shared__ int found;
  constexpr int V = 16 / (int)sizeof(T), kLoads = kBeamEach / V;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row = blockIdx.y;
  pdl_wait();
  pdl_trigger();
  if (a.finished && a.finished[row]) return;
  // the row from the 16-byte boundary at or before it: logit t is `lead` + t in its pieces
  const T *x = static_cast<const T *>(a.logits) + row * a.row_stride;
  const int lead = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  x -= lead;
  const int64_t end = lead + a.vocab, pieces = (end + kBeamPiece - 1) / kBeamPiece;
  const int first = (int)(pieces * blockIdx.x / gridDim.x), last = (int)(pieces * (blockIdx.x + 1) / gridDim.x);
  // keep distinct logits are at least the smallest of the maxima of as many groups of lanes
  int group = 32;
  while (kBeamThreads / group < a.keep) group >>= 1;
  auto stage = [&](int piece) {
    return reinterpret_cast<uint4 *>(stages) + (piece - first) % kBeamStages * (kLoads * kBeamThreads) + tid;
  };
  // place in its piece of logit j of load i
  auto place = [&](int i, int j) { return (i * kBeamThreads + tid) * V + j; };
  auto fetch = [&](int piece) {
    if (piece >= last) return;
    const int64_t base = (int64_t)piece * kBeamPiece;
    uint4 *to = stage(piece);
    if (base >= lead && base + kBeamPiece <= end) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) cp_async16(to + i * kBeamThreads, x + base + place(i, 0));
      return;
    }
#pragma unroll 1
    for (int i = 0; i < kLoads; ++i) {  // the row's first or last piece: -inf outside of it
      const int64_t at = base + place(i, 0);
      T *e = reinterpret_cast<T *>(to + i * kBeamThreads);
      if (at >= lead && at + V <= end) cp_async16(e, x + at);
      else
#pragma unroll
        for (int j = 0; j < V; ++j) e[j] = at + j >= lead && at + j < end ? x[at + j] : lowest_logit<T>();
    }
  };
#pragma unroll
  for (int s = 0; s < kBeamStages; ++s) {
    fetch(first + s);
    cp_async_commit();
  }
  if (tid == 0) found = 0;
  constexpr float kLog2e = 1.4426950408889634f;
  float top = -INFINITY;         // this thread's largest so far
  float all = -INFINITY;         // the chunk's
  float bar = -3.402823466e38f;  // what a candidate has to reach
  float floor = -INFINITY;       // and what it has to exceed
  double sum = 0.0;              // this thread's, of e^(v - all)
  int kept = 0;                  // candidates of the pieces before
  for (int piece = first; piece < last; ++piece) {
    cp_async_wait<kBeamStages - 1>();
    const uint4 *held = stage(piece);
    float v[kBeamEach];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint4 w = held[i * kBeamThreads];
      const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
      for (int j = 0; j < V; ++j) v[i * V + j] = load_logit(e + j);
    }
    float tops[4];  // of every fourth logit (maxima pass NaNs by)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      tops[q] = max3(v[q], v[q + 4], v[q + 8]);
      tops[q] = max3(tops[q], v[q + 12], v[q + 16]);
      tops[q] = max3(tops[q], v[q + 20], v[q + 24]);
      tops[q] = max3(tops[q], v[q + 28], -INFINITY);
    }
    const float own = max3(fmaxf(tops[0], tops[1]), tops[2], tops[3]);
    top = fmaxf(top, own);
    float most = top;
    for (int m = 1; m < group; m <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, m));
    float least = most;
    for (int m = group; m < 32; m <<= 1) {
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, m));
      least = fminf(least, __shfl_xor_sync(0xffffffffu, least, m));
    }
    if (lane == 0) warp_top[warp] = most, warp_least[warp] = least;
    __syncthreads();
    const float before = all;
    all = warp_top[0], least = warp_least[0];
#pragma unroll
    for (int w = 1; w < kBeamWarps; ++w) all = fmaxf(all, warp_top[w]), least = fminf(least, warp_least[w]);
    bar = floor == INFINITY ? float_above(floor) : fmaxf(least, float_above(floor));
    if (own >= bar) {
      uint32_t reach = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (tops[q] >= bar)
#pragma unroll
          for (int i = q; i < kBeamEach; i += 4) reach |= v[i] >= bar ? 1u << i : 0u;
      int at = atomicAdd(&found, __popc(reach));
      for (; reach; reach &= reach - 1, ++at) {
        const int i = (__ffs(reach) - 1) / V, j = (__ffs(reach) - 1) % V;
        if (at < kBeamList)
          list[at] = beam_key(load_logit(reinterpret_cast<const T *>(held + i * kBeamThreads) + j),
                              (uint32_t)(piece * kBeamPiece + place(i, j) - lead));
      }
    }
    const float shift = all == -INFINITY ? 0.0f : all;
    if (all != before && before > -INFINITY) sum *= exp2f((before - all) * kLog2e);
    // e^(v - shift) as 2^(v L + off), off = -shift L rounded and L log2 e in 32
    // bits, which makes it 2^(shift L + off) too large: one factor for the sum
    const float off = -shift * kLog2e, extra = __fmaf_rn(shift, kLog2e, off);
    float2 sums[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
#pragma unroll
    for (int i = 0; i < kBeamEach; i += 2) {
      float2 y = __ffma2_rn(make_float2(v[i], v[i + 1]), make_float2(kLog2e, kLog2e), make_float2(off, off));
      asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(y.x));
      asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(y.y));
      sums[i / 2 & 1] = __fadd2_rn(sums[i / 2 & 1], y);
    }
    float part = ((sums[0].x + sums[0].y) + (sums[1].x + sums[1].y)) * exp2f(-extra);
    if (!(part < INFINITY) || fabsf(shift) > 1e6f) {
      // a NaN, which is left out (an infinite logit makes its row's sum one), or a
      // shift whose product with L is too coarse
      part = 0.0f;
#pragma unroll 1
      for (int i = 0; i < kLoads; ++i)
#pragma unroll 1
        for (int j = 0; j < V; ++j) {
          const float y = load_logit(reinterpret_cast<const T *>(held + i * kBeamThreads) + j);
          if (!isnan(y)) part += exp2f((y - shift) * kLog2e);
        }
    }
    sum += (double)part;
    __syncthreads();
    if (found > kBeamList) {
      // more logits reach the bar than the list holds: the best of the list and
      // this piece, one after another; of later pieces only larger ones count
      uint64_t below = ~0ull;
      for (int r = 0; r < a.keep; ++r) {
        uint64_t best = 0;
#pragma unroll 1
        for (int i = 0; i < kLoads; ++i)
#pragma unroll 1
          for (int j = 0; j < V; ++j) {
            const float y = load_logit(reinterpret_cast<const T *>(held + i * kBeamThreads) + j);
            const uint64_t k = y >= bar ? beam_key(y, (uint32_t)(piece * kBeamPiece + place(i, j) - lead)) : 0;
            if (k < below && k > best) best = k;
          }
        for (int i = tid; i < kept; i += kBeamThreads)
          if (list[i] < below && list[i] > best) best = list[i];
        below = block_max<kBeamWarps>(best, scratch);
        if (tid == 0) best_keys[r] = below;
      }
      __syncthreads();
      if (tid < a.keep) list[tid] = best_keys[tid];
      if (tid == 0) found = a.keep;
      floor = key_value(below);
      __syncthreads();
    }
    kept = found;
    fetch(piece + kBeamStages);
    cp_async_commit();
  }
  cp_async_wait<0>();
#pragma unroll
  for (int m = 16; m; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  if (lane == 0) warp_sum[warp] = sum;
  __syncthreads();
  const int64_t chunk = row * gridDim.x + blockIdx.x;
  if (tid == 0) {
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < kBeamWarps; ++w) s += warp_sum[w];
    chunks[chunk] = {all, (float)s};
  }
  uint64_t *out = keys + chunk * a.keep;
  for (int i = warp; i < kept; i += kBeamWarps) {  // a warp a candidate: its rank is its place
    const uint64_t k = list[i];
    if (floor == -INFINITY && !(key_value(k) >= bar)) continue;  // an earlier, lower bar let it in
    int rank = 0;
    for (int j = 0; j < kept; j += 32) {
      const int at = j + lane;
      rank += __popc(__ballot_sync(0xffffffffu, at < kept && list[at] > k));
    }
    if (lane == 0 && rank < a.keep) out[rank] = k;
  }
  for (int i = kept + tid; i < a.keep; i += kBeamThreads) out[i] = 0;
}

// One CTA per search: the chunks' sums joined, then the best of all beams.
// Bound by latency: a few hundred to a few thousand candidates, of which a
// thread keeps up to kPickEach in registers.  16 searches of 8 beams: 9.8 us
// alone, of which a launch with nothing to do takes about 4.
__global__ void __launch_bounds__(kPickThreads) k_beam_pick(const BeamArgs a, const BeamChunk *chunks,
                                                           const uint64_t *keys, int n_chunks) {
  constexpr int WARPS = kPickThreads / 32;
  __shared__ double norm[kBeamMaxBeams], base[kBeamMaxBeams];
  __shared__ bool done[kBeamMaxBeams];
  __shared__ uint64_t score[kBeamList];  // as score_key()
  __shared__ uint64_t place[kBeamList];  // beam and token: the lower wins among equals
  __shared__ unsigned long long column[64];
  __shared__ double scratch[WARPS];
  __shared__ uint64_t pscratch[WARPS];
  __shared__ int found;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t search = blockIdx.x, row0 = search * a.beams;
  pdl_wait();
  pdl_trigger();
  if (tid == 0) found = 0;
  const uint32_t per_beam = (uint32_t)n_chunks * a.keep, total = per_beam * (uint32_t)a.beams;
  const uint64_t *own_keys = keys + row0 * per_beam;
  uint64_t mine[kPickEach];  // (those of a finished beam are not looked at: nobody wrote them)
#pragma unroll
  for (int x = 0; x < kPickEach; ++x) {
    const uint32_t i = tid + x * kPickThreads;
    mine[x] = i < total ? __ldcg(own_keys + i) : 0;
  }
  for (int j = warp; j < a.beams; j += WARPS) {
    const bool over = a.finished && a.finished[row0 + j];
    if (lane == 0) done[j] = over, base[j] = (double)a.scores[row0 + j];
    if (over) continue;
    const BeamChunk *c = chunks + (row0 + j) * n_chunks;
    float top = -INFINITY;
    for (int i = lane; i < n_chunks; i += 32) top = fmaxf(top, c[i].top);
    top = warp_max(top);
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
    if (i >= total) return false;
    const uint32_t j = i / per_beam;
    if (done[j]) {
      *s = base[j];
      *p = (uint64_t)j << 32 | (uint32_t)a.end_token;
      return i == j * per_beam && *s > -INFINITY;
    }
    *s = ((double)key_value(k) - norm[j]) + base[j];
    *p = (uint64_t)j << 32 | key_token(k);
    return k != 0 && *s > -INFINITY;
  };
  double best = -INFINITY, s;
  uint64_t p;
#pragma unroll
  for (int x = 0; x < kPickEach; ++x)
    if (candidate(tid + x * kPickThreads, mine[x], &s, &p) && s > best) best = s;
  for (uint32_t i = tid + kPickEach * kPickThreads; i < total; i += kPickThreads)
    if (candidate(i, __ldcg(own_keys + i), &s, &p) && s > best) best = s;
  // keep distinct scores are at least `least`: half of keep, rounded up, of the
  // maxima in either half of 64 columns (a chunk's keys come in order: they are
  // spread over the columns)
  const uint64_t nothing = score_key(-INFINITY);
  if (tid < 64) column[tid] = nothing;
  __syncthreads();
  atomicMax(&column[(tid + (uint32_t)tid / (uint32_t)a.keep) & 63], (unsigned long long)score_key(best));
  __syncthreads();
  const int half = (a.keep + 1) / 2;
  const uint64_t one = warp_nth((uint64_t)column[lane], half), two = warp_nth((uint64_t)column[32 + lane], half);
  const uint64_t least = one < two ? one : two;
  auto take = [&](uint32_t i, uint64_t k) {
    if (!candidate(i, k, &s, &p) || score_key(s) < least) return;
    const int at = atomicAdd(&found, 1);
    if (at < kBeamList) score[at] = score_key(s), place[at] = p;
  };
#pragma unroll
  for (int x = 0; x < kPickEach; ++x) take(tid + x * kPickThreads, mine[x]);
  for (uint32_t i = tid + kPickEach * kPickThreads; i < total; i += kPickThreads) take(i, __ldcg(own_keys + i));
  __syncthreads();
  const int n = found;
  auto put = [&](int r, double sc, uint64_t pl, bool any) {
    a.out_scores[search * a.keep + r] = any ? (float)sc : -INFINITY;
    a.out_parents[search * a.keep + r] = any ? (int32_t)(pl >> 32) : -1;
    a.out_tokens[search * a.keep + r] = any ? (int32_t)(uint32_t)pl : -1;
  };
  if (n <= kBeamList) {
    for (int i = warp; i < n; i += WARPS) {
      const uint64_t si = score[i];
      const uint64_t pi = place[i];
      int rank = 0;
      for (int j = 0; j < n; j += 32) {
        const int at = j + lane;
        rank += __popc(__ballot_sync(0xffffffffu, at < n && (score[at] > si || (score[at] == si && place[at] < pi))));
      }
      if (lane == 0 && rank < a.keep) put(rank, key_score(si), pi, true);
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
      if (!candidate(i, __ldcg(own_keys + i), &s, &p)) continue;
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

template <typename T>
cudaError_t launch_rows(const BeamArgs &a, cudaStream_t stream) {
  const int64_t rows = a.batch * a.beams;
  if (rows > 65535) return cudaErrorInvalidValue;
  BeamChunk *c = static_cast<BeamChunk *>(a.work);
  uint64_t *keys = reinterpret_cast<uint64_t *>(c + rows * a.chunks);
  constexpr int kSmem = kBeamStages * kBeamPiece * (int)sizeof(T);
  cudaError_t e = opt_in_smem(k_beam_chunk<T>, kSmem);
  if (e != cudaSuccess) return e;
  e = launch_pdl(k_beam_chunk<T>, dim3((unsigned)a.chunks, (unsigned)rows), dim3(kBeamThreads), kSmem, stream, a, c, keys);
  if (e != cudaSuccess) return e;
  return launch_pdl(k_beam_pick, dim3((unsigned)a.batch), dim3(kPickThreads), 0, stream, a,
                    static_cast<const BeamChunk *>(c), static_cast<const uint64_t *>(keys), a.chunks);
}

}  // namespace

// As few chunks as fill the GPU, by the pieces that the busiest CTA slot goes
// through, one more a CTA for its start and end.  128 rows of 201,088 logits:
// 3 to 8 chunks a row within 1 us of one another, 2 chunks 6 us slower, 25
// (one piece each) 11 us; 4 rows: 25 chunks 25.7 us with what follows, 8 26.2.
int beam_chunks(int64_t rows, int64_t vocab, int sm_count) {
  const int64_t slots = (int64_t)sm_count * kBeamCtas, pieces = (vocab + kBeamPiece - 1) / kBeamPiece;
  int64_t best = INT64_MAX;
  int chunks = 1;
  for (int64_t n = 1; n <= pieces && n <= kBeamMaxChunks; ++n) {
    const int64_t cost = (rows * n + slots - 1) / slots * ((pieces + n - 1) / n + 1);
    if (cost < best) best = cost, chunks = (int)n;
  }
  return chunks;
}

size_t beam_workspace_bytes(int64_t rows, int chunks, int keep) {
  return (size_t)(rows * chunks) * (sizeof(BeamChunk) + (size_t)keep * sizeof(uint64_t));
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
