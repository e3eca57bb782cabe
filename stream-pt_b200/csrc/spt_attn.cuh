// spt_attn.cuh -- what the attention kernels share: a CTA's share of a ragged
// batch, the cache's codes as f16 pairs, and a row's end.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "spt_device.cuh"
#include "spt_internal.cuh"
#include "spt_kv.cuh"
#include "spt_ptx.cuh"

namespace spt {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t bits(__half2 v) { return *reinterpret_cast<uint32_t *>(&v); }
__device__ __forceinline__ __half2 half2_of(uint32_t v) { return *reinterpret_cast<__half2 *>(&v); }
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) { return bits(__floats2half2_rn(lo, hi)); }

// The eight codes of a word as four f16 pairs of n - 8, exactly: pair i holds
// nibbles i and i + 4.  A nibble under the exponent of 1024 is 1024 + n (or,
// four bits higher, 1024 + 16 n).
__device__ __forceinline__ void decode_word(uint32_t w, uint32_t (&e)[4]) {
  const __half2 low = half2_of(0x64086408u);                      // 1032
  const __half2 sixteenth = half2_of(0x2c002c00u), off = half2_of(0xd480d480u);  // 1/16, -72
  const uint32_t v = w >> 8;
  e[0] = bits(__hsub2(half2_of((w & 0x000f000fu) | 0x64006400u), low));
  e[1] = bits(__hfma2(half2_of((w & 0x00f000f0u) | 0x64006400u), sixteenth, off));
  e[2] = bits(__hsub2(half2_of((v & 0x000f000fu) | 0x64006400u), low));
  e[3] = bits(__hfma2(half2_of((v & 0x00f000f0u) | 0x64006400u), sixteenth, off));
}

template <typename IO>
__device__ __forceinline__ float row_float(IO v) {
  if constexpr (sizeof(IO) == 4) return v;
  else return static_cast<float>(v);
}
template <typename IO>
__device__ __forceinline__ IO row_round(float v) {
  if constexpr (sizeof(IO) == 4) return v;
  else if constexpr (std::is_same<IO, __half>::value) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}
// N consecutive elements of a row, N * sizeof(IO) a multiple of 16; `vec`: they
// start on 16 bytes.
template <typename IO, int N>
__device__ __forceinline__ void load_row(const IO *p, bool vec, float (&x)[N]) {
  constexpr int W = N * (int)sizeof(IO) / 16, E = 16 / (int)sizeof(IO);
  if (vec) {
    uint4 w[W];
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = *reinterpret_cast<const uint4 *>(p + i * E);
    const IO *e = reinterpret_cast<const IO *>(w);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = row_float<IO>(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = row_float<IO>(p[i]);
  }
}
// Four consecutive elements; `vec`: they start on 4 * sizeof(IO) bytes.
template <typename IO>
__device__ __forceinline__ void store_row4(IO *p, bool vec, const float (&x)[4]) {
  IO e[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = row_round<IO>(x[i]);
  if (vec) {
    if constexpr (sizeof(IO) == 4) *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(e);
    else *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(e);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = e[i];
  }
}

// A bounded wait for another role of this CTA, short as a rule: the clock and the
// CTA's word for a role that has given up are looked at every 64th try only (an
// error that an earlier call left in a.err ends no wait of this one; the CTA
// records its own there in the end).  One atomic here keeps the sites short: a flag
// in shared memory beside a.err took f16 chunks of 12 sequences from 227 to 245 us.
__device__ __forceinline__ bool brief_wait(uint64_t *bar, uint32_t parity, const AttnArgs &a, int code) {
  if (mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  for (uint32_t i = 1;; ++i) {
    if (mbar_try(bar, parity)) return true;
    if ((i & 63u) == 0u) {
      if (*(volatile int32_t *)(a.gave_up + blockIdx.x)) return false;
      if (clock64() - t0 > (1ll << a.wait_shift)) {
        atomicCAS(a.gave_up + blockIdx.x, 0, code);
        return false;
      }
    }
  }
}

// The same for copies that the calling warp started itself.
__device__ __forceinline__ bool own_wait(uint64_t *bar, uint32_t parity, const AttnArgs &a, int code) {
  if (mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  for (uint32_t i = 1;; ++i) {
    if (mbar_try(bar, parity)) return true;
    if ((i & 63u) == 0u && clock64() - t0 > (1ll << a.wait_shift)) {
      atomicCAS(a.err, 0, code);
      return false;
    }
  }
}

// a / b for non-negative a, which seldom need 64 bits.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return ((uint64_t)a | (uint64_t)b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

// A sequence's new rows.
struct SeqRows {
  int start, len, n;
};
__device__ __forceinline__ SeqRows seq_rows(const AttnArgs &a, int64_t b) {
  SeqRows s;
  s.len = a.r.lengths[b];
  if (s.len < 0) s.len = 0;
  if (!a.r.offsets) {
    s.start = (int)b;
    s.n = b < a.r.tokens ? 1 : 0;
  } else {
    s.start = a.r.offsets[b];
    const int end = a.r.offsets[b + 1];
    s.n = s.start < 0 || end > a.r.tokens || end < s.start ? 0 : end - s.start;
  }
  return s;
}

// Tiles of KEYS keys, [first, last), that row block rb of a sequence sees: a
// block is ROWS consecutive (new row, head of the group) pairs.  [lo, hi) are the
// keys that any of its rows sees.
struct KeyTiles {
  int first, last, lo, hi;
};
template <int ROWS, int KEYS>
__device__ __forceinline__ KeyTiles key_tiles(const AttnArgs &a, const SeqRows &s, int rb) {
  // (tokens * group is below 2^31: launch_attention)
  const int i0 = (int)((uint32_t)(rb * ROWS) / (uint32_t)a.group);
  int i1 = (int)(((uint32_t)(rb * ROWS) + ROWS - 1) / (uint32_t)a.group);
  if (i1 > s.n - 1) i1 = s.n - 1;
  int64_t hi = (int64_t)s.len - s.n + i1 + 1;
  const int64_t cap = a.r.max_pages * a.c.page_tokens;
  if (hi > cap) hi = cap;
  int64_t lo = a.window > 0 ? (int64_t)s.len - s.n + i0 - a.window + 1 : 0;
  if (lo < 0) lo = 0;
  KeyTiles t = {0, 0, 0, 0};
  if (hi > lo) t.first = (int)(lo / KEYS), t.last = (int)((hi + KEYS - 1) / KEYS), t.lo = (int)lo, t.hi = (int)hi;
  return t;
}
template <int ROWS>
__device__ __forceinline__ int row_blocks(const AttnArgs &a, const SeqRows &s) {
  return (int)(((uint32_t)(s.n * a.group) + ROWS - 1) / ROWS);
}

// The walk of a CTA or a warp over its share of the work.  Items are (sequence, key head, row
// block), in that order; an item counts HEAD units for its beginning and end
// and one for each of its key tiles.  All items' units in a row are cut into
// equal shares, one a CTA (or warp), so ragged batches load every SM alike and
// a long sequence is split over all of them.
template <int ROWS, int KEYS, int HEAD>
struct AttnWalk {
  int64_t unit, item_begin, end, share;
  int b, rb, head;
  SeqRows seq;
  KeyTiles tiles;

  __device__ static int cost(const KeyTiles &t) { return t.last - t.first + HEAD; }
  // Units of row blocks [from, to) of a head, every step-th.
  __device__ static int64_t block_units(const AttnArgs &a, const SeqRows &s, int from, int to, int step) {
    int64_t u = 0;
    for (int i = from; i < to; i += step) u += cost(key_tiles<ROWS, KEYS>(a, s, i));
    return u;
  }
  __device__ static int64_t warp_sum(int64_t v) {
#pragma unroll
    for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
  }
  __device__ static int64_t warp_scan(int64_t v, int lane) {
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const int64_t o = __shfl_up_sync(0xffffffffu, v, m);
      if (lane >= m) v += o;
    }
    return v;
  }

  // Finds share `index` of `count` (the same for a warp's threads; every thread of
  // the CTA takes part); false where it is empty.  Sequences are weighed THREADS
  // at a time: by a thread each where they have a row block or two, by a warp
  // each where they have many.
  template <int THREADS>
  __device__ bool begin(const AttnArgs &a, int64_t min_share, int index, int count) {
    constexpr int WARPS = THREADS / 32;
    __shared__ int64_t scratch[WARPS];
    __shared__ int64_t weight[THREADS], before_of[THREADS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool wide = a.r.tokens * a.group > 2 * ROWS * a.r.sequences;
    auto weigh = [&](int64_t b0) {  // units of sequence b0 + tid
      if (!wide) {
        if (b0 + tid >= a.r.sequences) return (int64_t)0;
        const SeqRows s = seq_rows(a, b0 + tid);
        return block_units(a, s, 0, row_blocks<ROWS>(a, s), 1) * a.c.kv_heads;
      }
      for (int64_t i = b0 + warp; i < b0 + THREADS && i < a.r.sequences; i += WARPS) {
        const SeqRows s = seq_rows(a, i);
        const int64_t u = warp_sum(block_units(a, s, lane, row_blocks<ROWS>(a, s), 32)) * a.c.kv_heads;
        if (lane == 0) weight[i - b0] = u;
      }
      __syncthreads();
      const int64_t mine = b0 + tid < a.r.sequences ? weight[tid] : 0;
      __syncthreads();
      return mine;
    };
    // sums over the warps before this one, and over all
    auto block_scan = [&](int64_t up, int64_t *all) {
      if (lane == 31) scratch[warp] = up;
      __syncthreads();
      int64_t sum = 0, below = 0;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        if (w == warp) below = sum;
        sum += scratch[w];
      }
      __syncthreads();
      *all = sum;
      return below;
    };
    const int64_t mine = weigh(0);
    int64_t total = mine;
    for (int64_t b0 = THREADS; b0 < a.r.sequences; b0 += THREADS) total += weigh(b0);
    block_scan(warp_sum(total), &total);
    share = quotient(total + count - 1, count);
    if (share < min_share) share = min_share;
    unit = (int64_t)index * share;
    end = unit + share < total ? unit + share : total;
    int64_t per_head = 1, before = 0;
    b = -1;
    for (int64_t b0 = 0; b0 < a.r.sequences; b0 += THREADS) {
      const int64_t v = b0 == 0 ? mine : weigh(b0);
      const int64_t up = warp_scan(v, lane);
      int64_t all;
      const int64_t below = block_scan(up, &all);
      weight[tid] = v;
      before_of[tid] = before + below + up - v;
      __syncthreads();
      if (b < 0 && unit >= before && unit < before + all)  // the sequence that holds `unit`
        for (int i = 0; i < WARPS; ++i) {
          const int64_t at = before_of[i * 32 + lane], n = weight[i * 32 + lane];
          const uint32_t hit = __ballot_sync(0xffffffffu, unit >= at && unit < at + n);
          if (hit) {
            const int x = i * 32 + __ffs(hit) - 1;
            b = (int)(b0 + x);
            item_begin = before_of[x];
            per_head = quotient(weight[x], a.c.kv_heads);
            break;
          }
        }
      before += all;
      __syncthreads();
    }
    if (unit >= total) return false;
    seq = seq_rows(a, b);
    head = (int)quotient(unit - item_begin, per_head);
    item_begin += head * per_head;
    // the row block that holds `unit`: 32 at a time
    const int blocks = row_blocks<ROWS>(a, seq);
    for (rb = 0;; rb += 32) {
      const int64_t v = rb + lane < blocks ? cost(key_tiles<ROWS, KEYS>(a, seq, rb + lane)) : 0;
      const int64_t up = warp_scan(v, lane);
      const int64_t all = __shfl_sync(0xffffffffu, up, 31);
      if (item_begin + all > unit || rb + 32 >= blocks) {
        const uint32_t behind = __ballot_sync(0xffffffffu, item_begin + up > unit);
        const int at = behind ? __ffs(behind) - 1 : 0;
        item_begin += __shfl_sync(0xffffffffu, up - v, at);
        rb += at;
        break;
      }
      item_begin += all;
    }
    tiles = key_tiles<ROWS, KEYS>(a, seq, rb);
    return true;
  }

  // This share's part of the current item: units, and tiles [first_tile(), last_tile()).
  __device__ int units() const { return cost(tiles); }
  __device__ int take() const {
    const int left = units() - (int)(unit - item_begin);
    return left < end - unit ? left : (int)(end - unit);
  }
  __device__ int tile_at(int64_t u) const {
    const int past = (int)(u - item_begin) - HEAD;
    return tiles.first + (past > 0 ? past : 0);
  }
  __device__ int first_tile() const { return tile_at(unit); }
  __device__ int last_tile() const { return tile_at(unit + take()); }
  __device__ bool whole() const { return take() == units(); }
  __device__ int first_share() const { return (int)quotient(item_begin, share); }
  __device__ int last_share() const { return (int)quotient(item_begin + units() - 1, share); }

  __device__ bool next(const AttnArgs &a) {
    const int t = take();
    item_begin += units();
    unit += t;
    if (unit >= end) return false;
    if (++rb >= row_blocks<ROWS>(a, seq)) {
      rb = 0;
      if (++head >= a.c.kv_heads) {
        head = 0;
        do seq = seq_rows(a, ++b);
        while (seq.n == 0);
      }
    }
    tiles = key_tiles<ROWS, KEYS>(a, seq, rb);
    return true;
  }
};

// An item in several shares: the first keeps its part in its slot 1, every
// other in its slot 0; the last to arrive joins the parts in the order of the
// shares, so that the order of arrival changes nothing.
template <int ROWS, int DIM>
__device__ __forceinline__ float *part_slot(const AttnArgs &a, int share, int first) {
  return a.partial + ((int64_t)share * 2 + (share == first)) * (ROWS * (DIM + 2));
}
// Counts a part; whether it was the last.
template <typename Walk>
__device__ __forceinline__ bool arrive(const AttnArgs &a, const Walk &w) {
  const int first = w.first_share();
  const bool last = atomicAdd(&a.arrive[first], 1) == w.last_share() - first;
  if (last) a.arrive[first] = 0;
  return last;
}

// What a row's sums, which stand for 2^ref times their value, are multiplied by
// in the end; 0 where the row has seen nothing.
__device__ __forceinline__ float row_factor(const AttnArgs &a, int head, float ref, float l) {
  float up = 1.0f, below = l;
  if (a.sinks) {
    const float sink = a.sinks[head] * kLog2e;
    const float top = fmaxf(ref, sink);
    if (top > -INFINITY) {
      up = exp2f(ref - top);
      below = l * up + exp2f(sink - top);
    }
    if (!(sink < INFINITY)) below = sink;  // (infinite: every weight is 0)
  }
  return below == 0.0f ? 0.0f : up / below;
}

}  // namespace
}  // namespace spt
