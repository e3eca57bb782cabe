// spt_kv.cu -- the 4-bit KV cache: quantising rows as they are written,
// reading them back, and the beam reorder (spt_kv.cuh has the format and the
// layout).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "spt_device.cuh"
#include "spt_internal.cuh"
#include "spt_kv.cuh"

namespace spt {
namespace {

constexpr int kKvThreads = 256, kKvWarps = kKvThreads / 32;

// A warp's work: the new rows of a sequence that fall into one 16-token tile,
// for one head, keys or values.  Tiles are numbered so that a search finds
// them: sequence b has the slots from offsets[b] / 16 + 2 b on, which are as
// many as its rows can need wherever they start (n / 16 + 2).
struct KvUnit {
  int seq, tile, lo, hi;  // tokens [lo, hi) of the tile are new
  int row;                // of token lo
};
inline int64_t kv_slots(const KvRows &r) {
  return r.offsets ? r.tokens / kKvTile + 2 * r.sequences + 1 : r.sequences < r.tokens ? r.sequences : r.tokens;
}
// (slots fit 31 bits: the callers' row counts are checked for it)
__device__ __forceinline__ bool kv_unit(const KvRows &r, uint32_t slot, KvUnit *u) {
  int len, start, n;
  uint32_t first;  // the slot, counted from the sequence's first
  if (!r.offsets) {
    if (slot >= r.sequences || slot >= r.tokens) return false;
    u->seq = (int)slot;
    len = r.lengths[slot], start = (int)slot, n = 1, first = 0;
  } else {
    // the last sequence whose slots start at or before `slot`: 32 of them are looked at at once
    uint32_t lo = 0;
    for (uint32_t left = (uint32_t)r.sequences; left > 1;) {
      const uint32_t step = (left + 31) >> 5, at = lo + (threadIdx.x & 31) * step;
      const bool before = at < lo + left && (uint32_t)(r.offsets[at] >> 4) + 2 * at <= slot;
      const int hits = __popc(__ballot_sync(0xffffffffu, before));
      if (hits == 0) return false;
      const uint32_t past = (uint32_t)(hits - 1) * step;
      lo += past;
      left = min(left - past, step);
    }
    u->seq = (int)lo;
    len = r.lengths[lo], start = r.offsets[lo];
    const int end = r.offsets[lo + 1];
    if (start < 0 || end > r.tokens || end <= start) return false;
    n = end - start;
    first = slot - ((uint32_t)start / kKvTile + 2 * lo);
    if (first > (uint32_t)n / kKvTile + 1) return false;  // (before the first slot: beyond any)
  }
  const int64_t pos0 = (int64_t)len - n;  // (rows before position 0 have no place)
  const uint32_t p0 = pos0 > 0 ? (uint32_t)pos0 : 0, tile = p0 / kKvTile + first, from = tile * kKvTile;
  const int64_t lo = from > p0 ? from : p0, hi = len < (int64_t)from + kKvTile ? len : (int64_t)from + kKvTile;
  u->tile = (int)tile;
  u->lo = (int)lo;
  u->hi = (int)hi;
  u->row = start + (int)(lo - pos0);
  return lo < hi;
}

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float(float v) { return v; }
template <>
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }

// N consecutive elements, 4 or 8; VEC: they start on as many bytes as they have.
template <typename T, int N, bool VEC>
__device__ __forceinline__ void load_n(const T *p, float (&x)[N]) {
  if constexpr (VEC && N * sizeof(T) == 32) {
    asm("ld.global.L1::no_allocate.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
        : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7])
        : "l"(p)
        : "memory");
  } else if constexpr (VEC) {
    constexpr int B = N * (int)sizeof(T);  // 8, 16 or 32 bytes
    using W = typename std::conditional<B == 8, uint2, uint4>::type;
    W w[B / sizeof(W)];
#pragma unroll
    for (int i = 0; i < B / (int)sizeof(W); ++i) w[i] = __ldcs(reinterpret_cast<const W *>(p) + i);
    const T *e = reinterpret_cast<const T *>(w);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_float<T>(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_float<T>(p[i]);
  }
}
template <typename T, int N, bool VEC>
__device__ __forceinline__ void store_n(T *p, const float (&x)[N]) {
  if constexpr (VEC && N * sizeof(T) == 32) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]),
                 "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
                 : "memory");
  } else if constexpr (VEC) {
    constexpr int B = N * (int)sizeof(T);
    using W = typename std::conditional<B == 8, uint2, uint4>::type;
    W w[B / sizeof(W)];
    T *e = reinterpret_cast<T *>(w);
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = from_float<T>(x[i]);
#pragma unroll
    for (int i = 0; i < B / (int)sizeof(W); ++i) __stcs(reinterpret_cast<W *>(p) + i, w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = from_float<T>(x[i]);
  }
}

// Scale and codes of a block held by four neighbouring lanes, eight values
// each; nibble i of the result is value i of this lane, `quarter` the lane's
// place in the block.
__device__ __forceinline__ uint32_t kv_quantise(const float (&x)[8], int quarter, __half *scale) {
  constexpr int N = 8;
  float high = x[0], low = x[0];
  int nan = isnan(x[0]);
#pragma unroll
  for (int i = 1; i < N; ++i) {
    nan |= isnan(x[i]);
    high = fmaxf(high, x[i]), low = fminf(low, x[i]);
  }
#pragma unroll
  for (int m = 1; m < 4; m <<= 1) {
    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, m));
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, m));
    nan |= __shfl_xor_sync(0xffffffffu, nan, m);
  }
  float top = high >= -low ? high : low;
  if (__any_sync(0xffffffffu, high == -low)) {  // both signs have the largest magnitude: the first element that has it
    int at = 2 * 32;  // twice its place, and one more where it is negative
#pragma unroll
    for (int i = N - 1; i >= 0; --i)
      if (fabsf(x[i]) == high) at = 2 * (quarter * N + i) + (x[i] < 0.0f);
#pragma unroll
    for (int m = 1; m < 4; m <<= 1) at = min(at, __shfl_xor_sync(0xffffffffu, at, m));
    if (high == -low) top = at & 1 ? low : high;
  }
  const float wide = fminf(fmaxf(top * -0.125f, -65504.0f), 65504.0f);
  const __half d = nan ? __ushort_as_half(0x7fff) : __float2half_rn(wide);
  *scale = d;
  const float step = __half2float(d);
  const float inv = step != 0.0f && !nan ? __fdiv_rn(1.0f, step) : 0.0f;
  // x * inv is within 8.5 * 2^-23 of the quotient: its rounding is the
  // quotient's unless it lies that near a half.  Adding 1.5 * 2^23 rounds to
  // even, and leaves the integer in the low bits.
  constexpr float kMagic = 12582912.0f;
  float k[N], near = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float q = fminf(fmaxf(__fmul_rn(x[i], inv), -8.0f), 7.0f);  // (a NaN becomes -8; its block has no codes)
    k[i] = __fadd_rn(q, kMagic);
    near = fmaxf(near, fabsf(__fsub_rn(q, __fsub_rn(k[i], kMagic))));
  }
  uint32_t codes = 0;
  if (__any_sync(0xffffffffu, near > 0.499996f)) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      // the remainder x - n d is exact; beyond half a step, or on it with an odd n, the next n is right
      float n = __fsub_rn(k[i], kMagic);
      const float e = __fmaf_rn(-n, step, x[i]);
      const float over = __fsub_rn(2.0f * fabsf(e), fabsf(step));
      if (over > 0.0f || (over == 0.0f && (__float_as_uint(k[i]) & 1u)))
        n = __fadd_rn(n, (e < 0.0f) == (step < 0.0f) ? 1.0f : -1.0f);
      k[i] = __fadd_rn(fminf(fmaxf(n, -8.0f), 7.0f), kMagic);
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) codes |= ((__float_as_uint(k[i]) + 8u) & 15u) << (4 * i);
  return nan || step == 0.0f ? 0x88888888u >> (32 - 4 * N) : codes;
}

struct KvMove {
  KvLayer c;
  KvRows r;
  const void *src[2];
  void *dst[2];
  int64_t stride[2];
  int64_t units;
};

// This warp's unit and its tile's record; null where there is nothing to do.
__device__ __forceinline__ uint8_t *kv_record(const KvMove &a, KvUnit *u, int *head) {
  const int64_t id = (int64_t)blockIdx.x * kKvWarps + (threadIdx.x >> 5);
  if (id >= a.units) return nullptr;
  const uint32_t slot = (uint32_t)id / (uint32_t)a.c.kv_heads;
  *head = (int)((uint32_t)id - slot * a.c.kv_heads);
  if (!kv_unit(a.r, slot, u)) return nullptr;
  const int tiles = a.c.page_tokens / kKvTile, entry = (int)((uint32_t)u->tile / (uint32_t)tiles);
  if (entry >= a.r.max_pages) return nullptr;
  const int64_t page = a.r.table[u->seq * a.r.max_pages + entry];
  if (page < 0 || page >= a.c.pages) return nullptr;
  return a.c.base + kv_tile_offset(a.c, page, *head, (u->tile - entry * tiles) * kKvTile);
}

// Rows are read once and the records written once; bound by instructions on the
// way, 29 for a value of each lane, and in small calls by latency (24 prompts,
// 17,700 f32 tokens of 8 heads of 64 dims: 27 us under a profiler, 3.1 TB/s, at
// 0.68 instructions a clock).  A tile is a warp's, as its record is what the attention reads
// whole.  Lane 4 g +
// t quantises dims 8 t on of each block of tokens g and g + 8; that is the
// keys' layout, and for the values' two lanes' words are exchanged for their
// halves.  A tile whose 16 tokens are all new leaves as 16-byte pieces; else
// every token's codes are stored by themselves.
template <typename T, int NB, bool VEC>
__global__ void __launch_bounds__(kKvThreads) k_kv_append(const KvMove a) {
  pdl_wait();
  pdl_trigger();
  KvUnit u;
  int head;
  uint8_t *const rec = kv_record(a, &u, &head);
  if (!rec) return;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const bool value = blockIdx.y != 0;
  const int first = u.lo - u.tile * kKvTile, end = u.hi - u.tile * kKvTile;  // new tokens of the tile
  const bool all = end - first == kKvTile;
  const int64_t stride = value ? a.stride[1] : a.stride[0];
  const T *src = static_cast<const T *>(value ? a.src[1] : a.src[0]) + (int64_t)(u.row - first) * stride + head * (NB * 32);
  float x[NB][2][8];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int token = g + 8 * h;
      if (token >= first && token < end) load_n<T, 8, VEC>(src + token * stride + b * 32 + t * 8, x[b][h]);
      else
#pragma unroll
        for (int i = 0; i < 8; ++i) x[b][h][i] = 0.0f;
    }
  uint32_t w[NB][2];
  uint8_t *const codes = rec + (value ? kv_value_codes(NB) : 0), *const scales = rec + (value ? kv_value_scales(NB) : kv_key_scales(NB));
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int token = g + 8 * h;
      __half d;
      w[b][h] = kv_quantise(x[b][h], t, &d);
      if (t == 0 && token >= first && token < end) *reinterpret_cast<__half *>(scales + kv_scale(NB, b, token)) = d;
    }
  if (value) {
    // this lane's word: dims 4 g on of tokens 2 t and 2 t + 1, from the lanes of those with dims 8 (g / 2) on
    const int from = 8 * t + (g >> 1);
    const uint32_t halves = g & 1 ? 0x7632u : 0x5410u;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t even = __shfl_sync(0xffffffffu, w[b][h], from), odd = __shfl_sync(0xffffffffu, w[b][h], from + 4);
        w[b][h] = __byte_perm(even, odd, halves);
      }
  }
  if (all) {
#pragma unroll
    for (int b = 0; b + 1 < NB; b += 2)
      *reinterpret_cast<uint4 *>(codes + kv_word(NB, b, lane, 0)) = make_uint4(w[b][0], w[b][1], w[b + 1][0], w[b + 1][1]);
    if constexpr (NB % 2 == 1)
      *reinterpret_cast<uint2 *>(codes + kv_word(NB, NB - 1, lane, 0)) = make_uint2(w[NB - 1][0], w[NB - 1][1]);
    return;
  }
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint8_t *to = codes + kv_word(NB, b, lane, h);
      auto is_new = [&](int token) { return token >= first && token < end; };
      if (!value) {
        if (is_new(g + 8 * h)) *reinterpret_cast<uint32_t *>(to) = w[b][h];
      } else {
        if (is_new(2 * t + 8 * h)) *reinterpret_cast<uint16_t *>(to) = (uint16_t)w[b][h];
        if (is_new(2 * t + 1 + 8 * h)) *reinterpret_cast<uint16_t *>(to + 2) = (uint16_t)(w[b][h] >> 16);
      }
    }
}

// (n - 8) d of the code n in nibble P (2 to 4) of a word, in two instructions:
// the nibble in the mantissa of 2^E, E = 23 - 4 P, makes the float 2^E + n, and
// (2^E + n) d - (2^E + 8) d is exact, as (2^E + 8) d has 23 bits at most.
struct KvScale {
  float d, off[3];
  __device__ __forceinline__ explicit KvScale(float scale) : d(scale) {
#pragma unroll
    for (int i = 0; i < 3; ++i) off[i] = -((float)(1 << (15 - 4 * i)) + 8.0f) * scale;
  }
  template <int P>
  __device__ __forceinline__ float times(uint32_t word) const {
    return __fmaf_rn(__uint_as_float((word & 15u << (4 * P)) | (uint32_t)(127 + 23 - 4 * P) << 23), d, off[P - 2]);
  }
};

// The records are read once and the rows written once: 18 us under a profiler for
// the tokens above, 4.6 TB/s, at 0.62 instructions a clock.  Keys and values are
// different warps': by one warp in turn, a beam search step with four layers' reads
// took 88 us instead of 82, bound by the latency of finding a warp's rows.
template <typename T, int NB, bool VEC>
__global__ void __launch_bounds__(kKvThreads) k_kv_read(const KvMove a) {
  pdl_wait();
  pdl_trigger();
  const bool value = blockIdx.y != 0;
  void *const out = value ? a.dst[1] : a.dst[0];
  KvUnit u;
  int head;
  const uint8_t *const rec = out ? kv_record(a, &u, &head) : nullptr;
  if (!rec) return;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int first = u.lo - u.tile * kKvTile, end = u.hi - u.tile * kKvTile;
  const int64_t stride = value ? a.stride[1] : a.stride[0];
  T *dst = static_cast<T *>(out) + (int64_t)(u.row - first) * stride + head * (NB * 32);
  uint2 w[NB], s[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    w[b] = *reinterpret_cast<const uint2 *>(rec + (value ? kv_value_codes(NB) : 0) + kv_word(NB, b, lane, 0));
    // the four scales of this lane's tokens: 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of values, those of g & ~1 for keys
    s[b] = *reinterpret_cast<const uint2 *>(rec + (value ? kv_value_scales(NB) : kv_key_scales(NB)) +
                                               (value ? t : g >> 1) * NB * 8 + b * 8);
  }
  auto scale_of = [&](int b, int h, int odd) {
    const uint32_t pair = h ? s[b].y : s[b].x;
    return __half2float(__ushort_as_half((unsigned short)(odd ? pair >> 16 : pair)));
  };
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t word = h ? w[b].y : w[b].x;
      if (!value) {
        const int token = g + 8 * h;
        if (token < first || token >= end) continue;
        const KvScale d(scale_of(b, h, g & 1));
        const uint32_t up = word << 8, down = word >> 12;
        const float x[8] = {d.times<2>(up),   d.times<3>(up),   d.times<2>(word), d.times<3>(word),
                            d.times<4>(word), d.times<2>(down), d.times<3>(down), d.times<4>(down)};
        store_n<T, 8, VEC>(dst + token * stride + b * 32 + t * 8, x);
      } else {
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
          const int token = 2 * t + odd + 8 * h;
          if (token < first || token >= end) continue;
          const KvScale d(scale_of(b, h, odd));
          const uint32_t low = odd ? word >> 8 : word << 8, high = odd ? word >> 16 : word;
          const float x[4] = {d.times<2>(low), d.times<3>(low), d.times<2>(high), d.times<3>(high)};
          store_n<T, 4, VEC>(dst + token * stride + b * 32 + g * 4, x);
        }
      }
    }
}

// Accesses of eight elements need rows that start on as many bytes (a head's
// share is a multiple of 64 bytes in every type).
bool vectors(const void *p, int64_t stride, int size) {
  return reinterpret_cast<uintptr_t>(p) % (8 * size) == 0 && stride % 8 == 0;
}

template <typename T, int NB>
cudaError_t launch_blocks(const KvMove &a, bool append, cudaStream_t stream) {
  const dim3 grid((unsigned)((a.units + kKvWarps - 1) / kKvWarps), 2), block(kKvThreads);
  bool vec = true;
  for (int i = 0; i < 2; ++i) vec = vec && vectors(append ? a.src[i] : a.dst[i], a.stride[i], sizeof(T));
  if (append)
    return vec ? launch_pdl(k_kv_append<T, NB, true>, grid, block, 0, stream, a)
               : launch_pdl(k_kv_append<T, NB, false>, grid, block, 0, stream, a);
  return vec ? launch_pdl(k_kv_read<T, NB, true>, grid, block, 0, stream, a)
             : launch_pdl(k_kv_read<T, NB, false>, grid, block, 0, stream, a);
}

template <typename T>
cudaError_t launch_move(const KvMove &a, bool append, cudaStream_t stream) {
  switch (a.c.nb) {
    case 1: return launch_blocks<T, 1>(a, append, stream);
    case 2: return launch_blocks<T, 2>(a, append, stream);
    case 3: return launch_blocks<T, 3>(a, append, stream);
    case 4: return launch_blocks<T, 4>(a, append, stream);
  }
  return cudaErrorInvalidValue;
}

cudaError_t launch_typed(KvMove a, int type, bool append, cudaStream_t stream) {
  if (a.r.tokens <= 0 || a.r.sequences <= 0) return cudaSuccess;
  a.units = kv_slots(a.r) * a.c.kv_heads;
  if (a.units > 0x7fffffffll) return cudaErrorInvalidValue;
  switch (type) {
    case kKvF32: return launch_move<float>(a, append, stream);
    case kKvF16: return launch_move<__half>(a, append, stream);
    case kKvBF16: return launch_move<__nv_bfloat16>(a, append, stream);
  }
  return cudaErrorInvalidValue;
}

// One CTA row per sequence (blockIdx.x) and share of the copy (blockIdx.y).
// A child takes its parent's whole pages by number; the parent's partial last
// page goes to its first child, every later child gets a copy of the tiles in
// use, on every layer.  Bound by latency: a chain of table look-ups before a copy
// of a few KB (128 beams, 4 layers: 9.4 us alone; a launch that copies nothing
// takes about 4).
__global__ void __launch_bounds__(kKvThreads) k_kv_reorder(uint8_t *pool, int64_t layers, int64_t layer_bytes,
                                                          const KvLayer c, const KvReorder a) {
  pdl_wait();
  pdl_trigger();
  const int64_t s = blockIdx.x, b = s / a.beams, j = s - b * a.beams;
  const int32_t *parents = a.parents + b * a.parents_stride;
  const int64_t parent = parents[j];
  const bool valid = parent >= 0 && parent < a.beams;
  const int64_t from = valid ? b * a.beams + parent : 0;
  int64_t len = valid ? a.lengths[from] : 0;
  len = len < 0 ? 0 : len > a.max_pages * c.page_tokens ? a.max_pages * c.page_tokens : len;
  const int64_t full = (uint32_t)len / (uint32_t)c.page_tokens;  // (len is an int32)
  const int rest = (int)(len - full * c.page_tokens);
  bool later = false;
  for (int64_t i = 0; i < j; ++i) later |= parents[i] == parent;
  const int64_t old = rest ? a.table[from * a.max_pages + full] : -1;
  // a page outside the pool has nothing to copy: every child keeps its number, and no spare page is taken
  const bool held = old >= 0 && old < c.pages;
  const int64_t own = later && held ? a.spare[s] : old;
  const bool copy = rest && later && held && own >= 0 && own < c.pages;
  if (blockIdx.y == 0) {
    for (int64_t i = threadIdx.x; i < a.max_pages; i += kKvThreads)
      a.table_out[s * a.max_pages + i] =
          i < full ? a.table[from * a.max_pages + i] : i == full && rest ? (int32_t)own : -1;
    if (threadIdx.x == 0) {
      a.lengths_out[s] = (int32_t)len;
      if (a.copied) a.copied[s] = copy;
    }
  }
  if (!copy || old == own) return;
  const int per_head = (rest + kKvTile - 1) / kKvTile * (kv_tile_bytes(c.nb) / 16);  // 16-byte words
  const uint32_t words = (uint32_t)layers * c.kv_heads * per_head;
  for (uint32_t w = blockIdx.y * kKvThreads + threadIdx.x; w < words; w += gridDim.y * kKvThreads) {
    const uint32_t lh = w / per_head, layer = lh / c.kv_heads;
    const int head = (int)(lh - layer * c.kv_heads), at = (int)(w - lh * per_head);
    uint8_t *base = pool + layer * layer_bytes + (int64_t)at * 16;
    *reinterpret_cast<uint4 *>(base + kv_tile_offset(c, own, head, 0)) =
        *reinterpret_cast<const uint4 *>(base + kv_tile_offset(c, old, head, 0));
  }
}

}  // namespace

cudaError_t launch_kv_append(const KvLayer &c, const KvRows &r, int type, const void *k, int64_t k_stride,
                             const void *v, int64_t v_stride, cudaStream_t stream) {
  const KvMove a = {c, r, {k, v}, {nullptr, nullptr}, {k_stride, v_stride}, 0};
  return launch_typed(a, type, true, stream);
}

cudaError_t launch_kv_read(const KvLayer &c, const KvRows &r, int type, void *k, int64_t k_stride, void *v,
                           int64_t v_stride, cudaStream_t stream) {
  const KvMove a = {c, r, {nullptr, nullptr}, {k, v}, {k_stride, v_stride}, 0};
  return launch_typed(a, type, false, stream);
}

cudaError_t launch_kv_reorder(uint8_t *pool, int64_t layers, int64_t layer_bytes, const KvLayer &c,
                              const KvReorder &r, cudaStream_t stream) {
  const int64_t rows = r.batch * r.beams;
  if (rows <= 0) return cudaSuccess;
  if (rows > 0x7fffffffll) return cudaErrorInvalidValue;
  // a page's bytes over 16 KB a CTA, at most 64 CTAs a sequence
  const int64_t page = layers * c.kv_heads * (c.page_tokens / kKvTile) * (int64_t)kv_tile_bytes(c.nb);
  const int64_t parts = page / 16384 < 1 ? 1 : page / 16384 > 64 ? 64 : page / 16384;
  return launch_pdl(k_kv_reorder, dim3((unsigned)rows, (unsigned)parts), dim3(kKvThreads), 0, stream, pool, layers,
                    layer_bytes, c, r);
}

}  // namespace spt
