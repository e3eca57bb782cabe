// spt_kv.cu -- the 4-bit KV cache: quantising rows as they are written,
// reading them back, and the beam reorder (spt_kv.cuh has the format and the
// layout).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "spt_device.cuh"
#include "spt_internal.cuh"
#include "spt_kv.cuh"

namespace spt {
namespace {

constexpr int kKvThreads = 256;
constexpr int kKvSpan = 8;  // values a thread quantises; four threads share a block

// Sequence and position of a new row; false where the row belongs to none or
// its position has no place in the table.
__device__ __forceinline__ bool kv_locate(const KvRows &r, int64_t row, int64_t places, int64_t *seq, int64_t *pos) {
  if (!r.offsets) {
    if (row >= r.sequences) return false;
    *seq = row;
    *pos = (int64_t)r.lengths[row] - 1;
  } else {
    if (row < r.offsets[0] || row >= r.offsets[r.sequences]) return false;
    int64_t lo = 0, hi = r.sequences - 1;  // the first sequence whose rows end behind `row`
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (r.offsets[mid + 1] > row) hi = mid;
      else lo = mid + 1;
    }
    *seq = lo;
    *pos = (int64_t)r.lengths[lo] - r.offsets[lo + 1] + row;
  }
  return *pos >= 0 && *pos < places;
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

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T *p, float (&x)[kKvSpan]) {
  if constexpr (VEC) {
    constexpr int W = sizeof(T) * kKvSpan / 16;
    uint4 w[W];
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
    const T *e = reinterpret_cast<const T *>(w);
#pragma unroll
    for (int i = 0; i < kKvSpan; ++i) x[i] = to_float<T>(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kKvSpan; ++i) x[i] = to_float<T>(p[i]);
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T *p, const float (&x)[kKvSpan]) {
  if constexpr (VEC) {
    constexpr int W = sizeof(T) * kKvSpan / 16;
    uint4 w[W];
    T *e = reinterpret_cast<T *>(w);
#pragma unroll
    for (int i = 0; i < kKvSpan; ++i) e[i] = from_float<T>(x[i]);
#pragma unroll
    for (int i = 0; i < W; ++i) __stcs(reinterpret_cast<uint4 *>(p) + i, w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kKvSpan; ++i) p[i] = from_float<T>(x[i]);
  }
}

// Scale and codes of a block held by four neighbouring lanes, eight values
// each; nibble i of the result is value i of this lane.
__device__ __forceinline__ uint32_t kv_quantise(const float (&x)[kKvSpan], int quarter, __half *scale) {
  float top = x[0];
  bool nan = isnan(x[0]);
  int at = 0;
#pragma unroll
  for (int i = 1; i < kKvSpan; ++i) {
    nan |= isnan(x[i]);
    if (fabsf(x[i]) > fabsf(top)) top = x[i], at = i;
  }
  at += quarter * kKvSpan;
  int any = nan;
#pragma unroll
  for (int m = 1; m < 4; m <<= 1) {
    const float o = __shfl_xor_sync(0xffffffffu, top, m);
    const int oat = __shfl_xor_sync(0xffffffffu, at, m);
    any |= __shfl_xor_sync(0xffffffffu, any, m);
    if (fabsf(o) > fabsf(top) || (fabsf(o) == fabsf(top) && oat < at)) top = o, at = oat;
  }
  const float wide = fminf(fmaxf(top * -0.125f, -65504.0f), 65504.0f);
  const __half d = any ? __ushort_as_half(0x7fff) : __float2half_rn(wide);
  *scale = d;
  const float step = __half2float(d);
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < kKvSpan; ++i) {
    const float q = step != 0.0f ? rintf(__fdiv_rn(x[i], step)) : 0.0f;
    const int n = any ? 8 : (int)fminf(fmaxf(q, -8.0f), 7.0f) + 8;
    codes |= (uint32_t)n << (4 * i);
  }
  return codes;
}

struct KvMove {
  KvLayer c;
  KvRows r;
  const void *src[2];
  void *dst[2];
  int64_t stride[2];
};

// One thread: eight consecutive values of one row's key or value (blockIdx.y).
// Bound by memory: each row is read once and 9/16 byte a value written.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kKvThreads) k_kv_append(const KvMove a) {
  pdl_wait();
  pdl_trigger();
  const KvLayer &c = a.c;
  const int per_row = c.kv_heads * c.nb * 4;
  const int64_t id = (int64_t)blockIdx.x * kKvThreads + threadIdx.x;
  const int64_t row = id / per_row;
  const bool value = blockIdx.y != 0;
  int64_t seq = 0, pos = 0;
  bool live = row < a.r.tokens && kv_locate(a.r, row, a.r.max_pages * c.page_tokens, &seq, &pos);
  int64_t page = 0;
  if (live) {
    page = a.r.table[seq * a.r.max_pages + pos / c.page_tokens];
    live = page >= 0 && page < c.pages;
  }
  const int part = (int)(id - row * per_row);
  const int head = part / (c.nb * 4), block = part / 4 % c.nb, quarter = part & 3;
  float x[kKvSpan] = {};
  if (live)
    load8<T, VEC>(static_cast<const T *>(a.src[value]) + row * a.stride[value] +
                      (int64_t)head * c.nb * kKvBlock + block * kKvBlock + quarter * kKvSpan, x);
  __half d;
  const uint32_t codes = kv_quantise(x, quarter, &d);
  if (!live) return;
  const int place = (int)(pos % c.page_tokens), token = place % kKvTile;
  uint8_t *tile = c.base + kv_tile_offset(c, page, head, place);
  if (!value) {
    *reinterpret_cast<uint32_t *>(tile + kv_word(c.nb, block, (token & 7) * 4 + quarter, token >> 3)) = codes;
  } else {
    uint8_t *v = tile + kv_value_codes(c.nb) + 2 * (token & 1);
    const int t = (token & 7) >> 1, h = token >> 3;
    *reinterpret_cast<uint16_t *>(v + kv_word(c.nb, block, (2 * quarter) * 4 + t, h)) = (uint16_t)codes;
    *reinterpret_cast<uint16_t *>(v + kv_word(c.nb, block, (2 * quarter + 1) * 4 + t, h)) = (uint16_t)(codes >> 16);
  }
  if (quarter == 0)
    *reinterpret_cast<__half *>(tile + (value ? kv_value_scales(c.nb) : kv_key_scales(c.nb)) +
                                kv_scale(c.nb, block, token)) = d;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kKvThreads) k_kv_read(const KvMove a) {
  pdl_wait();
  pdl_trigger();
  const KvLayer &c = a.c;
  const int per_row = c.kv_heads * c.nb * 4;
  const int64_t id = (int64_t)blockIdx.x * kKvThreads + threadIdx.x;
  const int64_t row = id / per_row;
  const bool value = blockIdx.y != 0;
  if (!a.dst[value] || row >= a.r.tokens) return;
  int64_t seq, pos;
  if (!kv_locate(a.r, row, a.r.max_pages * c.page_tokens, &seq, &pos)) return;
  const int64_t page = a.r.table[seq * a.r.max_pages + pos / c.page_tokens];
  if (page < 0 || page >= c.pages) return;
  const int part = (int)(id - row * per_row);
  const int head = part / (c.nb * 4), block = part / 4 % c.nb, quarter = part & 3;
  const int place = (int)(pos % c.page_tokens), token = place % kKvTile;
  const uint8_t *tile = c.base + kv_tile_offset(c, page, head, place);
  uint32_t codes;
  if (!value) {
    codes = *reinterpret_cast<const uint32_t *>(tile + kv_word(c.nb, block, (token & 7) * 4 + quarter, token >> 3));
  } else {
    const uint8_t *v = tile + kv_value_codes(c.nb) + 2 * (token & 1);
    const int t = (token & 7) >> 1, h = token >> 3;
    codes = *reinterpret_cast<const uint16_t *>(v + kv_word(c.nb, block, (2 * quarter) * 4 + t, h)) |
            (uint32_t) * reinterpret_cast<const uint16_t *>(v + kv_word(c.nb, block, (2 * quarter + 1) * 4 + t, h)) << 16;
  }
  const float d = __half2float(*reinterpret_cast<const __half *>(
      tile + (value ? kv_value_scales(c.nb) : kv_key_scales(c.nb)) + kv_scale(c.nb, block, token)));
  float x[kKvSpan];
#pragma unroll
  for (int i = 0; i < kKvSpan; ++i) x[i] = (float)((int)(codes >> (4 * i) & 15u) - 8) * d;
  store8<T, VEC>(static_cast<T *>(a.dst[value]) + row * a.stride[value] + (int64_t)head * c.nb * kKvBlock +
                     block * kKvBlock + quarter * kKvSpan, x);
}

// 16-byte accesses need rows that start on 16 bytes (a head's and a thread's
// share are multiples of 16 bytes in every type).
bool vectors(const void *p, int64_t stride, int size) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (stride * size) % 16 == 0;
}

template <typename T>
cudaError_t launch_move(const KvMove &a, bool append, cudaStream_t stream) {
  const int64_t threads = a.r.tokens * a.c.kv_heads * a.c.nb * 4;
  const int64_t blocks = (threads + kKvThreads - 1) / kKvThreads;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)blocks, 2), block(kKvThreads);
  bool vec = true;
  for (int i = 0; i < 2; ++i) vec = vec && vectors(append ? a.src[i] : a.dst[i], a.stride[i], sizeof(T));
  if (append)
    return vec ? launch_pdl(k_kv_append<T, true>, grid, block, 0, stream, a)
               : launch_pdl(k_kv_append<T, false>, grid, block, 0, stream, a);
  return vec ? launch_pdl(k_kv_read<T, true>, grid, block, 0, stream, a)
             : launch_pdl(k_kv_read<T, false>, grid, block, 0, stream, a);
}

cudaError_t launch_typed(const KvMove &a, int type, bool append, cudaStream_t stream) {
  if (a.r.tokens <= 0 || a.r.sequences <= 0) return cudaSuccess;
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
// use, on every layer.
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
  const int64_t full = len / c.page_tokens;
  const int rest = (int)(len - full * c.page_tokens);
  bool later = false;
  for (int64_t i = 0; i < j; ++i) later |= parents[i] == parent;
  const int64_t old = rest ? a.table[from * a.max_pages + full] : -1;
  const int64_t own = later ? a.spare[s] : old;
  const bool copy = rest && later && old >= 0 && old < c.pages && own >= 0 && own < c.pages;
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
  const int64_t words = layers * c.kv_heads * per_head;
  for (int64_t w = (int64_t)blockIdx.y * kKvThreads + threadIdx.x; w < words; w += (int64_t)gridDim.y * kKvThreads) {
    const int64_t lh = w / per_head, layer = lh / c.kv_heads;
    const int head = (int)(lh - layer * c.kv_heads), at = (int)(w - lh * per_head);
    uint8_t *base = pool + layer * layer_bytes + (int64_t)at * 16;
    *reinterpret_cast<uint4 *>(base + kv_tile_offset(c, own, head, 0)) =
        *reinterpret_cast<const uint4 *>(base + kv_tile_offset(c, old, head, 0));
  }
}

}  // namespace

cudaError_t launch_kv_append(const KvLayer &c, const KvRows &r, int type, const void *k, int64_t k_stride,
                             const void *v, int64_t v_stride, cudaStream_t stream) {
  const KvMove a = {c, r, {k, v}, {nullptr, nullptr}, {k_stride, v_stride}};
  return launch_typed(a, type, true, stream);
}

cudaError_t launch_kv_read(const KvLayer &c, const KvRows &r, int type, void *k, int64_t k_stride, void *v,
                           int64_t v_stride, cudaStream_t stream) {
  const KvMove a = {c, r, {nullptr, nullptr}, {k, v}, {k_stride, v_stride}};
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
