// spt_attn.cu -- attention over the 4-bit KV cache (spt_kv.cuh).
//
// For query row i of a sequence (position p), head h and the keys
// max(0, p - window + 1) <= j <= p of its key head:
//
//   s_j = scale * q . k_j,   out = sum_j e^(s_j) v_j / (sum_j e^(s_j) + e^(sink_h))
//
// in one pass over the cache with a running maximum and sum.  A row without
// keys gives 0.
#include "spt_attn.cuh"

namespace spt {
namespace {

constexpr int kAttnWarps = 8;
constexpr int kAttnThreads = kAttnWarps * 32;
constexpr int kAttnStages = 3;
constexpr int kAttnCtasPerSm = 2;
constexpr int kAttnMinTiles = 8;     // a CTA's smallest share of the keys: a tile for each warp
constexpr int kAttnHead = 4;         // an item's beginning and end, in tiles' time
constexpr int kAttnMaxRows = 16;

// D (16 x 8, f32) += A (16 x 16, f16) * B (16 x 8, f16)
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// The work, B = NB blocks of 32 dims, TERMS f16 terms of q and of the softmax
// weights (2 for f32 rows: 22 bits each; 1 for f16 and bf16 rows), NT blocks
// of 8 rows.
//
// Within its share of the 16-key tiles (AttnWalk) a CTA's warps take steps of
// up to KS tiles in turn, each warp with its own cp.async ring and its own
// running maximum and sum; they meet in shared memory at the item's end.
//
// Products.  S (rows x keys) = Q K^T with the rows' two f16 terms stacked
// along M (TERMS 2) or two row blocks stacked (TERMS 1), codes n - 8 exact in
// f16, and the keys' scales applied to the f32 sums of each 32-dim block.
// O^T (dims x rows) = V^T P^T with the values' scales applied to the weights
// of each 32-dim block before their split into f16 terms.  S's fragment is
// the layout that P^T's operand needs.
template <int NB, typename IO, int NT>
struct Attn {
  static constexpr int kTerms = sizeof(IO) == 4 ? 2 : 1;
  static constexpr int kDim = NB * 32, kRows = NT * 8;
  static constexpr int kTile = kv_tile_bytes(NB);
  static constexpr int kSteps = NB <= 2 ? 4 : 2;  // tiles in a step at most
  static constexpr int kRing = kAttnStages * kSteps * kTile;
  static constexpr int kRedBytes = kAttnWarps * kRows * (kDim + 2) * 4;
  static constexpr int kSmem = kAttnWarps * kRing > kRedBytes ? kAttnWarps * kRing : kRedBytes;
  static constexpr int kMinCtas = NB <= 2 && kTerms * NT < 4 ? 2 : 1;
  static constexpr int kQ = kTerms == 2 ? NT : (NT + 1) / 2;  // A operands of 16 rows
};

template <typename IO>
__device__ __forceinline__ void finish4(const AttnArgs &a, int64_t row, int head, int dim, float ref, float l,
                                        const float (&acc)[4], int head_dim) {
  const float f = row_factor(a, head, ref, l);
  const float o[4] = {acc[0] * f, acc[1] * f, acc[2] * f, acc[3] * f};
  store_row4(static_cast<IO *>(a.out) + row * a.out_stride + (int64_t)head * head_dim + dim, a.out_vec, o);
}

template <int NB, typename IO, int NT>
__global__ void __launch_bounds__(kAttnThreads, Attn<NB, IO, NT>::kMinCtas) k_attn(const AttnArgs a) {
  using C = Attn<NB, IO, NT>;
  constexpr int TERMS = C::kTerms, ROWS = C::kRows, DIM = C::kDim, KS = C::kSteps, TILE = C::kTile, W = kAttnWarps;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int last_cta;
  __shared__ uint32_t okmask[kAttnWarps][kAttnStages];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint8_t *ring = smem + warp * C::kRing;
  float *red = reinterpret_cast<float *>(smem);  // [W][ROWS][DIM], then ref [W][ROWS], l [W][ROWS]
  float *red_ref = red + W * ROWS * DIM, *red_l = red_ref + W * ROWS;
  pdl_wait();
  pdl_trigger();

  AttnWalk<ROWS, kKvTile, kAttnHead> w;
  if (!w.template begin<kAttnThreads>(a, kAttnMinTiles)) return;
  do {
    const SeqRows &seq = w.seq;
    const int64_t rb = w.rb, ta = w.first_tile(), tb = w.last_tile();  // tiles [ta, tb) of the item are this CTA's
    const int head = w.head;

    // this lane's rows, one of each row block: position limits and q
    int64_t key_lo[NT], key_hi[NT];
    float ref[NT], l[NT], cs[NT];
    bool fresh[NT];
    uint32_t qa[C::kQ][NB * 2][4];
#pragma unroll
    for (int i = 0; i < C::kQ; ++i)
#pragma unroll
      for (int k = 0; k < NB * 2; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) qa[i][k][j] = 0;
    int64_t all_lo = 0, all_hi = INT64_MAX;  // keys that every row of the warp sees
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int64_t r = rb * ROWS + nt * 8 + g, i = (uint32_t)r / (uint32_t)a.group;
      const bool live = i < seq.n;
      const int qh = head * a.group + (int)(r - i * a.group);
      key_hi[nt] = live ? (int64_t)seq.len - seq.n + i + 1 : 0;
      key_lo[nt] = a.window > 0 && live ? key_hi[nt] - a.window : 0;
      if (live) {
        all_lo = key_lo[nt] > all_lo ? key_lo[nt] : all_lo;
        all_hi = key_hi[nt] < all_hi ? key_hi[nt] : all_hi;
      }
      ref[nt] = 0.0f, l[nt] = 0.0f, fresh[nt] = true;
      // a power of two brings the row's largest magnitude to [2^14, 2^15), so
      // that the f16 terms keep 39 bits below it
      float x[NB][8], top = 0.0f;
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        if (live)
          load_row<IO, 8>(static_cast<const IO *>(a.q) + (seq.start + i) * a.q_stride + (int64_t)qh * DIM + k * 32 + t * 8, a.q_vec, x[k]);
        else
#pragma unroll
          for (int j = 0; j < 8; ++j) x[k][j] = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[k][j]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      int e = 14 - ((int)(__float_as_uint(top) >> 23) - 127);
      if (top == 0.0f) e = 0;
      if (e > 100) e = 100;
      const float up = __uint_as_float((uint32_t)(e + 127) << 23);
      cs[nt] = a.scale * kLog2e * __uint_as_float((uint32_t)(127 - e) << 23);
      if (top == INFINITY) cs[nt] = __int_as_float(0x7fffffff);  // every score of the row is a NaN
#pragma unroll
      for (int k = 0; k < NB; ++k)
#pragma unroll
        for (int s = 0; s < 2; ++s)  // k16 step: pairs 2s and 2s + 1 of the word
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float x0 = x[k][2 * s + j] * up, x1 = x[k][2 * s + j + 4] * up;
            const __half2 hi = __floats2half2_rn(x0, x1);
            if constexpr (TERMS == 2) {
              const float2 f = __half22float2(hi);
              qa[nt][k * 2 + s][2 * j] = bits(hi);
              qa[nt][k * 2 + s][2 * j + 1] = pack_half2(x0 - f.x, x1 - f.y);
            } else {
              qa[nt / 2][k * 2 + s][2 * j + (nt & 1)] = bits(hi);
            }
          }
    }
#pragma unroll
    for (int m = 4; m < 32; m <<= 1) {
      const int64_t lo = __shfl_xor_sync(0xffffffffu, all_lo, m), hi = __shfl_xor_sync(0xffffffffu, all_hi, m);
      all_lo = lo > all_lo ? lo : all_lo;
      all_hi = hi < all_hi ? hi : all_hi;
    }
    float o[NT][NB][2][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < NB; ++k)
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[nt][k][m][j] = 0.0f;
    // values' scales seen so far are at most 2^vexp; a weight stands for
    // 2^(s - ref) with ref = max + vexp - 7, so weight * scale stays within
    // f16 until a later key exceeds the maximum by 2^8
    int vexp = -24;

    // ---- steps ------------------------------------------------------------------
    const int64_t count = tb - ta;
    const int per_step = count >= (int64_t)KS * W ? KS : count <= W ? 1 : (int)((count + W - 1) / W);
    const int64_t steps = (count + per_step - 1) / per_step;
    const int tiles_per_page = a.c.page_tokens / kKvTile;
    const int32_t *pages = a.r.table + w.b * a.r.max_pages;
    auto page_of = [&](int64_t j) -> int32_t {  // lane i: page of tile i of this warp's step j
      const int64_t step = warp + j * W, tile = ta + step * per_step + lane;
      return step < steps && lane < per_step && tile < tb ? pages[tile / tiles_per_page] : -1;
    };
    auto issue = [&](int64_t j, int32_t page) {
      const int64_t step = warp + j * W, tile0 = ta + step * per_step;
      const int stage = (int)(j % kAttnStages);
      const uint32_t ok = __ballot_sync(0xffffffffu, page >= 0 && page < a.c.pages);
      if (lane == 0) okmask[warp][stage] = ok;
      if (step < steps) {
        for (int i = 0; i < per_step && tile0 + i < tb; ++i) {
          const int32_t p = __shfl_sync(0xffffffffu, page, i);
          if (!(ok >> i & 1)) continue;
          const uint8_t *src = a.c.base + kv_tile_offset(a.c, p, head, (int)((tile0 + i) % tiles_per_page) * kKvTile);
          uint8_t *dst = ring + (stage * KS + i) * TILE;
#pragma unroll
          for (int c = 0; c < (TILE / 16 + 31) / 32; ++c)
            if (c * 32 + lane < TILE / 16) cp_async16(dst + (c * 32 + lane) * 16, src + (c * 32 + lane) * 16);
        }
      }
      cp_async_commit();
    };
    int32_t page_next = page_of(0);
#pragma unroll
    for (int j = 0; j < kAttnStages - 1; ++j) {
      issue(j, page_next);
      page_next = page_of(j + 1);
    }
    for (int64_t j = 0; warp + j * W < steps; ++j) {
      cp_async_wait<kAttnStages - 2>();
      __syncwarp();
      issue(j + kAttnStages - 1, page_next);
      page_next = page_of(j + kAttnStages);
      const int stage = (int)(j % kAttnStages);
      const int64_t tile0 = ta + (warp + j * W) * per_step;
      const int64_t key0 = tile0 * kKvTile;
      const uint32_t ok = okmask[warp][stage];
      const uint8_t *buf = ring + stage * KS * TILE;
      const int n_tiles = (int)(tb - tile0 < per_step ? tb - tile0 : per_step);
      const bool edge = key0 < all_lo || key0 + n_tiles * kKvTile > all_hi || ok != (1u << n_tiles) - 1u;

      // S = Q K^T of the step, and the largest value scale of it
      float s[KS][NT][4];
      uint32_t vmax = 0;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[i][nt][x] = 0.0f;
        if (i >= n_tiles || !(ok >> i & 1)) continue;
        const uint8_t *tile = buf + i * TILE;
#pragma unroll
        for (int k = 0; k < NB; ++k) {
          const uint2 kd = *reinterpret_cast<const uint2 *>(tile + kv_key_scales(NB) + t * NB * 8 + k * 8);
          const uint2 vd = *reinterpret_cast<const uint2 *>(tile + kv_value_scales(NB) + t * NB * 8 + k * 8);
          vmax = bits(__hmax2(half2_of(vmax), __hmax2(half2_of(vd.x & 0x7fff7fffu), half2_of(vd.y & 0x7fff7fffu))));
          const uint2 w = *reinterpret_cast<const uint2 *>(tile + kv_word(NB, k, lane, 0));
          const float2 d[2] = {__half22float2(half2_of(kd.x)), __half22float2(half2_of(kd.y))};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t e[4];
            decode_word(h ? w.y : w.x, e);
#pragma unroll
            for (int q = 0; q < C::kQ; ++q) {
              float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
              mma16816(c, qa[q][k * 2], e[0], e[1]);
              mma16816(c, qa[q][k * 2 + 1], e[2], e[3]);
              if constexpr (TERMS == 2) {
                s[i][q][2 * h] = fmaf(c[0] + c[2], d[h].x, s[i][q][2 * h]);
                s[i][q][2 * h + 1] = fmaf(c[1] + c[3], d[h].y, s[i][q][2 * h + 1]);
              } else {
                s[i][2 * q][2 * h] = fmaf(c[0], d[h].x, s[i][2 * q][2 * h]);
                s[i][2 * q][2 * h + 1] = fmaf(c[1], d[h].y, s[i][2 * q][2 * h + 1]);
                if constexpr (NT > 1) {
                  s[i][2 * q + 1][2 * h] = fmaf(c[2], d[h].x, s[i][2 * q + 1][2 * h]);
                  s[i][2 * q + 1][2 * h + 1] = fmaf(c[3], d[h].y, s[i][2 * q + 1][2 * h + 1]);
                }
              }
            }
          }
        }
      }
      // weights: x = log2 of the weight
      bool high = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            float v = fmaf(s[i][nt][x], cs[nt], -ref[nt]);
            if (i >= n_tiles) v = -INFINITY;
            if (edge) {
              const int64_t key = key0 + i * kKvTile + 2 * t + (x & 1) + (x >> 1) * 8;
              if (key < key_lo[nt] || key >= key_hi[nt] || !(ok >> i & 1)) v = -INFINITY;
            }
            s[i][nt][x] = v;
            top = fmaxf(top, v);
          }
        high |= top > (fresh[nt] ? -INFINITY : (float)(15 - vexp));
      }
      const float2 vm = __half22float2(half2_of(vmax));
      const float vtop = fmaxf(vm.x, vm.y);
      high |= vtop > __uint_as_float((uint32_t)(vexp + 127) << 23);
      if (__any_sync(0xffffffffu, high)) {  // a new maximum: rare after the first steps
        float vw = vtop;
#pragma unroll
        for (int m = 1; m < 32; m <<= 1) vw = fmaxf(vw, __shfl_xor_sync(0xffffffffu, vw, m));
        int ve = (int)(__float_as_uint(vw) >> 23) - 126;  // vw < 2^ve
        if (ve > 17) ve = 17;                             // an infinite scale: not written by append
        if (ve < vexp) ve = vexp;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float top = -INFINITY;
#pragma unroll
          for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) top = fmaxf(top, s[i][nt][x]);
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          float most = top + ref[nt];
          if (!fresh[nt]) most = fmaxf(most, ref[nt] - (float)(vexp - 7));
          const bool none = most == -INFINITY;
          const float now = none ? 0.0f : most + (float)(ve - 7);
          const float factor = fresh[nt] ? 1.0f : exp2f(ref[nt] - now);
#pragma unroll
          for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) s[i][nt][x] += ref[nt] - now;
          l[nt] *= factor;
          ref[nt] = now;
          fresh[nt] = none;
          const float f0 = __shfl_sync(0xffffffffu, factor, 8 * t), f1 = __shfl_sync(0xffffffffu, factor, 8 * t + 4);
#pragma unroll
          for (int k = 0; k < NB; ++k)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              o[nt][k][m][0] *= f0, o[nt][k][m][1] *= f1;
              o[nt][k][m][2] *= f0, o[nt][k][m][3] *= f1;
            }
        }
        vexp = ve;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            s[i][nt][x] = exp2_fast(s[i][nt][x]);
            l[nt] += s[i][nt][x];
          }
      // O^T += V^T P^T.  With two terms the step's products are summed from
      // zero and added in f32: the tensor cores' own additions lose bits of a
      // long sum.
      float oc[NT][NB][2][4];
      if constexpr (TERMS == 2) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < NB; ++k)
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
              for (int x = 0; x < 4; ++x) oc[nt][k][m][x] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        if (i >= n_tiles || !(ok >> i & 1)) continue;
        const uint8_t *tile = buf + i * TILE;
#pragma unroll
        for (int k = 0; k < NB; ++k) {
          const uint2 vd = *reinterpret_cast<const uint2 *>(tile + kv_value_scales(NB) + t * NB * 8 + k * 8);
          const uint2 w = *reinterpret_cast<const uint2 *>(tile + kv_value_codes(NB) + kv_word(NB, k, lane, 0));
          uint32_t e0[4], e1[4];
          decode_word(w.x, e0);
          decode_word(w.y, e1);
          const uint32_t a0[4] = {e0[0], e0[1], e1[0], e1[1]}, a1[4] = {e0[2], e0[3], e1[2], e1[3]};
          const float2 d0 = __half22float2(half2_of(vd.x)), d1 = __half22float2(half2_of(vd.y));
          const float d[4] = {d0.x, d0.y, d1.x, d1.y};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float p[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              p[x] = s[i][nt][x] * d[x];
              if (edge) {  // a masked key's scale may be anything
                const int64_t key = key0 + i * kKvTile + 2 * t + (x & 1) + (x >> 1) * 8;
                if (key < key_lo[nt] || key >= key_hi[nt]) p[x] = 0.0f;
              }
            }
            if constexpr (TERMS == 2) {
              float hi[4];
#pragma unroll
              for (int x = 0; x < 4; ++x) hi[x] = __uint_as_float(__float_as_uint(p[x]) & 0xffffe000u);
              const uint32_t b0 = pack_half2(hi[0], hi[1]), b1 = pack_half2(hi[2], hi[3]);
              const uint32_t c0 = pack_half2(p[0] - hi[0], p[1] - hi[1]), c1 = pack_half2(p[2] - hi[2], p[3] - hi[3]);
              mma16816(oc[nt][k][0], a0, b0, b1);
              mma16816(oc[nt][k][1], a1, b0, b1);
              mma16816(oc[nt][k][0], a0, c0, c1);
              mma16816(oc[nt][k][1], a1, c0, c1);
            } else {
              // one term: 2^-11 of each weight at most, no more than the rounding of f16 and bf16 rows
              const uint32_t b0 = pack_half2(p[0], p[1]), b1 = pack_half2(p[2], p[3]);
              mma16816(o[nt][k][0], a0, b0, b1);
              mma16816(o[nt][k][1], a1, b0, b1);
            }
          }
        }
      }
      if constexpr (TERMS == 2) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < NB; ++k)
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
              for (int x = 0; x < 4; ++x) o[nt][k][m][x] += oc[nt][k][m][x];
      }
    }
    cp_async_wait<0>();
    __syncthreads();

    // ---- the warps' sums meet ----------------------------------------------------
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float sum = l[nt];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if (t == 0) {
        red_ref[warp * ROWS + nt * 8 + g] = fresh[nt] && sum == 0.0f ? -INFINITY : ref[nt];
        red_l[warp * ROWS + nt * 8 + g] = sum;
      }
#pragma unroll
      for (int k = 0; k < NB; ++k)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          *reinterpret_cast<float4 *>(red + (warp * ROWS + nt * 8 + 2 * t + x) * DIM + k * 32 + 4 * g) =
              make_float4(o[nt][k][0][x], o[nt][k][0][2 + x], o[nt][k][1][x], o[nt][k][1][2 + x]);
    }
    __syncthreads();
    const bool whole = w.whole();
    const int64_t first_cta = w.first_cta(), last_share = w.last_cta();
    float *slot = part_slot<ROWS, DIM>(a, blockIdx.x, first_cta);
    for (int x = tid; x < ROWS * DIM / 4; x += kAttnThreads) {
      const int r = x / (DIM / 4), dim = x % (DIM / 4) * 4;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) top = fmaxf(top, red_ref[w * ROWS + r]);
      float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float rw = red_ref[w * ROWS + r];
        const float f = rw == -INFINITY ? 0.0f : exp2f(rw - top);
        const float4 v = *reinterpret_cast<const float4 *>(red + (w * ROWS + r) * DIM + dim);
        sum += red_l[w * ROWS + r] * f;
        acc[0] += v.x * f, acc[1] += v.y * f, acc[2] += v.z * f, acc[3] += v.w * f;
      }
      if (whole) {
        const int64_t rr = rb * ROWS + r, i = (uint32_t)rr / (uint32_t)a.group;
        if (i < seq.n)
          finish4<IO>(a, seq.start + i, head * a.group + (int)(rr - i * a.group), dim, top, sum, acc, DIM);
      } else {
        *reinterpret_cast<float4 *>(slot + r * DIM + dim) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        if (dim == 0) slot[ROWS * DIM + r] = top, slot[ROWS * DIM + ROWS + r] = sum;
      }
    }
    if (!whole) {
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        const int32_t parts = (int32_t)(last_share - first_cta + 1);
        last_cta = atomicAdd(&a.arrive[first_cta], 1) == parts - 1;
        if (last_cta) a.arrive[first_cta] = 0;
      }
      __syncthreads();
      if (last_cta) {
        __threadfence();
        for (int x = tid; x < ROWS * DIM / 4; x += kAttnThreads) {
          const int r = x / (DIM / 4), dim = x % (DIM / 4) * 4;
          const int64_t rr = rb * ROWS + r, i = (uint32_t)rr / (uint32_t)a.group;
          if (i >= seq.n) continue;
          float top = -INFINITY;
          for (int64_t c = first_cta; c <= last_share; ++c)
            top = fmaxf(top, __ldcg(part_slot<ROWS, DIM>(a, c, first_cta) + ROWS * DIM + r));
          float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sum = 0.0f;
          for (int64_t c = first_cta; c <= last_share; ++c) {
            const float *p = part_slot<ROWS, DIM>(a, c, first_cta);
            const float rw = __ldcg(p + ROWS * DIM + r);
            const float f = rw == -INFINITY ? 0.0f : exp2f(rw - top);
            const float4 v = __ldcg(reinterpret_cast<const float4 *>(p + r * DIM + dim));
            sum += __ldcg(p + ROWS * DIM + ROWS + r) * f;
            acc[0] += v.x * f, acc[1] += v.y * f, acc[2] += v.z * f, acc[3] += v.w * f;
          }
          finish4<IO>(a, seq.start + i, head * a.group + (int)(rr - i * a.group), dim, top, sum, acc, DIM);
        }
      }
    }
    __syncthreads();
  } while (w.next(a));
}

template <int NB, typename IO, int NT>
cudaError_t launch(const AttnArgs &a, cudaStream_t stream) {
  using C = Attn<NB, IO, NT>;
  const cudaError_t e = opt_in_smem(k_attn<NB, IO, NT>, C::kSmem);
  if (e != cudaSuccess) return e;
  return launch_pdl(k_attn<NB, IO, NT>, dim3(a.sm_count * C::kMinCtas), dim3(kAttnThreads), C::kSmem, stream, a);
}

template <typename IO>
cudaError_t launch_dims(const AttnArgs &a, cudaStream_t stream) {
  const bool two = a.r.offsets || a.group > 8;
  switch (a.c.nb) {
    case 1: return two ? launch<1, IO, 2>(a, stream) : launch<1, IO, 1>(a, stream);
    case 2: return two ? launch<2, IO, 2>(a, stream) : launch<2, IO, 1>(a, stream);
    case 3: return two ? launch<3, IO, 2>(a, stream) : launch<3, IO, 1>(a, stream);
    case 4: return two ? launch<4, IO, 2>(a, stream) : launch<4, IO, 1>(a, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

size_t attn_workspace_bytes(int sm_count, int nb) {
  return (size_t)sm_count * kAttnCtasPerSm * 2 * kAttnMaxRows * (nb * 32 + 2) * sizeof(float);
}
size_t attn_counter_bytes(int sm_count) { return (size_t)sm_count * kAttnCtasPerSm * sizeof(int32_t); }

cudaError_t launch_attention(const AttnArgs &args, cudaStream_t stream) {
  AttnArgs a = args;
  if (a.r.tokens <= 0 || a.r.sequences <= 0) return cudaSuccess;
  if (a.r.tokens > INT32_MAX / a.group) return cudaErrorInvalidValue;
  const int size = a.type == kKvF32 ? 4 : 2;
  a.q_vec = ((reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)(a.q_stride * size)) & 15) == 0;
  a.out_vec = ((reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)(a.out_stride * size)) & 15) == 0;
  if (a.r.offsets && a.r.tokens * a.group > 32 * a.r.sequences) return launch_attention_mma(a, stream);
  switch (a.type) {
    case kKvF32: return launch_dims<float>(a, stream);
    case kKvF16: return launch_dims<__half>(a, stream);
    case kKvBF16: return launch_dims<__nv_bfloat16>(a, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace spt
