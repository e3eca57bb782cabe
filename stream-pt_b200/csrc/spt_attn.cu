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
constexpr int kAttnMinTiles = 12;    // a CTA's smallest share: a tile for each warp
// An item's beginning and end, in tiles' time.  One f32 token on 2,047 keys, 64 f32
// and 64 bf16 sequences of up to 8,192 keys, 48 of a window of 128, us: at 1 17.0,
// 88.0, 91.2, 20.5; at 4 13.1, 87.2, 90.5, 19.1; at 8 14.6, 85.9, 89.1, 19.2; at 16
// 12.5, 84.5, 87.5, 19.3.
constexpr int kAttnHead = 4;

// D (16 x 8, f32) += A (16 x 16, f16) * B (16 x 8, f16)
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The work, B = NB blocks of 32 dims, TERMS f16 terms of q (2 for f32 rows: 22
// bits; 1 holds f16 and bf16 rows), two terms of the softmax weights, NT blocks of
// 8 rows.
//
// Within its share of the 16-key tiles (AttnWalk) a CTA's warps take steps of
// up to KS tiles in turn, each warp with its own ring of bulk copies and its own
// running maximum and sum; they meet in shared memory at the item's end.  (With
// a share a warp and no meeting, a long sequence left hundreds of parts to be
// joined: one of 131,000 tokens took 212 us instead of 62.)
//
// Products.  S (rows x keys) = Q K^T with the rows' two f16 terms stacked
// along M (TERMS 2) or two row blocks stacked (TERMS 1), codes n - 8 exact in
// f16, and the keys' scales applied to the f32 sums of each 32-dim block.
// O^T (dims x rows) = V^T P^T with the values' scales applied to the weights
// of each 32-dim block before their split into f16 terms.  S's fragment is
// the layout that P^T's operand needs.
//
// Bound by instructions and the latency of one behind another, as neither issue
// slots nor a pipe are full and there are 4 warps a scheduler (2 at 128 dims) to
// change between: 64 f32 sequences of up to 8,192 tokens, 8 heads of 64 dims and 8
// queries each, read 187 MB in 87 us (2.1 TB/s, 0.55 instructions a clock, the ALU
// 46% busy with codes becoming f16); 64 such bf16 sequences take 90 us, one bf16
// sequence of 131,000 tokens and 128 dims 72 us for 151 MB (2.1 TB/s, 0.45
// instructions a clock).  Three CTAs an SM of steps of two tiles took 110 us
// instead of 87, steps of two tiles on two CTAs 92; at 128 dims two CTAs an SM took
// 18% longer than one.  What exactness and safety cost bf16 rows of 64 and of 128
// dims: the weights' second f16 term 82 -> 88 us and 65 -> 70, scales by what each
// row sees and waits that are looked at 88 -> 90 and 70 -> 72.
template <int NB, typename IO, int NT>
struct Attn {
  static constexpr int kTerms = sizeof(IO) == 4 ? 2 : 1;
  static constexpr int kDim = NB * 32, kRows = NT * 8;
  static constexpr int kTile = kv_tile_bytes(NB);
  static constexpr int kSteps = NB <= 2 ? 4 : 2;  // tiles in a step at most
  static constexpr int kRing = kAttnStages * kSteps * kTile;
  static constexpr int kRedBytes = kAttnWarps * kRows * (kDim + 2) * 4;
  static constexpr int kSmem = kAttnWarps * kRing > kRedBytes ? kAttnWarps * kRing : kRedBytes;
  static constexpr int kSub = 2;                  // tiles of a step whose weights are taken at once
  // CTAs on an SM: 16 warps of 128 registers, where that holds the fragments (bf16
  // rows at 64 dims, two row blocks: 143 us on two CTAs with spills, 135 on one)
  static constexpr int kMinCtas = (NT == 1 ? NB <= 2 : NB == 1 && kTerms == 1) ? 2 : 1;
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
  __shared__ uint64_t bars[kAttnWarps][kAttnStages];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint8_t *ring = smem + warp * C::kRing;
  float *red = reinterpret_cast<float *>(smem);  // [W][ROWS][DIM], then ref [W][ROWS], l [W][ROWS]
  float *red_ref = red + W * ROWS * DIM, *red_l = red_ref + W * ROWS;
  pdl_wait();
  pdl_trigger();

  AttnWalk<ROWS, kKvTile, kAttnHead> w;
  if (tid < W * kAttnStages) mbar_init(&bars[tid / kAttnStages][tid % kAttnStages], 1);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  __syncthreads();
  if (!w.template begin<kAttnThreads>(a, kAttnMinTiles, blockIdx.x, gridDim.x)) return;
  const uint32_t tiles_per_page = (uint32_t)a.c.page_tokens / kKvTile;
  int stage = 0;  // of this warp's ring: the step to be read next
  uint32_t phase = 0;
  // A warp whose wait runs out takes no more steps: it waits for its copies in
  // flight, whose bytes would else land in the sums that follow or in another CTA's
  // shared memory, and comes to the meetings and the arrivals as the others do.
  bool gave_up = false;
  uint32_t steps = 0;  // that this warp has asked for
  do {
    const SeqRows &seq = w.seq;
    const int rb = w.rb, ta = w.first_tile(), tb = w.last_tile();  // tiles [ta, tb) of the item are this CTA's
    const int head = w.head;

    // this lane's rows, one of each row block: position limits and q
    int key_lo[NT], key_hi[NT];
    float ref[NT], l[NT], cs[NT];
    bool fresh[NT];
    uint32_t qa[C::kQ][NB * 2][4];
#pragma unroll
    for (int i = 0; i < C::kQ; ++i)
#pragma unroll
      for (int k = 0; k < NB * 2; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) qa[i][k][j] = 0;
    int all_lo = 0, all_hi = INT32_MAX;  // keys that every row of the warp sees
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = rb * ROWS + nt * 8 + g, i = (int)((uint32_t)r / (uint32_t)a.group);
      const bool live = i < seq.n;
      const int qh = head * a.group + r - i * a.group;
      key_hi[nt] = live ? max(seq.len - seq.n + i + 1, 0) : 0;
      key_lo[nt] = a.window > 0 && key_hi[nt] > a.window ? key_hi[nt] - (int)a.window : 0;
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
          load_row<IO, 8>(static_cast<const IO *>(a.q) + (int64_t)(seq.start + i) * a.q_stride + (int64_t)qh * DIM + k * 32 + t * 8, a.q_vec, x[k]);
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
      const int lo = __shfl_xor_sync(0xffffffffu, all_lo, m), hi = __shfl_xor_sync(0xffffffffu, all_hi, m);
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
    // the scales of the values that a row has seen are at most 2^vexp; a weight
    // stands for 2^(s - ref) with ref = max + vexp - 7, so weight * scale stays
    // within f16 until a later key exceeds the maximum by 2^8.  Keys that the row
    // does not see count for nothing: a page's tail may hold anything.
    int vexp[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) vexp[nt] = -24;

    // ---- steps ------------------------------------------------------------------
    // step j of this warp: tiles ta + (warp + j W) per_step on.  Lane i of it looks
    // after tile i: its page, read a step ahead, and its copy; tiles that follow
    // one another in a page are copied at once.
    const int count = tb - ta;
    const int per_step = count >= KS * W ? KS : count <= W ? 1 : (count + W - 1) / W;
    const int32_t *pages = a.r.table + (int64_t)w.b * a.r.max_pages;
    int32_t page = -1;
    uint32_t place = 0;
    int asked = ta + warp * per_step, read = asked;  // first tiles of the step asked for next, read next
    auto ask = [&](int tile0) {
      const uint32_t tile = (uint32_t)(tile0 + lane), p = tile / tiles_per_page;
      place = tile - p * tiles_per_page;
      page = lane < per_step && (int)tile < tb ? __ldcg(pages + p) : -1;
    };
    int left_out = -1;
    auto fetch = [&](int to) {  // the step that was asked for, into ring slot `to`
      const bool good = page >= 0 && page < a.c.pages;
      if (blockIdx.x == 0 && warp == 0 && steps++ == (uint32_t)a.fault_tile) {
        left_out = to;
        return 0u;
      }
      const uint32_t ok = __ballot_sync(0xffffffffu, good);
      const uint32_t starts = __ballot_sync(0xffffffffu, good && (place == 0 || lane == 0 || !(ok >> (lane - 1) & 1)));
      if (lane == 0) mbar_expect_tx(&bars[warp][to], __popc(ok) * TILE);
      __syncwarp();
      if (starts >> lane & 1) {  // up to the next start or bad page
        const uint32_t ends = (starts | ~ok) >> lane >> 1;
        bulk_load(ring + (to * KS + lane) * TILE, a.c.base + kv_tile_offset(a.c, page, head, (int)place * kKvTile),
                  (uint32_t)__ffs(ends) * TILE, &bars[warp][to]);
      }
      return ok;
    };
    uint32_t ok_now = 0, ok_next = 0;  // good pages of the steps under way
    int slot = stage;
    if (asked < tb && !gave_up) {
      ask(asked);
      ok_now = fetch(slot);
      asked += W * per_step;
      ask(asked);
      if (++slot == kAttnStages) slot = 0;
      if (asked < tb) ok_next = fetch(slot);
      asked += W * per_step;
      ask(asked);
      if (++slot == kAttnStages) slot = 0;
    }
    // KU tiles, all of whose keys every row sees, or any
    constexpr int KU = C::kSub;
    auto step = [&](auto full_step, const uint8_t *buf, int key0, int n_tiles, uint32_t ok) {
      constexpr bool FULL = decltype(full_step)::value;
      // S = Q K^T of the step, and the largest value scale of it
      float2 s[KU][NT][2];  // of keys 2 t, 2 t + 1 and 2 t + 8, 2 t + 9
      // the largest value scales: of these four keys each, or of all where all are seen
      uint32_t vmax[FULL ? 1 : KU][FULL ? 1 : 2] = {};
#pragma unroll
      for (int i = 0; i < KU; ++i) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[i][nt][0] = s[i][nt][1] = make_float2(0.0f, 0.0f);
        if (!FULL && (i >= n_tiles || !(ok >> i & 1))) continue;
        const uint8_t *tile = buf + i * TILE;
#pragma unroll
        for (int k = 0; k < NB; ++k) {
          const uint2 kd = *reinterpret_cast<const uint2 *>(tile + kv_key_scales(NB) + t * NB * 8 + k * 8);
          const uint2 vd = *reinterpret_cast<const uint2 *>(tile + kv_value_scales(NB) + t * NB * 8 + k * 8);
          const __half2 v0 = half2_of(vd.x & 0x7fff7fffu), v1 = half2_of(vd.y & 0x7fff7fffu);
          if constexpr (FULL) {
            vmax[0][0] = bits(__hmax2(half2_of(vmax[0][0]), __hmax2(v0, v1)));
          } else {
            vmax[i][0] = bits(__hmax2(half2_of(vmax[i][0]), v0));
            vmax[i][1] = bits(__hmax2(half2_of(vmax[i][1]), v1));
          }
          const uint2 word = *reinterpret_cast<const uint2 *>(tile + kv_word(NB, k, lane, 0));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 d = __half22float2(half2_of(h ? kd.y : kd.x));
            uint32_t e[4];
            decode_word(h ? word.y : word.x, e);
#pragma unroll
            for (int q = 0; q < C::kQ; ++q) {
              float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
              mma16816(c, qa[q][k * 2], e[0], e[1]);
              mma16816(c, qa[q][k * 2 + 1], e[2], e[3]);
              const float2 c0 = make_float2(c[0], c[1]), c1 = make_float2(c[2], c[3]);
              if constexpr (TERMS == 2) {
                s[i][q][h] = __ffma2_rn(__fadd2_rn(c0, c1), d, s[i][q][h]);
              } else {
                s[i][2 * q][h] = __ffma2_rn(c0, d, s[i][2 * q][h]);
                if constexpr (NT > 1) s[i][2 * q + 1][h] = __ffma2_rn(c1, d, s[i][2 * q + 1][h]);
              }
            }
          }
        }
      }
      // a key of this lane: pair h of tile i, its x-th
      auto hidden = [&](int nt, int i, int h, int x) {
        const int key = key0 + i * kKvTile + 2 * t + 8 * h + x;
        return key < key_lo[nt] || key >= key_hi[nt] || i >= n_tiles || !(ok >> i & 1);
      };
      // s becomes log2 of the weight
      float vtop[NT];  // the largest value scale of this lane's keys that its row sees
      const float2 vm = __half22float2(half2_of(vmax[0][0]));
      bool high = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float2 scale = make_float2(cs[nt], cs[nt]), off = make_float2(-ref[nt], -ref[nt]);
        float top = -INFINITY;
        vtop[nt] = FULL ? fmaxf(vm.x, vm.y) : 0.0f;
#pragma unroll
        for (int i = 0; i < KU; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float2 v = __ffma2_rn(s[i][nt][h], scale, off);
            if constexpr (!FULL) {
              const float2 d = __half22float2(half2_of(vmax[i][h]));
              if (hidden(nt, i, h, 0)) v.x = -INFINITY;
              else vtop[nt] = fmaxf(vtop[nt], d.x);
              if (hidden(nt, i, h, 1)) v.y = -INFINITY;
              else vtop[nt] = fmaxf(vtop[nt], d.y);
            }
            s[i][nt][h] = v;
            top = fmaxf(top, fmaxf(v.x, v.y));
          }
        high |= top > (fresh[nt] ? -INFINITY : (float)(15 - vexp[nt]));
        high |= vtop[nt] > __uint_as_float((uint32_t)(vexp[nt] + 127) << 23);
      }
      if (__any_sync(0xffffffffu, high)) {  // a new maximum: rare after the first steps
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float vw = vtop[nt];
          vw = fmaxf(vw, __shfl_xor_sync(0xffffffffu, vw, 1));
          vw = fmaxf(vw, __shfl_xor_sync(0xffffffffu, vw, 2));
          int ve = (int)(__float_as_uint(vw) >> 23) - 126;  // vw < 2^ve
          if (ve > 17) ve = 17;                             // an infinite scale: not written by append
          if (ve < vexp[nt]) ve = vexp[nt];
          float top = -INFINITY;
#pragma unroll
          for (int i = 0; i < KU; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) top = fmaxf(top, fmaxf(s[i][nt][h].x, s[i][nt][h].y));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          // (a row whose own maxima stand keeps its reference, whatever the others')
          const bool up = top > (fresh[nt] ? -INFINITY : (float)(15 - vexp[nt])) ||
                          vw > __uint_as_float((uint32_t)(vexp[nt] + 127) << 23);
          float most = top + ref[nt];
          if (!fresh[nt]) most = fmaxf(most, ref[nt] - (float)(vexp[nt] - 7));
          const bool none = most == -INFINITY;
          const float now = !up ? ref[nt] : none ? 0.0f : most + (float)(ve - 7);
          const float factor = fresh[nt] ? 1.0f : exp2f(ref[nt] - now);
          const float2 move = make_float2(ref[nt] - now, ref[nt] - now);
#pragma unroll
          for (int i = 0; i < KU; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) s[i][nt][h] = __fadd2_rn(s[i][nt][h], move);
          l[nt] *= factor;
          ref[nt] = now;
          fresh[nt] = none;
          if (up) vexp[nt] = ve;
          const float f0 = __shfl_sync(0xffffffffu, factor, 8 * t), f1 = __shfl_sync(0xffffffffu, factor, 8 * t + 4);
#pragma unroll
          for (int k = 0; k < NB; ++k)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              o[nt][k][m][0] *= f0, o[nt][k][m][1] *= f1;
              o[nt][k][m][2] *= f0, o[nt][k][m][3] *= f1;
            }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < KU; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            s[i][nt][h] = make_float2(exp2_fast(s[i][nt][h].x), exp2_fast(s[i][nt][h].y));
            sum = __fadd2_rn(sum, s[i][nt][h]);
          }
        l[nt] += sum.x + sum.y;
      }
      // O^T += V^T P^T.  A weight times its value's scale is two f16 terms whatever
      // the rows' type: one would be 2^-11 of it off, as much as the rounding of an
      // f16 row, and more where the values nearly cancel.  The step's products are
      // summed from zero and added in f32: the tensor cores' own additions lose bits
      // of a long sum.
      float oc[NT][NB][2][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < NB; ++k)
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int x = 0; x < 4; ++x) oc[nt][k][m][x] = 0.0f;
#pragma unroll
      for (int i = 0; i < KU; ++i) {
        if (!FULL && (i >= n_tiles || !(ok >> i & 1))) continue;
        const uint8_t *tile = buf + i * TILE;
#pragma unroll
        for (int k = 0; k < NB; ++k) {
          const uint2 vd = *reinterpret_cast<const uint2 *>(tile + kv_value_scales(NB) + t * NB * 8 + k * 8);
          const uint2 word = *reinterpret_cast<const uint2 *>(tile + kv_value_codes(NB) + kv_word(NB, k, lane, 0));
          uint32_t e0[4], e1[4];
          decode_word(word.x, e0);
          decode_word(word.y, e1);
          const uint32_t a0[4] = {e0[0], e0[1], e1[0], e1[1]}, a1[4] = {e0[2], e0[3], e1[2], e1[3]};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            uint32_t hi[2], lo[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float2 p = __fmul2_rn(s[i][nt][h], __half22float2(half2_of(h ? vd.y : vd.x)));
              if (!FULL) {  // a masked key's scale may be anything
                if (hidden(nt, i, h, 0)) p.x = 0.0f;
                if (hidden(nt, i, h, 1)) p.y = 0.0f;
              }
              const __half2 r = __floats2half2_rn(p.x, p.y);
              const float2 rest = __ffma2_rn(__half22float2(r), make_float2(-1.0f, -1.0f), p);
              hi[h] = bits(r);
              lo[h] = pack_half2(rest.x, rest.y);
            }
            mma16816(oc[nt][k][0], a0, lo[0], lo[1]);
            mma16816(oc[nt][k][1], a1, lo[0], lo[1]);
            mma16816(oc[nt][k][0], a0, hi[0], hi[1]);
            mma16816(oc[nt][k][1], a1, hi[0], hi[1]);
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < NB; ++k)
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int x = 0; x < 4; x += 2) {
              const float2 v = __fadd2_rn(make_float2(o[nt][k][m][x], o[nt][k][m][x + 1]),
                                          make_float2(oc[nt][k][m][x], oc[nt][k][m][x + 1]));
              o[nt][k][m][x] = v.x, o[nt][k][m][x + 1] = v.y;
            }
    };
#pragma unroll 1
    for (; read < tb && !gave_up; read += W * per_step) {
      if (!__all_sync(0xffffffffu, own_wait(&bars[warp][stage], phase, a, 46))) {
        gave_up = true;  // the step of this slot and the next are in flight
        if (stage != left_out) mbar_wait_own(&bars[warp][stage], phase);
        if (++stage == kAttnStages) stage = 0, phase ^= 1u;
        if (read + W * per_step < tb && stage != left_out) mbar_wait_own(&bars[warp][stage], phase);
        break;
      }
      __syncwarp();  // the slot read last is free: the step after the next goes there
      uint32_t ok_then = 0;
      if (asked < tb) ok_then = fetch(slot);
      asked += W * per_step;
      ask(asked);
      if (++slot == kAttnStages) slot = 0;
      int key0 = read * kKvTile, n_tiles = tb - read < per_step ? tb - read : per_step;
      const uint8_t *buf = ring + stage * KS * TILE;
      uint32_t ok = ok_now;
#pragma unroll 1
      for (; n_tiles > 0; n_tiles -= KU, key0 += KU * kKvTile, buf += KU * TILE, ok >>= KU) {
        constexpr uint32_t all = (1u << KU) - 1u;
        if (n_tiles >= KU && (ok & all) == all && key0 >= all_lo && all_hi - key0 >= KU * kKvTile)
          step(std::true_type{}, buf, key0, KU, all);
        else
          step(std::false_type{}, buf, key0, n_tiles, ok);
      }
      ok_now = ok_next, ok_next = ok_then;
      if (++stage == kAttnStages) stage = 0, phase ^= 1u;
    }
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
    const int first = w.first_share(), last = w.last_share();
    float *part = part_slot<ROWS, DIM>(a, blockIdx.x, first);
    for (int x = tid; x < ROWS * DIM / 4; x += kAttnThreads) {
      const int r = x / (DIM / 4), dim = x % (DIM / 4) * 4;
      float top = -INFINITY;
#pragma unroll
      for (int v = 0; v < W; ++v) top = fmaxf(top, red_ref[v * ROWS + r]);
      float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sum = 0.0f;
#pragma unroll
      for (int v = 0; v < W; ++v) {
        const float rw = red_ref[v * ROWS + r];
        const float f = rw == -INFINITY ? 0.0f : exp2_fast(rw - top);
        const float4 u = *reinterpret_cast<const float4 *>(red + (v * ROWS + r) * DIM + dim);
        sum = fmaf(red_l[v * ROWS + r], f, sum);
        acc[0] = fmaf(u.x, f, acc[0]), acc[1] = fmaf(u.y, f, acc[1]);
        acc[2] = fmaf(u.z, f, acc[2]), acc[3] = fmaf(u.w, f, acc[3]);
      }
      if (whole) {
        const int rr = rb * ROWS + r, i = (int)((uint32_t)rr / (uint32_t)a.group);
        if (i < seq.n) finish4<IO>(a, seq.start + i, head * a.group + rr - i * a.group, dim, top, sum, acc, DIM);
      } else {
        *reinterpret_cast<float4 *>(part + r * DIM + dim) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        if (dim == 0) part[ROWS * DIM + r] = top, part[ROWS * DIM + ROWS + r] = sum;
      }
    }
    if (!whole) {
      __threadfence();
      __syncthreads();
      if (tid == 0) last_cta = arrive(a, w);
      __syncthreads();
      if (last_cta) {
        __threadfence();
        for (int x = tid; x < ROWS * DIM / 4; x += kAttnThreads) {
          const int r = x / (DIM / 4), dim = x % (DIM / 4) * 4;
          const int rr = rb * ROWS + r, i = (int)((uint32_t)rr / (uint32_t)a.group);
          if (i >= seq.n) continue;
          float top = -INFINITY;
#pragma unroll 4
          for (int c = first; c <= last; ++c) top = fmaxf(top, __ldcg(part_slot<ROWS, DIM>(a, c, first) + ROWS * DIM + r));
          float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sum = 0.0f;
#pragma unroll 4
          for (int c = first; c <= last; ++c) {
            const float *p = part_slot<ROWS, DIM>(a, c, first);
            const float rw = __ldcg(p + ROWS * DIM + r);
            const float f = rw == -INFINITY ? 0.0f : exp2_fast(rw - top);
            const float4 v = __ldcg(reinterpret_cast<const float4 *>(p + r * DIM + dim));
            sum = fmaf(__ldcg(p + ROWS * DIM + ROWS + r), f, sum);
            acc[0] = fmaf(v.x, f, acc[0]), acc[1] = fmaf(v.y, f, acc[1]);
            acc[2] = fmaf(v.z, f, acc[2]), acc[3] = fmaf(v.w, f, acc[3]);
          }
          finish4<IO>(a, seq.start + i, head * a.group + rr - i * a.group, dim, top, sum, acc, DIM);
        }
      }
    }
    // the next item's copies write where these sums lay
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
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
  // Two blocks of 8 rows where a key head has more than 8 on average: without
  // offsets it has `group`.  64 sequences of 8,000 keys, 8 rows each, took 142 us
  // (f32) and 135 us (bf16) with two, half of them empty, 87 and 88 with one.
  const bool two = a.group > 8 || (a.r.offsets && a.r.tokens * a.group > 8 * a.r.sequences);
  switch (a.c.nb) {
    case 1: return two ? launch<1, IO, 2>(a, stream) : launch<1, IO, 1>(a, stream);
    case 2: return two ? launch<2, IO, 2>(a, stream) : launch<2, IO, 1>(a, stream);
    case 3: return two ? launch<3, IO, 2>(a, stream) : launch<3, IO, 1>(a, stream);
    case 4: return two ? launch<4, IO, 2>(a, stream) : launch<4, IO, 1>(a, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

// two slots a CTA
size_t attn_workspace_bytes(int sm_count, int nb) {
  return (size_t)sm_count * kAttnCtasPerSm * 2 * 16 * (nb * 32 + 2) * sizeof(float);
}
// a counter a CTA, and a flag for each CTA of the many-row kernel
size_t attn_counter_bytes(int sm_count) { return (size_t)sm_count * (kAttnCtasPerSm + 1) * sizeof(int32_t); }

cudaError_t launch_attention(const AttnArgs &args, cudaStream_t stream) {
  AttnArgs a = args;
  if (a.r.tokens <= 0 || a.r.sequences <= 0) return cudaSuccess;
  if (a.r.tokens > INT32_MAX / a.group) return cudaErrorInvalidValue;
  a.gave_up = a.arrive + a.sm_count * kAttnCtasPerSm;
  const int size = a.type == kKvF32 ? 4 : 2;
  a.q_vec = ((reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)(a.q_stride * size)) & 15) == 0;
  a.out_vec = ((reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)(a.out_stride * size)) & 15) == 0;
  // Query rows a sequence and key head, on average over the call, from which the
  // tensor cores' 128-row tiles pay although most of a tile may be empty.  16
  // sequences of 8,000 keys, 8 key heads, this kernel against those tiles, us: dim
  // 64, f32, 32 rows 96 : 219, 64 rows 180 : 216, 128 rows 343 : 185; bf16 64 rows
  // 169 : 215, 128 rows 322 : 180; dim 128, f32, 32 rows 194 : 235, 64 rows 367 :
  // 239; bf16 32 rows 162 : 238, 64 rows 305 : 239.  A batch of both kinds has one of
  // them in the wrong kernel: 60 single tokens on 8,000 keys each beside 512 rows
  // on 2,000 take 882 us there and would take 449 here, 300 single tokens on 2,000
  // beside a prompt of 2,000 take 1,695 here and would take 1,382 there; in two calls
  // these are 181 and 318.
  const int64_t few = a.c.nb > 2 ? 32 : 64;
  if (a.r.offsets && a.r.tokens * a.group > few * a.r.sequences) {
    const cudaError_t e = launch_attention_mma(a, stream);
    if (e != cudaErrorNotSupported) return e;
  }
  switch (a.type) {
    case kKvF32: return launch_dims<float>(a, stream);
    case kKvF16: return launch_dims<__half>(a, stream);
    case kKvBF16: return launch_dims<__nv_bfloat16>(a, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace spt
