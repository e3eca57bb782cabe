// spt_attn_mma.cu -- attention of many query rows over the 4-bit KV cache on
// the tcgen05 tensor cores (spt_attn.cu has the formula, and the kernel for
// few rows).
//
// A CTA takes up to 256 rows of one key head (new tokens x heads of the group;
// 128 above head_dim 64) and runs down their keys 64 at a time, with four
// kinds of warps:
//
//   loader     copies the tiles' records to shared memory (bulk copies) and
//              looks at their scales
//   dequant    six warps, write keys and values as f16 pairs hi + lo: a code
//              times its scale has 15 bits, so hi + lo is exact (a power of two
//              for the tile brings the largest scale that a row of the CTA sees to
//              2^11; scales down to 2^-25 of it keep all their bits, smaller ones
//              are at most 2^-36 of it off).  What no row sees is written as zeros.
//   issuer     S = Q K^T and O = P V into TMEM, from Q and P in TMEM, 128 rows each
//   softmax    one row a thread: the weights 2^(s - ref) of S's row back into
//              TMEM as f16 terms, O's row added up in registers
//
// f32 rows take two f16 terms of q: S = Qlo Khi + Qhi Klo + Qhi Khi, every product
// but lo * lo (2^-22 of it); f16 and bf16 rows are one term, S = Q Klo + Q Khi.  The
// weights are two terms whatever the rows' type, O = Plo Vhi + Phi Vlo + Phi Vhi:
// one would be 2^-11 of a weight off, as much as the rounding of an f16 row, and
// more where the values nearly cancel.  O starts from zero for each tile and is
// added in f32: the tensor cores' own long sums lose bits.  S is double
// buffered, so that the next tile's products run under a tile's softmax.
//
// Bound, for 256 rows x 64 keys at head_dim 64: 1,024 clocks of exponentials
// (16 a clock on an SM), 1,584 of MMA for f32 rows (48 of 33 clocks) and 1,320
// for 16-bit rows (40).  A tile takes some 3,300 clocks, those of the softmax
// warps' own chain: 200 to wait, 350 to fetch S, 300 for its maximum, 1,650 for the
// weights, 650 to add O, two warps a scheduler.  A prompt of 2,000 f32 rows (64
// heads on 8 of 64 dims) takes 161 us, tensor cores active in 28% of the cycles;
// f16 chunks of 12 sequences, 3,000 tokens each, 231 us.  Maxima of three instead
// of two, or each MMA's S right behind its own O, changed neither by 1%.
//
// The four roles' code together strains the instruction caches (0.6 to 0.8 warps
// an issue stall for want of an instruction), so that a few instructions more in
// one role can cost another 5%: the same change to the loader left prompts of 64
// dims alone and took f16 ones of 128 dims from 157 to 167 us.  Every instance
// spills 276 to 320 bytes a thread; the local loads and stores are 0.2 to 0.4% of
// the instructions executed.
#include "spt_attn.cuh"

namespace spt {
namespace {

constexpr int kMmaRows = 128, kMmaKeys = 64;  // of one MMA
constexpr int64_t kMmaMinTiles = 6;           // a CTA's smallest share
constexpr int kMmaHead = 3;                   // an item's beginning and end, in tiles' time

template <int NB, typename IO>
struct MmaTile {
  static constexpr int kDim = NB * 32;
  static constexpr int kTerms = sizeof(IO) == 4 ? 2 : 1;        // f16 terms of q
  static constexpr int kM = NB <= 2 ? 2 : 1;                    // 128-row MMAs of a CTA: a row's O fills the registers above
  static constexpr int kRows = kM * kMmaRows;
  static constexpr int kSoftmaxWarps = 4 * kM;
  static constexpr int kDequant = 6;                            // warps
  static constexpr int kThreads = 32 * (kSoftmaxWarps + 2 + kDequant);
  static constexpr int kAtoms = (kDim + 63) / 64;               // 128-byte swizzle atoms in a row of dims
  static constexpr int kKTerm = kAtoms * kMmaKeys * 128;
  static constexpr int kVTerm = kDim * 128;                     // 64 keys: one atom
  static constexpr int kStages = NB <= 2 ? 3 : 2;               // of keys, and of values
  static constexpr int kOffV = kStages * 2 * kKTerm;
  static constexpr int kRaw = NB <= 2 ? 4 : 3;                  // tiles' records
  static constexpr int kRecord = kv_tile_bytes(NB), kRawTile = 4 * kRecord;
  static constexpr int kOffRaw = kOffV + kStages * 2 * kVTerm;
  // rows on their way between global memory and a thread each: q's terms, out
  static constexpr int kPitch = kDim * (int)sizeof(IO), kPieces = kPitch / 16;
  static constexpr int kOffRows = kOffRaw + kRaw * kRawTile;
  static constexpr int kSmem = kOffRows + kRows * kPitch + 1024;  // + alignment
  static constexpr int kUnits = 4 * NB;                         // (16 keys, block) pieces of a tile
  // TMEM of one MMA's rows: S twice (64 columns), O, q's terms
  static constexpr int kColO = 2 * kMmaKeys, kColQ = kColO + kDim;
  static constexpr int kColsM = kColQ + kTerms * kDim / 2;
  static constexpr uint32_t kCols = kM * kColsM <= 256 ? 256 : 512;
  // The softmax warpgroups take registers from the others; the sum is no more
  // than what the block was launched with (checked before the first launch).
  static constexpr int kLaunchRegs = kM == 2 ? 128 : 168;
  static constexpr int kSoftmaxRegs = kM == 2 ? 168 : 240, kOtherRegs = kM == 2 ? 88 : 128;
  static_assert(kSoftmaxWarps * kSoftmaxRegs + (2 + kDequant) * kOtherRegs <= (kThreads / 32) * kLaunchRegs, "registers");
  static_assert(kSmem <= 226 * 1024 && kM * kColsM <= 512, "shared memory, TMEM");
};

__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t leader, uint64_t *bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(leader)
      : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// K-major operand with the 128-byte swizzle: rows of 128 bytes, 8-row groups
// 1024 bytes apart.  The descriptor's low half holds the address; it advances
// by 2 for 16 elements of a row.
__device__ __forceinline__ uint32_t swizzled_desc(uint32_t addr) { return addr >> 4 | 1u << 16; }
constexpr uint32_t kDescHigh = (1024 >> 4) | 1u << 14 | 2u << 29;
// kind::f16, A and B f16 and K-major, D f32, M = 128.
__device__ __forceinline__ constexpr uint32_t f16_idesc(int n) {
  return 1u << 4 | (uint32_t)(n >> 3) << 17 | (uint32_t)(128 >> 4) << 24;
}
// D (+)= A (TMEM) * B (shared memory).  The whole warp runs up to here with the
// same operands and `leader` alone issues: with uniform operands an MMA of M =
// 128, N = 64 takes its 33 clocks, from a single thread's branch (where each
// operand has to be moved to a uniform register) 80 or more.
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                       uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 bd;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 bd, {%2, %3};\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], bd, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "n"(kDescHigh), "r"(idesc), "r"(add), "r"(leader)
      : "memory");
}
// 64 or 32 columns of this warp's 32 TMEM lanes (and the wait).
__device__ __forceinline__ void tmem_load(uint32_t taddr, float (&v)[64]) {
  uint32_t r[64];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_load(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_store8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// brief_wait for a whole warp, which passes or gives up together.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, const AttnArgs &a, int code) {
  return __all_sync(0xffffffffu, brief_wait(bar, parity, a, code));
}

__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// What the loader says of a tile to the softmax warps ...
struct TileInfoAttn {
  float k_unit, v_unit;              // keys and values are in these units
  uint32_t ok;                       // bit i: keys 16 i .. 16 i + 15 lie on a page of the pool
  uint32_t any_nan;                  // some value block is a NaN
  unsigned long long nan[kKvMaxBlocks];  // of block b: keys whose values are NaNs (held as zeros)
};
// ... and to the dequant warps.
struct RawInfo {
  float k_up, v_up;
  uint32_t ok;
  int end;     // no tile: there are no more
  int lo, hi;  // the loader's: keys [lo, hi) of the tile are seen by rows of the item
};

// The scales of tokens `token`, + 1, + 8 and + 9 of a tile, zero outside [lo, hi).
__device__ __forceinline__ uint2 seen_scales(uint2 d, int token, int lo, int hi) {
  auto pair = [&](int t) { return (t >= lo && t < hi ? 0xffffu : 0u) | (t + 1 >= lo && t + 1 < hi ? 0xffff0000u : 0u); };
  return make_uint2(d.x & pair(token), d.y & pair(token + 8));
}

// A tile's information is overwritten by that of the tile kInfos on, which is
// loaded when the raw slot kRaw tiles before it is free, that is behind the PV
// of the tile kStages before that: behind every reader.
constexpr int kInfos = 8;

template <int NB, typename IO>
using MmaWalk = AttnWalk<MmaTile<NB, IO>::kRows, kMmaKeys, kMmaHead>;

template <int NB, typename IO>
struct MmaCta {
  using T = MmaTile<NB, IO>;
  static_assert(kInfos > T::kRaw + T::kStages, "tile information ring");
  uint64_t raw_full[T::kRaw], raw_ready[T::kRaw], raw_empty[T::kRaw];
  uint64_t k_full[T::kStages], k_empty[T::kStages], v_full[T::kStages], v_empty[T::kStages];
  uint64_t info_full[kInfos];
  uint64_t s_full[T::kM][2], p_full[T::kM][2], o_full[T::kM], o_empty[T::kM], q_full[T::kM], meet, told, drain;
  TileInfoAttn info[kInfos];
  RawInfo raw[T::kRaw];
  uint32_t tmem;
  int last;
};

// The MMAs of an item that have rows: the first always.
template <int NB, typename IO>
__device__ __forceinline__ int live_mmas(const AttnArgs &a, const MmaWalk<NB, IO> &w) {
  const int rows = w.seq.n * a.group - w.rb * MmaTile<NB, IO>::kRows;
  return MmaTile<NB, IO>::kM == 2 && rows > kMmaRows ? 2 : 1;
}

// The loader warp: records of the walk's tiles, kRaw - 1 ahead of the one whose
// scales it looks at.
template <int NB, typename IO>
__device__ __forceinline__ void load_tiles(const AttnArgs &a, MmaCta<NB, IO> &s, uint8_t *smem, MmaWalk<NB, IO> &w,
                                           int lane) {
  using T = MmaTile<NB, IO>;
  constexpr int kChunks = (16 * NB + 31) / 32;  // 8-byte pieces of the tile's scales a lane looks at
  const uint32_t tiles_per_page = (uint32_t)a.c.page_tokens / kKvTile;
  const int64_t page_tiles = a.r.max_pages * tiles_per_page;  // (a sequence has fewer than 2^28)
  uint8_t *const raw = smem + T::kOffRaw;
  // lane i (mod 4): the page of keys 16 i .. of a tile
  auto page_of = [&](int tile) {
    const uint32_t t16 = (uint32_t)(tile * (kMmaKeys / kKvTile)) + (lane & 3);
    return t16 < page_tiles ? __ldcg(a.r.table + w.b * a.r.max_pages + t16 / tiles_per_page) : -1;
  };
  int at = w.first_tile(), last = w.last_tile();
  bool more = true, page_known = false;
  int32_t page = 0;
  uint32_t oks = 0;            // 4 bits a tile under way, and one more where keys of it are seen by no row: the oldest lowest
  int ahead = 0, put = 0, get = 0, left_out = -1;
  uint32_t put_phase = 0, get_phase = 0, jt = 0;
  // starts the next tile's copies; false where a wait gave up
  auto start = [&]() {
    while (more && at >= last) {
      more = w.next(a);
      page_known = false;
      if (more) at = w.first_tile(), last = w.last_tile();
    }
    if (!more) return true;
    if (!page_known) page = page_of(at);
    if (!warp_wait(&s.raw_empty[put], put_phase ^ 1u, a, 30)) return false;
    const bool good = page >= 0 && page < a.c.pages;
    const uint32_t ok = __ballot_sync(0xffffffffu, good) & 15u;
    const bool fault = blockIdx.x == 0 && jt + ahead == (uint32_t)a.fault_tile;
    if (fault) left_out = put;
    if (lane == 0 && !fault) mbar_expect_tx(&s.raw_full[put], __popc(ok) * T::kRecord);
    __syncwarp();
    if (lane < 4 && good && !fault) {
      const uint32_t place = ((uint32_t)(at * (kMmaKeys / kKvTile)) + lane) % tiles_per_page;
      bulk_load(raw + put * T::kRawTile + lane * T::kRecord,
                a.c.base + kv_tile_offset(a.c, page, w.head, (int)place * kKvTile), T::kRecord, &s.raw_full[put]);
    }
    const int lo = w.tiles.lo - at * kMmaKeys, hi = w.tiles.hi - at * kMmaKeys;
    const bool edge = lo > 0 || hi < kMmaKeys;
    if (edge && lane == 0) s.raw[put].lo = lo, s.raw[put].hi = hi;
    oks |= (ok | (edge ? 16u : 0u)) << (5 * ahead);
    if (++put == T::kRaw) put = 0, put_phase ^= 1u;
    ++ahead;
    page = page_of(++at);  // of the item's next tile, if it has one
    page_known = true;
    return true;
  };
  bool fine = true;
#pragma unroll 1
  for (int i = 0; fine && i < T::kRaw - 1; ++i) fine = start();
#pragma unroll 1
  while (fine && ahead > 0) {
    if (!warp_wait(&s.raw_full[get], get_phase, a, 43)) break;
    const uint32_t ok = oks & 15u;
    uint8_t *from = raw + get * T::kRawTile;
    if (oks & 16u) {  // what no row sees counts as zeros, here and for the dequant warps
      const int lo = s.raw[get].lo, hi = s.raw[get].hi;
#pragma unroll 1
      for (int c = lane; c < 16 * NB; c += 32) {
        const int sub = c / (4 * NB), token = sub * kKvTile + c % (4 * NB) / NB * 2;
        uint2 *d = reinterpret_cast<uint2 *>(from + sub * T::kRecord + kv_key_scales(NB) + c % (4 * NB) * 8);
        d[0] = seen_scales(d[0], token, lo, hi);
        d[4 * NB] = seen_scales(d[4 * NB], token, lo, hi);  // (the values' come behind the keys')
      }
      fence_async_smem();  // the slot's next copy comes behind these writes
    }
    // largest scales of keys (low half) and values (high), NaNs aside; values' NaNs
    __half2 top = half2_of(0);
    uint32_t nan = 0;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int c = lane + 32 * i, sub = c / (4 * NB);
      if (sub >= 4 || !(ok >> sub & 1)) continue;
      const uint8_t *p = from + sub * T::kRecord + c % (4 * NB) * 8;
      const uint2 k = *reinterpret_cast<const uint2 *>(p + kv_key_scales(NB));
      const uint2 v = *reinterpret_cast<const uint2 *>(p + kv_value_scales(NB));
      const __half2 mk = __hmax2(half2_of(k.x & 0x7fff7fffu), half2_of(k.y & 0x7fff7fffu));
      const __half2 mv = __hmax2(half2_of(v.x & 0x7fff7fffu), half2_of(v.y & 0x7fff7fffu));
      top = __hmax2(top, __hmax2(__lows2half2(mk, mv), __highs2half2(mk, mv)));
#pragma unroll
      for (int x = 0; x < 4; ++x)
        nan |= (uint32_t)(((x < 2 ? v.x : v.y) >> (16 * (x & 1)) & 0x7fffu) > 0x7c00u) << (4 * i + x);
    }
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) top = __hmax2(top, half2_of(__shfl_xor_sync(0xffffffffu, bits(top), i)));
    const uint32_t any = __ballot_sync(0xffffffffu, nan != 0);
    // scaled by 2^(11 - its exponent), the largest lies in [2^11, 2^12)
    const float2 f = __half22float2(top);
    const int ke = f.x == 0.0f ? 0 : 11 - ((int)(__float_as_uint(f.x) >> 23) - 127);
    const int ve = f.y == 0.0f ? 0 : 11 - ((int)(__float_as_uint(f.y) >> 23) - 127);
    TileInfoAttn &info = s.info[jt % kInfos];
    if (lane == 0) {
      info.k_unit = exp2_int(-ke);
      info.v_unit = exp2_int(-ve);
      info.ok = ok;
      info.any_nan = any;
      s.raw[get] = {exp2_int(ke), exp2_int(ve), ok, 0, 0, 0};
    }
    if (any) {
      if (lane < kKvMaxBlocks) info.nan[lane] = 0;
      __syncwarp();
      for (int i = 0; i < 4 * kChunks; ++i)
        if (nan >> i & 1) {
          const int c = lane + 32 * (i / 4), x = i % 4, sub = c / (4 * NB), tt = c % (4 * NB) / NB, blk = c % NB;
          atomicOr(&info.nan[blk], 1ull << (sub * 16 + 2 * tt + (x & 1) + 8 * (x >> 1)));
        }
    }
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(&s.raw_ready[get]);
      mbar_arrive(&s.info_full[jt % kInfos]);
    }
    ++jt;
    oks >>= 5;
    --ahead;
    if (++get == T::kRaw) get = 0, get_phase ^= 1u;
    fine = start();
  }
  if (fine && ahead == 0) {  // the end, in a slot of its own
    if (warp_wait(&s.raw_empty[put], put_phase ^ 1u, a, 44)) {
      if (lane == 0) {
        s.raw[put].end = 1;
        mbar_arrive(&s.raw_ready[put]);
      }
      __syncwarp();
    }
  }
  // after a wait that gave up: no copy may land when the CTA has gone
  for (; ahead > 0; --ahead) {
    if (get != left_out) mbar_wait_own(&s.raw_full[get], get_phase);  // (about a second at most, whatever the option says)
    if (++get == T::kRaw) get = 0, get_phase ^= 1u;
  }
}

// A dequant warp: keys and values of the loaded tiles as f16 pairs.
template <int NB, typename IO>
__device__ __forceinline__ void dequantise(const AttnArgs &a, MmaCta<NB, IO> &s, uint8_t *smem, int dw, int lane) {
  using T = MmaTile<NB, IO>;
  const int g = lane >> 2, t = lane & 3;
  const int dv = (dw + T::kDequant - T::kUnits % T::kDequant) % T::kDequant;  // who took one piece of the keys more takes one of the values less
  int slot = 0, stage = 0;
  uint32_t slot_phase = 0, phase = 0;
#pragma unroll 1
  while (true) {
    if (!warp_wait(&s.raw_ready[slot], slot_phase, a, 45)) return;
    const RawInfo info = s.raw[slot];
    if (info.end) return;
    const uint8_t *raw = smem + T::kOffRaw + slot * T::kRawTile;
    // ---- keys ----
    if (!warp_wait(&s.k_empty[stage], phase ^ 1u, a, 31)) return;
    uint8_t *kb = smem + stage * 2 * T::kKTerm;
#pragma unroll 1
    for (int u = dw; u < T::kUnits; u += T::kDequant) {
      const int sub = u / NB, blk = u % NB;
      const uint8_t *rec = raw + sub * T::kRecord;
      uint2 codes = make_uint2(0, 0), d = make_uint2(0, 0);
      if (info.ok >> sub & 1) {
        codes = *reinterpret_cast<const uint2 *>(rec + (blk >> 1) * 512 + ((blk | 1) < NB ? lane * 16 + (blk & 1) * 8 : lane * 8));
        d = *reinterpret_cast<const uint2 *>(rec + kv_key_scales(NB) + (g >> 1) * NB * 8 + blk * 8);
      }
      const int chunk = blk * 4 + t;
      uint8_t *to = kb + (chunk >> 3) * (kMmaKeys * 128) + (sub * 16 + g) * 128 + (((chunk & 7) ^ g) << 4);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t pair = h ? d.y : d.x;
        const float scale = __half2float(__ushort_as_half((unsigned short)(g & 1 ? pair >> 16 : pair)));
        const __half2 dn = __float2half2_rn(scale * info.k_up);
        uint32_t e[4], hi[4], lo[4];
        decode_word(h ? codes.y : codes.x, e);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const __half2 v = __hmul2(half2_of(e[x]), dn);
          hi[x] = bits(v);
          lo[x] = bits(__hfma2(half2_of(e[x]), dn, __hneg2(v)));
        }
        *reinterpret_cast<uint4 *>(to + h * 1024) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4 *>(to + h * 1024 + T::kKTerm) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
    fence_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&s.k_full[stage]);
    // ---- values ----
    if (!warp_wait(&s.v_empty[stage], phase ^ 1u, a, 32)) return;
    uint8_t *vb = smem + T::kOffV + stage * 2 * T::kVTerm;
#pragma unroll 1
    for (int u = dv; u < T::kUnits; u += T::kDequant) {
      const int sub = u / NB, blk = u % NB;
      const uint8_t *rec = raw + sub * T::kRecord + kv_value_codes(NB);
      uint2 codes = make_uint2(0, 0), d = make_uint2(0, 0);
      if (info.ok >> sub & 1) {
        codes = *reinterpret_cast<const uint2 *>(rec + (blk >> 1) * 512 + ((blk | 1) < NB ? lane * 16 + (blk & 1) * 8 : lane * 8));
        d = *reinterpret_cast<const uint2 *>(rec + (kv_value_scales(NB) - kv_value_codes(NB)) + t * NB * 8 + blk * 8);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float2 f = __half22float2(half2_of(h ? d.y : d.x));
        // a NaN is said in the tile's information: in the product it would reach every row
        f.x = isnan(f.x) ? 0.0f : f.x * info.v_up;
        f.y = isnan(f.y) ? 0.0f : f.y * info.v_up;
        const __half2 dn = __floats2half2_rn(f.x, f.y);
        uint32_t e[4];
        decode_word(h ? codes.y : codes.x, e);
        // dim 32 blk + 4 g + x lies in row 32 blk + 8 x + g
        uint8_t *to = vb + (32 * blk + g) * 128 + (((sub * 2 + h) ^ g) << 4) + t * 4;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const __half2 v = __hmul2(half2_of(e[x]), dn);
          *reinterpret_cast<uint32_t *>(to + x * 1024) = bits(v);
          *reinterpret_cast<uint32_t *>(to + x * 1024 + T::kVTerm) = bits(__hfma2(half2_of(e[x]), dn, __hneg2(v)));
        }
      }
    }
    fence_async_smem();
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(&s.v_full[stage]);
      mbar_arrive(&s.raw_empty[slot]);
    }
    if (++stage == T::kStages) stage = 0, phase ^= 1u;
    if (++slot == T::kRaw) slot = 0, slot_phase ^= 1u;
  }
}

// The issuer, a whole warp of which one lane (`leader`) issues.
template <int NB, typename IO>
__device__ __forceinline__ bool issue(const AttnArgs &a, MmaCta<NB, IO> &s, uint32_t smem, MmaWalk<NB, IO> &w,
                                      uint32_t leader) {
  using T = MmaTile<NB, IO>;
  constexpr uint32_t s_desc = f16_idesc(kMmaKeys), o_desc = f16_idesc(T::kDim);
  const uint32_t tmem = __shfl_sync(0xffffffffu, s.tmem, 0);
  uint32_t items0 = 0, items1 = 0, turn0 = 0, turn1 = 0;  // of each MMA: items, tiles
  int k_stage = 0, v_stage = 0;
  uint32_t k_phase = 0, v_phase = 0;
  do {
    const int n = w.last_tile() - w.first_tile();
    if (n <= 0) continue;
    const int mmas = live_mmas<NB, IO>(a, w);
    if (!warp_wait(&s.q_full[0], items0++ & 1u, a, 35)) return false;
    if (mmas == 2 && !warp_wait(&s.q_full[T::kM - 1], items1++ & 1u, a, 35)) return false;
    auto values = [&]() {  // O of the tile whose weights come next
      if (!warp_wait(&s.v_full[v_stage], v_phase, a, 32)) return false;
      const uint32_t v = swizzled_desc(smem + T::kOffV + v_stage * 2 * T::kVTerm);
#pragma unroll 1
      for (int m = 0; m < mmas; ++m) {
        const uint32_t turn = m ? turn1 : turn0;
        if (!warp_wait(&s.p_full[m][turn & 1], turn >> 1 & 1u, a, 33)) return false;
        if (!warp_wait(&s.o_empty[m], (turn & 1u) ^ 1u, a, 34)) return false;
        tc_after();
        const uint32_t o = tmem + m * T::kColsM + T::kColO, p = tmem + m * T::kColsM + (turn & 1) * kMmaKeys;
        // the weights of 16 keys: 8 columns of each term, side by side
#pragma unroll 1
        for (int x = 0; x < 3; ++x) {  // Plo Vhi, Phi Vlo, Phi Vhi
          const uint32_t pt = p + (x == 0 ? 8 : 0), vt = v + (x == 1 ? T::kVTerm / 16 : 0);
#pragma unroll
          for (int k = 0; k < kMmaKeys / 16; ++k) mma_ts(leader, o, pt + k * 16, vt + k * 2, o_desc, x + k > 0);
        }
        tc_commit(leader, &s.o_full[m]);
      }
      ++turn0;
      if (mmas == 2) ++turn1;
      tc_commit(leader, &s.v_empty[v_stage]);
      if (++v_stage == T::kStages) v_stage = 0, v_phase ^= 1u;
      return true;
    };
    for (int i = 0; i < n; ++i) {
      if (!warp_wait(&s.k_full[k_stage], k_phase, a, 36)) return false;
      tc_after();
      const uint32_t kd = swizzled_desc(smem + k_stage * 2 * T::kKTerm);
#pragma unroll 1
      for (int m = 0; m < mmas; ++m) {
        // this MMA's tile `turn` is computed while its tile turn - 1 waits for its weights
        const uint32_t buf = ((m ? turn1 : turn0) + (i > 0)) & 1;
        const uint32_t q = tmem + m * T::kColsM + T::kColQ, to = tmem + m * T::kColsM + buf * kMmaKeys;
#pragma unroll 1
        for (int x = 3 - T::kTerms - 1; x < 3; ++x) {  // Qlo Khi (two terms), Qhi Klo, Qhi Khi
          const uint32_t qt = q + (x == 0 ? T::kDim / 2 : 0), kt = kd + (x == 1 ? T::kKTerm / 16 : 0);
#pragma unroll
          for (int k = 0; k < T::kDim / 16; ++k)
            mma_ts(leader, to, qt + k * 8, kt + (k >> 2) * (kMmaKeys * 128 / 16) + (k & 3) * 2, s_desc, x + k > 2 - T::kTerms);
        }
        tc_commit(leader, &s.s_full[m][buf]);
      }
      tc_commit(leader, &s.k_empty[k_stage]);
      if (++k_stage == T::kStages) k_stage = 0, k_phase ^= 1u;
      if (i > 0 && !values()) return false;
    }
    if (!values()) return false;
  } while (w.next(a));
  return true;
}

// The softmax warps: thread = row.  `arrived`: the current item's part is
// counted.
template <int NB, typename IO>
__device__ __forceinline__ bool softmax(const AttnArgs &a, MmaCta<NB, IO> &s, uint8_t *smem, MmaWalk<NB, IO> &w,
                                        int warp, int lane, bool &arrived) {
  using T = MmaTile<NB, IO>;
  constexpr int DIM = T::kDim, ROWS = T::kRows;
  const int row = warp * 32 + lane, m = warp >> 2;
  const uint32_t cols = s.tmem + m * T::kColsM + ((uint32_t)((warp & 3) * 32) << 16);
  // this warp's 32 rows under way: 16-byte piece p of row r
  uint8_t *const rows = smem + T::kOffRows + warp * 32 * T::kPitch;
  auto piece = [&](int r, int p) {
    return rows + r * T::kPitch + ((p ^ (r & (T::kPieces % 8 == 0 ? 7 : 3))) << 4);
  };
  uint32_t jt = 0, turn = 0, parts = 0;  // tiles, this MMA's tiles, items shared with other CTAs so far
  do {
    const SeqRows &seq = w.seq;
    const int r = w.rb * ROWS + row, i = (int)((uint32_t)r / (uint32_t)a.group);
    const bool live = i < seq.n;
    const int head = w.head * a.group + r - i * a.group;
    const int first = w.first_tile(), last = w.last_tile();
    // positions are below 2^31, a tile's end may not be
    const int key_hi = live ? max(seq.len - seq.n + i + 1, 0) : 0;
    const int key_lo = a.window > 0 && key_hi > a.window ? key_hi - (int)a.window : 0;
    float ref = 0.0f, l = 0.0f;
    bool fresh = true;
    float2 o[DIM / 2];
#pragma unroll
    for (int x = 0; x < DIM / 2; ++x) o[x] = make_float2(0.0f, 0.0f);
    if (last > first && m < live_mmas<NB, IO>(a, w)) {
      // q as f16 terms: rows to shared memory whole, then a thread each (the
      // issuer has read the last item's when its last S was seen)
      constexpr int kElems = 16 / (int)sizeof(IO);
      const IO *q = static_cast<const IO *>(a.q);
#pragma unroll 4
      for (int x = lane; x < 32 * T::kPieces; x += 32) {
        const int rr = x / T::kPieces, p = x % T::kPieces;
        const int from = w.rb * ROWS + warp * 32 + rr, fi = (int)((uint32_t)from / (uint32_t)a.group);
        const IO *src = q + (int64_t)(seq.start + fi) * a.q_stride + (int64_t)(w.head * a.group + from - fi * a.group) * DIM + p * kElems;
        if (fi >= seq.n) {
          *reinterpret_cast<uint4 *>(piece(rr, p)) = make_uint4(0, 0, 0, 0);
        } else if (a.q_vec) {
          cp_async16(piece(rr, p), src);
        } else {
          IO e[kElems];
#pragma unroll
          for (int y = 0; y < kElems; ++y) e[y] = src[y];
          *reinterpret_cast<uint4 *>(piece(rr, p)) = *reinterpret_cast<const uint4 *>(e);
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
      float top = 0.0f;
#pragma unroll 4
      for (int x = 0; x < T::kPieces; ++x) {
        const uint4 u = *reinterpret_cast<const uint4 *>(piece(lane, x));
        const IO *e = reinterpret_cast<const IO *>(&u);
#pragma unroll
        for (int y = 0; y < kElems; ++y) top = fmaxf(top, fabsf(row_float<IO>(e[y])));
      }
      // a power of two brings the row's largest magnitude to [2^14, 2^15)
      int e2 = 14 - ((int)(__float_as_uint(top) >> 23) - 127);
      if (top == 0.0f) e2 = 0;
      if (e2 > 100) e2 = 100;
      // an infinity makes every score of its row a NaN
      const float up = top == INFINITY ? __int_as_float(0x7fffffff) : exp2_int(e2);
      const float c = a.scale * kLog2e * exp2_int(-e2);
#pragma unroll 1
      for (int x = 0; x < DIM / 16; ++x) {
        constexpr int kSpan = 16 / kElems;  // pieces of 16 dims
        uint4 u[kSpan];
#pragma unroll
        for (int y = 0; y < kSpan; ++y) u[y] = *reinterpret_cast<const uint4 *>(piece(lane, x * kSpan + y));
        const IO *e = reinterpret_cast<const IO *>(u);
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int y = 0; y < 8; ++y) {  // the order of the keys' words: dims z and z + 4 of eight make a pair
          const int z = (y & 4) * 2 + (y & 3);
          const float x0 = row_float<IO>(e[z]) * up, x1 = row_float<IO>(e[z + 4]) * up;
          const __half2 h = __floats2half2_rn(x0, x1);
          const float2 f = __half22float2(h);
          hi[y] = bits(h);
          lo[y] = pack_half2(x0 - f.x, x1 - f.y);
        }
        tmem_store8(cols + T::kColQ + x * 8, hi);
        if (T::kTerms == 2) tmem_store8(cols + T::kColQ + DIM / 2 + x * 8, lo);
      }
      tmem_store_wait();
      tc_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.q_full[m]);

      float v_unit = 0.0f;  // of the tile whose O is to be added next, times what ref has moved since
      auto add_o = [&](uint32_t j) {
        if (!warp_wait(&s.o_full[m], j & 1u, a, 37)) return false;
        tc_after();
        const float2 unit = make_float2(v_unit, v_unit);
        constexpr int kSpan = DIM % 64 == 0 ? 64 : 32;
#pragma unroll
        for (int x = 0; x < DIM; x += kSpan) {
          float v[kSpan];
          tmem_load(cols + T::kColO + x, v);
#pragma unroll
          for (int y = 0; y < kSpan / 2; ++y)
            o[x / 2 + y] = __ffma2_rn(make_float2(v[2 * y], v[2 * y + 1]), unit, o[x / 2 + y]);
        }
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.o_empty[m]);
        return true;
      };
      int key0 = first * kMmaKeys;
#pragma unroll 1
      for (int tile = first; tile < last; ++tile, ++jt, ++turn, key0 += kMmaKeys) {
        const uint32_t sc = cols + (turn & 1) * kMmaKeys;
        // S first: only then is info_full in the phase that its parity names, as
        // warps whose MMA had no rows in the last items come here early
        if (!__all_sync(0xffffffffu, mbar_try(&s.s_full[m][turn & 1], turn >> 1 & 1u) &&
                                         mbar_try(&s.info_full[jt % kInfos], jt / kInfos & 1u))) {
          if (!warp_wait(&s.s_full[m][turn & 1], turn >> 1 & 1u, a, 39)) return false;
          if (!warp_wait(&s.info_full[jt % kInfos], jt / kInfos & 1u, a, 38)) return false;
        }
        tc_after();
        const TileInfoAttn &info = s.info[jt % kInfos];
        // (never 0: a masked score of -inf has to stay one)
        const float scale = fmaxf(c * info.k_unit, 1.2e-38f), next_unit = info.v_unit;
        const uint32_t ok = info.ok, any_nan = info.any_nan;
        const bool edge = __any_sync(0xffffffffu, key_lo > key0 || key_hi - key0 < kMmaKeys || ok != 15u);
        float v[kMmaKeys];
        tmem_load(sc, v);
        if (edge || any_nan) {  // keys of the tile that this row does not see: their scores become -inf
          const int lo = key_lo - key0, hi = key_hi - key0;
          unsigned long long seen = hi > 0 ? ~0ull >> (hi < kMmaKeys ? kMmaKeys - hi : 0) : 0;
          seen &= lo > 0 ? lo < kMmaKeys ? ~0ull << lo : 0 : ~0ull;
          for (int x = 0; x < 4; ++x)
            if (!(ok >> x & 1)) seen &= ~(0xffffull << (16 * x));
          const uint32_t half[2] = {(uint32_t)seen, (uint32_t)(seen >> 32)};
#pragma unroll
          for (int x = 0; x < kMmaKeys; ++x) v[x] = half[x / 32] >> (x % 32) & 1 ? v[x] : -INFINITY;
          if (any_nan)
#pragma unroll
            for (int x = 0; x < NB; ++x)
              if (info.nan[x] & seen)
#pragma unroll
                for (int y = 0; y < 16; ++y) o[x * 16 + y].x = o[x * 16 + y].y = __int_as_float(0x7fffffff);
        }
        float tops[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
        for (int x = 4; x < kMmaKeys; ++x) tops[x & 3] = fmaxf(tops[x & 3], v[x]);
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        // weights are 2^(s - ref), ref the maximum less 7 until a score exceeds it by 8 more:
        // at most 2^15, and f16 terms down to 2^-24
        const float most = top * scale;
        if (most > (fresh ? -INFINITY : ref + 15.0f)) {
          const float now = most - 7.0f;
          const float factor = fresh ? 1.0f : exp2f(ref - now);
          ref = now;
          fresh = false;
          l *= factor;
          v_unit *= factor;
          const float2 f2 = make_float2(factor, factor);
#pragma unroll
          for (int x = 0; x < DIM / 2; ++x) o[x] = __fmul2_rn(o[x], f2);
        }
        const float2 scale2 = make_float2(scale, scale), ref2 = make_float2(-ref, -ref), minus = make_float2(-1.0f, -1.0f);
        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t ph[8], pl[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            float2 p = __ffma2_rn(make_float2(v[16 * q + 2 * x], v[16 * q + 2 * x + 1]), scale2, ref2);
            p.x = exp2_fast(p.x), p.y = exp2_fast(p.y);
            sum = __fadd2_rn(sum, p);
            const float2 f = make_float2(__uint_as_float(__float_as_uint(p.x) & 0xffffe000u),
                                         __uint_as_float(__float_as_uint(p.y) & 0xffffe000u));
            const float2 low = __ffma2_rn(f, minus, p);
            ph[x] = pack_half2(f.x, f.y);
            pl[x] = pack_half2(low.x, low.y);
          }
          tmem_store8(sc + 16 * q, ph);
          tmem_store8(sc + 16 * q + 8, pl);
        }
        l += sum.x + sum.y;
        tmem_store_wait();
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.p_full[m][turn & 1]);
        if (tile > first && !add_o(turn - 1)) return false;
        v_unit = next_unit;
      }
      if (!add_o(turn - 1)) return false;
    } else {
      jt += (uint32_t)(last - first);
    }

    // ---- the rows' end -------------------------------------------------------------
    float end_ref = fresh && l == 0.0f ? -INFINITY : ref;
    bool write = true;
    if (!w.whole()) {
      const int first_cta = w.first_share(), last_cta = w.last_share();
      float *slot = part_slot<ROWS, DIM>(a, blockIdx.x, first_cta);
#pragma unroll
      for (int x = 0; x < DIM / 2; x += 2)  // column groups first: neighbouring rows lie side by side
        *reinterpret_cast<float4 *>(slot + (x / 2 * ROWS + row) * 4) = make_float4(o[x].x, o[x].y, o[x + 1].x, o[x + 1].y);
      slot[ROWS * DIM + row] = end_ref;
      slot[ROWS * (DIM + 1) + row] = l;
      __threadfence();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.meet);
      if (!warp_wait(&s.meet, parts & 1u, a, 41)) return false;
      if (row == 0) {
        s.last = arrive(a, w);
        mbar_arrive(&s.told);
      }
      arrived = true;
      if (!warp_wait(&s.told, parts & 1u, a, 42)) return false;
      ++parts;
      write = s.last;
      if (write) {
        __threadfence();
        float top = -INFINITY;
        for (int x = first_cta; x <= last_cta; ++x)
          top = fmaxf(top, __ldcg(part_slot<ROWS, DIM>(a, x, first_cta) + ROWS * DIM + row));
        l = 0.0f;
#pragma unroll
        for (int x = 0; x < DIM / 2; ++x) o[x] = make_float2(0.0f, 0.0f);
#pragma unroll 1
        for (int x = first_cta; x <= last_cta; ++x) {
          const float *p = part_slot<ROWS, DIM>(a, x, first_cta);
          const float pr = __ldcg(p + ROWS * DIM + row);
          const float f = pr == -INFINITY ? 0.0f : exp2f(pr - top);
          l += __ldcg(p + ROWS * (DIM + 1) + row) * f;
          const float2 f2 = make_float2(f, f);
#pragma unroll
          for (int y = 0; y < DIM / 2; y += 2) {
            const float4 v = __ldcg(reinterpret_cast<const float4 *>(p + (y / 2 * ROWS + row) * 4));
            o[y] = __ffma2_rn(make_float2(v.x, v.y), f2, o[y]);
            o[y + 1] = __ffma2_rn(make_float2(v.z, v.w), f2, o[y + 1]);
          }
        }
        end_ref = top;
      }
    }
    if (write) {
      // through shared memory, so that rows are written whole
      const float end = live ? row_factor(a, head, end_ref, l) : 0.0f;
      constexpr int kPieces = T::kPieces, kElems = 16 / (int)sizeof(IO);
#pragma unroll
      for (int x = 0; x < kPieces; ++x) {
        IO e[kElems];
#pragma unroll
        for (int y = 0; y < kElems; ++y) {  // dim 32 b + 4 g + z is column 32 b + 8 z + g
          const int out = x * kElems + y, col = (out & ~31) + 8 * (out & 3) + ((out & 31) >> 2);
          e[y] = row_round<IO>((col & 1 ? o[col / 2].y : o[col / 2].x) * end);
        }
        *reinterpret_cast<uint4 *>(piece(lane, x)) = *reinterpret_cast<const uint4 *>(e);
      }
      __syncwarp();
#pragma unroll 2
      for (int x = lane; x < 32 * kPieces; x += 32) {
        const int rr = x / kPieces, p = x % kPieces;
        const int to = w.rb * ROWS + warp * 32 + rr, ti = (int)((uint32_t)to / (uint32_t)a.group);
        if (ti >= seq.n) continue;
        IO *out = static_cast<IO *>(a.out) + (int64_t)(seq.start + ti) * a.out_stride +
                  (int64_t)(w.head * a.group + to - ti * a.group) * DIM + p * kElems;
        const uint4 v = *reinterpret_cast<const uint4 *>(piece(rr, p));
        if (a.out_vec) {
          *reinterpret_cast<uint4 *>(out) = v;
        } else {
          const IO *e = reinterpret_cast<const IO *>(&v);
#pragma unroll
          for (int y = 0; y < kElems; ++y) out[y] = e[y];
        }
      }
      __syncwarp();
    }
    arrived = false;
  } while (w.next(a));
  return true;
}

template <int NB, typename IO>
__global__ void __launch_bounds__(MmaTile<NB, IO>::kThreads, 1) k_attn_mma(const AttnArgs a) {
  using T = MmaTile<NB, IO>;
  extern __shared__ uint8_t raw[];
  __shared__ MmaCta<NB, IO> s;
  uint8_t *smem = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  MmaWalk<NB, IO> w;
  if (!w.template begin<T::kThreads>(a, kMmaMinTiles, blockIdx.x, gridDim.x)) return;
  if (threadIdx.x == 0) {
    a.gave_up[blockIdx.x] = 0;
    for (int i = 0; i < T::kRaw; ++i) {
      mbar_init(&s.raw_full[i], 1);
      mbar_init(&s.raw_ready[i], 1);
      mbar_init(&s.raw_empty[i], T::kDequant);
    }
    for (int i = 0; i < T::kStages; ++i) {
      mbar_init(&s.k_full[i], T::kDequant);
      mbar_init(&s.v_full[i], T::kDequant);
      mbar_init(&s.k_empty[i], 1);
      mbar_init(&s.v_empty[i], 1);
    }
    for (int i = 0; i < kInfos; ++i) mbar_init(&s.info_full[i], 1);
    for (int m = 0; m < T::kM; ++m) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s.s_full[m][i], 1);
        mbar_init(&s.p_full[m][i], 4);
      }
      mbar_init(&s.o_full[m], 1);
      mbar_init(&s.o_empty[m], 4);
      mbar_init(&s.q_full[m], 4);
    }
    mbar_init(&s.meet, T::kSoftmaxWarps);
    mbar_init(&s.told, 1);
    mbar_init(&s.drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == T::kSoftmaxWarps) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s.tmem)),
                 "r"(T::kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  if (warp < T::kSoftmaxWarps) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(T::kSoftmaxRegs));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(T::kOtherRegs));
  if (warp < T::kSoftmaxWarps) {
    bool arrived = false;
    if (!softmax<NB, IO>(a, s, smem, w, warp, lane, arrived) && threadIdx.x == 0) {
      // a wait gave up: the parts that are left still count, so that the counters end at zero
      do {
        if (!arrived && !w.whole()) arrive(a, w);
        arrived = false;
      } while (w.next(a));
    }
  } else if (warp == T::kSoftmaxWarps + 1) {
    load_tiles<NB, IO>(a, s, smem, w, lane);
  } else if (warp > T::kSoftmaxWarps + 1) {
    dequantise<NB, IO>(a, s, smem, warp - T::kSoftmaxWarps - 2, lane);
  } else {
    uint32_t leader;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(leader));
    issue<NB, IO>(a, s, smem_u32(smem), w, leader);
    // nothing of the tensor cores' may be in flight when TMEM is freed
    tc_commit(leader, &s.drain);
    if (!mbar_wait_own(&s.drain, 0)) atomicCAS(a.err, 0, 40);
  }
  tc_before();
  __syncthreads();
  tc_after();
  if (threadIdx.x == 0) {
    const int code = *(volatile int32_t *)(a.gave_up + blockIdx.x);
    if (code != 0) atomicCAS(a.err, 0, code);
  }
  if (warp == T::kSoftmaxWarps)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s.tmem), "r"(T::kCols) : "memory");
}

template <int NB, typename IO>
cudaError_t launch(const AttnArgs &a, cudaStream_t stream) {
  using T = MmaTile<NB, IO>;
  cudaError_t e = opt_in_smem(k_attn_mma<NB, IO>, T::kSmem);
  if (e != cudaSuccess) return e;
  // the register split waits for ever where the block was launched with fewer:
  // another compiler's build is left to the kernel for few rows
  static std::atomic<int> regs{0};
  if (regs.load() == 0) {
    cudaFuncAttributes at;
    if ((e = cudaFuncGetAttributes(&at, k_attn_mma<NB, IO>)) != cudaSuccess) return e;
    regs.store(at.numRegs);
  }
  if (regs.load() != T::kLaunchRegs) return cudaErrorNotSupported;
  return launch_pdl(k_attn_mma<NB, IO>, dim3(a.sm_count), dim3(T::kThreads), T::kSmem, stream, a);
}

template <typename IO>
cudaError_t launch_dims(const AttnArgs &a, cudaStream_t stream) {
  switch (a.c.nb) {
    case 1: return launch<1, IO>(a, stream);
    case 2: return launch<2, IO>(a, stream);
    case 3: return launch<3, IO>(a, stream);
    case 4: return launch<4, IO>(a, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

size_t attn_mma_workspace_bytes(int sm_count, int nb) {
  return (size_t)sm_count * 2 * (nb <= 2 ? 2 : 1) * kMmaRows * (nb * 32 + 2) * sizeof(float);
}

cudaError_t launch_attention_mma(const AttnArgs &a, cudaStream_t stream) {
  switch (a.type) {
    case kKvF32: return launch_dims<float>(a, stream);
    case kKvF16: return launch_dims<__half>(a, stream);
    case kKvBF16: return launch_dims<__nv_bfloat16>(a, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace spt
