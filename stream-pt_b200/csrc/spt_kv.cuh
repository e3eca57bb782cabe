// spt_kv.cuh -- the 4-bit KV cache: block format, HBM layout and launchers.
//
// Format.  A block is 32 consecutive dims of one head of one token (keys and
// values alike).  With m its element of largest magnitude (the first among
// equals), d = f16(m / -8) saturated to +-65504, the block holds d and 4-bit
// codes n = clamp(rint(x / d) + 8, 0, 15) (n = 8 where d = 0); it stands for
// (n - 8) * d.  A block with a NaN has d = NaN.  rint(fl32(x / d)) is the
// rounding of the exact quotient: a halfway point (k + 1/2) d has at most 15
// significant bits, so x differs from it by nothing or by at least ulp(x),
// more than half an ulp of the quotient.
//
// Layout.  Tokens live in pages of `page_tokens` (a multiple of 16); a page
// holds, for each head, its 16-token tiles one after another:
//
//   [layer][page][kv_head][page_tokens / 16] tiles of NB * 576 bytes, NB = head_dim / 32
//
// and a tile holds key codes (NB * 256 bytes), value codes (NB * 256), key
// scales (NB * 32), value scales (NB * 32).  The codes lie in the order in
// which a warp's m16n8k16 fragments want them, so that a lane takes its share
// of a tile with 16-byte loads and no shuffle.  With lane = 4 g + t:
//
//   key word   (block b, lane, h):  token g + 8 h, dims 32 b + 8 t + i in nibble i
//   value word (block b, lane, h):  low half token 2 t + 8 h, high half token 2 t + 1 + 8 h,
//                                   dims 32 b + 4 g + i in nibble i of each half
//   words of blocks 2 c and 2 c + 1: byte c * 512 + lane * 16 + ((b & 1) * 2 + h) * 4;
//   an odd last block:               byte c * 512 + lane * 8 + h * 4
//   scale      (block b, token):     byte t * NB * 8 + b * 8 + (2 h + (token & 1)) * 2, for token = 2 t + (token & 1) + 8 h
//
// Nibbles i and i + 4 of a word are the two halves of one f16 pair, and no
// byte is shared by two tokens, so tokens of one tile may be written by
// different threads.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace spt {

constexpr int kKvTile = 16;        // tokens in a tile
constexpr int kKvBlock = 32;       // values that share a scale
constexpr int kKvMaxBlocks = 4;    // head_dim <= 128

enum KvType : int { kKvF32 = 0, kKvF16 = 1, kKvBF16 = 30 };  // GGML type numbers

// One layer's share of the pool.
struct KvLayer {
  uint8_t *base = nullptr;
  int64_t pages = 0;
  int kv_heads = 0, nb = 0;
  int page_tokens = 0;
};

// What a call works on (device pointers).  Sequence b's new rows are
// offsets[b] .. offsets[b+1] (row b alone without offsets), at positions
// lengths[b] - n .. lengths[b] - 1.
struct KvRows {
  const int32_t *table = nullptr;    // [sequences][max_pages]
  const int32_t *lengths = nullptr;  // [sequences]
  const int32_t *offsets = nullptr;  // [sequences + 1] or null
  int64_t sequences = 0, tokens = 0, max_pages = 0;
};

__host__ __device__ constexpr int kv_tile_bytes(int nb) { return nb * 576; }
__host__ __device__ constexpr int kv_value_codes(int nb) { return nb * 256; }
__host__ __device__ constexpr int kv_key_scales(int nb) { return nb * 512; }
__host__ __device__ constexpr int kv_value_scales(int nb) { return nb * 544; }

// Byte of word (block b, lane, h) within the key or value codes.
__host__ __device__ constexpr int kv_word(int nb, int b, int lane, int h) {
  return (b >> 1) * 512 + ((b | 1) < nb ? lane * 16 + ((b & 1) * 2 + h) * 4 : lane * 8 + h * 4);
}
// Byte of the scale of (block b, token) within the key or value scales.
__host__ __device__ constexpr int kv_scale(int nb, int b, int token) {
  return ((token & 7) >> 1) * nb * 8 + b * 8 + ((token >> 3) * 2 + (token & 1)) * 2;
}

// Tile of (page, head, place in the page).
__host__ __device__ inline int64_t kv_tile_offset(const KvLayer &c, int64_t page, int head, int place) {
  const int64_t tiles = c.page_tokens / kKvTile;
  return ((page * c.kv_heads + head) * tiles + place / kKvTile) * (int64_t)kv_tile_bytes(c.nb);
}

// Rows of k and v ([tokens][stride] elements of `type`, head h at h * head_dim)
// into the cache; rows whose position or page lies outside it are skipped.
cudaError_t launch_kv_append(const KvLayer &c, const KvRows &r, int type, const void *k, int64_t k_stride,
                             const void *v, int64_t v_stride, cudaStream_t stream);
// The same rows out of the cache (k or v may be null); rows outside it are left as they were.
cudaError_t launch_kv_read(const KvLayer &c, const KvRows &r, int type, void *k, int64_t k_stride, void *v,
                           int64_t v_stride, cudaStream_t stream);

// Beam reorder: the tables and lengths of batch * beams sequences put in the
// order of their parents, and partial last pages copied where a second child
// needs one of its own.
struct KvReorder {
  const int32_t *parents = nullptr;  // [batch][parents_stride], the first `beams` of each row count
  int64_t parents_stride = 0;
  const int32_t *table = nullptr;    // [batch * beams][max_pages]
  const int32_t *lengths = nullptr;  // [batch * beams]
  const int32_t *spare = nullptr;    // [batch * beams]
  int32_t *table_out = nullptr, *lengths_out = nullptr;
  uint8_t *copied = nullptr;
  int64_t batch = 0, beams = 0, max_pages = 0;
};
cudaError_t launch_kv_reorder(uint8_t *pool, int64_t layers, int64_t layer_bytes, const KvLayer &c,
                              const KvReorder &r, cudaStream_t stream);

// Attention over the cache (spt_attn.cu).
struct AttnArgs {
  KvLayer c;
  KvRows r;
  const void *q = nullptr;
  void *out = nullptr;
  int64_t q_stride = 0, out_stride = 0;
  const float *sinks = nullptr;  // [heads] or null
  float scale = 1.0f;
  int64_t window = 0;            // keys a row sees at most; 0: all
  int heads = 0, group = 0;
  int type = kKvF32;
  bool q_vec = false, out_vec = false;  // rows start on 16 bytes
  float *partial = nullptr;      // attn_workspace_bytes()
  int32_t *arrive = nullptr;     // attn_counter_bytes(): counters, zero between launches
  int32_t *gave_up = nullptr;    // the many-row kernel's, behind them: a word a CTA, set when one of its waits gives up
  int32_t *err = nullptr;        // set when a bounded wait gives up
  int wait_shift = 31;
  int fault_tile = -1;           // a test's: CTA 0 leaves out this tile's (its first warp's step's) copies
  int sm_count = 148;
};
cudaError_t launch_attention(const AttnArgs &a, cudaStream_t stream);
// The kernel for many rows of a key head (spt_attn_mma.cu), which launch_attention
// picks; cudaErrorNotSupported where it was built with other registers than it needs.
cudaError_t launch_attention_mma(const AttnArgs &a, cudaStream_t stream);
size_t attn_mma_workspace_bytes(int sm_count, int nb);
size_t attn_workspace_bytes(int sm_count, int nb);
size_t attn_counter_bytes(int sm_count);

// Beam selection (spt_beam.cu).
constexpr int kBeamMaxKeep = 64;
constexpr int kBeamMaxBeams = 64;
struct BeamArgs {
  const void *logits = nullptr;  // [batch * beams][row_stride] of `type`
  int64_t row_stride = 0;
  const float *scores = nullptr;
  const uint8_t *finished = nullptr;
  int type = kKvF32;
  int64_t batch = 0, beams = 0, vocab = 0;
  int keep = 0;
  int64_t end_token = 0;
  float *out_scores = nullptr;
  int32_t *out_parents = nullptr, *out_tokens = nullptr;
  void *work = nullptr;          // beam_workspace_bytes()
  int chunks = 1;                // beam_chunks()
};
int beam_chunks(int64_t rows, int64_t vocab, int sm_count);  // CTAs a row's logits are cut into
size_t beam_workspace_bytes(int64_t rows, int chunks, int keep);
cudaError_t launch_beam_select(const BeamArgs &a, cudaStream_t stream);

}  // namespace spt
