// Attention of drafted tokens over a paged cache (pa_tree; its contract is in llm_decoder.h).
//
// A workgroup of 4 waves (or 8: tree_plan) takes rows (tokens x heads of the group) of one key/value head and one
// split of its keys, in tiles of 16 rows and blocks of 32 keys.  One tile: the waves take its blocks
// in turn, from memory straight into registers one block ahead.  Up to 4 tiles: two waves of two
// tiles each take one block, two the next; up to 8: four waves, two tiles each, take the same
// block.  Keys that waves share go into LDS once, stages ahead (16 heads x 63 rows of 32768 e4m3
// tokens: each wave loading them for itself 94 us, L1 gave no more than L2).  Two tiles a wave share
// the conversions and exchanges of the keys.  Waves with the same rows are merged through LDS.
//   S^T[32 keys][16 rows] = K . Q^T       v_mfma_f32_16x16x32, two tiles of 16 keys
//   O^T[D][16 rows]      += V^T . P^T
// A lane (g = lane / 16, c = lane % 16) holds the scores of 8 keys (16 u + 4 g + r; u < 2,
// r < 4) of row c, which are the B operand of the second product once its k slots are taken in
// that order.  The A operand wants, in lane c, 8 keys of one dim: a lane loads the dims
// c D/16 .. of its 8 keys, 2 to 32 bytes a key and whole rows together, and exchanges
// bytes among its own registers (v_perm), so V^T needs no LDS.  Tile dd of O^T then has rows
// m = c for the dims c D/16 + dd: lane (g, c) ends with dims 4 g D/16 .. (4 g + 4) D/16 of row c.
//
// 8-bit codes become 16 bits on the way into the products, exactly: keys' fp16 (int8: 0x6400 | code ^ 0x80 is
// the fp16 number 1152 + code; e4m3: one conversion for two), values' bf16.  A key's scale multiplies its
// scores, a value's scale its probabilities.
//
// Precision: queries enter as parts of 16 bits (fp32 ones as two of fp16, three of bf16: 22 and
// 24 bits; others exactly), probabilities as two or three (launch_tree_parts), the rest is fp32.  The products
// keep subnormal numbers.  fp16 ones are kept away from its ends: a row of queries is scaled to 2^14 by a power of
// two, probabilities by 2^11 (they may grow to 2^15).  Quantised values' weights, probabilities times scales,
// are bf16, which has fp32's range.
//
// What bounds it: one tile, the memory (64 x 16 heads of 128 over up to 8192 int8 tokens, pages of 2 KB and
// their scales in any order: 241 us, 5.1 TB/s, vector instructions 43 % of it).  More tiles, the chain of one
// block (loads, scores, exponentials, products), which too few waves hide: 16 heads x 63 rows over 32768 e4m3 tokens
// 57 us, 2.4 TB/s and 300 TFLOP/s, with 1.3 waves a SIMD whose vector instructions take 42 % of the time and
// its products 17 %; 16 x 2 x 168 rows over up to 4096 bf16 33 us, where 278 of 704 workgroups have keys:
// 0.7 waves a SIMD, 16 % and 7 %.  Tiles of sums, queries and a block fill the registers of two waves a
// SIMD.  Short rows, a launch and its code (8 rows of 12 heads over 113 tokens: 5.6 us).
//
// Keys that a row does not see get the score -infinity.  Their V still meets a probability of 0
// in the product, and 0 times NaN is NaN: rows of V that nobody sees (behind the row's end, in
// missing pages) are zeroed, and what is not a number in a drafted token's V or its scale is
// taken as 0; if there was any, the rows that see it get their infinities and NaNs in a pass behind the
// others, from products of ones.
#pragma once

#include "common.hpp"
#include "paged_rows.hpp"

namespace llm {

struct TreeArgs {
  const void* q;
  void* out;
  int dtype;
  long long q_stride, out_stride;  // elements from token to token
  const uint8_t *k_pool, *v_pool;
  const float *k_scale, *v_scale;  // NULL: 1
  size_t page_stride, scale_stride;
  const int32_t* table;
  int num_pages, num_beams, kv_heads, max_tiles, page_size;
  const int32_t *beam_ids, *context_lens, *tree_lens;
  const uint32_t* mask;
  int mask_words;
  int B, N, H, G, T;  // G = H / kv_heads
  float scale2;       // sm_scale log2(e)
  int nsplit, split_keys, waves;
  float *acc, *ml;  // [row][split][D], [row][split][2], row = (b N + token) H + head
};

constexpr int kTreeKeys = 32;
constexpr int kTreeStep = 128;  // splits begin at multiples of it

// Committed and all tokens of row b, its drafts, and the keys of one of its splits: nsplit of
// them hold the row however long it is.
struct TreeRow {
  int n, C, L, split_len;
};
__device__ __forceinline__ TreeRow tree_row(const TreeArgs& a, int b) {
  TreeRow r;
  const int room = a.max_tiles * a.page_size;
  r.n = a.tree_lens ? clamp_int(a.tree_lens[b], 0, a.N) : a.N;
  r.C = clamp_int(a.context_lens ? a.context_lens[b] : a.T, 0, room);
  r.L = min(r.C + r.n, room);
  const int even = ((r.L + a.nsplit - 1) / a.nsplit + kTreeStep - 1) / kTreeStep * kTreeStep;
  r.split_len = max(a.split_keys, even);
  return r;
}

// Parts of a query: the products' type is bf16 over bf16 pools, else fp16.
constexpr int tree_parts(int kvt, int dtype) {
  return kvt == LLM_BF16 ? (dtype == LLM_F32 ? 3 : dtype == LLM_F16 ? 2 : 1) : dtype == LLM_F32 ? 2 : 1;
}
// Row tiles of a wave where a workgroup's keys come through LDS: queries and sums of two fit the
// registers of two waves a SIMD up to 128 dims of query parts.  And of a workgroup for `rows` rows.
constexpr int tree_wave_tiles(int D, int parts) { return D * parts <= 128 ? 2 : 1; }
inline int tree_tiles(int D, int parts, int rows) {
  return rows <= 16 ? 1 : rows <= 64 ? 4 : 4 * tree_wave_tiles(D, parts);
}

// Most waves of a workgroup of one row tile (heads of 256 leave a SIMD registers for one).
constexpr int tree_most_waves(int D) { return D == 256 ? 4 : 8; }

// pa_tree_*.hip
hipError_t launch_tree_f16(const TreeArgs& a, int D, int tiles, dim3 grid, hipStream_t st);
hipError_t launch_tree_bf16(const TreeArgs& a, int D, int tiles, dim3 grid, hipStream_t st);
hipError_t launch_tree_i8(const TreeArgs& a, int D, int tiles, dim3 grid, hipStream_t st);
hipError_t launch_tree_e4m3(const TreeArgs& a, int D, int tiles, dim3 grid, hipStream_t st);

}  // namespace llm
