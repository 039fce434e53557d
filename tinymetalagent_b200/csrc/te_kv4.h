// The 4-bit KV cache: record layout and kernel parameters, shared by
// te_api_kv4.cpp and k_kv4.cu.  Not installed; not part of the ABI.
//
// A key or value row of one kv head is head_dim / 32 GGUF Q4_0 blocks: a
// binary16 scale d and 32 codes c, each standing for (c - 8) d.  The pool is
// [layers][pages][kv_heads][page_tokens / 16] tiles of 16 tokens, keys and
// values together, so that one tile is one contiguous copy:
//
//   K codes | V codes | K scales | V scales      8 * hd, 8 * hd, hd, hd bytes
//
// Inside a tile the codes lie as the warp-level m16n8k16 product wants them:
// lane 4g + t of a warp (g < 8, t < 4) owns 16-byte aligned words, and each
// 32-bit word w yields its four f16 pairs by one mask each (w & 0x000f000f,
// w & 0x00f000f0, and the same of w >> 8).
//   K word (j, lane, b): token 8j + g, dims 32b + 8t .. +7; dim 8t + 2p + e
//     of the block is nibble p + 4e (p < 4, e < 2).
//   V word (j, lane, b): tokens 8j + 2t + e, dims 32b + 4g + p; nibble p + 4e
//     (so a token owns 16-bit halves of its own: appending it writes no
//     byte of its neighbour).
//   scale (j, t, b, e): token 8j + 2t + e, block b (binary16).
// With NB = head_dim / 32 blocks, word (j, lane, b) is at byte
//   head_dim 128: j * 512 + lane * 16 + b * 4;  head_dim 64: lane * 16 + j * 8 + b * 4
// and scale (j, t, b, e) at the same formula with t for lane, + e * 2 (and 64
// for 512).
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace te {

constexpr int kKv4Tile = 16;        // tokens of a tile
// A decode copy, and what a warp attends at a time: 64 tokens, 9 KB at head_dim 128.  Fewer leave too little
// independent work beside each product (28 layers x 32768 tokens of 128: 139 us, 32 tokens 147, 16 tokens 171 or
// more; 24 layers x 8192 of 64: 14.2, 32 tokens 15.7).
constexpr int kKv4StageTiles = 4, kKv4StageTokens = kKv4StageTiles * kKv4Tile;
// Warps of a decode CTA, each with its own copies; two CTAs fit an SM.
__host__ __device__ constexpr int kv4_warps(int hd) { return hd == 128 ? 4 : 8; }
// What a group's queries and merge cost, in units: the stream split counts them before the group's own (a ragged
// batch of 64: 52.5 us with one, 52.0 with two, 53.7 with three; 28 layers x 6000 tokens 35.6, 34.4, 38.3; the
// geometric mean of 28 ragged batches 20.6 us with none, 20.5, 20.4, 20.6).
constexpr int kKv4GroupUnits = 2;
// Work unit of the decode split: one copy for each warp.
__host__ __device__ constexpr int kv4_unit(int hd) { return kKv4StageTokens * kv4_warps(hd); }
constexpr int kKv4Heads = 8;        // query heads of a work group (larger groups take several)
constexpr int kKv4MaxSeqs = 64;     // sequences per decode launch

__host__ __device__ constexpr int kv4_code_bytes(int hd) { return 8 * hd; }   // one side's codes of a tile
__host__ __device__ constexpr int kv4_scale_bytes(int hd) { return hd; }      // one side's scales of a tile
__host__ __device__ constexpr int kv4_tile_bytes(int hd) { return 18 * hd; }
// Byte of word (j, lane, b) in a side's codes, and of scale (j, t, b, e) in its scales.
__host__ __device__ constexpr int kv4_word_at(int hd, int j, int lane, int b) {
  return hd == 128 ? j * 512 + lane * 16 + b * 4 : lane * 16 + j * 8 + b * 4;
}
__host__ __device__ constexpr int kv4_scale_at(int hd, int j, int t, int b, int e) {
  return (hd == 128 ? j * 64 + t * 16 + b * 4 : t * 16 + j * 8 + b * 4) + e * 2;
}

// Where a cache's tiles are.
struct Kv4Pool {
  unsigned char* base;
  int32_t num_pages;        // pages per layer
  int32_t kv_heads;
  int32_t tiles_per_page;
  uint32_t tpp_magic;       // ceil(2^32 / tiles_per_page)
  int32_t stages_per_page;  // decode copies of a page
  int32_t step_pages, step_in;  // kv4_warps stages on: whole pages, and stages past them
  int32_t page_tokens;
};

struct Kv4Seq {
  int32_t slot;        // row of the page table
  int32_t len;         // tokens cached before the call
  int32_t q_pos;       // RoPE position of the query
  int32_t new_pos;     // RoPE position of the appended token
  int32_t unit_begin;  // first work unit of this sequence within a (layer, kv head, head block)
  int32_t part_begin;  // aligned split: its first part within a (layer, kv head, head block)
  int32_t page_base;   // >= 0: the sequence's pages are page_base, page_base + 1, ...; -1: read the table
};
__host__ __device__ inline int kv4_units(int len, int hd) { return len > 0 ? (len + kv4_unit(hd) - 1) / kv4_unit(hd) : 1; }

struct Kv4DecodeParams {
  Kv4Pool pool;
  const int32_t* page_table;  // [max_seqs][max_pages_per_seq]
  const void* q;              // [n_layers][n_seqs][heads][hd], fp32 or f16
  const void* k_new;          // [n_layers][n_seqs][kv_heads][hd] or null
  const void* v_new;
  float* out;                 // [..][heads][hd], or partial records [..][heads][hd + 2]
  float* partials;            // records of split groups: [grid][2][kv4_record_floats]
  uint32_t* counters;         // one per group, zero between launches
  const float* rope_cos;      // [max_position][hd / 2]
  const float* rope_sin;
  const float* q_bias;        // null, or [cache layers][heads * hd]
  const float* k_bias;        // null, or [cache layers][kv_heads * hd]
  const float* v_bias;
  int* error;
  long long total_units;
  int32_t n_seqs, seq_total, seq_base;
  int32_t layer_begin, n_layers;
  int32_t group;              // query heads per kv head
  int32_t head_blocks;        // work groups per kv head: ceil(group / 8)
  int32_t block_heads;        // query heads of a work group: ceil(group / head_blocks)
  int32_t block_units;        // work units of one (layer, kv head, head block)
  int32_t block_parts;        // aligned split: CTAs of one (layer, kv head, head block); 0: stream split
  int32_t grid;
  int32_t max_pages_per_seq;
  int32_t rope, input_f16, partial_out;
  float scale_log2;           // log2(e) / sqrt(hd)
  Kv4Seq seqs[kKv4MaxSeqs];
};
static_assert(sizeof(Kv4DecodeParams) <= 4096, "decode parameters exceed the kernel parameter space");

// Record of a part of a split group: 8 heads' accumulators, m and l.
constexpr int kv4_record_floats(int hd) { return kKv4Heads * hd + 2 * kKv4Heads; }
// Plans the split of p's work over `slots` resident CTAs (fills the sequences' units and parts, block_units,
// block_parts, total_units, grid).
void plan_kv4_decode(Kv4DecodeParams& p, int head_dim, long long slots);
int kv4_decode_ctas_per_sm(int head_dim);
cudaError_t launch_kv4_decode(const Kv4DecodeParams& p, int head_dim, cudaStream_t s);

struct Kv4RowsParams {
  Kv4Pool pool;
  const int32_t* page_row;  // page table row of the sequence
  const void* k;            // append: [n_layers][n_tokens] rows of kv_heads * hd values, token_stride apart
  const void* v;
  void* k_rows;             // append: the rows as stored, or null; read: the rows (contiguous)
  void* v_rows;
  const float* rope_cos;
  const float* rope_sin;
  const float* k_bias;
  const float* v_bias;
  long long token_stride;   // append: values from one token's row to the next in k and v
  int32_t n_layers, layer_begin;
  int32_t first, n_tokens;  // local token range
  int32_t first_pos;        // RoPE position of the first token (append)
  int32_t rope;
  int32_t input_f16;        // append: k and v are binary16
  int32_t rows_f16;         // k_rows and v_rows are binary16
};
// Warps of an append or read call; the kernels index them in 32 bits.
inline long long kv4_row_items(const Kv4RowsParams& p) {
  const long long tiles = (long long)(p.first + p.n_tokens - 1) / kKv4Tile - p.first / kKv4Tile + 1;
  return tiles * p.pool.kv_heads * p.n_layers;
}
cudaError_t launch_kv4_append(const Kv4RowsParams& p, int head_dim, cudaStream_t s);
cudaError_t launch_kv4_read(const Kv4RowsParams& p, int head_dim, cudaStream_t s);
// Raw GGUF Q4_0 blocks [n_layers][n_tokens][kv_heads][hd / 32][18 bytes] into the pool (k, v) or out of it (k_rows, v_rows).
cudaError_t launch_kv4_raw(const Kv4RowsParams& p, int head_dim, bool to_pool, cudaStream_t s);

}  // namespace te
