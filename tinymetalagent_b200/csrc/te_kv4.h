// The 4-bit KV cache: record layout and kernel parameters, shared by
// te_api_kv4.cpp and k_kv4.cu.  Not installed; not part of the ABI.
//
// A key or value row of one kv head is NB = head_dim / 32 GGUF Q4_0 blocks: a
// binary16 scale d and 32 codes c, each standing for (c - 8) d.  The pool is
// [layers][pages][kv_heads][page_tokens / 64] units of 64 tokens, keys and
// values together, so that one unit is one contiguous copy of 72 hd bytes:
//
//   K codes | V codes | K scales | V scales      32 hd, 32 hd, 4 hd, 4 hd
//
// The codes lie as the tensor core's A operands want them, one row per thread
// and 8 codes a word; a word w holds code 2p + e (p < 4, e < 2) in nibble
// p + 4e, so that its four f16 pairs come from one mask each (w & 0x000f000f,
// w & 0x00f000f0, and the same of w >> 8).
//   K: a row is a token.  Word (r, b, t): token r, dims 32b + 8t .. + 7, at
//     byte (64b + r) 16 + 4t.
//   V: a row is a dim (V^T).  Word (d, y): dim d, tokens 8y .. + 7, at byte
//     ((y / 4) hd + d) 16 + 4 (y % 4).
//   scale (r, b): token r, block b, at byte 2 (r NB + b).
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace te {

constexpr int kKv4Unit = 64;        // tokens of a unit
constexpr int kKv4Stage = 128;      // tokens of a step of the decode kernel: the M of its matrix products
constexpr int kKv4Heads = 8;        // query heads of a work group (larger groups take several)
constexpr int kKv4MaxSeqs = 64;     // sequences per decode launch

__host__ __device__ constexpr int kv4_unit_bytes(int hd) { return 72 * hd; }
__host__ __device__ constexpr int kv4_v_off(int hd) { return 32 * hd; }
__host__ __device__ constexpr int kv4_ks_off(int hd) { return 64 * hd; }
__host__ __device__ constexpr int kv4_vs_off(int hd) { return 68 * hd; }
// Byte of K word (r, b, t), of V word (d, y) and of scale (r, b) in their parts.
__host__ __device__ constexpr int kv4_k_word(int r, int b, int t) { return (64 * b + r) * 16 + 4 * t; }
__host__ __device__ constexpr int kv4_v_word(int hd, int d, int y) { return ((y >> 2) * hd + d) * 16 + 4 * (y & 3); }
__host__ __device__ constexpr int kv4_scale(int hd, int r, int b) { return 2 * (r * (hd / 32) + b); }
// Nibble of code i (0..7) in its word.
__host__ __device__ constexpr int kv4_nibble(int i) { return (i >> 1) + 4 * (i & 1); }

// Where a cache's units are.
struct Kv4Pool {
  unsigned char* base;
  int32_t num_pages;        // pages per layer
  int32_t kv_heads;
  int32_t units_per_page;
  uint32_t upp_magic;       // ceil(2^32 / units_per_page), or 0 for one unit per page
};

struct Kv4Seq {
  int32_t slot;        // row of the page table
  int32_t len;         // tokens cached before the call
  int32_t q_pos;       // RoPE position of the query
  int32_t new_pos;     // RoPE position of the appended token
  int32_t stage_begin; // first stage of this sequence within a (layer, kv head, head block)
  int32_t part_begin;  // aligned split: its first part within a (layer, kv head, head block)
  int32_t page_base;   // >= 0: the sequence's pages are page_base, page_base + 1, ...; -1: read the table
};
// Stages of a sequence that attends n tokens (one at least: an empty sequence writes zeros).
__host__ __device__ inline int kv4_stages(int n) { return n > 0 ? (n + kKv4Stage - 1) / kKv4Stage : 1; }

struct Kv4DecodeParams {
  Kv4Pool pool;
  const int32_t* page_table;  // [max_seqs][max_pages_per_seq]
  const void* q;              // [n_layers][n_seqs][heads][hd], fp32 or f16
  const void* k_new;          // [n_layers][n_seqs][kv_heads][hd] or null
  const void* v_new;
  float* out;                 // [..][heads][hd], or partial records [..][heads][hd + 2]
  float* partials;            // records of split groups: [grid][2][kv4_record_floats] (aligned split: [grid])
  uint32_t* counters;         // one per group, zero between launches
  const float* rope_cos;      // [max_position][hd / 2]
  const float* rope_sin;
  const float* q_bias;        // null, or [cache layers][heads * hd]
  const float* k_bias;        // null, or [cache layers][kv_heads * hd]
  const float* v_bias;
  int* error;
  long long total_stages;
  int32_t n_seqs, seq_total, seq_base;
  int32_t layer_begin, n_layers;
  int32_t group;              // query heads per kv head
  int32_t head_blocks;        // work groups per kv head: ceil(group / 8)
  int32_t block_heads;        // query heads of a work group: ceil(group / head_blocks)
  int32_t block_stages;       // stages of one (layer, kv head, head block)
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
// Plans the split of p's work over `slots` resident CTAs (fills the sequences' stages and parts, block_stages,
// block_parts, total_stages, grid).
void plan_kv4_decode(Kv4DecodeParams& p, long long slots);
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
cudaError_t launch_kv4_append(const Kv4RowsParams& p, int head_dim, cudaStream_t s);
cudaError_t launch_kv4_read(const Kv4RowsParams& p, int head_dim, cudaStream_t s);
// Raw GGUF Q4_0 blocks [n_layers][n_tokens][kv_heads][hd / 32][18 bytes] into the pool (k, v) or out of it (k_rows, v_rows).
cudaError_t launch_kv4_raw(const Kv4RowsParams& p, int head_dim, bool to_pool, cudaStream_t s);

}  // namespace te
