// C-ABI layer of the 4-bit KV cache (te_kv4_*): argument validation, pages and
// lengths (a te_kv_cache's bookkeeping without its pools), work decomposition.
#include <cuda_runtime.h>

#include <cmath>
#include <cstring>
#include <new>

#include "../../include/tinyengine_attn.h"
#include "te_engine.h"
#include "te_internal.h"
#include "te_kv4.h"

using namespace te;

struct te_kv4_cache {
  te_kv_cache b;  // pages, lengths, RoPE table, biases; its pools stay null
  unsigned char* pool = nullptr;
  std::vector<uint32_t> seen;  // per sequence: the last decode call that named it
  uint32_t call = 0;
};

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool bad_layers(const te_kv4_cache* c, size_t begin, size_t n) {
  return n == 0 || n > c->b.d.layers || begin > c->b.d.layers - n;
}

Kv4Pool pool_of(const te_kv4_cache* c) {
  Kv4Pool p{};
  p.base = c->pool;
  p.num_pages = (int32_t)c->b.d.total_pages;
  p.kv_heads = (int32_t)c->b.d.kv_heads;
  p.page_tokens = (int32_t)c->b.d.page_tokens;
  p.tiles_per_page = (int32_t)(c->b.d.page_tokens / kKv4Tile);
  p.tpp_magic = (uint32_t)(((1ull << 32) + (uint64_t)p.tiles_per_page - 1) / (uint64_t)p.tiles_per_page);
  p.stages_per_page = p.tiles_per_page / kKv4StageTiles;
  p.step_pages = kv4_warps((int)c->b.d.head_dim) / p.stages_per_page;
  p.step_in = kv4_warps((int)c->b.d.head_dim) % p.stages_per_page;
  return p;
}

// Token rows of one sequence: the parameters shared by the append, read and raw kernels.
Kv4RowsParams rows_params(const te_kv4_cache* c, size_t layer_begin, size_t n_layers, size_t seq, size_t first,
                          size_t n_tokens) {
  Kv4RowsParams p{};
  p.pool = pool_of(c);
  p.page_row = c->b.d_page_table + seq * c->b.pages_per_seq;
  p.n_layers = (int32_t)n_layers;
  p.layer_begin = (int32_t)layer_begin;
  p.first = (int32_t)first;
  p.n_tokens = (int32_t)n_tokens;
  p.token_stride = (long long)c->b.d.kv_heads * c->b.d.head_dim;
  return p;
}

// Closes a launch: its profile event, its error, the launch count.
te_status queue(te_attn_engine* e, cudaError_t err, int prof, const char* what) {
  prof_end(e, prof);
  if (err != cudaSuccess) return cuda_fail(e, err, what);
  e->launches++;
  return TE_STATUS_OK;
}

}  // namespace

extern "C" {

TE_API te_status te_kv4_cache_create(te_attn_engine* e, const te_kv_cache_desc* desc, te_kv4_cache** out) {
  if (!e || !desc || !out) return TE_STATUS_INVALID_ARGUMENT;
  *out = nullptr;
  if (desc->abi_version != TE_ATTN_ABI_VERSION) return fail(e, TE_STATUS_UNSUPPORTED, "cache desc ABI version");
  te_kv_cache_desc d = *desc;
  if (d.page_tokens == 0) d.page_tokens = 128;
  if (d.layers == 0 || d.max_seqs == 0 || d.max_tokens_per_seq == 0 || d.kv_heads == 0 || !(d.rope_theta > 0.0f) ||
      d.page_tokens % kStageTokens != 0) {
    return fail(e, TE_STATUS_INVALID_ARGUMENT, "invalid cache description");
  }
  if (d.head_dim != 64 && d.head_dim != 128) return fail(e, TE_STATUS_UNSUPPORTED, "head_dim must be 64 or 128");
  // token and page indices are 32-bit on the device, byte offsets 64-bit
  if (d.max_tokens_per_seq > (1u << 30) || d.page_tokens > (1u << 30)) {
    return fail(e, TE_STATUS_UNSUPPORTED, "more than 2^30 tokens per sequence");
  }
  const uint32_t pps = (d.max_tokens_per_seq + d.page_tokens - 1) / d.page_tokens;
  const uint64_t pages = d.total_pages ? d.total_pages : (uint64_t)d.max_seqs * pps;
  if (pages > (uint64_t)INT32_MAX || (uint64_t)d.layers * d.kv_heads > (uint64_t)INT32_MAX / 64) {
    return fail(e, TE_STATUS_UNSUPPORTED, "too many pages or heads");
  }
  d.total_pages = (uint32_t)pages;
  if (d.max_position == 0) d.max_position = d.max_tokens_per_seq;
  if (d.max_position > (uint32_t)INT32_MAX) return fail(e, TE_STATUS_UNSUPPORTED, "RoPE table too long");
  DeviceGuard dg(e->device);
  te_kv4_cache* c = nullptr;
  const size_t half = d.head_dim / 2;
  const size_t tab_floats = 2 * (size_t)d.max_position * half;
  const double pool_bytes = (double)d.layers * (double)pages * d.kv_heads * (d.page_tokens / kKv4Tile) *
                            kv4_tile_bytes((int)d.head_dim);
  if (pool_bytes > 1e13) return fail(e, TE_STATUS_OUT_OF_MEMORY, "4-bit KV pool too large");
  const size_t bytes = (size_t)d.layers * pages * d.kv_heads * (d.page_tokens / kKv4Tile) *
                       (size_t)kv4_tile_bytes((int)d.head_dim);
  try {
    c = new te_kv4_cache();
    te_kv_cache& b = c->b;
    b.eng = e;
    b.d = d;
    b.pages_per_seq = pps;
    b.h_page_table.assign((size_t)d.max_seqs * pps, -1);
    b.contig.assign(d.max_seqs, 0);
    b.len.assign(d.max_seqs, 0);
    b.offset.assign(d.max_seqs, 0);
    b.free_pages.resize(d.total_pages);
    for (uint32_t i = 0; i < d.total_pages; ++i) b.free_pages[i] = (int32_t)(d.total_pages - 1 - i);
    c->seen.assign(d.max_seqs, 0);
    cudaError_t err = cudaMalloc(reinterpret_cast<void**>(&c->pool), bytes);
    // zeros: a scale of 0 everywhere, until written
    if (err == cudaSuccess) err = cudaMemsetAsync(c->pool, 0, bytes, e->stream);
    if (err == cudaSuccess) {
      err = cudaMalloc(reinterpret_cast<void**>(&b.d_page_table), b.h_page_table.size() * sizeof(int32_t));
    }
    if (err == cudaSuccess) err = cudaMalloc(reinterpret_cast<void**>(&b.d_cos), tab_floats * sizeof(float));
    if (err != cudaSuccess) {
      te_kv4_cache_free(c);
      return cuda_fail(e, err, "4-bit KV cache allocation");
    }
    b.d_sin = b.d_cos + tab_floats / 2;
    std::vector<float> tab(tab_floats);
    te_host_rope_table(tab.data(), tab.data() + tab_floats / 2, 0, d.max_position, d.head_dim, d.rope_theta);
    err = cudaMemcpy(b.d_cos, tab.data(), tab_floats * sizeof(float), cudaMemcpyHostToDevice);
    if (err == cudaSuccess) {
      err = cudaMemcpy(b.d_page_table, b.h_page_table.data(), b.h_page_table.size() * sizeof(int32_t),
                       cudaMemcpyHostToDevice);
    }
    if (err == cudaSuccess) err = cudaStreamSynchronize(e->stream);
    if (err != cudaSuccess) {
      te_kv4_cache_free(c);
      return cuda_fail(e, err, "4-bit KV cache initialisation");
    }
  } catch (const std::bad_alloc&) {
    te_kv4_cache_free(c);
    return fail(e, TE_STATUS_OUT_OF_MEMORY, "4-bit KV cache bookkeeping");
  }
  *out = c;
  return TE_STATUS_OK;
}

TE_API void te_kv4_cache_free(te_kv4_cache* c) {
  if (!c) return;
  if (c->b.eng) {
    DeviceGuard dg(c->b.eng->device);
    cudaStreamSynchronize(c->b.eng->stream);
    cudaFree(c->pool);
    cudaFree(c->b.d_page_table);
    cudaFree(c->b.d_cos);
    cudaFree(c->b.d_kb);
  }
  delete c;
}

TE_API te_status te_kv4_cache_seq_reset(te_kv4_cache* c, size_t seq, size_t position_offset) {
  if (!c || position_offset > (size_t)INT32_MAX) return TE_STATUS_INVALID_ARGUMENT;
  return te_kv_cache_seq_reset(&c->b, seq, position_offset);
}
TE_API te_status te_kv4_cache_seq_truncate(te_kv4_cache* c, size_t seq, size_t length) {
  return te_kv_cache_seq_truncate(c ? &c->b : nullptr, seq, length);
}
TE_API te_status te_kv4_cache_seq_length(const te_kv4_cache* c, size_t seq, size_t* out_length) {
  return te_kv_cache_seq_length(c ? &c->b : nullptr, seq, out_length);
}
TE_API te_status te_kv4_cache_reserve(te_kv4_cache* c, size_t seq, size_t tokens) {
  return te_kv_cache_reserve(c ? &c->b : nullptr, seq, tokens);
}
TE_API te_status te_kv4_cache_set_qkv_bias(te_kv4_cache* c, size_t layer_begin, size_t n_layers, size_t heads,
                                           const float* q_bias, const float* k_bias, const float* v_bias) {
  if (!c || bad_layers(c, layer_begin, n_layers)) return TE_STATUS_INVALID_ARGUMENT;
  return te_kv_cache_set_qkv_bias(&c->b, layer_begin, n_layers, heads, q_bias, k_bias, v_bias);
}

TE_API te_status te_kv4_append(te_kv4_cache* c, size_t layer_begin, size_t n_layers, size_t seq, const void* k,
                               const void* v, size_t n_tokens, size_t token_stride, void* k_stored, void* v_stored,
                               uint32_t flags) {
  if (!c || !k || !v || n_tokens == 0 || seq >= c->b.d.max_seqs || bad_layers(c, layer_begin, n_layers) ||
      (k_stored == NULL) != (v_stored == NULL)) {
    return TE_STATUS_INVALID_ARGUMENT;
  }
  te_attn_engine* e = c->b.eng;
  if (flags & ~(TE_ATTN_ADVANCE | TE_ATTN_INPUT_F16 | TE_ATTN_OUTPUT_F16 | TE_ATTN_NO_ROPE | TE_ATTN_QKV_BIAS)) {
    return fail(e, TE_STATUS_INVALID_ARGUMENT, "unsupported flags for te_kv4_append");
  }
  if ((flags & TE_ATTN_QKV_BIAS) && !c->b.d_kb) {
    return fail(e, TE_STATUS_INVALID_ARGUMENT, "TE_ATTN_QKV_BIAS before te_kv4_cache_set_qkv_bias");
  }
  const size_t row = (size_t)c->b.d.kv_heads * c->b.d.head_dim;
  const size_t el = (flags & TE_ATTN_INPUT_F16) ? 2 : 4;
  if (token_stride == 0) token_stride = row;
  if (token_stride < row || (token_stride * el) % 16 != 0 || token_stride > ((size_t)1 << 40)) {
    return fail(e, TE_STATUS_INVALID_ARGUMENT, "token_stride must hold a row and be a multiple of 16 bytes");
  }
  if (!aligned16(k) || !aligned16(v) || !aligned16(k_stored) || !aligned16(v_stored)) {
    return fail(e, TE_STATUS_INVALID_ARGUMENT, "k, v, k_stored and v_stored must be 16-byte aligned");
  }
  const size_t first = (size_t)c->b.len[seq];
  if (n_tokens > c->b.d.max_tokens_per_seq - first) {
    return fail(e, TE_STATUS_INVALID_ARGUMENT, "sequence would exceed max_tokens_per_seq");
  }
  if ((uint64_t)c->b.offset[seq] + first + n_tokens > c->b.d.max_position) {
    return fail(e, TE_STATUS_INVALID_ARGUMENT, "RoPE position beyond max_position");
  }
  DeviceGuard dg(e->device);
  te_status st = ensure_pages(&c->b, seq, first + n_tokens);
  if (st != TE_STATUS_OK) return st;
  Kv4RowsParams p = rows_params(c, layer_begin, n_layers, seq, first, n_tokens);
  p.k = k;
  p.v = v;
  p.k_rows = k_stored;
  p.v_rows = v_stored;
  p.token_stride = (long long)token_stride;
  p.rope_cos = c->b.d_cos;
  p.rope_sin = c->b.d_sin;
  if (flags & TE_ATTN_QKV_BIAS) {
    p.k_bias = c->b.d_kb;
    p.v_bias = c->b.d_vb;
  }
  p.first_pos = (int32_t)(c->b.offset[seq] + (int64_t)first);
  p.rope = (flags & TE_ATTN_NO_ROPE) ? 0 : 1;
  p.input_f16 = (flags & TE_ATTN_INPUT_F16) ? 1 : 0;
  p.rows_f16 = (flags & TE_ATTN_OUTPUT_F16) ? 1 : 0;
  if (kv4_row_items(p) > (long long)INT32_MAX) return fail(e, TE_STATUS_UNSUPPORTED, "too many rows for one call");
  const int prof = prof_begin(e, PK_KV4_APPEND);
  st = queue(e, launch_kv4_append(p, (int)c->b.d.head_dim, e->stream), prof, "4-bit append launch");
  if (st == TE_STATUS_OK && (flags & TE_ATTN_ADVANCE)) c->b.len[seq] = (int64_t)(first + n_tokens);
  return st;
}

// The checks shared by the two reads: a non-empty range of cached tokens.
static te_status check_range(te_kv4_cache* c, size_t layer_begin, size_t n_layers, size_t seq, size_t token_begin,
                             size_t n_tokens, const void* k, const void* v) {
  if (!c || !k || !v || n_tokens == 0 || seq >= c->b.d.max_seqs || bad_layers(c, layer_begin, n_layers)) {
    return TE_STATUS_INVALID_ARGUMENT;
  }
  const size_t len = (size_t)c->b.len[seq];
  if (token_begin > len || n_tokens > len - token_begin) {
    return fail(c->b.eng, TE_STATUS_INVALID_ARGUMENT, "read past length");
  }
  return TE_STATUS_OK;
}

TE_API te_status te_kv4_cache_read(te_kv4_cache* c, size_t layer_begin, size_t n_layers, size_t seq,
                                   size_t token_begin, size_t n_tokens, void* k, void* v, uint32_t flags) {
  te_status st = check_range(c, layer_begin, n_layers, seq, token_begin, n_tokens, k, v);
  if (st != TE_STATUS_OK) return st;
  te_attn_engine* e = c->b.eng;
  if (flags & ~TE_ATTN_OUTPUT_F16) return fail(e, TE_STATUS_INVALID_ARGUMENT, "unsupported flags for te_kv4_cache_read");
  if (!aligned16(k) || !aligned16(v)) return fail(e, TE_STATUS_INVALID_ARGUMENT, "k and v must be 16-byte aligned");
  DeviceGuard dg(e->device);
  Kv4RowsParams p = rows_params(c, layer_begin, n_layers, seq, token_begin, n_tokens);
  p.k_rows = k;
  p.v_rows = v;
  p.rows_f16 = (flags & TE_ATTN_OUTPUT_F16) ? 1 : 0;
  if (kv4_row_items(p) > (long long)INT32_MAX) return fail(e, TE_STATUS_UNSUPPORTED, "too many rows for one call");
  const int prof = prof_begin(e, PK_KV4_READ);
  return queue(e, launch_kv4_read(p, (int)c->b.d.head_dim, e->stream), prof, "4-bit read launch");
}

TE_API te_status te_kv4_cache_read_q4_0(te_kv4_cache* c, size_t layer_begin, size_t n_layers, size_t seq,
                                        size_t token_begin, size_t n_tokens, void* k, void* v) {
  te_status st = check_range(c, layer_begin, n_layers, seq, token_begin, n_tokens, k, v);
  if (st != TE_STATUS_OK) return st;
  te_attn_engine* e = c->b.eng;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 1u) {
    return fail(e, TE_STATUS_INVALID_ARGUMENT, "blocks must be 2-byte aligned");
  }
  DeviceGuard dg(e->device);
  Kv4RowsParams p = rows_params(c, layer_begin, n_layers, seq, token_begin, n_tokens);
  p.k_rows = k;
  p.v_rows = v;
  const int prof = prof_begin(e, PK_KV4_READ);
  return queue(e, launch_kv4_raw(p, (int)c->b.d.head_dim, false, e->stream), prof, "4-bit block read launch");
}

TE_API te_status te_kv4_cache_write_q4_0(te_kv4_cache* c, size_t layer_begin, size_t n_layers, size_t seq,
                                         size_t token_begin, size_t n_tokens, const void* k, const void* v) {
  if (!c || !k || !v || n_tokens == 0 || seq >= c->b.d.max_seqs || bad_layers(c, layer_begin, n_layers)) {
    return TE_STATUS_INVALID_ARGUMENT;
  }
  te_attn_engine* e = c->b.eng;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 1u) {
    return fail(e, TE_STATUS_INVALID_ARGUMENT, "blocks must be 2-byte aligned");
  }
  if (token_begin > (size_t)c->b.len[seq]) {
    return fail(e, TE_STATUS_INVALID_ARGUMENT, "token_begin past the sequence's length");
  }
  if (n_tokens > c->b.d.max_tokens_per_seq - token_begin) {
    return fail(e, TE_STATUS_INVALID_ARGUMENT, "sequence would exceed max_tokens_per_seq");
  }
  DeviceGuard dg(e->device);
  te_status st = ensure_pages(&c->b, seq, token_begin + n_tokens);
  if (st != TE_STATUS_OK) return st;
  Kv4RowsParams p = rows_params(c, layer_begin, n_layers, seq, token_begin, n_tokens);
  p.k = k;
  p.v = v;
  const int prof = prof_begin(e, PK_KV4_APPEND);
  st = queue(e, launch_kv4_raw(p, (int)c->b.d.head_dim, true, e->stream), prof, "4-bit block write launch");
  if (st == TE_STATUS_OK) c->b.len[seq] = std::max<int64_t>(c->b.len[seq], (int64_t)(token_begin + n_tokens));
  return st;
}

TE_API te_status te_kv4_attention_decode(te_kv4_cache* c, size_t layer_begin, size_t n_layers,
                                         const uint32_t* seq_ids, size_t n_seqs, const int64_t* q_positions,
                                         const void* q, const void* k_new, const void* v_new, size_t heads, float* out,
                                         uint32_t flags) {
  if (!c || !seq_ids || !q || !out || n_seqs == 0 || heads == 0 || bad_layers(c, layer_begin, n_layers) ||
      (k_new == NULL) != (v_new == NULL)) {
    return TE_STATUS_INVALID_ARGUMENT;
  }
  te_kv_cache& b = c->b;
  te_attn_engine* e = b.eng;
  if (flags & ~(TE_ATTN_ADVANCE | TE_ATTN_PARTIAL | TE_ATTN_NO_ROPE | TE_ATTN_QKV_BIAS | TE_ATTN_INPUT_F16)) {
    return fail(e, TE_STATUS_INVALID_ARGUMENT, "unsupported flags for te_kv4_attention_decode");
  }
  const size_t hkv = b.d.kv_heads, hd = b.d.head_dim;
  if (heads % hkv != 0) return fail(e, TE_STATUS_INVALID_ARGUMENT, "heads must be a multiple of kv_heads");
  if (heads > (1u << 20)) return fail(e, TE_STATUS_UNSUPPORTED, "more than 2^20 query heads");
  if ((flags & TE_ATTN_QKV_BIAS) && (!b.d_qb || b.bias_heads != heads)) {
    return fail(e, TE_STATUS_INVALID_ARGUMENT, "TE_ATTN_QKV_BIAS needs te_kv4_cache_set_qkv_bias with these heads");
  }
  if (n_seqs > b.d.max_seqs) return TE_STATUS_INVALID_ARGUMENT;
  if (!aligned16(q) || !aligned16(k_new) || !aligned16(v_new) || !aligned16(out)) {
    return fail(e, TE_STATUS_INVALID_ARGUMENT, "q, k_new, v_new and out must be 16-byte aligned");
  }
  const bool append = k_new != NULL;

  // Every sequence is checked before anything is mapped or queued.
  const uint32_t call = ++c->call;
  if (call == 0) std::fill(c->seen.begin(), c->seen.end(), 0u), c->call = 1;
  for (size_t i = 0; i < n_seqs; ++i) {
    const uint32_t s = seq_ids[i];
    if (s >= b.d.max_seqs || c->seen[s] == c->call) {
      return fail(e, TE_STATUS_INVALID_ARGUMENT, "bad or repeated sequence id");
    }
    c->seen[s] = c->call;
    const int64_t len = b.len[s] + (append ? 1 : 0);
    if ((uint64_t)len > b.d.max_tokens_per_seq) return fail(e, TE_STATUS_INVALID_ARGUMENT, "sequence full");
    // an empty sequence that appends nothing has no position of its own
    const int64_t last = b.offset[s] + (len > 0 ? len - 1 : 0);
    const int64_t qpos = q_positions ? q_positions[i] : (len > 0 ? last : 0);
    if (qpos < 0 || (uint64_t)qpos >= b.d.max_position || (append && (uint64_t)last >= b.d.max_position)) {
      return fail(e, TE_STATUS_INVALID_ARGUMENT, "RoPE position beyond max_position");
    }
  }
  DeviceGuard dg(e->device);
  if (append) {
    // all of the step's pages or none: a refused step leaves the pool as it was
    size_t missing = 0;
    for (size_t i = 0; i < n_seqs; ++i) {
      const size_t s = seq_ids[i];
      missing += b.h_page_table[s * b.pages_per_seq + (size_t)b.len[s] / b.d.page_tokens] < 0 ? 1 : 0;
    }
    if (missing > b.free_pages.size()) return fail(e, TE_STATUS_OUT_OF_MEMORY, "KV page pool exhausted");
    for (size_t i = 0; i < n_seqs; ++i) {
      te_status st = ensure_pages(&b, seq_ids[i], (size_t)b.len[seq_ids[i]] + 1);
      if (st != TE_STATUS_OK) return st;
    }
  }

  Kv4DecodeParams p;
  std::memset(&p, 0, sizeof(p));
  p.pool = pool_of(c);
  p.page_table = b.d_page_table;
  p.q = q;
  p.k_new = k_new;
  p.v_new = v_new;
  p.out = out;
  p.rope_cos = b.d_cos;
  p.rope_sin = b.d_sin;
  if (flags & TE_ATTN_QKV_BIAS) {
    p.q_bias = b.d_qb;
    p.k_bias = b.d_kb;
    p.v_bias = b.d_vb;
  }
  p.error = e->d_error;
  p.seq_total = (int32_t)n_seqs;
  p.layer_begin = (int32_t)layer_begin;
  p.n_layers = (int32_t)n_layers;
  p.group = (int32_t)(heads / hkv);
  p.head_blocks = (p.group + kKv4Heads - 1) / kKv4Heads;
  p.block_heads = (p.group + p.head_blocks - 1) / p.head_blocks;
  p.max_pages_per_seq = (int32_t)b.pages_per_seq;
  p.rope = (flags & TE_ATTN_NO_ROPE) ? 0 : 1;
  p.input_f16 = (flags & TE_ATTN_INPUT_F16) ? 1 : 0;
  p.partial_out = (flags & TE_ATTN_PARTIAL) ? 1 : 0;
  p.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)hd));

  for (size_t base = 0; base < n_seqs; base += kKv4MaxSeqs) {
    const size_t nb = std::min<size_t>(kKv4MaxSeqs, n_seqs - base);
    for (size_t i = 0; i < nb; ++i) {
      const uint32_t s = seq_ids[base + i];
      Kv4Seq& w = p.seqs[i];
      const int64_t len = b.len[s] + (append ? 1 : 0);
      const int64_t last = b.offset[s] + (len > 0 ? len - 1 : 0);
      w.slot = (int32_t)s;
      w.len = (int32_t)b.len[s];
      w.q_pos = (int32_t)(q_positions ? q_positions[base + i] : (len > 0 ? last : 0));
      w.new_pos = append ? (int32_t)last : -1;
      w.page_base = contiguous_base(&b, s, (size_t)len);
    }
    p.n_seqs = (int32_t)nb;
    p.seq_base = (int32_t)base;
    plan_kv4_decode(p, (int)hd, (long long)e->sm_count * kv4_decode_ctas_per_sm((int)hd));
    const size_t groups = n_layers * hkv * (size_t)p.head_blocks * nb;
    if (p.total_units > (long long)INT32_MAX || groups > (size_t)INT32_MAX) {
      return fail(e, TE_STATUS_UNSUPPORTED, "decode call too large");
    }
    const size_t part_bytes = (size_t)p.grid * 2 * kv4_record_floats((int)hd) * sizeof(float);
    const cudaError_t err = grow_decode_scratch(e, part_bytes, groups);
    if (err != cudaSuccess) return cuda_fail(e, err, "decode scratch allocation");
    p.partials = e->partials;
    p.counters = e->counters;
    const int prof = prof_begin(e, PK_KV4_DECODE);
    const te_status st = queue(e, launch_kv4_decode(p, (int)hd, e->stream), prof, "4-bit decode launch");
    if (st != TE_STATUS_OK) return st;
  }
  if (append && (flags & TE_ATTN_ADVANCE)) {
    for (size_t i = 0; i < n_seqs; ++i) b.len[seq_ids[i]] += 1;
  }
  return TE_STATUS_OK;
}

}  // extern "C"
