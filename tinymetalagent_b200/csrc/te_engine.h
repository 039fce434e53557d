// The engine and the paged cache's bookkeeping, shared by the translation
// units of the C-ABI layer (te_api.cpp, te_api_kv4.cpp), with their helpers:
// error reporting, the launch profile, scratch growth, page mapping.  Not
// installed; not part of the ABI.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdio>
#include <string>
#include <vector>

#include "te_internal.h"

extern "C" void te_host_rope_table(float* cos_table, float* sin_table, size_t first_position, size_t positions,
                                   size_t head_dim, float theta);

struct te_attn_engine {
  int device = 0;
  cudaStream_t stream = nullptr;
  bool own_stream = false;
  int sm_count = 148;
  uint32_t decode_chunk = 0;
  float* partials = nullptr;
  size_t partials_bytes = 0;
  uint32_t* counters = nullptr;
  size_t counters_count = 0;
  int* d_error = nullptr;
  void* io = nullptr;  // device staging for TE_ATTN_HOST_BUFFERS
  size_t io_bytes = 0;
  void* qh = nullptr;  // prefill: rotated f16 queries
  size_t qh_bytes = 0;
  uint32_t* tile_counter = nullptr;
  // decode scratch (partials, counters) that a larger one took the place of: recorded CUDA graphs still hold its
  // address, so it lives as long as the engine.  Sizes at least double, so all of it is no larger than what replaced it.
  static constexpr int kMaxRetired = 64;
  void* retired[kMaxRetired] = {};
  int n_retired = 0;
  uint64_t launches = 0;
  std::string last_error;
  bool time_kernels = false;  // te_attn_engine_time_kernels
  bool kernel_timed = false;
  cudaEvent_t ev_k0 = nullptr, ev_k1 = nullptr;
  uint64_t wait_ns = 2000000000ull;  // bound of the exchange kernel's waits for other GPUs

  // Per-kernel device-time profile (te_attn_engine_profile, TINYENGINE_PROFILE=1):
  // an event pair around every launch, resolved when the engine synchronises.
  bool profile = false;
  bool profile_env = false;  // enabled by TINYENGINE_PROFILE: printed to stderr when the engine is freed
  struct ProfPair {
    int kind;
    cudaEvent_t a, b;
  };
  std::vector<ProfPair> prof_pending;
  std::vector<ProfPair> prof_free;
  static constexpr int kProfKinds = 16;
  double prof_ms[kProfKinds] = {};  // per ProfKind
  uint64_t prof_calls[kProfKinds] = {};
};

struct te_kv_cache {
  te_attn_engine* eng = nullptr;
  te_kv_cache_desc d{};
  uint32_t pages_per_seq = 0;
  uint16_t* k_pool = nullptr;
  uint16_t* v_pool = nullptr;
  int32_t* d_page_table = nullptr;
  std::vector<int32_t> h_page_table;  // [max_seqs][pages_per_seq], -1 = unmapped
  std::vector<uint32_t> contig;       // per sequence: leading pages that are consecutive in the pool
  std::vector<int64_t> len, offset;
  std::vector<int32_t> free_pages;
  float* d_cos = nullptr;
  float* d_sin = nullptr;
  CUtensorMap tmap_k{}, tmap_v{};
  // projection biases (te_kv_cache_set_qkv_bias): [layers][bias_heads * hd] for q,
  // [layers][kv_heads * hd] for k and v; null until set
  float* d_qb = nullptr;
  float* d_kb = nullptr;
  float* d_vb = nullptr;
  uint32_t bias_heads = 0;
};

namespace te {

// Switches to a device for the duration of a call and restores the caller's.
struct DeviceGuard {
  int prev = -1;
  explicit DeviceGuard(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev != dev) cudaSetDevice(dev);
  }
  ~DeviceGuard() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

inline te_status fail(te_attn_engine* e, te_status st, const std::string& msg) {
  if (e) e->last_error = msg;
  return st;
}

inline te_status cuda_fail(te_attn_engine* e, cudaError_t err, const char* what) {
  (void)cudaGetLastError();  // reported here: the next launch must not report it again
  std::string m = std::string(what) + ": " + cudaGetErrorString(err);
  if (e) e->last_error = m;
  return err == cudaErrorMemoryAllocation ? TE_STATUS_OUT_OF_MEMORY : TE_STATUS_RUNTIME_ERROR;
}

inline bool cuda_device_available() {
  int n = 0;
  return cudaGetDeviceCount(&n) == cudaSuccess && n > 0;
}

// Kernel families of the profile, in report order.
enum ProfKind {
  PK_DECODE = 0, PK_APPEND, PK_MERGE, PK_PREFILL_PREP, PK_PREFILL_ATTN, PK_MATVEC, PK_EXCHANGE, PK_STEP,
  PK_KV4_DECODE, PK_KV4_APPEND, PK_KV4_READ, PK_COUNT
};
inline const char* const kProfNames[PK_COUNT] = {"decode",       "append", "merge",    "prefill_prep",
                                                 "prefill_attn", "matvec", "exchange", "step",
                                                 "kv4_decode",   "kv4_append", "kv4_read"};

static_assert(PK_COUNT <= te_attn_engine::kProfKinds, "profile totals too small");

// Opens a profiled launch: records the first event of a pair on the engine's
// stream and returns its slot, or -1 when profiling is off or the stream is
// being captured into a graph (event timing does not apply to replays).
inline int prof_begin(te_attn_engine* e, int kind) {
  if (!e->profile) return -1;
  cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(e->stream, &cs) != cudaSuccess || cs != cudaStreamCaptureStatusNone) return -1;
  te_attn_engine::ProfPair pp;
  if (!e->prof_free.empty()) {
    pp = e->prof_free.back();
    e->prof_free.pop_back();
  } else if (cudaEventCreate(&pp.a) != cudaSuccess || cudaEventCreate(&pp.b) != cudaSuccess) {
    return -1;
  }
  pp.kind = kind;
  cudaEventRecord(pp.a, e->stream);
  e->prof_pending.push_back(pp);
  return (int)e->prof_pending.size() - 1;
}

inline void prof_end(te_attn_engine* e, int slot) {
  if (slot >= 0) cudaEventRecord(e->prof_pending[(size_t)slot].b, e->stream);
}

// Folds every completed pair into the per-kind totals (waits for none).
inline void prof_collect(te_attn_engine* e) {
  std::vector<te_attn_engine::ProfPair> keep;
  for (const auto& pp : e->prof_pending) {
    if (cudaEventQuery(pp.b) != cudaSuccess) {
      keep.push_back(pp);
      continue;
    }
    float ms = 0.f;
    if (cudaEventElapsedTime(&ms, pp.a, pp.b) == cudaSuccess) {
      e->prof_ms[pp.kind] += ms;
      e->prof_calls[pp.kind] += 1;
    }
    e->prof_free.push_back(pp);
  }
  e->prof_pending.swap(keep);
  (void)cudaGetLastError();  // a query of a not-yet-complete event is not an error
}

inline std::string prof_line(const te_attn_engine* e) {
  double total = 0.0;
  for (int k = 0; k < PK_COUNT; ++k) total += e->prof_ms[k];
  std::string out;
  char buf[96];
  std::snprintf(buf, sizeof(buf), "tinyengine_profile: device_ms=%.3f", total);
  out += buf;
  for (int k = 0; k < PK_COUNT; ++k) {
    // the 4-bit cache's kinds only where they ran: without it the line is what its readers' buffers were made for
    if (k >= PK_KV4_DECODE && e->prof_calls[k] == 0) continue;
    std::snprintf(buf, sizeof(buf), " %s=%.3f/%llu", kProfNames[k], e->prof_ms[k],
                  (unsigned long long)e->prof_calls[k]);
    out += buf;
  }
  return out;
}

// Grows a device buffer; the stream is drained first so no queued kernel uses the old one.
inline cudaError_t grow(te_attn_engine* e, void** buf, size_t* cap, size_t need) {
  if (need <= *cap) return cudaSuccess;
  cudaError_t err = cudaStreamSynchronize(e->stream);
  if (err != cudaSuccess) return err;
  if (*buf) cudaFree(*buf);
  *buf = nullptr;
  *cap = 0;
  const size_t sz = std::max(2 * need, (size_t)1 << 20);  // a call that needs slightly more never reallocates each time
  err = cudaMalloc(buf, sz);
  if (err == cudaSuccess) *cap = sz;
  return err;
}

// Grows the decode kernels' scratch to `part_bytes` of partial records and `counters` group counters (zero between
// launches).  The old buffers are retired, not freed: decode calls can be recorded into CUDA graphs.
inline cudaError_t grow_decode_scratch(te_attn_engine* e, size_t part_bytes, size_t counters) {
  auto larger = [&](void** buf, size_t* cap, size_t need, bool zero) -> cudaError_t {
    if (need <= *cap) return cudaSuccess;
    if (e->n_retired == te_attn_engine::kMaxRetired) return cudaErrorMemoryAllocation;
    cudaError_t err = cudaStreamSynchronize(e->stream);  // refuses a stream that is being captured, whatever the mode
    if (err != cudaSuccess) return err;
    const size_t sz = std::max(2 * need, (size_t)1 << 20);
    void* fresh = nullptr;
    err = cudaMalloc(&fresh, sz);
    if (err == cudaSuccess && zero) err = cudaMemsetAsync(fresh, 0, sz, e->stream);  // before the kernels that use it
    if (err != cudaSuccess) {
      cudaFree(fresh);
      return err;
    }
    if (*buf) e->retired[e->n_retired++] = *buf;
    *buf = fresh;
    *cap = sz;
    return cudaSuccess;
  };
  cudaError_t err = larger(reinterpret_cast<void**>(&e->partials), &e->partials_bytes, part_bytes, false);
  if (err != cudaSuccess) return err;
  size_t bytes = e->counters_count * sizeof(uint32_t);
  err = larger(reinterpret_cast<void**>(&e->counters), &bytes, counters * sizeof(uint32_t), true);
  e->counters_count = bytes / sizeof(uint32_t);
  return err;
}

// Maps pages so that sequence `seq` can hold `tokens` tokens.
inline te_status ensure_pages(te_kv_cache* c, size_t seq, size_t tokens) {
  if (tokens > c->d.max_tokens_per_seq) {
    return fail(c->eng, TE_STATUS_INVALID_ARGUMENT, "sequence would exceed max_tokens_per_seq");
  }
  const size_t need = (tokens + c->d.page_tokens - 1) / c->d.page_tokens;
  int32_t* row = c->h_page_table.data() + seq * c->pages_per_seq;
  // All or nothing: a page mapped here but never uploaded would be missing from the device's table later.
  size_t missing = 0;
  for (size_t i = 0; i < need; ++i) missing += row[i] < 0 ? 1 : 0;
  if (missing > c->free_pages.size()) return fail(c->eng, TE_STATUS_OUT_OF_MEMORY, "KV page pool exhausted");
  size_t first_new = need, last_new = 0;
  for (size_t i = 0; i < need && missing > 0; ++i) {
    if (row[i] >= 0) continue;
    row[i] = c->free_pages.back();
    c->free_pages.pop_back();
    --missing;
    first_new = std::min(first_new, i);
    last_new = i;
  }
  if (first_new < need) {
    cudaError_t err = cudaMemcpyAsync(c->d_page_table + seq * c->pages_per_seq + first_new, row + first_new,
                                      (last_new - first_new + 1) * sizeof(int32_t), cudaMemcpyHostToDevice,
                                      c->eng->stream);
    if (err != cudaSuccess) return cuda_fail(c->eng, err, "page table upload");
  }
  uint32_t& run = c->contig[seq];
  while (run < need && row[run] == row[0] + (int32_t)run) ++run;
  return TE_STATUS_OK;
}

// First page of `seq` when its pages covering `tokens` are consecutive in the
// pool (the kernel then computes page ids instead of reading the table), or -1.
inline int32_t contiguous_base(const te_kv_cache* c, size_t seq, size_t tokens) {
  const size_t need = (tokens + c->d.page_tokens - 1) / c->d.page_tokens;
  return need > 0 && c->contig[seq] >= need ? c->h_page_table[seq * c->pages_per_seq] : -1;
}

}  // namespace te
