// Kernels of the 4-bit KV cache (layout: te_kv4.h): the quantising append,
// the read-back, the raw Q4_0 import/export, and the decode attention on the
// tensor cores (tcgen05), which widens the codes only on their way into TMEM.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>

#include "te_internal.h"
#include "te_kv4.h"
#include "te_ptx.cuh"
#include "te_rope.cuh"

#ifndef KV4_CTAS
#define KV4_CTAS 3
#endif

namespace te {
namespace {

// ---- quantising one row -----------------------------------------------------

// Codes and scale of the 32-value block held by 8 consecutive lanes, 4 values
// each: m = the value of largest magnitude (the lowest index on ties), d =
// f16(m / -8) saturated to the finite range, c = clamp(rint(x / d), -8, 7) + 8
// with the correctly rounded quotient.  d is held as the cache holds it, so a
// value is off by at most |d| / 2 (|d| at the far end of the block's range).
// A block with a value that is not finite gets d = NaN: it stands for no
// number, and what reads it shows that.
__device__ __forceinline__ void q4_quantise(const float (&x)[4], int lane, uint32_t (&c)[4], __half& d) {
  auto mag = [](float v) { return __float_as_uint(v) & 0x7fffffffu; };
  float m = x[0];
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    if (mag(x[i]) > mag(m)) m = x[i];
  }
#pragma unroll
  for (int off = 1; off < 8; off <<= 1) {
    const float o = __shfl_xor_sync(0xffffffffu, m, off);
    if (mag(o) > mag(m) || (mag(o) == mag(m) && (lane & off))) m = o;
  }
  const bool finite = mag(m) < 0x7f800000u;
  d = finite ? __float2half_rn(fminf(fmaxf(m * -0.125f, -65504.f), 65504.f)) : __ushort_as_half((unsigned short)0x7fff);
  const float df = __half2float(d);
  const bool zero = !finite || df == 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float r = fminf(fmaxf(rintf(__fdiv_rn(x[i], df)), -8.f), 7.f);
    c[i] = zero ? 8u : (uint32_t)((int)r + 8);
  }
}

// The value a code stands for (exact in fp32: 4 by 11 bits).
__device__ __forceinline__ float q4_value(uint32_t c, float d) { return (float)((int)c - 8) * d; }

// Bits of 4 consecutive codes in their K word: h = 0 the lower 4 of the word's 8 codes, 1 the upper.
__device__ __forceinline__ uint32_t k_bits(const uint32_t (&c)[4], int h) {
  return (c[0] | c[1] << 16 | c[2] << 4 | c[3] << 20) << (8 * h);
}

// One token's key and value row, spread over a warp: lane l holds 4 values
// of each.  head_dim 128: dims 4l .. 4l+3 of the key and of the value;
// head_dim 64: the key in lanes 0-15, the value in lanes 16-31 (k unused in
// the upper lanes, v in the lower).
template <int HD>
struct RowDims {
  static constexpr int kLanes = HD / 4;
  static __device__ __forceinline__ int dim(int lane) { return (lane % kLanes) * 4; }
  static __device__ __forceinline__ bool has_k(int lane) { return HD == 128 || lane < 16; }
  static __device__ __forceinline__ bool has_v(int lane) { return HD == 128 || lane >= 16; }
};

__device__ __forceinline__ void load4(const void* base, size_t idx, int f16, float (&v)[4]) {
  if (f16) {
    const uint2 u = *reinterpret_cast<const uint2*>(reinterpret_cast<const __half*>(base) + idx);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
  } else {
    const float4 a = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + idx);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  }
}
__device__ __forceinline__ void store4(void* base, size_t idx, int f16, const float (&v)[4]) {
  if (f16) {
    *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(base) + idx) =
        make_uint2(pack_half2(v[0], v[1]), pack_half2(v[2], v[3]));
  } else {
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + idx) = make_float4(v[0], v[1], v[2], v[3]);
  }
}
__device__ __forceinline__ void add_bias4(float (&v)[4], const float* b) {
  const float4 x = *reinterpret_cast<const float4*>(b);
  v[0] = __fadd_rn(v[0], x.x); v[1] = __fadd_rn(v[1], x.y); v[2] = __fadd_rn(v[2], x.z); v[3] = __fadd_rn(v[3], x.w);
}

// Rotates the key row (4 dims a lane) at cos/sin rows c, s with the
// reference's fp32 expressions; the partner dim is half a row of lanes away.
template <int HD>
__device__ __forceinline__ void rope4(float (&k)[4], const float* cr, const float* sr, int lane) {
  constexpr int half_lanes = HD / 8;
  const bool upper = (lane & half_lanes) != 0;
  const int d = RowDims<HD>::dim(lane) % (HD / 2);
  const float4 c = *reinterpret_cast<const float4*>(cr + d);
  const float4 s = *reinterpret_cast<const float4*>(sr + d);
  const float cv[4] = {c.x, c.y, c.z, c.w}, sv[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float o = __shfl_xor_sync(0xffffffffu, k[i], half_lanes);
    k[i] = upper ? rope_hi(o, k[i], cv[i], sv[i]) : rope_lo(k[i], o, cv[i], sv[i]);
  }
}

// Quantises a token's rows: kw = its K word (complete in both lanes of a pair), vc its V codes, and the scales
// (in every lane of a block).  The whole warp calls it.  On return k and v hold the values the codes stand for.
// At head_dim 64 the key's results are in lanes 0-15, the value's in lanes 16-31.
template <int HD>
__device__ __forceinline__ void quantise_row(int lane, float (&k)[4], float (&v)[4], uint32_t& kw, __half& kd,
                                             uint32_t (&vc)[4], __half& vd) {
  using R = RowDims<HD>;
  uint32_t c[4];
  if constexpr (HD == 128) {
    q4_quantise(k, lane, c, kd);
    q4_quantise(v, lane, vc, vd);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      k[i] = q4_value(c[i], __half2float(kd));
      v[i] = q4_value(vc[i], __half2float(vd));
    }
  } else {
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = R::has_k(lane) ? k[i] : v[i];
    q4_quantise(x, lane, c, kd);
    vd = kd;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      vc[i] = c[i];
      k[i] = v[i] = q4_value(c[i], __half2float(kd));
    }
  }
  kw = k_bits(c, lane & 1);
  kw |= __shfl_xor_sync(0xffffffffu, kw, 1);
}

// A token's raw key and value rows at element offset `at`.
template <int HD>
__device__ __forceinline__ void fetch_row(const void* kp, const void* vp, size_t at, int f16, int lane, float (&k)[4],
                                          float (&v)[4]) {
  using R = RowDims<HD>;
#pragma unroll
  for (int i = 0; i < 4; ++i) k[i] = v[i] = 0.f;
  if (R::has_k(lane)) load4(kp, at + R::dim(lane), f16, k);
  if (R::has_v(lane)) load4(vp, at + R::dim(lane), f16, v);
}
// Their bias and RoPE (null pointers: none).
template <int HD>
__device__ __forceinline__ void prepare_row(const float* kb, const float* vb, const float* cr, const float* sr,
                                            int lane, float (&k)[4], float (&v)[4]) {
  using R = RowDims<HD>;
  if (kb) {
    if (R::has_k(lane)) add_bias4(k, kb + R::dim(lane));
    if (R::has_v(lane)) add_bias4(v, vb + R::dim(lane));
  }
  if (cr) rope4<HD>(k, cr, sr, lane);
}

// Quotient of a unit index by units_per_page: the product with the rounded-up
// reciprocal is at most one too large (its excess is below unit / 2^32 < 1).
__device__ __forceinline__ int kv4_page_of(const Kv4Pool& p, int unit) {
  if (p.upp_magic == 0) return unit;
  int q = (int)__umulhi((uint32_t)unit, p.upp_magic);
  if (q * p.units_per_page > unit) --q;
  return q;
}
__device__ __forceinline__ unsigned char* unit_ptr(const Kv4Pool& p, const int32_t* page_row, int layer, int kvh,
                                                   int unit, int unit_bytes) {
  const int page = kv4_page_of(p, unit);
  const int in = unit - page * p.units_per_page;
  const long long rec = ((long long)layer * p.num_pages + page_row[page]) * p.kv_heads + kvh;
  return p.base + (rec * p.units_per_page + in) * unit_bytes;
}

// ---- append -------------------------------------------------------------------

// One CTA per (layer, kv head, 32 tokens), a warp per 8 of them (a V word): the half unit is assembled in shared
// memory, with the tokens it already holds if the new ones do not fill it, and written in 16-byte pieces.
template <int HD>
__global__ void __launch_bounds__(128) kv4_append_kernel(const Kv4RowsParams p) {
  constexpr int UB = kv4_unit_bytes(HD), NB = HD / 32;
  constexpr int kSc = 32 * NB * 2;  // bytes of one side's scales
  __shared__ __align__(16) unsigned char sk[NB * 512], sv[HD * 16], sc[2 * kSc];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h0 = p.first / 32;
  const int n_half = (p.first + p.n_tokens - 1) / 32 - h0 + 1;
  const long long item = blockIdx.x;
  const int kvh = (int)(item % p.pool.kv_heads);
  const long long r = item / p.pool.kv_heads;
  const int half = h0 + (int)(r % n_half);
  const int ll = (int)(r / n_half);
  const int layer = p.layer_begin + ll;
  const int lo = max(p.first - half * 32, 0), hi = min(p.first + p.n_tokens - half * 32, 32);
  using R = RowDims<HD>;

  // this warp's tokens: all rows in flight before the first is used
  float k[8][4], v[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int t = 8 * warp + i;
    if (t >= lo && t < hi) {
      const long long row = (long long)ll * p.n_tokens + (half * 32 + t - p.first);
      fetch_row<HD>(p.k, p.v, (size_t)(row * p.token_stride) + (size_t)kvh * HD, p.input_f16, lane, k[i], v[i]);
    }
  }
  unsigned char* unit = unit_ptr(p.pool, p.page_row, layer, kvh, half / 2, UB);
  // global pieces of this thread: (b, token) of the K codes, dim of the V codes, 16 bytes of scales
  const int h32 = (half & 1) * 32;
  unsigned char* gk = unit + ((int)(threadIdx.x >> 5) * 64 + h32 + (int)(threadIdx.x & 31)) * 16;
  unsigned char* gv = unit + kv4_v_off(HD) + ((half & 1) * HD + (int)threadIdx.x) * 16;
  const int si = (int)threadIdx.x * 16;  // of [K scales | V scales]
  unsigned char* gs = unit + (si < kSc ? kv4_ks_off(HD) + kv4_scale(HD, h32, 0) + si
                                       : kv4_vs_off(HD) + kv4_scale(HD, h32, 0) + si - kSc);
  const bool has_k = threadIdx.x < NB * 32, has_v = threadIdx.x < HD, has_s = si < 2 * kSc;
  if (lo > 0 || hi < 32) {
    if (has_k) *reinterpret_cast<uint4*>(sk + threadIdx.x * 16) = *reinterpret_cast<const uint4*>(gk);
    if (has_v) *reinterpret_cast<uint4*>(sv + threadIdx.x * 16) = *reinterpret_cast<const uint4*>(gv);
    if (has_s) *reinterpret_cast<uint4*>(sc + si) = *reinterpret_cast<const uint4*>(gs);
    __syncthreads();
  }
  const size_t brow = ((size_t)layer * p.pool.kv_heads + kvh) * HD;
  const float* kb = p.k_bias ? p.k_bias + brow : nullptr;
  const float* vb = p.k_bias ? p.v_bias + brow : nullptr;
  const int dim = R::dim(lane), b = dim >> 5;
  uint32_t vw[4] = {0u, 0u, 0u, 0u}, mask = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int t = 8 * warp + i;
    if (t < lo || t >= hi) continue;  // the same for the whole warp
    const int tok = half * 32 + t - p.first;
    const float* cr = p.rope ? p.rope_cos + (size_t)(p.first_pos + tok) * (HD / 2) : nullptr;
    const float* sr = p.rope ? p.rope_sin + (size_t)(p.first_pos + tok) * (HD / 2) : nullptr;
    prepare_row<HD>(kb, vb, cr, sr, lane, k[i], v[i]);
    uint32_t kw, vc[4];
    __half kd, vd;
    quantise_row<HD>(lane, k[i], v[i], kw, kd, vc, vd);
#pragma unroll
    for (int j = 0; j < 4; ++j) vw[j] |= vc[j] << (4 * kv4_nibble(i));
    mask |= 15u << (4 * kv4_nibble(i));
    if (R::has_k(lane) && (lane & 1) == 0) {
      *reinterpret_cast<uint32_t*>(sk + (b * 32 + t) * 16 + ((dim & 31) >> 3) * 4) = kw;
    }
    if ((lane & 7) == 0) {
      if (R::has_k(lane)) *reinterpret_cast<__half*>(sc + kv4_scale(HD, t, b)) = kd;
      if (R::has_v(lane)) *reinterpret_cast<__half*>(sc + kSc + kv4_scale(HD, t, b)) = vd;
    }
    if (p.k_rows) {
      const size_t o = (((size_t)ll * p.n_tokens + tok) * p.pool.kv_heads + kvh) * HD + dim;
      if (R::has_k(lane)) store4(p.k_rows, o, p.rows_f16, k[i]);
      if (R::has_v(lane)) store4(p.v_rows, o, p.rows_f16, v[i]);
    }
  }
  if (R::has_v(lane) && mask != 0u) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t* w = reinterpret_cast<uint32_t*>(sv + (dim + j) * 16 + warp * 4);
      *w = mask == 0xffffffffu ? vw[j] : (*w & ~mask) | vw[j];
    }
  }
  __syncthreads();
  if (has_k) *reinterpret_cast<uint4*>(gk) = *reinterpret_cast<const uint4*>(sk + threadIdx.x * 16);
  if (has_v) *reinterpret_cast<uint4*>(gv) = *reinterpret_cast<const uint4*>(sv + threadIdx.x * 16);
  if (has_s) *reinterpret_cast<uint4*>(gs) = *reinterpret_cast<const uint4*>(sc + si);
}

// ---- read ---------------------------------------------------------------------

// One CTA per (layer, kv head, 32 tokens), a warp per 8 of them; a lane holds 4 dims, so that a token's row leaves
// as one contiguous store.
template <int HD>
__global__ void __launch_bounds__(128) kv4_read_kernel(const Kv4RowsParams p) {
  constexpr int UB = kv4_unit_bytes(HD);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h0 = p.first / 32;
  const int n_half = (p.first + p.n_tokens - 1) / 32 - h0 + 1;
  const long long item = blockIdx.x;
  const int kvh = (int)(item % p.pool.kv_heads);
  const long long r = item / p.pool.kv_heads;
  const int half = h0 + (int)(r % n_half);
  const int ll = (int)(r / n_half);
  const unsigned char* unit = unit_ptr(p.pool, p.page_row, p.layer_begin + ll, kvh, half / 2, UB);
  using R = RowDims<HD>;
  const int dim = R::dim(lane), b = dim >> 5;
  const int r0 = (half & 1) * 32 + 8 * warp;  // this warp's first token in the unit
  uint32_t vw[4];
  if (R::has_v(lane)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      vw[j] = *reinterpret_cast<const uint32_t*>(unit + kv4_v_off(HD) + kv4_v_word(HD, dim + j, r0 >> 3));
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int tok = half * 32 + 8 * warp + i - p.first;
    if (tok < 0 || tok >= p.n_tokens) continue;
    const size_t o = (((size_t)ll * p.n_tokens + tok) * p.pool.kv_heads + kvh) * HD + dim;
    float x[4];
    if (R::has_k(lane)) {
      const uint32_t w =
          *reinterpret_cast<const uint32_t*>(unit + kv4_k_word(r0 + i, b, (dim & 31) >> 3)) >> (8 * (lane & 1));
      const float d = __half2float(*reinterpret_cast<const __half*>(unit + kv4_ks_off(HD) + kv4_scale(HD, r0 + i, b)));
      x[0] = q4_value(w & 15u, d);
      x[1] = q4_value((w >> 16) & 15u, d);
      x[2] = q4_value((w >> 4) & 15u, d);
      x[3] = q4_value((w >> 20) & 15u, d);
      store4(p.k_rows, o, p.rows_f16, x);
    }
    if (R::has_v(lane)) {
      const float d = __half2float(*reinterpret_cast<const __half*>(unit + kv4_vs_off(HD) + kv4_scale(HD, r0 + i, b)));
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = q4_value((vw[j] >> (4 * kv4_nibble(i))) & 15u, d);
      store4(p.v_rows, o, p.rows_f16, x);
    }
  }
}

// ---- raw Q4_0 blocks ------------------------------------------------------------

// One thread per (layer, kv head, 8 tokens, block): both sides.  A raw block is 18 bytes, 2-byte aligned: the
// scale, then byte i = code i | code (i + 16) << 4.
template <int HD>
__global__ void __launch_bounds__(128) kv4_raw_kernel(const Kv4RowsParams p, int to_pool) {
  constexpr int UB = kv4_unit_bytes(HD), NB = HD / 32;
  const int g0 = p.first / 8;
  const int n_groups = (p.first + p.n_tokens - 1) / 8 - g0 + 1;
  const long long n = (long long)p.n_layers * n_groups * p.pool.kv_heads * NB;
  const long long id = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (id >= n) return;
  const int b = (int)(id % NB);
  long long r = id / NB;
  const int kvh = (int)(r % p.pool.kv_heads);
  r /= p.pool.kv_heads;
  const int group = g0 + (int)(r % n_groups);
  const int ll = (int)(r / n_groups);
  unsigned char* unit = unit_ptr(p.pool, p.page_row, p.layer_begin + ll, kvh, group / 8, UB);
  const int y = group % 8;
  const int lo = max(p.first - group * 8, 0), hi = min(p.first + p.n_tokens - group * 8, 8);
  auto raw_at = [&](int i) {  // raw block of the group's token i, in 2-byte units
    const long long tok = (long long)ll * p.n_tokens + (group * 8 + i - p.first);
    return ((tok * p.pool.kv_heads + kvh) * NB + b) * 9;
  };
  auto v_word = [&](int c) {
    return reinterpret_cast<uint32_t*>(unit + kv4_v_off(HD) + kv4_v_word(HD, 32 * b + c, y));
  };
  uint32_t vw[32];
  if (to_pool) {
    uint32_t mask = 0u;
#pragma unroll
    for (int c = 0; c < 32; ++c) vw[c] = 0u;
    for (int i = lo; i < hi; ++i) {
      const uint16_t* kr = reinterpret_cast<const uint16_t*>(p.k) + raw_at(i);
      const uint16_t* vr = reinterpret_cast<const uint16_t*>(p.v) + raw_at(i);
      const int tok = 8 * y + i, sh = 4 * kv4_nibble(i);
      uint32_t kc[32];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const uint32_t kx = kr[1 + q], vx = vr[1 + q];
        kc[2 * q] = kx & 15u;
        kc[2 * q + 1] = (kx >> 8) & 15u;
        kc[2 * q + 16] = (kx >> 4) & 15u;
        kc[2 * q + 17] = kx >> 12;
        vw[2 * q] |= (vx & 15u) << sh;
        vw[2 * q + 1] |= ((vx >> 8) & 15u) << sh;
        vw[2 * q + 16] |= ((vx >> 4) & 15u) << sh;
        vw[2 * q + 17] |= (vx >> 12) << sh;
      }
      mask |= 15u << sh;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint32_t a[4] = {kc[8 * t], kc[8 * t + 1], kc[8 * t + 2], kc[8 * t + 3]};
        const uint32_t c[4] = {kc[8 * t + 4], kc[8 * t + 5], kc[8 * t + 6], kc[8 * t + 7]};
        *reinterpret_cast<uint32_t*>(unit + kv4_k_word(tok, b, t)) = k_bits(a, 0) | k_bits(c, 1);
      }
      *reinterpret_cast<uint16_t*>(unit + kv4_ks_off(HD) + kv4_scale(HD, tok, b)) = kr[0];
      *reinterpret_cast<uint16_t*>(unit + kv4_vs_off(HD) + kv4_scale(HD, tok, b)) = vr[0];
    }
#pragma unroll
    for (int c = 0; c < 32; ++c) *v_word(c) = mask == 0xffffffffu ? vw[c] : (*v_word(c) & ~mask) | vw[c];
  } else {
#pragma unroll
    for (int c = 0; c < 32; ++c) vw[c] = *v_word(c);
    for (int i = lo; i < hi; ++i) {
      uint16_t* kr = reinterpret_cast<uint16_t*>(p.k_rows) + raw_at(i);
      uint16_t* vr = reinterpret_cast<uint16_t*>(p.v_rows) + raw_at(i);
      const int tok = 8 * y + i, sh = 4 * kv4_nibble(i);
      uint32_t kc[32];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(unit + kv4_k_word(tok, b, t));
#pragma unroll
        for (int c = 0; c < 8; ++c) kc[8 * t + c] = (w >> (4 * kv4_nibble(c))) & 15u;
      }
      kr[0] = *reinterpret_cast<const uint16_t*>(unit + kv4_ks_off(HD) + kv4_scale(HD, tok, b));
      vr[0] = *reinterpret_cast<const uint16_t*>(unit + kv4_vs_off(HD) + kv4_scale(HD, tok, b));
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        kr[1 + q] = (uint16_t)(kc[2 * q] | kc[2 * q + 16] << 4 | kc[2 * q + 1] << 8 | kc[2 * q + 17] << 12);
        vr[1 + q] = (uint16_t)(((vw[2 * q] >> sh) & 15u) | ((vw[2 * q + 16] >> sh) & 15u) << 4 |
                               ((vw[2 * q + 1] >> sh) & 15u) << 8 | ((vw[2 * q + 17] >> sh) & 15u) << 12);
      }
    }
  }
}

// ---- decode attention -------------------------------------------------------------
//
// out = softmax(q K^T / sqrt(hd)) V per query head, over a group's cached tokens and the token the call appends.
// A CTA of 128 threads takes 128 tokens a step (two units), one token a thread, and up to 8 query heads:
//
//   S = K q^T: A = the K codes minus 8, widened to f16 and put into TMEM by the thread whose token they are;
//      B = the queries in shared memory, f16 hi and lo parts of 8 heads (N = 16), scaled by a power of two per head;
//      one product per block of 32 dims, so that the thread multiplies by its token's scales on the way out:
//      score = sum_b d_b (hi + lo), fp32.
//   O^T = V^T P: A = the V codes minus 8 (M = dims, the same TMEM columns); B = the weights in shared memory:
//      P d for each block of dims, f16 hi + lo parts by an error-free product (hi = f16(P d), lo = f16 of the
//      rest, about 22 bits), N = blocks * 16.  The rows of block b need its 16 columns only; the rest of the
//      product is computed and not read -- the tensor pipe is far from its limit (at head_dim 64 the rows are
//      the dims of the step's two units, each with columns of its own).
//
// Each product starts from zero and is added to fp32 registers: a long accumulation inside the tensor core
// truncates at every step.  The online softmax keeps a reference exponent per head for the whole CTA and moves it
// only when a score exceeds it by more than 2^3.
template <int HD>
struct Dec {
  static constexpr int kThreads = 128, kCtas = KV4_CTAS, kRing = 2;
  static constexpr int NB = HD / 32;
  static constexpr int UB = kv4_unit_bytes(HD);
  static constexpr int kStageBytes = 2 * UB;
  static constexpr int kPRows = HD == 128 ? 128 : 64;  // K extent of the second product
  static constexpr int kColA = 0, kColD = 64;          // TMEM columns: the A operand, the products
  static constexpr int p_off = 0;                      // weights: rows of 128 bytes, 128B swizzle
  static constexpr int q_off = kPRows * 128;           // queries: (HD / 64) chunks of 16 rows of 128 bytes, 128B swizzle
  static constexpr int ring_off = q_off + (HD / 64) * 2048;
  static constexpr int f_off = ring_off + kRing * kStageBytes;  // per head: S f = score in exp2 units
  static constexpr int mb_off = f_off + 32;                     // per head: kWeightExp - reference exponent
  static constexpr int red_off = mb_off + 32;                   // [4 warps][9]
  static constexpr int flag_off = red_off + 160;                // fold flags [2], abort, TMEM address
  static constexpr int bar_off = flag_off + 16;                 // full[kRing], product 1, product 2
  static constexpr int pend_off = bar_off + (kRing + 2) * 8;    // two Seg
  static constexpr int smem = pend_off + 2 * 64;
};
static_assert((Dec<128>::smem + 1024) * Dec<128>::kCtas <= 228 * 1024 && Dec<128>::kCtas * 128 <= 512, "CTAs per SM");

constexpr float kSlack = 3.f;       // scores may exceed the reference by this before it moves
constexpr float kWeightExp = 11.f;  // weights are 2^(score - m + 11): at most 2^14, products with a scale at most 2^15

struct Seg {
  int ll, kvh, hb, si;  // local layer, kv head, head block, sequence
  int s0, s1, n;        // stages of the segment, stages of its group
  int next;             // the CTA's next stage (global index), its end when there is none
  int parts, c0;        // CTAs that share the group, the first of them
  int gb;               // stream split: the group's first stage (global index)
  int group_id;
};

static_assert(sizeof(Seg) <= 64, "pending segments");

// Stream split: the CTA whose range [b T / G, (b + 1) T / G) holds stage u.
__device__ __forceinline__ int kv4_cta_of(int u, long long total, int grid) {
  return (int)div_nonneg((long long)(u + 1) * grid - 1, total);
}

// The segment of this CTA that begins at u (stream split), or its only one (aligned split).
__device__ __forceinline__ Seg kv4_seg_at(const Kv4DecodeParams& p, int u, int u1) {
  Seg s;
  const bool aligned = p.block_parts != 0;
  const int per = aligned ? p.block_parts : p.block_stages;
  const int at = aligned ? (int)blockIdx.x : u;
  const uint32_t blk = (uint32_t)at / (uint32_t)per;
  const int rem = at - (int)blk * per;
  int lo = 0, hi = p.n_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    const int begin = aligned ? p.seqs[mid].part_begin : p.seqs[mid].stage_begin;
    if (begin <= rem) lo = mid; else hi = mid - 1;
  }
  s.si = lo;
  s.n = kv4_stages(p.seqs[lo].len + (p.k_new ? 1 : 0));
  if (aligned) {
    const int part = rem - p.seqs[lo].part_begin;
    s.parts = (lo + 1 < p.n_seqs ? p.seqs[lo + 1].part_begin : per) - p.seqs[lo].part_begin;
    s.c0 = (int)blockIdx.x - part;
    s.s0 = (int)div_nonneg((long long)part * s.n, s.parts);
    s.s1 = (int)div_nonneg((long long)(part + 1) * s.n, s.parts);
    s.gb = 0;
    s.next = u1;
  } else {
    s.gb = (int)blk * per + p.seqs[lo].stage_begin;
    s.next = min(s.gb + s.n, u1);
    s.s0 = u - s.gb;
    s.s1 = s.next - s.gb;
    s.c0 = kv4_cta_of(s.gb, p.total_stages, p.grid);
    s.parts = kv4_cta_of(s.gb + s.n - 1, p.total_stages, p.grid) - s.c0 + 1;
  }
  if (p.seqs[lo].len == 0 && !p.k_new) s.s1 = s.s0;  // nothing to attend: zeros
  const uint32_t lk = blk / (uint32_t)p.head_blocks;
  s.hb = (int)(blk - lk * (uint32_t)p.head_blocks);
  s.ll = (int)(lk / (uint32_t)p.pool.kv_heads);
  s.kvh = (int)lk - s.ll * p.pool.kv_heads;
  s.group_id = (int)blk * p.n_seqs + lo;
  return s;
}

__device__ __forceinline__ uint32_t h2_add(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// a b - c in f16x2, one rounding.
__device__ __forceinline__ uint32_t h2_fms(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("{\n\t.reg .b32 n;\n\tneg.f16x2 n, %3;\n\tfma.rn.f16x2 %0, %1, %2, n;\n\t}" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t h2_maxabs(uint32_t a, uint32_t b) {
  const __half2 x = __habs2(*reinterpret_cast<const __half2*>(&a));
  const __half2 y = __habs2(*reinterpret_cast<const __half2*>(&b));
  const __half2 m = __hmax2(x, y);
  return *reinterpret_cast<const uint32_t*>(&m);
}
// 2^k as fp32, -126 <= k <= 127.
__device__ __forceinline__ float pow2i(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }
__device__ __forceinline__ int exponent_of(float x) { return (int)((__float_as_uint(x) >> 23) & 255u) - 127; }

// (x & m) | o as one operation: o comes in a register, since an instruction holds one immediate.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t m, uint32_t o) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(x), "r"(m), "r"(o));
  return d;
}
__device__ __forceinline__ uint32_t code_magic() {  // opaque to the compiler, so that it stays in a register
  uint32_t m;
  asm volatile("mov.b32 %0, 0x64006400;" : "=r"(m));
  return m;
}
// The four f16 pairs of a word: c - 8, and 16 (c - 8) for the odd pairs, exactly: a code under the exponent of
// 1024 is 1024 + c (or + 16 c), and one subtraction leaves a normal number.  Codes read as f16 subnormals would
// need no subtraction, but the tensor core aligns the products of a step by their operands' nominal exponents:
// subnormals lose 7 to 10 bits of the fp32 sum (measured: the output was 8e-6 off, against 1e-6).
__device__ __forceinline__ void centred(uint32_t x, uint32_t magic, uint32_t* c) {
  const uint32_t y = x >> 8;
  c[0] = h2_add(and_or(x, 0x000f000fu, magic), 0xe408e408u);
  c[1] = h2_add(and_or(x, 0x00f000f0u, magic), 0xe480e480u);
  c[2] = h2_add(and_or(y, 0x000f000fu, magic), 0xe408e408u);
  c[3] = h2_add(and_or(y, 0x00f000f0u, magic), 0xe480e480u);
}
// The 16 f16 pairs of a 16-byte chunk.
__device__ __forceinline__ void centred_chunk(uint32_t addr, uint32_t magic, uint32_t* c) {
  const uint4 x = lds128(addr);
  centred(x.x, magic, c);
  centred(x.y, magic, c + 4);
  centred(x.z, magic, c + 8);
  centred(x.w, magic, c + 12);
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]),
        "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&r)[16]) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
      : "r"(taddr));
}
// D[tmem] (+)= A[tmem] * B[smem desc], kind::f16, one CTA.
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// A query head's raw row, 4 dims a lane (lanes 0-15 at head_dim 64); zeros for a head the group has not.
template <int HD>
__device__ __forceinline__ void fetch_query(const Kv4DecodeParams& p, const Seg& s, int h, int lane, float (&v)[4]) {
  const int hg = s.hb * p.block_heads + h;
  v[0] = v[1] = v[2] = v[3] = 0.f;
  if (h < p.block_heads && hg < p.group && lane < HD / 4) {
    const size_t row = ((size_t)s.ll * p.seq_total + p.seq_base + s.si) * (p.pool.kv_heads * p.group) +
                       s.kvh * p.group + hg;
    load4(p.q, row * HD + 4 * lane, p.input_f16, v);
  }
}

// Bias, RoPE, the head's power of two (largest value in [2^11, 2^12)) and the f16 hi / lo split: writes rows h and
// 8 + h of the B operand (dims of odd pairs divided by 16: their codes come as 16 c) and the factor that turns S
// into exp2 units.
template <int HD>
__device__ __forceinline__ void stage_query(const Kv4DecodeParams& p, const Seg& s, int h, int lane, float (&v)[4],
                                            unsigned char* qs, float* f) {
  const int hg = s.hb * p.block_heads + h;
  const bool have = h < p.block_heads && hg < p.group;
  if (have && p.q_bias && lane < HD / 4) {
    add_bias4(v, p.q_bias + ((size_t)(p.layer_begin + s.ll) * (p.pool.kv_heads * p.group) + s.kvh * p.group + hg) * HD +
                     4 * lane);
  }
  if (p.rope) {
    rope4<HD>(v, p.rope_cos + (size_t)p.seqs[s.si].q_pos * (HD / 2), p.rope_sin + (size_t)p.seqs[s.si].q_pos * (HD / 2),
              lane);
  }
  float top = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
  for (int off = 1; off < HD / 4; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  const int k = top > 0.f ? min(max(11 - exponent_of(top), -100), 126) : 0;
  const float sc = pow2i(k);
  if (lane == 0) f[h] = p.scale_log2 * pow2i(-k);
  uint32_t hi[2], lo[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const float mul = r ? 0.0625f : 1.f;
    const float x = v[2 * r] * sc * mul, y = v[2 * r + 1] * sc * mul;
    const __half2 a = __floats2half2_rn(x, y);
    const float2 af = __half22float2(a);
    hi[r] = *reinterpret_cast<const uint32_t*>(&a);
    lo[r] = pack_half2(x - af.x, y - af.y);
  }
  if (lane < HD / 4) {
    const int d = 4 * lane;
    unsigned char* at = qs + (d >> 6) * 2048 + h * 128 + ((((d & 63) >> 3) ^ h) * 16) + (d & 7) * 2;
    *reinterpret_cast<uint2*>(at) = make_uint2(hi[0], hi[1]);
    *reinterpret_cast<uint2*>(at + 1024) = make_uint2(lo[0], lo[1]);
  }
}

// The copies of a CTA: the stages of its segments in order, across segments (kept by thread 0).
struct Feed {
  int u, u1;                  // next segment's first stage, end of the CTA's range
  int stage, s1;              // next stage and end of the current segment
  int units;                  // units of the sequence that hold attended tokens
  const unsigned char* base;  // page 0 of the segment's layer, at its kv head
  const int32_t* row;
  int page_base;
};

template <int HD>
__device__ __forceinline__ void feed_issue(const Kv4DecodeParams& p, Feed& f, unsigned char* dst, uint64_t* bar) {
  using D = Dec<HD>;
  while (f.stage >= f.s1) {
    if (f.u >= f.u1) return;
    const Seg s = kv4_seg_at(p, f.u, f.u1);
    f.u = s.next;
    f.stage = s.s0;
    f.s1 = s.s1;
    f.units = (p.seqs[s.si].len + (p.k_new ? 1 : 0) + kKv4Unit - 1) / kKv4Unit;
    const long long rec = (long long)(p.layer_begin + s.ll) * p.pool.num_pages * p.pool.kv_heads + s.kvh;
    f.base = p.pool.base + rec * p.pool.units_per_page * D::UB;
    f.row = p.page_table + (size_t)p.seqs[s.si].slot * p.max_pages_per_seq;
    f.page_base = p.seqs[s.si].page_base;
  }
  const int u0 = 2 * f.stage;
  const int n = min(2, f.units - u0);
  mbar_arrive_expect_tx(bar, n * D::UB);
  for (int i = 0; i < n; ++i) {
    const int page = kv4_page_of(p.pool, u0 + i);
    const int in = u0 + i - page * p.pool.units_per_page;
    const int id = f.page_base >= 0 ? f.page_base + page : f.row[page];
    bulk_load(dst + i * D::UB,
              f.base + ((long long)id * p.pool.kv_heads * p.pool.units_per_page + in) * D::UB, D::UB, bar);
  }
  ++f.stage;
}

// Quantises the appended token (warp 0): into its slot of the stage in shared memory, so that the step attends it
// as stored, and (first head block) into the cache.
template <int HD>
__device__ __forceinline__ void place_new_token(const Kv4DecodeParams& p, const Seg& s, unsigned char* stage, int lane) {
  using R = RowDims<HD>;
  constexpr int UB = kv4_unit_bytes(HD);
  const Kv4Seq& sq = p.seqs[s.si];
  const size_t at = (((size_t)s.ll * p.seq_total + p.seq_base + s.si) * p.pool.kv_heads + s.kvh) * HD;
  const size_t brow = ((size_t)(p.layer_begin + s.ll) * p.pool.kv_heads + s.kvh) * HD;
  float k[4], v[4];
  fetch_row<HD>(p.k_new, p.v_new, at, p.input_f16, lane, k, v);
  prepare_row<HD>(p.k_bias ? p.k_bias + brow : nullptr, p.k_bias ? p.v_bias + brow : nullptr,
                  p.rope ? p.rope_cos + (size_t)sq.new_pos * (HD / 2) : nullptr,
                  p.rope ? p.rope_sin + (size_t)sq.new_pos * (HD / 2) : nullptr, lane, k, v);
  uint32_t kw, vc[4];
  __half kd, vd;
  quantise_row<HD>(lane, k, v, kw, kd, vc, vd);
  const int unit = sq.len / kKv4Unit, r = sq.len % kKv4Unit;
  unsigned char* sm = stage + (unit & 1) * UB;
  unsigned char* gm = s.hb == 0 ? unit_ptr(p.pool, p.page_table + (size_t)sq.slot * p.max_pages_per_seq,
                                           p.layer_begin + s.ll, s.kvh, unit, UB)
                                : nullptr;
  const int dim = R::dim(lane), b = dim >> 5;
  if (R::has_k(lane) && (lane & 1) == 0) {
    const int o = kv4_k_word(r, b, (dim & 31) >> 3);
    *reinterpret_cast<uint32_t*>(sm + o) = kw;
    if (gm) *reinterpret_cast<uint32_t*>(gm + o) = kw;
  }
  if (R::has_v(lane)) {
    // the token's nibble of each dim's word: its byte also holds the token two places on or back, which the stage has
    const int nib = kv4_nibble(r & 7);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int o = kv4_v_off(HD) + kv4_v_word(HD, dim + j, r >> 3) + (nib >> 1);
      const uint32_t old = sm[o];
      const unsigned char byte = (unsigned char)((nib & 1) ? (old & 0x0fu) | vc[j] << 4 : (old & 0xf0u) | vc[j]);
      sm[o] = byte;
      if (gm) gm[o] = byte;
    }
  }
  if ((lane & 7) == 0) {
    if (R::has_k(lane)) {
      const int o = kv4_ks_off(HD) + kv4_scale(HD, r, b);
      *reinterpret_cast<__half*>(sm + o) = kd;
      if (gm) *reinterpret_cast<__half*>(gm + o) = kd;
    }
    if (R::has_v(lane)) {
      const int o = kv4_vs_off(HD) + kv4_scale(HD, r, b);
      *reinterpret_cast<__half*>(sm + o) = vd;
      if (gm) *reinterpret_cast<__half*>(gm + o) = vd;
    }
  }
}

template <int HD>
__global__ void __launch_bounds__(128, KV4_CTAS) kv4_decode_kernel(const __grid_constant__ Kv4DecodeParams p) {
  using D = Dec<HD>;
  constexpr int NB = D::NB, UB = D::UB, H = kKv4Heads;
  constexpr int rec = kv4_record_floats(HD);
  extern __shared__ __align__(1024) unsigned char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  unsigned char* ps = smem + D::p_off;
  unsigned char* qs = smem + D::q_off;
  unsigned char* ring = smem + D::ring_off;
  float* sm_f = reinterpret_cast<float*>(smem + D::f_off);
  float* sm_mb = reinterpret_cast<float*>(smem + D::mb_off);
  float* sm_red = reinterpret_cast<float*>(smem + D::red_off);
  volatile int* sm_flag = reinterpret_cast<volatile int*>(smem + D::flag_off);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + D::bar_off);
  uint64_t* done1 = full + D::kRing;
  uint64_t* done2 = done1 + 1;
  Seg* pending = reinterpret_cast<Seg*>(smem + D::pend_off);

  // the CTA's range of stages (stream split; an aligned CTA has one segment)
  const bool aligned = p.block_parts != 0;
  const int u_begin = aligned ? 0 : (int)stage_start(blockIdx.x, p.total_stages, p.grid);
  const int u1 = aligned ? 1 : (int)stage_start(blockIdx.x + 1, p.total_stages, p.grid);
  Feed feed{};
  feed.u = u_begin;
  feed.u1 = u1;
  if (tid == 0) {
    for (int i = 0; i < D::kRing + 2; ++i) mbar_init(&full[i], 1);
    sm_flag[2] = 0;
    fence_mbarrier_init();
    fence_proxy_async_shared();
  }
  __syncwarp();
  if (warp == 0) {
    tmem_alloc(reinterpret_cast<uint32_t*>(smem + D::flag_off) + 3, 128);
    tmem_relinquish();
    tc_fence_before();
  }
  griddep_launch_dependents();
  griddep_wait();  // below: the first access to global memory
  int issued = 0;
  if (tid == 0) {
    for (; issued < D::kRing; ++issued) feed_issue<HD>(p, feed, ring + issued * D::kStageBytes, &full[issued]);
  }
  Seg s = kv4_seg_at(p, u_begin, u1);
  float qr[2][4];
#pragma unroll
  for (int i = 0; i < 2; ++i) fetch_query<HD>(p, s, 2 * warp + i, lane, qr[i]);
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *(reinterpret_cast<uint32_t*>(smem + D::flag_off) + 3);
  const uint32_t my_a = tmem + ((uint32_t)(warp * 32) << 16) + D::kColA;
  const uint32_t my_d = tmem + ((uint32_t)(warp * 32) << 16) + D::kColD;
  const uint32_t magic = code_magic();
  // A wait that runs out sets the error word and the CTA's abort flag; the CTA then goes through the rest of its
  // steps without waiting (its results are void), so that every barrier below stays matched.
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (!mbar_try_wait(bar, parity) && !sm_flag[2] && !mbar_wait(bar, parity)) {
      sm_flag[2] = 1;
      set_error(p.error, 60);
    }
    __syncwarp();  // warp-collective TMEM accesses follow
  };

  const int row = tid & 63, unit = tid >> 6;  // this thread's token in the stage
  const int k_scale = unit * UB + kv4_ks_off(HD) + kv4_scale(HD, row, 0);
  const int v_scale = unit * UB + kv4_vs_off(HD) + kv4_scale(HD, row, 0);
  // this thread's row of the weights, and its chunks' swizzle; odd pairs of tokens meet 16 (c - 8)
  const int prow = HD == 128 ? tid : row;
  const uint32_t p_addr = smem_u32(ps) + prow * 128;
  const int p_chunk = HD == 128 ? 0 : unit * 4;
  const float v_div = (tid & 2) ? 0.0625f : 1.f;

  int slot = 0;
  uint32_t phase = 0, phase1 = 0, phase2 = 0;
  int n_pending = 0;   // partial segments of this CTA, whose groups may be its to fold (kept in shared memory)

  while (true) {
#pragma unroll
    for (int i = 0; i < 2; ++i) stage_query<HD>(p, s, 2 * warp + i, lane, qr[i], qs, sm_f);
    if (tid < H) sm_mb[tid] = INFINITY;
    fence_proxy_async_shared();
    const int attended = p.seqs[s.si].len + (p.k_new ? 1 : 0);
    const bool more = s.next < u1;
    Seg nx = s;
    if (more) {  // the next segment's query rows travel while this one is attended
      nx = kv4_seg_at(p, s.next, u1);
#pragma unroll
      for (int i = 0; i < 2; ++i) fetch_query<HD>(p, nx, 2 * warp + i, lane, qr[i]);
    }
    float o[H];
    uint64_t l2[H / 2];
#pragma unroll
    for (int h = 0; h < H; ++h) o[h] = 0.f;
#pragma unroll
    for (int h = 0; h < H / 2; ++h) l2[h] = 0;
    float vlim = 0.f;     // largest |V scale| the current vexp allows
    uint32_t vmul = 0;    // 2^vexp (over 16 for odd pairs of tokens), twice, f16
    int vexp = 0;
    bool open = false;    // a second product is in flight
    auto take_o = [&]() {
      wait(done2, phase2);
      phase2 ^= 1u;
      tc_fence_after();
      float d[16];
      tmem_ld16(my_d + 16 * warp, d);
      tmem_wait_ld();
#pragma unroll
      for (int h = 0; h < H; ++h) o[h] += d[h] + d[8 + h];
    };

    for (int st = s.s0; st < s.s1; ++st) {
      unsigned char* stage = ring + slot * D::kStageBytes;
      const uint32_t sa = smem_u32(stage);
      wait(&full[slot], phase);
      if (p.k_new && st == s.n - 1) {
        __syncthreads();  // every thread has seen the copy land
        if (warp == 0) place_new_token<HD>(p, s, stage, lane);
        fence_proxy_async_shared();  // before a later copy into this slot
        __syncthreads();
      }
      const int left = attended - st * kKv4Stage;  // tokens of this stage that are attended

      // K codes -> TMEM, one token a row
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        uint32_t c[16];
        centred_chunk(sa + unit * UB + kv4_k_word(row, b, 0), magic, c);
        if (b == 0 && open) take_o();  // the A columns and D are free once the last second product is done
        tmem_st16(my_a + 16 * b, c);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncthreads();
      if (tid == 0) {
        tc_fence_after();
        constexpr uint32_t idesc = idesc_f16_f32(128, 16, false, false);
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const uint64_t b = smem_desc_sw128(smem_u32(qs) + (k >> 2) * 2048 + (k & 3) * 32, 16, 1024);
          umma_ts(tmem + D::kColD + (k >> 1) * 16, tmem + D::kColA + k * 8, b, idesc, k & 1);
        }
        umma_commit(done1);
      }

      // V codes: this thread's dim (head_dim 64: of its unit), widened while the product runs
      uint32_t vr[HD / 2];
      if constexpr (HD == 128) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          centred_chunk(sa + (i >> 1) * UB + kv4_v_off(HD) + kv4_v_word(HD, tid, 4 * (i & 1)), magic, vr + 16 * i);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          centred_chunk(sa + unit * UB + kv4_v_off(HD) + kv4_v_word(HD, row, 4 * i), magic, vr + 16 * i);
        }
      }
      uint32_t ks[NB / 2], vs[NB / 2];
#pragma unroll
      for (int i = 0; i < NB / 2; ++i) {
        ks[i] = *reinterpret_cast<const uint32_t*>(stage + k_scale + 4 * i);
        vs[i] = *reinterpret_cast<const uint32_t*>(stage + v_scale + 4 * i);
      }
      wait(done1, phase1);
      phase1 ^= 1u;
      tc_fence_after();
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) tmem_st16(my_a + 16 * i, vr + 16 * i);

      // scores of this thread's token, 8 heads in pairs
      uint64_t x2[H / 2];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float d[16];
        tmem_ld16(my_d + 16 * b, d);
        tmem_wait_ld();
        const float2 kf = __half22float2(*reinterpret_cast<const __half2*>(&ks[b >> 1]));
        const float kd = (b & 1) ? kf.y : kf.x;
        const uint64_t kd2 = f2_pack(kd, kd);
#pragma unroll
        for (int h = 0; h < H / 2; ++h) {
          const uint64_t sum = f2_add(f2_pack(d[2 * h], d[2 * h + 1]), f2_pack(d[8 + 2 * h], d[9 + 2 * h]));
          x2[h] = b == 0 ? f2_mul(kd2, sum) : f2_fma(kd2, sum, x2[h]);
        }
      }
      const bool in = tid < left;
      if (!in) {  // a token past the sequence: no weight, whatever its place holds
        const uint64_t none = f2_pack(-INFINITY, -INFINITY);
#pragma unroll
        for (int h = 0; h < H / 2; ++h) x2[h] = none;
#pragma unroll
        for (int i = 0; i < NB / 2; ++i) vs[i] = 0u;
      }
      float mb[H];
      bool need = false;
      {
        const uint4 a = lds128(smem_u32(sm_mb)), b = lds128(smem_u32(sm_mb) + 16);
        const uint4 c = lds128(smem_u32(sm_f)), e = lds128(smem_u32(sm_f) + 16);
        const uint32_t mw[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}, fw[8] = {c.x, c.y, c.z, c.w, e.x, e.y, e.z, e.w};
#pragma unroll
        for (int h = 0; h < H; ++h) mb[h] = __uint_as_float(mw[h]);
#pragma unroll
        for (int h = 0; h < H / 2; ++h) {
          x2[h] = f2_mul(x2[h], f2_pack(__uint_as_float(fw[2 * h]), __uint_as_float(fw[2 * h + 1])));
        }
      }
      uint32_t vm = h2_maxabs(vs[0], vs[NB / 2 - 1]);
      const float2 vmf = __half22float2(*reinterpret_cast<const __half2*>(&vm));
      const float vtop = fmaxf(vmf.x, vmf.y);
      need = vtop > vlim;
#pragma unroll
      for (int h = 0; h < H / 2; ++h) {
        float x, y;
        f2_unpack(x2[h], x, y);
        need = need || x + mb[2 * h] > kWeightExp + kSlack || y + mb[2 * h + 1] > kWeightExp + kSlack;
      }
      if (__syncthreads_or(need ? 1 : 0)) {
        // the largest score of each head and the largest V scale over the stage
        float mx[H + 1];
#pragma unroll
        for (int h = 0; h < H / 2; ++h) f2_unpack(x2[h], mx[2 * h], mx[2 * h + 1]);
        mx[H] = vtop;
#pragma unroll
        for (int h = 0; h <= H; ++h) {
#pragma unroll
          for (int off = 16; off > 0; off >>= 1) mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], off));
          if (lane == 0) sm_red[warp * (H + 1) + h] = mx[h];
        }
        __syncthreads();
        float vx = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) vx = fmaxf(vx, sm_red[i * (H + 1) + H]);
        float beta = 1.f;
        if (vx > vlim) {
          const int e = min(exponent_of(vx), 15);
          const int k = min(max(-1 - e, -16), 15);  // |V scale| 2^k in [0.5, 1) now, at most 2 until it moves again
          beta = vlim > 0.f ? pow2i(k - vexp) : 1.f;
          vexp = k;
          vlim = pow2i(e + 2);
          const __half2 m = __float2half2_rn(pow2i(k) * v_div);
          vmul = *reinterpret_cast<const uint32_t*>(&m);
        }
#pragma unroll
        for (int h = 0; h < H; ++h) {
          float top = -INFINITY;
#pragma unroll
          for (int i = 0; i < 4; ++i) top = fmaxf(top, sm_red[i * (H + 1) + h]);
          float alpha = 1.f;
          if (top + mb[h] > kWeightExp + kSlack) {
            alpha = ex2(kWeightExp - top - mb[h]);  // 0 from the first reference (mb = +inf)
            mb[h] = kWeightExp - top;
          }
          o[h] *= alpha * beta;
          float x, y;
          f2_unpack(l2[h >> 1], x, y);
          if (h & 1) y *= alpha; else x *= alpha;
          l2[h >> 1] = f2_pack(x, y);
        }
        __syncthreads();  // every thread has read the old references
        if (tid == 0) {
#pragma unroll
          for (int h = 0; h < H; ++h) sm_mb[h] = mb[h];
        }
      }

      // weights, and their products with the token's V scales as f16 hi + lo
      uint32_t ph[H / 2], pl[H / 2];
#pragma unroll
      for (int h = 0; h < H / 2; ++h) {
        float x, y;
        f2_unpack(f2_add(x2[h], f2_pack(mb[2 * h], mb[2 * h + 1])), x, y);
        const float p0 = ex2(x), p1 = ex2(y);
        l2[h] = f2_add(l2[h], f2_pack(p0, p1));
        const __half2 a = __floats2half2_rn(p0, p1);
        const float2 af = __half22float2(a);
        ph[h] = *reinterpret_cast<const uint32_t*>(&a);
        pl[h] = pack_half2(p0 - af.x, p1 - af.y);
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const uint32_t d2 = h2_mul(vs[b >> 1], vmul);
        const uint32_t d = prmt(d2, d2, (b & 1) ? 0x3232 : 0x1010);
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          hi[h] = h2_mul(ph[h], d);
          lo[h] = h2_fma(pl[h], d, h2_fms(ph[h], d, hi[h]));
        }
        sts128(p_addr + (((p_chunk + 2 * b) ^ (prow & 7)) * 16), hi[0], hi[1], hi[2], hi[3]);
        sts128(p_addr + (((p_chunk + 2 * b + 1) ^ (prow & 7)) * 16), lo[0], lo[1], lo[2], lo[3]);
      }
      fence_proxy_async_shared();
      tmem_wait_st();
      tc_fence_before();
      __syncthreads();
      if (tid == 0) {
        tc_fence_after();
        constexpr uint32_t idesc = idesc_f16_f32(128, 64, false, true);
#pragma unroll
        for (int k = 0; k < D::kPRows / 16; ++k) {
          const uint64_t b = smem_desc_sw128(smem_u32(ps) + k * 2048, 8192, 1024);
          umma_ts(tmem + D::kColD, tmem + D::kColA + k * 8, b, idesc, k > 0);
        }
        umma_commit(done2);
        if (!sm_flag[2]) feed_issue<HD>(p, feed, stage, &full[slot]);  // every read of the slot is behind the barrier
      }
      open = true;
      if (++slot == D::kRing) {
        slot = 0;
        phase ^= 1u;
      }
    }
    if (open) take_o();

    // sums of the weights over the threads
    float l[H];
#pragma unroll
    for (int h = 0; h < H / 2; ++h) f2_unpack(l2[h], l[2 * h], l[2 * h + 1]);
#pragma unroll
    for (int h = 0; h < H; ++h) {
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], off);
    }
    if (lane == 0) {
#pragma unroll
      for (int h = 0; h < H; ++h) sm_red[warp * (H + 1) + h] = l[h];
    }
    const float vs = pow2i(-vexp);
    if constexpr (HD == 64) {  // the two units' halves of each dim
      float* half = reinterpret_cast<float*>(ps);  // the second product has been taken
      if (unit == 1) {
#pragma unroll
        for (int h = 0; h < H; ++h) half[h * 64 + row] = o[h];
      }
      __syncthreads();
      if (unit == 0) {
#pragma unroll
        for (int h = 0; h < H; ++h) o[h] += half[h * 64 + row];
      }
    } else {
      __syncthreads();
    }
    const size_t out_row = ((size_t)s.ll * p.seq_total + p.seq_base + s.si) * (p.pool.kv_heads * p.group) +
                           s.kvh * p.group + s.hb * p.block_heads;
    const int heads = min(p.block_heads, p.group - s.hb * p.block_heads);
    const bool dim_mine = HD == 128 || unit == 0;
    const int dim = HD == 128 ? tid : row;
    // a CTA's first segment uses its slot 0, its last another one: at most two of its segments are parts of groups
    float* mine = p.partials + ((size_t)blockIdx.x * 2 + (aligned || s.gb + s.s0 == u_begin ? 0 : 1)) * rec;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const float sum = (sm_red[h] + sm_red[(H + 1) + h]) + (sm_red[2 * (H + 1) + h] + sm_red[3 * (H + 1) + h]);
      const float acc = o[h] * vs;
      const float m = kWeightExp - sm_mb[h];
      if (s.parts > 1) {
        if (dim_mine) mine[h * HD + dim] = acc;
        if (tid == 0) {
          mine[H * HD + h] = m;
          mine[H * HD + H + h] = sum;
        }
      } else if (h < heads && dim_mine) {
        if (p.partial_out) {
          constexpr float k = 0x1p-11f;  // 2^-kWeightExp
          float* dst = p.out + (out_row + h) * (HD + 2);
          dst[dim] = acc * k;
          if (dim == 0) {
            dst[HD] = m;
            dst[HD + 1] = sum * k;
          }
        } else {
          p.out[(out_row + h) * HD + dim] = sum == 0.f ? 0.f : acc / sum;  // no token at all: zeros
        }
      }
    }
    if (s.parts > 1) {
      if (tid == 0) pending[n_pending] = s;
      ++n_pending;
    }
    __syncthreads();  // the reduction buffers are free again
    if (!more) break;
    s = nx;
  }

  // Groups shared with other CTAs: the last of a group's CTAs to arrive folds its records, in part order.
  if (n_pending > 0) {
    if (tid == 0) {
      __threadfence();
      for (int i = 0; i < n_pending; ++i) {
        const Seg& q = pending[i];
        sm_flag[i] = atomicAdd(&p.counters[q.group_id], 1u) == (uint32_t)q.parts - 1u;
      }
      __threadfence();
    }
    __syncthreads();
    for (int i = 0; i < n_pending; ++i) {
      if (sm_flag[i] == 0) continue;
      const Seg& q = pending[i];
      // part k is CTA c0 + k's: its first segment unless (stream split) its range began before the group
      auto rec_of = [&](int k) {
        const int c = q.c0 + k;
        const int sl = aligned || stage_start(c, p.total_stages, p.grid) >= q.gb ? 0 : 1;
        return p.partials + ((size_t)c * 2 + sl) * rec;
      };
      float* wt = reinterpret_cast<float*>(ring);  // [parts][8] m, then weights; [parts][8] l (no copy in flight now)
      float* tot = sm_red;                         // [8] sums, [8] reference exponents
      __syncthreads();
      for (int j = tid; j < q.parts * 2 * H; j += 128) {
        const int k = j / (2 * H), e = j - k * 2 * H;
        wt[(e < H ? 0 : q.parts * H) + k * H + (e & 7)] = __ldcg(rec_of(k) + H * HD + e);
      }
      __syncthreads();
      if (tid < H) {
        float all = -INFINITY, sum = 0.f;
        for (int k = 0; k < q.parts; ++k) all = fmaxf(all, wt[k * H + tid]);
        for (int k = 0; k < q.parts; ++k) {
          const float m = wt[k * H + tid];
          const float e = m == -INFINITY ? 0.f : ex2(m - all);
          wt[k * H + tid] = e;
          sum = fmaf(e, wt[(q.parts + k) * H + tid], sum);
        }
        tot[tid] = sum;
        tot[H + tid] = all;
      }
      __syncthreads();
      const size_t out_row = ((size_t)q.ll * p.seq_total + p.seq_base + q.si) * (p.pool.kv_heads * p.group) +
                             q.kvh * p.group + q.hb * p.block_heads;
      const int heads = min(p.block_heads, p.group - q.hb * p.block_heads);
      constexpr int kPer = HD / 16;  // heads of a thread: all 8, or 4 at head_dim 64
      const int h0 = HD == 128 ? 0 : unit * 4, dim = HD == 128 ? tid : row;
      float acc[kPer];
#pragma unroll
      for (int h = 0; h < kPer; ++h) acc[h] = 0.f;
#pragma unroll 4
      for (int k = 0; k < q.parts; ++k) {
        const float* r = rec_of(k);
#pragma unroll
        for (int h = 0; h < kPer; ++h) acc[h] = fmaf(wt[k * H + h0 + h], __ldcg(r + (h0 + h) * HD + dim), acc[h]);
      }
#pragma unroll
      for (int h = 0; h < kPer; ++h) {
        if (h0 + h >= heads) continue;
        const float sum = tot[h0 + h];
        if (p.partial_out) {
          constexpr float k = 0x1p-11f;
          float* dst = p.out + (out_row + h0 + h) * (HD + 2);
          dst[dim] = acc[h] * k;
          if (dim == 0) {
            dst[HD] = tot[H + h0 + h];
            dst[HD + 1] = sum * k;
          }
        } else {
          p.out[(out_row + h0 + h) * HD + dim] = sum == 0.f ? 0.f : acc[h] / sum;
        }
      }
      if (tid == 0) p.counters[q.group_id] = 0;
    }
  }
  __syncthreads();
  if (sm_flag[2]) {
    // a wait ran out: copies and products may still be in flight; let them land before the CTA leaves
    for (int i = 0; i < D::kRing; ++i) (void)mbar_wait(&full[i], phase ^ (i < slot ? 1u : 0u));
    (void)mbar_wait(done1, phase1);
    (void)mbar_wait(done2, phase2);
    __syncthreads();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 128);
  }
}

template <int HD>
cudaError_t launch_decode_t(const Kv4DecodeParams& p, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  cudaError_t e = set_smem_limit_once(done, reinterpret_cast<const void*>(kv4_decode_kernel<HD>), Dec<HD>::smem);
  if (e != cudaSuccess) return e;
  // Programmatic dependent launch: the CTAs set up their barriers and TMEM while the previous kernel drains, and
  // wait for it before touching global memory.
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)p.grid);
  cfg.blockDim = dim3(Dec<HD>::kThreads);
  cfg.dynamicSmemBytes = Dec<HD>::smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv4_decode_kernel<HD>, p);
}

// Work items of the append and read kernels: (layer, kv head, 32 tokens).
long long half_items(const Kv4RowsParams& p) {
  return (long long)((p.first + p.n_tokens - 1) / 32 - p.first / 32 + 1) * p.pool.kv_heads * p.n_layers;
}

}  // namespace

int kv4_decode_ctas_per_sm(int) { return KV4_CTAS; }

void plan_kv4_decode(Kv4DecodeParams& p, long long slots) {
  const int extra = p.k_new ? 1 : 0;
  const long long reps = (long long)p.n_layers * p.pool.kv_heads * p.head_blocks;
  int acc = 0, longest = 1;
  for (int i = 0; i < p.n_seqs; ++i) {
    const int n = kv4_stages(p.seqs[i].len + extra);
    p.seqs[i].stage_begin = acc;
    acc += n;
    longest = n > longest ? n : longest;
  }
  p.block_stages = acc;
  p.total_stages = reps * acc;
  // Aligned split: every group in equal parts of at most `most` stages, one part a CTA, all resident at once.
  auto parts_for = [&](int most) {
    long long c = 0;
    for (int i = 0; i < p.n_seqs; ++i) c += (kv4_stages(p.seqs[i].len + extra) + most - 1) / most;
    return c * reps;
  };
  const long long ideal = (p.total_stages + slots - 1) / slots;
  int lo = 1, hi = longest;
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (parts_for(mid) <= slots) hi = mid; else lo = mid + 1;
  }
  if (lo < 2 && longest >= 2) lo = 2;
  if (parts_for(lo) <= slots && lo <= ideal + ideal / 8 + 1) {
    int parts = 0;
    for (int i = 0; i < p.n_seqs; ++i) {
      p.seqs[i].part_begin = parts;
      parts += (kv4_stages(p.seqs[i].len + extra) + lo - 1) / lo;
    }
    p.block_parts = parts;
    p.grid = (int32_t)(reps * parts);
    return;
  }
  p.block_parts = 0;
  p.grid = (int32_t)(p.total_stages < slots ? p.total_stages : slots);
}

cudaError_t launch_kv4_decode(const Kv4DecodeParams& p, int head_dim, cudaStream_t s) {
  return head_dim == 128 ? launch_decode_t<128>(p, s) : launch_decode_t<64>(p, s);
}

cudaError_t launch_kv4_append(const Kv4RowsParams& p, int head_dim, cudaStream_t s) {
  const unsigned grid = (unsigned)half_items(p);
  if (head_dim == 128) kv4_append_kernel<128><<<grid, 128, 0, s>>>(p);
  else kv4_append_kernel<64><<<grid, 128, 0, s>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_kv4_read(const Kv4RowsParams& p, int head_dim, cudaStream_t s) {
  const unsigned grid = (unsigned)half_items(p);
  if (head_dim == 128) kv4_read_kernel<128><<<grid, 128, 0, s>>>(p);
  else kv4_read_kernel<64><<<grid, 128, 0, s>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_kv4_raw(const Kv4RowsParams& p, int head_dim, bool to_pool, cudaStream_t s) {
  const long long groups = (p.first + p.n_tokens - 1) / 8 - p.first / 8 + 1;
  const long long n = groups * p.n_layers * p.pool.kv_heads * (head_dim / 32);
  const unsigned grid = (unsigned)((n + 127) / 128);
  if (head_dim == 128) kv4_raw_kernel<128><<<grid, 128, 0, s>>>(p, to_pool ? 1 : 0);
  else kv4_raw_kernel<64><<<grid, 128, 0, s>>>(p, to_pool ? 1 : 0);
  return cudaGetLastError();
}

}  // namespace te
