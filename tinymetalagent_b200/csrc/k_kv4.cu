// Kernels of the 4-bit KV cache (layout: te_kv4.h): the quantising append,
// the read-back, the raw Q4_0 import/export, and the decode attention that
// consumes the codes on the tensor cores without widening the cache.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <type_traits>

#include "te_internal.h"
#include "te_kv4.h"
#include "te_ptx.cuh"
#include "te_rope.cuh"

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

// Bits of 4 consecutive codes in their K word (dims 8t + 4h .. + 3, h the half
// of the word's 8 dims) and in their V halfword.
__device__ __forceinline__ uint32_t k_bits(const uint32_t (&c)[4], int h) {
  return (c[0] | c[1] << 16 | c[2] << 4 | c[3] << 20) << (8 * h);
}
__device__ __forceinline__ uint32_t v_bits(const uint32_t (&c)[4]) {
  return c[0] | c[1] << 4 | c[2] << 8 | c[3] << 12;
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

// Quantises the row and writes its codes and scales at token slot `tok` of the
// tile at `tile` (shared or global memory).  The whole warp calls it.  On
// return k and v hold the values the codes stand for.
template <int HD>
__device__ __forceinline__ void store_row(unsigned char* tile, int tok, int lane, float (&k)[4], float (&v)[4]) {
  constexpr int CB = kv4_code_bytes(HD), SB = kv4_scale_bytes(HD);
  using R = RowDims<HD>;
  const int j = tok >> 3, g = tok & 7, tp = (tok & 7) >> 1, e = tok & 1;
  const int dim = R::dim(lane), b = dim >> 5;
  auto put_k = [&](const uint32_t(&c)[4], __half d) {
    uint32_t w = k_bits(c, lane & 1);
    w |= __shfl_xor_sync(0xffffffffu, w, 1);
    if (R::has_k(lane)) {
      if ((lane & 1) == 0) {
        *reinterpret_cast<uint32_t*>(tile + kv4_word_at(HD, j, 4 * g + ((dim & 31) >> 3), b)) = w;
      }
      if ((lane & 7) == 0) {
        *reinterpret_cast<__half*>(tile + 2 * CB + kv4_scale_at(HD, j, tp, b, e)) = d;
      }
    }
  };
  auto put_v = [&](const uint32_t(&c)[4], __half d) {
    if (R::has_v(lane)) {
      *reinterpret_cast<uint16_t*>(tile + CB + kv4_word_at(HD, j, 4 * ((dim & 31) >> 2) + tp, b) + 2 * e) =
          (uint16_t)v_bits(c);
      if ((lane & 7) == 0) {
        *reinterpret_cast<__half*>(tile + 2 * CB + SB + kv4_scale_at(HD, j, tp, b, e)) = d;
      }
    }
  };
  uint32_t c[4];
  __half d;
  if constexpr (HD == 128) {
    q4_quantise(k, lane, c, d);
    put_k(c, d);
#pragma unroll
    for (int i = 0; i < 4; ++i) k[i] = q4_value(c[i], __half2float(d));
    q4_quantise(v, lane, c, d);
    put_v(c, d);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = q4_value(c[i], __half2float(d));
  } else {
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = R::has_k(lane) ? k[i] : v[i];
    q4_quantise(x, lane, c, d);
    put_k(c, d);
    put_v(c, d);
#pragma unroll
    for (int i = 0; i < 4; ++i) k[i] = v[i] = q4_value(c[i], __half2float(d));
  }
}

// A token's raw key and value rows at element offset `at`, with bias and RoPE.
template <int HD>
__device__ __forceinline__ void load_row(const void* kp, const void* vp, size_t at, int f16, const float* kb,
                                         const float* vb, const float* cr, const float* sr, int lane, float (&k)[4],
                                         float (&v)[4]) {
  using R = RowDims<HD>;
  const int dim = R::dim(lane);
#pragma unroll
  for (int i = 0; i < 4; ++i) k[i] = v[i] = 0.f;
  if (R::has_k(lane)) load4(kp, at + dim, f16, k);
  if (R::has_v(lane)) load4(vp, at + dim, f16, v);
  if (kb) {
    if (R::has_k(lane)) add_bias4(k, kb + dim);
    if (R::has_v(lane)) add_bias4(v, vb + dim);
  }
  if (cr) rope4<HD>(k, cr, sr, lane);
}

// Quotient of a tile index by tiles_per_page: the product with the rounded-up
// reciprocal is at most one too large (its excess is below t / 2^32 < 1).
__device__ __forceinline__ int kv4_page_of(const Kv4Pool& p, int tile) {
  int q = (int)__umulhi((uint32_t)tile, p.tpp_magic);
  if (q * p.tiles_per_page > tile) --q;
  return q;
}

__device__ __forceinline__ unsigned char* tile_ptr(const Kv4Pool& p, const int32_t* page_row, int layer, int kvh,
                                                   int tile, int tile_bytes) {
  const int page = kv4_page_of(p, tile);
  const int in = tile - page * p.tiles_per_page;
  const long long rec = ((long long)layer * p.num_pages + page_row[page]) * p.kv_heads + kvh;
  return p.base + (rec * p.tiles_per_page + in) * tile_bytes;
}

// ---- append -------------------------------------------------------------------

constexpr int kRowWarps = 4;

__device__ __forceinline__ float fmax3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float fmin3_nan(float a, float b, float c) {
  float d;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// One block in one thread: x becomes c - 8 (fp32), the result is d; q4_quantise's values, without its shuffles.
//
// The quotients are correctly rounded by Markstein's step: with y = RN(1 / d), q = RN(x y) and r = x - q d (exact
// in an fma), RN(q + r y) is RN(x / d); two values at a time that is three packed operations a pair, where a
// division is some ten instructions a value.  Adding 1.5 2^23 rounds to an integer, half to even.
__device__ __forceinline__ __half q4_quantise32(float (&x)[32]) {
  float mx = x[0], mn = x[0];
#pragma unroll
  for (int i = 1; i + 1 < 32; i += 2) {
    mx = fmax3_nan(mx, x[i], x[i + 1]);
    mn = fmin3_nan(mn, x[i], x[i + 1]);
  }
  mx = fmax3_nan(mx, x[31], x[31]);
  mn = fmin3_nan(mn, x[31], x[31]);
  float m = mx > -mn ? mx : mn;
  if (mx == -mn) {  // both signs reach the largest magnitude (or all are zero): the lowest index decides
    m = x[31];
#pragma unroll
    for (int i = 30; i >= 0; --i) {
      if (fabsf(x[i]) == mx) m = x[i];
    }
  }
  const bool finite = mx < INFINITY && mn > -INFINITY;  // false for NaN too
  const __half d =
      finite ? __float2half_rn(fminf(fmaxf(m * -0.125f, -65504.f), 65504.f)) : __ushort_as_half((unsigned short)0x7fff);
  const float df = __half2float(d);
  if (!finite || df == 0.f) {
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = 0.f;
    return d;
  }
  if (fabsf(df) < 0x1p-14f || fabsf(df) == 65504.f) {
    // subnormal or saturated: quotients may lie far outside the codes' range
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = fminf(fmaxf(rintf(__fdiv_rn(x[i], df)), -8.f), 7.f);
    return d;
  }
  // d is within 2^-11 of m / -8: every quotient rounds to -8 .. 8
  const float inv = __frcp_rn(df);
  const uint64_t inv2 = f2_pack(inv, inv), neg2 = f2_pack(-df, -df);
  constexpr float kMagic = 12582912.f;
  const uint64_t magic2 = f2_pack(kMagic, kMagic);
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    const uint64_t v = f2_pack(x[i], x[i + 1]);
    const uint64_t q = f2_mul(v, inv2);
    const uint64_t r = f2_fma(q, neg2, v);
    float a, b;
    f2_unpack(f2_sub(f2_add(f2_fma(r, inv2, q), magic2), magic2), a, b);
    x[i] = fminf(a, 7.f);  // 8 where x is as large as m and of the other sign
    x[i + 1] = fminf(b, 7.f);
  }
  return d;
}

// Four codes as the low 16 bits of an fp32 number, from c - 8 in fp32: 2^23 + sum 16^i (c_i - 8 + 8) is exact.
constexpr float kNibbles = 8388608.f + 0x8888;
__device__ __forceinline__ uint32_t q4_half(float a, float b, float c, float d) {
  return __float_as_uint(fmaf(d, 4096.f, fmaf(c, 256.f, fmaf(b, 16.f, a + kNibbles))));
}
// The K word of dims x[i0] .. x[i0 + 7]: even dims in its low half, odd ones in its high half.
__device__ __forceinline__ uint32_t q4_word(const float (&x)[32], int i0) {
  uint64_t v = f2_add(f2_pack(x[i0], x[i0 + 1]), f2_pack(kNibbles, kNibbles));
  v = f2_fma(f2_pack(x[i0 + 2], x[i0 + 3]), f2_pack(16.f, 16.f), v);
  v = f2_fma(f2_pack(x[i0 + 4], x[i0 + 5]), f2_pack(256.f, 256.f), v);
  v = f2_fma(f2_pack(x[i0 + 6], x[i0 + 7]), f2_pack(4096.f, 4096.f), v);
  float lo, hi;
  f2_unpack(v, lo, hi);
  return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x5410);
}

// 32 consecutive values of a binary16 (64 bytes) or fp32 (128 bytes) row, as read and as fp32.
template <bool F16>
__device__ __forceinline__ void widen32(const uint4 (&u)[F16 ? 4 : 8], float (&x)[32]) {
  if constexpr (F16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float v[8];
      unpack8(u[i], v);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[8 * i + e] = v[e];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[4 * i] = __uint_as_float(u[i].x);
      x[4 * i + 1] = __uint_as_float(u[i].y);
      x[4 * i + 2] = __uint_as_float(u[i].z);
      x[4 * i + 3] = __uint_as_float(u[i].w);
    }
  }
}
// Byte of piece i % C of block i / C in a step's rows: C pieces of 16 bytes a block, swizzled so that neither a warp's 32
// consecutive pieces nor the pieces of the same number of its 32 blocks meet in a bank.
template <int C>
__device__ __forceinline__ int row_piece(int i) {
  const int l = i / C;
  return (l * C + ((i % C) ^ (C == 4 ? (l >> 1) & 3 : l & 7))) * 16;
}
// The lane's block into a step's rows.
template <bool F16>
__device__ __forceinline__ void put32(unsigned char* buf, int lane, const float (&x)[32]) {
  constexpr int C = F16 ? 4 : 8;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    uint4 u;
    if constexpr (F16) {
      u = make_uint4(pack_half2(x[8 * i], x[8 * i + 1]), pack_half2(x[8 * i + 2], x[8 * i + 3]),
                     pack_half2(x[8 * i + 4], x[8 * i + 5]), pack_half2(x[8 * i + 6], x[8 * i + 7]));
    } else {
      u = make_uint4(__float_as_uint(x[4 * i]), __float_as_uint(x[4 * i + 1]), __float_as_uint(x[4 * i + 2]),
                     __float_as_uint(x[4 * i + 3]));
    }
    *reinterpret_cast<uint4*>(buf + row_piece<C>(lane * C + i)) = u;
  }
}
// An fp32 block straight to memory.
__device__ __forceinline__ void store32(void* base, size_t idx, const float (&x)[32]) {
  float4* p = reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + idx);
#pragma unroll
  for (int i = 0; i < 8; ++i) p[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
}

// One warp per (layer, kv head, tile of 16 tokens), one block a lane: the tile is assembled in shared memory (with
// the tokens it already holds, if the new ones do not fill it) and written whole.  Rows come in, and stored rows go
// out, through shared memory, so that a warp's accesses are whole rows while a lane's work is a block.
//
// Bound by bytes: 36 layers x 2048 tokens x 2 kv heads x 128 values, stored rows returned in the same type, take
// 33 to 35 us as binary16 (172 MB, 5.0 TB/s, 0.76 of a copy's rate; a seventh is ramp and tail) and 52.4 us as fp32
// (323 MB, 6.2 TB/s); at 64 dims 18.9 and 27.5 us.  Eight lanes a block with a division a value took 80 us for the
// first, a block a lane with Markstein's step 39, each lane reading its own block one step ahead 34.7 (fp32: 85.0,
// 64 dims 20.6 and 44.8), codes joined in the FMA pipe 34.2.  Four CTAs an SM: held to the registers of five or six,
// the values spill (37 to 43 us; at four, fp32 rows of 64 dims spill five words).  A single token (24 layers) is a
// launch: 2 us on the device.
template <int HD, bool F16>
__global__ void __launch_bounds__(32 * kRowWarps, 4) kv4_append_kernel(const Kv4RowsParams p) {
  constexpr int TB = kv4_tile_bytes(HD), CB = kv4_code_bytes(HD), SB = kv4_scale_bytes(HD), NB = HD / 32;
  constexpr int kTokens = 32 / NB;  // tokens of a warp's step
  // rows come in by asynchronous copies of 16-byte pieces, whole rows at a time, kBufs steps ahead
  constexpr int kChunks = F16 ? 4 : 8, kStepBytes = 32 * 16 * kChunks, kBufs = F16 ? 4 : 2;
  __shared__ __align__(16) unsigned char tiles[kRowWarps][TB];
  __shared__ __align__(16) unsigned char bufs[kRowWarps][kBufs][kStepBytes];
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t0 = p.first / kKv4Tile;
  const uint32_t n_tiles = (uint32_t)((p.first + p.n_tokens - 1) / kKv4Tile - t0 + 1);
  const uint32_t item = blockIdx.x * kRowWarps + warp;
  const uint32_t r = item / (uint32_t)p.pool.kv_heads;
  const int kvh = (int)(item - r * (uint32_t)p.pool.kv_heads);
  const int ll = (int)(r / n_tiles);
  const int tile = t0 + (int)(r - (uint32_t)ll * n_tiles);
  if (ll >= p.n_layers) return;
  const int layer = p.layer_begin + ll;
  unsigned char* dst = tile_ptr(p.pool, p.page_row, layer, kvh, tile, TB);
  unsigned char* sm = tiles[warp];
  const int lo = max(p.first - tile * kKv4Tile, 0);
  const int hi = min(p.first + p.n_tokens - tile * kKv4Tile, kKv4Tile);
  if (lo > 0 || hi < kKv4Tile) {
    for (int i = lane * 16; i < TB; i += 512) {
      *reinterpret_cast<uint4*>(sm + i) = *reinterpret_cast<const uint4*>(dst + i);
    }
    __syncwarp();
  }
  const int b = lane % NB;
  const size_t brow = ((size_t)layer * p.pool.kv_heads + kvh) * HD + 32 * b;
  constexpr int kSteps = 2 * kKv4Tile / kTokens;
  // the pieces of a step's rows that this lane copies in or out, C to a block: calls f(its byte in the buffer, token
  // row, byte from the head's first value)
  auto pieces = [&](auto chunks, int step, auto f) {
    constexpr int C = chunks;
#pragma unroll
    for (int n = 0; n < C; ++n) {
      const int i = n * 32 + lane, slot = (step % (kSteps / 2)) * kTokens + i / (NB * C);
      if (slot >= lo && slot < hi) {
        f(row_piece<C>(i), (long long)ll * p.n_tokens + (tile * kKv4Tile + slot - p.first), i % (NB * C) * 16);
      }
    }
  };
  using In = std::integral_constant<int, kChunks>;
  constexpr int kEl = F16 ? 2 : 4;
  auto fetch = [&](int step) {
    if (step < kSteps) {
      const unsigned char* src = static_cast<const unsigned char*>(step >= kSteps / 2 ? p.v : p.k);
      unsigned char* buf = bufs[warp][step % kBufs];
      pieces(In(), step, [&](int at, long long row, int byte) {
        cp_async_cg16(smem_u32(buf + at), src + (row * p.token_stride + (long long)kvh * HD) * kEl + byte);
      });
    }
    cp_async_commit();
  };
  // returned rows leave through the step's buffer too, unless they are larger than what came in
  const bool buffered = p.k_rows && (p.rows_f16 || !F16);
#pragma unroll
  for (int i = 0; i < kBufs; ++i) fetch(i);
#pragma unroll 1
  for (int step = 0; step < kSteps; ++step) {
    const bool value = step >= kSteps / 2;
    const int slot = (step % (kSteps / 2)) * kTokens + lane / NB;  // token of the tile
    const bool in = slot >= lo && slot < hi;
    const int tok = tile * kKv4Tile + slot - p.first;  // index among the new tokens
    if (__all_sync(0xffffffffu, !in)) {
      fetch(step + kBufs);
      continue;
    }
    unsigned char* buf = bufs[warp][step % kBufs];
    cp_async_wait<kBufs - 1>();
    __syncwarp();
    float x[32];
    if (in) {
      uint4 raw[kChunks];
#pragma unroll
      for (int i = 0; i < kChunks; ++i) raw[i] = *reinterpret_cast<const uint4*>(buf + row_piece<kChunks>(lane * kChunks + i));
      widen32<F16>(raw, x);
      if (p.k_bias) {
        const float* br = (value ? p.v_bias : p.k_bias) + brow;
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 v = *reinterpret_cast<const float4*>(br + i);
          x[i] = __fadd_rn(x[i], v.x);
          x[i + 1] = __fadd_rn(x[i + 1], v.y);
          x[i + 2] = __fadd_rn(x[i + 2], v.z);
          x[i + 3] = __fadd_rn(x[i + 3], v.w);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) x[i] = 0.f;
    }
    if (!value && p.rope) {  // the partner dims are another lane's block of the same token
      const size_t at = (size_t)(p.first_pos + (in ? tok : 0)) * (HD / 2) + 32 * (b % (NB / 2));
      const bool upper = b >= NB / 2;
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        const float4 c = *reinterpret_cast<const float4*>(p.rope_cos + at + i);
        const float4 s = *reinterpret_cast<const float4*>(p.rope_sin + at + i);
        const float cv[4] = {c.x, c.y, c.z, c.w}, sv[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float o = __shfl_xor_sync(0xffffffffu, x[i + e], NB / 2);
          x[i + e] = upper ? rope_hi(o, x[i + e], cv[e], sv[e]) : rope_lo(x[i + e], o, cv[e], sv[e]);
        }
      }
    }
    __syncwarp();  // every lane has read its block
    if (in) {
      const __half d = q4_quantise32(x);
      const int j = slot >> 3, g = slot & 7;
      if (!value) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          *reinterpret_cast<uint32_t*>(sm + kv4_word_at(HD, j, 4 * g + t, b)) = q4_word(x, 8 * t);
        }
        *reinterpret_cast<__half*>(sm + 2 * CB + kv4_scale_at(HD, j, g >> 1, b, g & 1)) = d;
      } else {
#pragma unroll
        for (int gg = 0; gg < 8; ++gg) {
          *reinterpret_cast<uint16_t*>(sm + CB + kv4_word_at(HD, j, 4 * gg + (g >> 1), b) + 2 * (g & 1)) =
              (uint16_t)q4_half(x[4 * gg], x[4 * gg + 1], x[4 * gg + 2], x[4 * gg + 3]);
        }
        *reinterpret_cast<__half*>(sm + 2 * CB + SB + kv4_scale_at(HD, j, g >> 1, b, g & 1)) = d;
      }
      if (p.k_rows) {
        const float df = __half2float(d);
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] *= df;
        if (buffered) {
          if (F16 || p.rows_f16) put32<true>(buf, lane, x); else put32<false>(buf, lane, x);
        } else {
          store32(value ? p.v_rows : p.k_rows, (((size_t)ll * p.n_tokens + tok) * p.pool.kv_heads + kvh) * HD + 32 * b, x);
        }
      }
    }
    if (buffered) {
      __syncwarp();
      auto leave = [&](auto chunks) {
        unsigned char* out = static_cast<unsigned char*>(value ? p.v_rows : p.k_rows);
        pieces(chunks, step, [&](int at, long long row, int byte) {
          *reinterpret_cast<uint4*>(out + (row * p.pool.kv_heads + kvh) * (HD / 2) * chunks() + byte) =
              *reinterpret_cast<const uint4*>(buf + at);
        });
      };
      if (F16 || p.rows_f16) leave(std::integral_constant<int, 4>()); else leave(In());
    }
    __syncwarp();
    fetch(step + kBufs);
  }
  __syncwarp();
  for (int i = lane * 16; i < TB; i += 512) {
    *reinterpret_cast<uint4*>(dst + i) = *reinterpret_cast<const uint4*>(sm + i);
  }
}

// ---- read ---------------------------------------------------------------------

// One warp per (layer, kv head, tile): lane 4g + t expands its K words (dims 8t.. of token g) and V words (dims
// 4g.. of tokens 2t, 2t + 1), read 16 bytes at a time; a row's pieces leave as whole 32-byte sectors.
//
// Bound by the rows it writes: 28 layers x 16384 tokens x 4 kv heads x 128 values as binary16, 1.2 GB in all, take
// 186 to 192 us (6.3 to 6.5 TB/s, a plain copy's rate); 29 MB of odd range as fp32 6.7 us.  Read a word at a time where it
// was needed, the large case took 228 us.
template <int HD>
__global__ void __launch_bounds__(32 * kRowWarps) kv4_read_kernel(const Kv4RowsParams p) {
  constexpr int TB = kv4_tile_bytes(HD), CB = kv4_code_bytes(HD), SB = kv4_scale_bytes(HD), NB = HD / 32;
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int t0 = p.first / kKv4Tile;
  const uint32_t n_tiles = (uint32_t)((p.first + p.n_tokens - 1) / kKv4Tile - t0 + 1);
  const uint32_t item = blockIdx.x * kRowWarps + warp;
  const uint32_t r = item / (uint32_t)p.pool.kv_heads;
  const int kvh = (int)(item - r * (uint32_t)p.pool.kv_heads);
  const int ll = (int)(r / n_tiles);
  const int tile = t0 + (int)(r - (uint32_t)ll * n_tiles);
  if (ll >= p.n_layers) return;
  const unsigned char* src = tile_ptr(p.pool, p.page_row, p.layer_begin + ll, kvh, tile, TB);
  auto row_of = [&](int tok) -> long long {  // element offset of tile token tok's row, or -1 outside the range
    const int i = tile * kKv4Tile + tok - p.first;
    return i >= 0 && i < p.n_tokens ? (((long long)ll * p.n_tokens + i) * p.pool.kv_heads + kvh) * HD : -1;
  };
  // every word of the lane, and its tokens' scales
  uint32_t kw[2][NB], vw[2][NB], vs[2][NB];
  uint16_t ks[2][NB];
  auto words = [&](int at, int stride, int who, uint32_t(&w)[2][NB]) {
    if constexpr (HD == 128) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint4 v = *reinterpret_cast<const uint4*>(src + at + j * stride + who * 16);
        w[j][0] = v.x; w[j][1] = v.y; w[j][2] = v.z; w[j][3] = v.w;
      }
    } else {
      const uint4 v = *reinterpret_cast<const uint4*>(src + at + who * 16);
      w[0][0] = v.x; w[0][1] = v.y; w[1][0] = v.z; w[1][1] = v.w;
    }
  };
  words(0, 512, lane, kw);
  words(CB, 512, lane, vw);
  words(2 * CB + SB, 64, t, vs);
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      ks[j][b] = *reinterpret_cast<const uint16_t*>(src + 2 * CB + kv4_scale_at(HD, j, g >> 1, b, g & 1));
    }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const long long kr = row_of(8 * j + g);
    const long long v0 = row_of(8 * j + 2 * t), v1 = row_of(8 * j + 2 * t + 1);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      if (kr >= 0) {
        const float d = __half2float(__ushort_as_half(ks[j][b]));
        float x[8];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          x[2 * q] = q4_value((kw[j][b] >> (4 * q)) & 15u, d);
          x[2 * q + 1] = q4_value((kw[j][b] >> (4 * q + 16)) & 15u, d);
        }
        const size_t at = (size_t)kr + 32 * b + 8 * t;
        if (p.rows_f16) {
          *reinterpret_cast<uint4*>(reinterpret_cast<__half*>(p.k_rows) + at) = pack8(x);
        } else {
          float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(p.k_rows) + at);
          o[0] = make_float4(x[0], x[1], x[2], x[3]);
          o[1] = make_float4(x[4], x[5], x[6], x[7]);
        }
      }
      const float2 d = __half22float2(*reinterpret_cast<const __half2*>(&vs[j][b]));
      float x[4], y[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        x[q] = q4_value((vw[j][b] >> (4 * q)) & 15u, d.x);
        y[q] = q4_value((vw[j][b] >> (4 * q + 16)) & 15u, d.y);
      }
      if (v0 >= 0) store4(p.v_rows, (size_t)v0 + 32 * b + 4 * g, p.rows_f16, x);
      if (v1 >= 0) store4(p.v_rows, (size_t)v1 + 32 * b + 4 * g, p.rows_f16, y);
    }
  }
}

// ---- raw Q4_0 blocks ------------------------------------------------------------

// One thread per (layer, token, kv head, block): both sides.  A raw block is
// 18 bytes, 2-byte aligned: the scale, then byte i = code i | code (i + 16) << 4.
// For saving and restoring a session; not tuned.
template <int HD>
__global__ void __launch_bounds__(128) kv4_raw_kernel(const Kv4RowsParams p, int to_pool) {
  constexpr int TB = kv4_tile_bytes(HD), CB = kv4_code_bytes(HD), SB = kv4_scale_bytes(HD), NB = HD / 32;
  const long long n = (long long)p.n_layers * p.n_tokens * p.pool.kv_heads * NB;
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int b = (int)(i % NB);
  long long r = i / NB;
  const int kvh = (int)(r % p.pool.kv_heads);
  r /= p.pool.kv_heads;
  const int tok = p.first + (int)(r % p.n_tokens);
  const int layer = p.layer_begin + (int)(r / p.n_tokens);
  unsigned char* tile = tile_ptr(p.pool, p.page_row, layer, kvh, tok / kKv4Tile, TB);
  const int s = tok % kKv4Tile, j = s >> 3, g = s & 7, tp = g >> 1, e = s & 1;
  // code index of the block -> its word (byte offset) and nibble shift
  auto k_word = [&](int t) { return reinterpret_cast<uint32_t*>(tile + kv4_word_at(HD, j, 4 * g + t, b)); };
  auto v_half = [&](int gg) {
    return reinterpret_cast<uint16_t*>(tile + CB + kv4_word_at(HD, j, 4 * gg + tp, b) + 2 * e);
  };
  uint16_t* kd = reinterpret_cast<uint16_t*>(tile + 2 * CB + kv4_scale_at(HD, j, tp, b, e));
  uint16_t* vd = reinterpret_cast<uint16_t*>(tile + 2 * CB + SB + kv4_scale_at(HD, j, tp, b, e));
  if (to_pool) {
    const uint16_t* kr = reinterpret_cast<const uint16_t*>(p.k) + i * 9;
    const uint16_t* vr = reinterpret_cast<const uint16_t*>(p.v) + i * 9;
    uint32_t kc[32], vc[32];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const uint32_t kx = kr[1 + q], vx = vr[1 + q];
      kc[2 * q] = kx & 15u; kc[2 * q + 1] = (kx >> 8) & 15u;
      kc[2 * q + 16] = (kx >> 4) & 15u; kc[2 * q + 17] = kx >> 12;
      vc[2 * q] = vx & 15u; vc[2 * q + 1] = (vx >> 8) & 15u;
      vc[2 * q + 16] = (vx >> 4) & 15u; vc[2 * q + 17] = vx >> 12;
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t a[4] = {kc[8 * t], kc[8 * t + 1], kc[8 * t + 2], kc[8 * t + 3]};
      const uint32_t c[4] = {kc[8 * t + 4], kc[8 * t + 5], kc[8 * t + 6], kc[8 * t + 7]};
      *k_word(t) = k_bits(a, 0) | k_bits(c, 1);
    }
#pragma unroll
    for (int gg = 0; gg < 8; ++gg) {
      const uint32_t a[4] = {vc[4 * gg], vc[4 * gg + 1], vc[4 * gg + 2], vc[4 * gg + 3]};
      *v_half(gg) = (uint16_t)v_bits(a);
    }
    *kd = kr[0];
    *vd = vr[0];
  } else {
    uint16_t* kr = reinterpret_cast<uint16_t*>(p.k_rows) + i * 9;
    uint16_t* vr = reinterpret_cast<uint16_t*>(p.v_rows) + i * 9;
    uint32_t kc[32], vc[32];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t w = *k_word(t);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        kc[8 * t + 2 * q] = (w >> (4 * q)) & 15u;
        kc[8 * t + 2 * q + 1] = (w >> (4 * q + 16)) & 15u;
      }
    }
#pragma unroll
    for (int gg = 0; gg < 8; ++gg) {
      const uint32_t w = *v_half(gg);
#pragma unroll
      for (int q = 0; q < 4; ++q) vc[4 * gg + q] = (w >> (4 * q)) & 15u;
    }
    kr[0] = *kd;
    vr[0] = *vd;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      kr[1 + q] = (uint16_t)(kc[2 * q] | kc[2 * q + 16] << 4 | kc[2 * q + 1] << 8 | kc[2 * q + 17] << 12);
      vr[1 + q] = (uint16_t)(vc[2 * q] | vc[2 * q + 16] << 4 | vc[2 * q + 1] << 8 | vc[2 * q + 17] << 12);
    }
  }
}

// ---- decode attention -------------------------------------------------------------
//
// out = softmax(q K^T / sqrt(hd)) V per query head, over a group's cached
// tokens and the token the call appends.  Both products run on mma.sync
// m16n8k16 with fp32 accumulators, fed with the codes themselves:
//
//   S: A = the group's queries as f16 hi (rows 0-7) and lo (rows 8-15) parts,
//      scaled by a power of two per head; B = K codes minus 8.
//      Per block of 32 dims S += d (A B) in fp32.
//   O^T: A = V codes minus 8, rows = dims; B = P d as f16 hi + lo parts (an
//      error-free product: hi = f16(P d), lo = f16 of the rest): about 22 bits
//      of a product that is not below 2^-14 of the copy's largest.
//
// The C fragment of S holds, in lane 4g + t, head g and tokens 2t, 2t + 1:
// exactly what the B fragment of O^T wants, so the weights never leave their
// registers.  A copy's weights are counted from its own largest score, a power
// of two per head, and its products join O by that power against the head's
// reference, which moves (rescaling O) only when a copy exceeds it by more than
// 2^5.  Counted from the head's reference instead, weights of 2^-17 (beside a
// token that takes nearly all of the weight) had their products with scales
// of 2^-7 on the grid of binary16's subnormals: where that token's values are
// zero the output was 6e-4 off, against less than 1e-5 now, at the same speed
// (147 and 50 to 51 us for the first two lines below, both ways in turn).
//
// Split: a warp streams copies of 64 tokens through a ring of its own, so no
// barrier stands in the loop; the CTA's warps merge at the end of a segment, and a group's CTAs through records that the last of them
// to arrive folds (plan_kv4_decode chooses who takes what).
//
// What bounds it is not the bytes but the conversion of the codes and the
// products they feed: a tile of 16 tokens costs a warp about 327 instructions,
// 32 of them matrix products of 9 clocks, and an SM some 160 clocks with the
// copies taken out, where HBM would deliver one in 99; with the arithmetic
// taken out the same loop streams 5.9 TB/s.  Measured at head_dim 128, 7 or 8
// heads a group:
//   28 layers x 4 kv heads x 32768 tokens  529 MB  135 to 148 us by GPU, 3.6 to 3.9 TB/s (copy rate: 81 us)
//   64 sequences, 8192 tokens at most      153 MB   50 us, 3.0 TB/s (23 us)
//   36 layers x 2 kv heads x 4097 tokens    43 MB   19 us, 2.3 TB/s (6.6 us)
//   24 layers x 2 kv heads x 1000 tokens of 64, appending  12 us (0.6 us: latency)
// Copies with scales outside 2^-14 .. 2 cost a tenth to a sixth more (all of
// them outside: 156 us for the first line where the others take 135).
// Shapes: at head_dim 128, four warps x 2 CTAs with 64 tokens a step and 255
// registers took 136 us for the first line, one CTA of eight warps 142 (58 and
// 19.5 for the next two); when the shape was chosen it took 138, 16 warps with
// 32 tokens 147 (12 warps 147 too), 20 and 24 warps with 16 tokens 171 and 180.
// At head_dim 64 eight warps x 2 CTAs take 14.1 us for 24 layers x 8192 tokens,
// four x 2 15.3, four x 4 15.7.  A tcgen05 form (128 rows of codes converted into shared
// memory, the heads as the N side) was slower: a product of M = 128 takes 53
// clocks however few heads there are, and the codes pass shared memory once
// more (178 to 194 us in four arrangements).  Integer products of the codes
// (m16n8k32) are as fast as these at twice the depth, but their sums' digits
// need the shifts and conversions that the codes then save.
template <int HD>
struct Dec {
  static constexpr int kWarps = kv4_warps(HD), kCtas = 2;
  static constexpr int kStageTiles = kKv4StageTiles, kStageTokens = kKv4StageTokens;
  static constexpr int TB = kv4_tile_bytes(HD), CB = kv4_code_bytes(HD), SB = kv4_scale_bytes(HD);
  static constexpr int kStageBytes = kStageTiles * TB;
  static constexpr int NB = HD / 32;
  static constexpr int kRing = 2;                       // stages in flight per warp
  static constexpr int kItems = NB * 2 * 32;           // float4 items of a warp's O
  static constexpr int ring_off = 0;
  static constexpr int new_off = kWarps * kRing * kStageBytes;  // a stage for the appended token
  static constexpr int q_off = new_off + kStageBytes;
  static constexpr int red_off = q_off + NB * 2 * 512;
  static constexpr int stat_off = red_off + (kWarps / 2) * kItems * 16;
  static constexpr int f_off = stat_off + 2 * kWarps * kKv4Heads * 4;
  static constexpr int flag_off = f_off + kKv4Heads * 4;
  static constexpr int seg_off = flag_off + 16;        // the current segment, the next, a pending one
  static constexpr int feed_off = seg_off + 3 * 64;
  static constexpr int bar_off = feed_off + kWarps * 64;
  static constexpr int smem = bar_off + kWarps * kRing * 8;
};
static_assert((Dec<128>::smem + 1024) * Dec<128>::kCtas <= 228 * 1024, "CTAs per SM");
static_assert((Dec<64>::smem + 1024) * Dec<64>::kCtas <= 228 * 1024, "CTAs per SM");

struct Seg {
  int next;            // the CTA's next unit (global index), its end when there is none
  int ll, kvh, hb, si; // local layer, kv head, head block, sequence
  int s0, s1;          // stages (copies) of the sequence in this segment
  int first;           // 1: the CTA's first segment
  int parts, c0;       // CTAs that share the group, the first of them
  int gb;              // stream split: the group's first unit (global index)
  int last;            // 1: holds the group's last unit (and so the appended token)
  int group_id;
  int blk;             // (layer, kv head, head block)
};

static_assert(sizeof(Seg) <= 64, "segments in shared memory");

// The sequence (of block-relative position rem) by its first unit or part.
__device__ __forceinline__ int kv4_seq_at(const Kv4DecodeParams& p, int rem, bool aligned) {
  int lo = 0, hi = p.n_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    const int begin = aligned ? p.seqs[mid].part_begin : p.seqs[mid].unit_begin;
    if (begin <= rem) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Stream split: where CTA b's range begins: at b T / grid, or at the start of that unit's group when the cut would
// leave the CTA before nothing but the group's fixed units (a part without a token).  The range may be empty.
__device__ __forceinline__ int kv4_cut(const Kv4DecodeParams& p, int b) {
  const int u = (int)stage_start(b, p.total_units, p.grid);
  if (u >= p.total_units) return u;
  const int blk = (int)((uint32_t)u / (uint32_t)p.block_units);
  const int gb = blk * p.block_units + p.seqs[kv4_seq_at(p, u - blk * p.block_units, false)].unit_begin;
  return u - gb <= kKv4GroupUnits ? gb : u;
}

// Stream split: the CTA whose range holds unit u, which is not one of its group's fixed units but the last.
__device__ __forceinline__ int kv4_cta_of(int u, long long total, int grid) {
  return (int)div_nonneg((long long)(u + 1) * grid - 1, total);
}

// The segment of this CTA that begins at u (stream split), or its only one (aligned split).
template <int HD>
__device__ __forceinline__ Seg kv4_seg_at(const Kv4DecodeParams& p, int u, int u_begin, int u1) {
  Seg s;
  const bool aligned = p.block_parts != 0;
  const int per = aligned ? p.block_parts : p.block_units;
  const int at = aligned ? (int)blockIdx.x : u;
  const uint32_t blk = (uint32_t)at / (uint32_t)per;
  const int rem = at - (int)blk * per;
  const int lo = kv4_seq_at(p, rem, aligned);
  s.si = lo;
  const int len = p.seqs[lo].len;
  const int n = kv4_units(len, HD);
  int a, b;  // units of the sequence in this segment
  if (aligned) {
    const int part = rem - p.seqs[lo].part_begin;
    s.parts = (lo + 1 < p.n_seqs ? p.seqs[lo + 1].part_begin : per) - p.seqs[lo].part_begin;
    s.c0 = (int)blockIdx.x - part;
    a = (int)div_nonneg((long long)part * n, s.parts);
    b = (int)div_nonneg((long long)(part + 1) * n, s.parts);
    s.gb = 0;
    s.next = u1;
    s.first = 1;
  } else {
    s.gb = (int)blk * per + p.seqs[lo].unit_begin;
    s.next = min(s.gb + n + kKv4GroupUnits, u1);
    a = max(u - s.gb - kKv4GroupUnits, 0);
    b = max(s.next - s.gb - kKv4GroupUnits, 0);
    s.c0 = kv4_cta_of(s.gb + kKv4GroupUnits, p.total_units, p.grid);
    s.parts = kv4_cta_of(s.gb + n + kKv4GroupUnits - 1, p.total_units, p.grid) - s.c0 + 1;
    s.first = u == u_begin;
  }
  constexpr int kUnitStages = kv4_warps(HD), kTokens = kKv4StageTokens;
  s.s0 = a * kUnitStages;
  s.s1 = min(b * kUnitStages, (len + kTokens - 1) / kTokens);
  s.last = b == n;
  const uint32_t lk = blk / (uint32_t)p.head_blocks;
  s.hb = (int)(blk - lk * (uint32_t)p.head_blocks);
  s.ll = (int)(lk / (uint32_t)p.pool.kv_heads);
  s.kvh = (int)lk - s.ll * p.pool.kv_heads;
  s.group_id = (int)blk * p.n_seqs + lo;
  s.blk = (int)blk;
  return s;
}

// Stream split: the segment after s, whose group begins inside this CTA's range, without kv4_seg_at's search.
template <int HD>
__device__ __forceinline__ void kv4_seg_after(const Kv4DecodeParams& p, const Seg& s, int u1, Seg& r) {
  r = s;
  r.gb = s.next;
  r.first = 0;
  if (++r.si == p.n_seqs) {
    r.si = 0;
    ++r.blk;
    if (++r.hb == p.head_blocks) {
      r.hb = 0;
      if (++r.kvh == p.pool.kv_heads) {
        r.kvh = 0;
        ++r.ll;
      }
    }
  }
  r.group_id = r.blk * p.n_seqs + r.si;
  const int len = p.seqs[r.si].len, n = kv4_units(len, HD), end = r.gb + n + kKv4GroupUnits;
  r.next = min(end, u1);
  const int b = max(r.next - r.gb - kKv4GroupUnits, 0);
  r.s0 = 0;
  r.s1 = min(b * kv4_warps(HD), (len + kKv4StageTokens - 1) / kKv4StageTokens);
  r.last = b == n;
  r.c0 = blockIdx.x;
  r.parts = end <= u1 ? 1 : kv4_cta_of(end - 1, p.total_units, p.grid) - r.c0 + 1;
}

__device__ __forceinline__ uint32_t h2_add(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
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
// The four f16 pairs of a word: c - 8, and 16 (c - 8) for the upper nibbles, exactly: a code under the exponent
// of 1024 is 1024 + c (or + 16 c), and one subtraction leaves a normal number.  Codes read as f16 subnormals
// would need no subtraction for the keys, but the tensor core aligns the 16 products of a step by their
// operands' nominal exponents: subnormals lose 7 to 10 bits of the fp32 sum (measured: the output was 8e-6
// off, against less than 1e-6 now).
__device__ __forceinline__ void centred(uint32_t x, uint32_t magic, uint32_t (&c)[4]) {
  const uint32_t y = x >> 8;
  c[0] = h2_add(and_or(x, 0x000f000fu, magic), 0xe408e408u);
  c[1] = h2_add(and_or(x, 0x00f000f0u, magic), 0xe480e480u);
  c[2] = h2_add(and_or(y, 0x000f000fu, magic), 0xe408e408u);
  c[3] = h2_add(and_or(y, 0x00f000f0u, magic), 0xe480e480u);
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
// D = A B (+ D), m16n8k16, f16 operands, f32 accumulators.
__device__ __forceinline__ void mma_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_add(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t h2_maxabs(uint32_t a, uint32_t b) {
  const __half2 x = __habs2(*reinterpret_cast<const __half2*>(&a));
  const __half2 y = __habs2(*reinterpret_cast<const __half2*>(&b));
  const __half2 m = __hmax2(x, y);
  return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t h2_min(uint32_t a, uint32_t b) {
  const __half2 m = __hmin2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
// 2^k as fp32, -126 <= k <= 127.
__device__ __forceinline__ float pow2i(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }
__device__ __forceinline__ int exponent_of(float x) { return (int)((__float_as_uint(x) >> 23) & 255u) - 127; }

template <int HD>
struct WarpState {
  float f;                // S f = score in exp2 units
  float o[HD / 32][2][4];    // O^T accumulators: block, m16 tile
  float m;                // head g: reference of the scores, an integer, so that rescaling is exact
  float l;                // sum of this lane's weights, head g
};

constexpr float kSlack = 5.f;       // a stage's reference may exceed the head's by this before that one moves
constexpr float kWeightExp = 14.f;  // weights are 2^(score - the stage's reference + 14): the largest is above 2^13
// Token scales (the largest of a row's block scales) for which weight times scale stays within f16: the stage's largest
// product is between 2^-1 and 2^15, and a product's two parts are off by 2^-25 and a part in 2^22 at most.
constexpr float kScaleMin = 0x1p-14f, kScaleMax = 2.f;
constexpr float kRefMax = 0x1p22f;  // references up to here leave 14 - reference exact

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

// Bias, RoPE, the head's power of two (largest value in [2^11, 2^12)) and the f16 hi / lo split: writes the row's
// part of the A fragments (lane 4h + t of block b, step st: {hi, lo, hi / 16, lo / 16} of 4 dims -- the codes of
// the second pair come as 16 c) and the factor that turns S into exp2 units.
template <int HD>
__device__ __forceinline__ void stage_query(const Kv4DecodeParams& p, const Seg& s, int h, int lane, float (&v)[4],
                                            unsigned char* qf, float* f) {
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
  const int k = top > 0.f ? min(max(11 - exponent_of(top), -116), 126) : 0;
  const float sc = pow2i(k);
  if (lane == 0) f[h] = p.scale_log2 * pow2i(-k);
  uint32_t w[4];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const float mul = r ? 0.0625f : 1.f;
    const float x = v[2 * r] * sc * mul, y = v[2 * r + 1] * sc * mul;
    const __half2 hi = __floats2half2_rn(x, y);
    const float2 hf = __half22float2(hi);
    w[2 * r] = *reinterpret_cast<const uint32_t*>(&hi);
    w[2 * r + 1] = pack_half2(x - hf.x, y - hf.y);
  }
  // dims 4 lane .. + 3: block lane / 8, lane t = (lane % 8) / 2 of the fragment, step lane % 2
  if (lane < HD / 4) {
    *reinterpret_cast<uint4*>(qf + ((lane >> 3) * 2 + (lane & 1)) * 512 + (4 * h + ((lane & 7) >> 1)) * 16) =
        make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <int HD>
__device__ __forceinline__ void reset_state(WarpState<HD>& w) {
#pragma unroll
  for (int b = 0; b < HD / 32; ++b)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) w.o[b][i][r] = 0.f;
  w.m = -INFINITY;
  w.l = 0.f;
}

// Words of a lane: NB per n8 half / token-pair half j.
template <int HD>
__device__ __forceinline__ void lds_words(uint32_t addr, int lane, uint32_t (&w)[2][HD / 32]) {
  if constexpr (HD == 128) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint4 v = lds128(addr + j * 512 + lane * 16);
      w[j][0] = v.x; w[j][1] = v.y; w[j][2] = v.z; w[j][3] = v.w;
    }
  } else {
    const uint4 v = lds128(addr + lane * 16);
    w[0][0] = v.x; w[0][1] = v.y; w[1][0] = v.z; w[1][1] = v.w;
  }
}
template <int HD>
__device__ __forceinline__ void lds_scales(uint32_t addr, int t, uint32_t (&w)[2][HD / 32]) {
  if constexpr (HD == 128) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint4 v = lds128(addr + j * 64 + t * 16);
      w[j][0] = v.x; w[j][1] = v.y; w[j][2] = v.z; w[j][3] = v.w;
    }
  } else {
    const uint4 v = lds128(addr + t * 16);
    w[0][0] = v.x; w[0][1] = v.y; w[1][0] = v.z; w[1][1] = v.w;
  }
}

// Attends the first `valid` tokens of T consecutive tiles at shared address `addr`; the queries' A fragments are
// at shared address `qf` (read again for each stage: 32 registers less in every warp, so that more warps fit).
template <int HD, int T>
__device__ __forceinline__ void attend(uint32_t addr, uint32_t qf, int valid, int lane, uint32_t magic,
                                       WarpState<HD>& w) {
  using D = Dec<HD>;
  constexpr int NB = D::NB;
  const int t = lane & 3;
  // s[i][2j + r]: tile i, token 8j + 2t + r, head g, in exp2 units
  float s[T][4];
  {
    uint32_t kw[T][2][NB], ks[T][2][NB];
#pragma unroll
    for (int i = 0; i < T; ++i) {
      lds_words<HD>(addr + i * D::TB, lane, kw[i]);
      lds_scales<HD>(addr + i * D::TB + 2 * D::CB, t, ks[i]);
    }
    uint64_t s2[T][2];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      uint32_t qa[2][4];
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const uint4 x = lds128(qf + (b * 2 + st) * 512 + lane * 16);
        qa[st][0] = x.x; qa[st][1] = x.y; qa[st][2] = x.z; qa[st][3] = x.w;
      }
      // all conversions of the block, then its products: the registers of a product's codes are not written
      // again right behind it (12 clocks a product instead of 9)
      uint32_t c[T][2][4];
      float acc[T][2][4];
#pragma unroll
      for (int i = 0; i < T; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) centred(kw[i][j][b], magic, c[i][j]);
#pragma unroll
      for (int i = 0; i < T; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) mma_zero(acc[i][j], qa[0], c[i][j][0], c[i][j][1]);
#pragma unroll
      for (int i = 0; i < T; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) mma_add(acc[i][j], qa[1], c[i][j][2], c[i][j][3]);
#pragma unroll
      for (int i = 0; i < T; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float2 d = __half22float2(*reinterpret_cast<const __half2*>(&ks[i][j][b]));
          const uint64_t d2 = f2_pack(d.x, d.y);
          const uint64_t hi = f2_pack(acc[i][j][0], acc[i][j][1]), lo = f2_pack(acc[i][j][2], acc[i][j][3]);
          s2[i][j] = f2_fma(d2, lo, b == 0 ? f2_mul(d2, hi) : f2_fma(d2, hi, s2[i][j]));
        }
    }
    // exp2 units, rounded: the reference and the weights have to see the same score, however large it is
    const uint64_t f2 = f2_pack(w.f, w.f);
#pragma unroll
    for (int i = 0; i < T; ++i) {
      f2_unpack(f2_mul(s2[i][0], f2), s[i][0], s[i][1]);
      f2_unpack(f2_mul(s2[i][1], f2), s[i][2], s[i][3]);
    }
  }
  uint32_t vs[T][2][NB];
#pragma unroll
  for (int i = 0; i < T; ++i) lds_scales<HD>(addr + i * D::TB + 2 * D::CB + D::SB, t, vs[i]);
  if (valid < kKv4Tile * T) {  // tokens past the sequence: no weight, whatever the tile holds there
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (kKv4Tile * i + 8 * (r >> 1) + 2 * t + (r & 1) >= valid) {
          s[i][r] = -INFINITY;
#pragma unroll
          for (int b = 0; b < NB; ++b) {  // a scale of 1
            uint32_t& d = vs[i][r >> 1][b];
            d = (r & 1) ? (d & 0x0000ffffu) | 0x3c000000u : (d & 0xffff0000u) | 0x3c00u;
          }
        }
      }
  }
  // Weights are counted from the stage's own largest score: a token's share of the stage keeps its bits however far
  // the stage lies below the reference, and O takes the stage in by one power of two a head.
  float top = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
#pragma unroll
  for (int i = 1; i < T; ++i) top = fmaxf(fmaxf(top, fmaxf(s[i][0], s[i][1])), fmaxf(s[i][2], s[i][3]));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  auto token_scale = [&](int i, int j) {  // the largest block scale of two tokens
    uint32_t d = vs[i][j][0];
#pragma unroll
    for (int b = 1; b < NB; ++b) d = h2_maxabs(d, vs[i][j][b]);
    return d;
  };
  uint32_t dmin = token_scale(0, 0), dmax = dmin;
#pragma unroll
  for (int i = 0; i < T; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (i + j == 0) continue;
      const uint32_t d = token_scale(i, j);
      dmin = h2_min(dmin, d);
      dmax = h2_maxabs(dmax, d);
    }
  const float2 lo2 = __half22float2(*reinterpret_cast<const __half2*>(&dmin));
  const float2 hi2 = __half22float2(*reinterpret_cast<const __half2*>(&dmax));
  const bool some = top > -INFINITY;  // false: every score is -inf or NaN
  const float ref = some ? ceilf(top) : 0.f;
  const bool move = some && ref > w.m + kSlack;
  bool odd = fminf(lo2.x, lo2.y) < kScaleMin || fmaxf(hi2.x, hi2.y) > kScaleMax || fabsf(ref) > kRefMax;
  auto pair_of = [&](float x) {  // head g's x for the two heads whose columns of O this lane holds
    return f2_pack(__shfl_sync(0xffffffffu, x, 8 * t), __shfl_sync(0xffffffffu, x, 8 * t + 4));
  };
  if (__any_sync(0xffffffffu, move)) {
    const float alpha = move ? ex2(w.m - ref) : 1.f;
    if (move) w.m = ref;
    w.l *= alpha;
    const uint64_t a2 = pair_of(alpha);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          f2_unpack(f2_mul(f2_pack(w.o[b][i][r], w.o[b][i][r + 1]), a2), w.o[b][i][r], w.o[b][i][r + 1]);
        }
  }
  float into_o = some ? ex2(ref - w.m) : 0.f, into_l = into_o;
  float mb = kWeightExp - ref;
  odd = __any_sync(0xffffffffu, odd);
  if (odd) {
    // A token whose scales lie outside the ordinary range (or scores so large that the offset cannot hold both the
    // reference and the 14): every token's scales are brought to [1, 2) by a power of two, which its weight takes
    // instead, and the weights are counted from the largest of these products.  The weights' sum has them without it.
    float sum = 0.f, vtop = -INFINITY;
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        sum += ex2((s[i][2 * j] - ref) + kWeightExp) + ex2((s[i][2 * j + 1] - ref) + kWeightExp);
        const uint32_t dm = token_scale(i, j);
        const float2 d = __half22float2(*reinterpret_cast<const __half2*>(&dm));
        const int e0 = min(max(exponent_of(d.x), -15), 15), e1 = min(max(exponent_of(d.y), -15), 15);
        const uint32_t k = pack_half2(pow2i(-e0), pow2i(-e1));
#pragma unroll
        for (int b = 0; b < NB; ++b) vs[i][j][b] = h2_mul(vs[i][j][b], k);
        // values of zero add nothing, whatever their weight
        s[i][2 * j] = d.x == 0.f ? -INFINITY : (s[i][2 * j] - ref) + (float)e0;
        s[i][2 * j + 1] = d.y == 0.f ? -INFINITY : (s[i][2 * j + 1] - ref) + (float)e1;
        vtop = fmaxf(vtop, fmaxf(s[i][2 * j], s[i][2 * j + 1]));
      }
    vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, 1));
    vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, 2));
    w.l += into_l * sum;
    into_l = 0.f;
    const float vref = vtop > -INFINITY ? ceilf(vtop) : 0.f;
    into_o *= ex2(vref);
    mb = kWeightExp - vref;
  }
  const uint64_t into2 = pair_of(into_o);
  float sum = 0.f;
  uint32_t ph[T][2], pl[T][2], vw[T][2][NB];
#pragma unroll
  for (int i = 0; i < T; ++i) {
    lds_words<HD>(addr + i * D::TB + D::CB, lane, vw[i]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float p0, p1;
      f2_unpack(f2_add(f2_pack(s[i][2 * j], s[i][2 * j + 1]), f2_pack(mb, mb)), p0, p1);
      p0 = ex2(p0);
      p1 = ex2(p1);
      sum += p0 + p1;
      const __half2 h = __floats2half2_rn(p0, p1);
      const float2 hf = __half22float2(h);
      ph[i][j] = *reinterpret_cast<const uint32_t*>(&h);
      pl[i][j] = pack_half2(p0 - hf.x, p1 - hf.y);
    }
  }
  w.l += into_l * sum;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    // the tiles' products start from zero and join O by a rounded fp32 FMA: a long accumulation inside
    // the tensor core truncates at every step
    float o0[4], o1[4];
    uint32_t hi[T][2], lo[T][2], ca[T][4], cc[T][4];  // as for the keys: all conversions first
#pragma unroll
    for (int i = 0; i < T; ++i) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t d = vs[i][j][b];
        hi[i][j] = h2_mul(ph[i][j], d);
        lo[i][j] = h2_fma(pl[i][j], d, h2_fms(ph[i][j], d, hi[i][j]));
      }
      uint32_t c0[4], c1[4];
      centred(vw[i][0][b], magic, c0);
      centred(vw[i][1][b], magic, c1);
      ca[i][0] = c0[0]; ca[i][1] = c0[1]; ca[i][2] = c1[0]; ca[i][3] = c1[1];
      cc[i][0] = c0[2]; cc[i][1] = c0[3]; cc[i][2] = c1[2]; cc[i][3] = c1[3];
    }
#pragma unroll
    for (int i = 0; i < T; ++i) {
      if (i == 0) {
        mma_zero(o0, ca[i], lo[i][0], lo[i][1]);
        mma_zero(o1, cc[i], lo[i][0], lo[i][1]);
      } else {
        mma_add(o0, ca[i], lo[i][0], lo[i][1]);
        mma_add(o1, cc[i], lo[i][0], lo[i][1]);
      }
      mma_add(o0, ca[i], hi[i][0], hi[i][1]);
      mma_add(o1, cc[i], hi[i][0], hi[i][1]);
    }
#pragma unroll
    for (int r = 0; r < 4; r += 2) {
      f2_unpack(f2_fma(f2_pack(o0[r], o0[r + 1]), into2, f2_pack(w.o[b][0][r], w.o[b][0][r + 1])), w.o[b][0][r],
                w.o[b][0][r + 1]);
      f2_unpack(f2_fma(f2_pack(o1[r], o1[r + 1]), into2, f2_pack(w.o[b][1][r], w.o[b][1][r + 1])), w.o[b][1][r],
                w.o[b][1][r + 1]);
    }
  }
}

// A warp's copies: stages s0 + warp, + kWarps, ... of each segment of the CTA's range, in order, across segments.
// Lane 0 keeps them, in shared memory: the other lanes' registers are the attention's.
struct Feed {
  int stage, s1;              // next stage and end of the current segment
  int page, in;               // the next stage's page and stage within it
  const unsigned char* base;  // page 0 of the segment's layer, at its kv head
  const int32_t* row;
  int u, page_base;           // next segment's first unit; as Kv4Seq
  long long page_bytes;       // from one page of this kv head to the next
  int blk, si;                // the segment's (layer, kv head, head block) and sequence
};
static_assert(sizeof(Feed) <= 56, "feeds in shared memory");

template <int HD>
__device__ __forceinline__ void feed_enter(const Kv4DecodeParams& p, Feed& f, const Seg& s, int warp) {
  using D = Dec<HD>;
  f.u = s.next;
  f.blk = s.blk;
  f.si = s.si;
  f.stage = s.s0 + warp;
  f.s1 = s.s1;
  const long long rec = (long long)(p.layer_begin + s.ll) * p.pool.num_pages * p.pool.kv_heads + s.kvh;
  f.base = p.pool.base + rec * p.pool.tiles_per_page * D::TB;
  f.page_bytes = (long long)p.pool.kv_heads * p.pool.tiles_per_page * D::TB;
  f.row = p.page_table + (size_t)p.seqs[s.si].slot * p.max_pages_per_seq;
  f.page_base = p.seqs[s.si].page_base;
  f.page = kv4_page_of(p.pool, f.stage * D::kStageTiles);
  f.in = f.stage - f.page * p.pool.stages_per_page;
}

// Moves f to a segment in which it has a stage left; false past the end of the CTA's range.
template <int HD>
__device__ __forceinline__ bool feed_seek(const Kv4DecodeParams& p, Feed& f, int warp, int u1) {
  using D = Dec<HD>;
  if (f.stage < f.s1) return true;
  int blk = f.blk, si = f.si, u = f.u, s1 = 0;
  do {
    if (u >= u1) {
      f.u = u;
      return false;
    }
    if (++si == p.n_seqs) si = 0, ++blk;
    const int len = p.seqs[si].len, end = min(u + kv4_units(len, HD) + kKv4GroupUnits, u1);
    s1 = min(max(end - u - kKv4GroupUnits, 0) * D::kWarps, (len + D::kStageTokens - 1) / D::kStageTokens);
    u = end;
  } while (warp >= s1);
  Seg s;
  s.next = u;
  s.blk = blk;
  s.si = si;
  s.s0 = 0;
  s.s1 = s1;
  const uint32_t lk = (uint32_t)blk / (uint32_t)p.head_blocks;
  s.ll = (int)(lk / (uint32_t)p.pool.kv_heads);
  s.kvh = (int)lk - s.ll * p.pool.kv_heads;
  feed_enter<HD>(p, f, s, warp);
  return true;
}

// Issues the copy of f's stage and steps past it.
template <int HD>
__device__ __forceinline__ void feed_issue(const Kv4DecodeParams& p, Feed& f, unsigned char* dst, uint64_t* bar) {
  using D = Dec<HD>;
  const int id = f.page_base >= 0 ? f.page_base + f.page : f.row[f.page];
  const unsigned char* src = f.base + id * f.page_bytes + (long long)f.in * D::kStageBytes;
  mbar_arrive_expect_tx(bar, D::kStageBytes);
  bulk_load(dst, src, D::kStageBytes, bar);
  f.stage += D::kWarps;
  f.page += p.pool.step_pages;
  f.in += p.pool.step_in;
  if (f.in >= p.pool.stages_per_page) {
    f.in -= p.pool.stages_per_page;
    ++f.page;
  }
}

template <int HD>
__global__ void __launch_bounds__(32 * Dec<HD>::kWarps, Dec<HD>::kCtas)
    kv4_decode_kernel(const __grid_constant__ Kv4DecodeParams p) {
  using D = Dec<HD>;
  constexpr int NB = D::NB, W = D::kWarps, H = kKv4Heads, HW = W / 2;
  constexpr int rec = kv4_record_floats(HD);
  static_assert(W % 2 == 0, "the merge pairs warps");
  extern __shared__ __align__(128) unsigned char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + D::bar_off) + warp * D::kRing;
  unsigned char* ring = smem + D::ring_off + warp * D::kRing * D::kStageBytes;
  unsigned char* new_stage = smem + D::new_off;
  unsigned char* qf = smem + D::q_off;
  float4* red = reinterpret_cast<float4*>(smem + D::red_off);
  float* sm_m = reinterpret_cast<float*>(smem + D::stat_off);  // [W][8]
  float* sm_l = sm_m + W * H;
  float* sm_f = reinterpret_cast<float*>(smem + D::f_off);
  int* sm_flag = reinterpret_cast<int*>(smem + D::flag_off);
  auto seg = [&](int i) -> Seg& { return *reinterpret_cast<Seg*>(smem + D::seg_off + 64 * i); };

  // Launched as a programmatic dependent: up to griddep_wait the previous kernel may still run, and nothing here
  // touches global memory.
  if (lane == 0) {
    for (int i = 0; i < D::kRing; ++i) mbar_init(&bars[i], 1);
    fence_mbarrier_init();
    fence_proxy_async_shared();
  }
  __syncwarp();
  const bool aligned = p.block_parts != 0;
  if (threadIdx.x == 0) {
    const int u0 = aligned ? 0 : kv4_cut(p, blockIdx.x), u1 = aligned ? 1 : kv4_cut(p, blockIdx.x + 1);
    sm_flag[2] = u1;
    sm_flag[3] = u0 < u1;
    if (u0 < u1) seg(0) = kv4_seg_at<HD>(p, u0, u0, u1);
  }
  Feed& feed = *reinterpret_cast<Feed*>(smem + D::feed_off + 64 * warp);
  int* sm_issued = reinterpret_cast<int*>(smem + D::feed_off + 64 * warp + 56);
  bool feeding = false;
  __syncthreads();
  const int u1 = sm_flag[2];
  if (sm_flag[3] == 0) return;  // an empty range
  if (lane == 0) {
    feed_enter<HD>(p, feed, seg(0), warp);
    *sm_issued = 0;
    feeding = feed_seek<HD>(p, feed, warp, u1);
    // L2 may fetch the first stage while the previous kernel drains (a hint, coherent with that kernel's writes)
    if (feeding && feed.page_base >= 0) {
      bulk_prefetch_l2(feed.base + (feed.page_base + feed.page) * feed.page_bytes + (long long)feed.in * D::kStageBytes,
                       D::kStageBytes);
    }
  }
  auto issue = [&](int slot) {  // lane 0
    if (!feeding) return;
    feed_issue<HD>(p, feed, ring + slot * D::kStageBytes, &bars[slot]);
    ++*sm_issued;
    feeding = feed_seek<HD>(p, feed, warp, u1);
  };
  griddep_launch_dependents();
  griddep_wait();
  constexpr int kRows = (H + W - 1) / W;  // query heads a warp prepares
  float qr[kRows][4];  // asked for before the stages, whose first wave fills the memory system for microseconds
#pragma unroll
  for (int i = 0; i < kRows; ++i) fetch_query<HD>(p, seg(0), warp + i * W, lane, qr[i]);
  if (lane == 0) {
    for (int i = 0; i < D::kRing; ++i) issue(i);
  }
  int used = 0;              // stages consumed by this warp
  int slot = 0;
  uint32_t phase = 0;
  bool ok = true;            // false: a wait ran out; the warp computes no more
  const uint32_t magic = code_magic();
  int n_pending = 0;         // segments of this CTA that are parts of shared groups
  int at_seg = 0;            // seg(at_seg): the current segment

  auto part_weight = [](float m, float top) { return m == -INFINITY ? 0.f : ex2(m - top); };
  // item i of an output: block i / 64, heads 2 (i % 4) + (i / 32) % 2, dims 4 ((i % 32) / 4) .. + 3 of the block
  auto write_out = [&](const Seg& q, int head, int dim, const float4& acc, float top, float sum) {
    const int hg = q.hb * p.block_heads + head;
    if (head >= p.block_heads || hg >= p.group) return;
    const size_t row =
        ((size_t)q.ll * p.seq_total + p.seq_base + q.si) * (p.pool.kv_heads * p.group) + q.kvh * p.group + hg;
    if (p.partial_out) {
      const float k = pow2i(-(int)kWeightExp);
      float* o = p.out + row * (HD + 2);
      o[dim] = acc.x * k;
      o[dim + 1] = acc.y * k;
      o[dim + 2] = acc.z * k;
      o[dim + 3] = acc.w * k;
      if (dim == 0) {
        o[HD] = top;
        o[HD + 1] = sum * k;
      }
    } else {
      const float r = sum == 0.f ? 0.f : 1.f / sum;  // no token at all: zeros
      *reinterpret_cast<float4*>(p.out + row * HD + dim) = make_float4(acc.x * r, acc.y * r, acc.z * r, acc.w * r);
    }
  };

  WarpState<HD> w;
  while (true) {
    const Seg& s = seg(at_seg);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (warp + i * W < H) stage_query<HD>(p, s, warp + i * W, lane, qr[i], qf, sm_f);
    }
    const Kv4Seq& sq = p.seqs[s.si];
    const int len = sq.len;
    const int n_stages = s.s1 - s.s0;
    const bool appender = p.k_new != nullptr && s.last && warp == n_stages % W;
    __syncthreads();  // the queries are in shared memory
    w.f = sm_f[g];
    reset_state<HD>(w);
    if (s.next < u1 && threadIdx.x == 32 * (W - 1)) kv4_seg_after<HD>(p, s, u1, seg(at_seg ^ 1));
    if (appender) {
      // the new token: quantised into the cache (by the first head block) and into a stage of its own here, by the
      // warp that has the fewest stages, while the others attend theirs
      const size_t at = (((size_t)s.ll * p.seq_total + p.seq_base + s.si) * p.pool.kv_heads + s.kvh) * HD;
      const size_t brow = ((size_t)(p.layer_begin + s.ll) * p.pool.kv_heads + s.kvh) * HD;
      float k[4], v[4];
      load_row<HD>(p.k_new, p.v_new, at, p.input_f16, p.k_bias ? p.k_bias + brow : nullptr,
                   p.k_bias ? p.v_bias + brow : nullptr,
                   p.rope ? p.rope_cos + (size_t)sq.new_pos * (HD / 2) : nullptr,
                   p.rope ? p.rope_sin + (size_t)sq.new_pos * (HD / 2) : nullptr, lane, k, v);
      float k2[4] = {k[0], k[1], k[2], k[3]}, v2[4] = {v[0], v[1], v[2], v[3]};
      store_row<HD>(new_stage, 0, lane, k, v);
      if (s.hb == 0) {
        unsigned char* dst = tile_ptr(p.pool, p.page_table + (size_t)sq.slot * p.max_pages_per_seq, p.layer_begin + s.ll,
                                      s.kvh, len / kKv4Tile, D::TB);
        store_row<HD>(dst, len % kKv4Tile, lane, k2, v2);
      }
      __syncwarp();
    }
    // the appended token's stage, then this warp's
    int st = s.s0 + warp;
    bool extra = appender;
    while (st < s.s1 || extra) {
      const bool cached = !extra;
      uint32_t addr = smem_u32(new_stage);
      int valid = 1;
      if (cached) {
        if (ok) ok = mbar_wait_warp(&bars[slot], phase);
        if (!ok) {
          if (lane == 0) set_error(p.error, 60);
          break;
        }
        addr = smem_u32(ring + slot * D::kStageBytes);
        valid = len - st * D::kStageTokens;
      } else {
        extra = false;
      }
      attend<HD, D::kStageTiles>(addr, smem_u32(qf), valid, lane, magic, w);
      if (cached) {
        __syncwarp();
        ++used;
        if (lane == 0) issue(slot);
        if (++slot == D::kRing) {
          slot = 0;
          phase ^= 1u;
        }
        st += W;
      }
    }

    // merge the warps' states: m and l per head first, then O in two rounds
    float l = w.l;
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (t == 0) {
      sm_m[warp * H + g] = w.m;
      sm_l[warp * H + g] = l;
    }
    __syncthreads();
    {
      float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        mx0 = fmaxf(mx0, sm_m[i * H + 2 * t]);
        mx1 = fmaxf(mx1, sm_m[i * H + 2 * t + 1]);
      }
      const float c0 = part_weight(sm_m[warp * H + 2 * t], mx0), c1 = part_weight(sm_m[warp * H + 2 * t + 1], mx1);
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          w.o[b][i][0] *= c0;
          w.o[b][i][1] *= c1;
          w.o[b][i][2] *= c0 * 0.0625f;
          w.o[b][i][3] *= c1 * 0.0625f;
        }
    }
    auto o_item = [&](int b, int c) {
      return make_float4(w.o[b][0][c], w.o[b][0][2 + c], w.o[b][1][c], w.o[b][1][2 + c]);
    };
    if (warp >= HW) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int c = 0; c < 2; ++c) red[(warp - HW) * D::kItems + (b * 2 + c) * 32 + lane] = o_item(b, c);
    }
    __syncthreads();
    if (warp < HW) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float4* sl = &red[warp * D::kItems + (b * 2 + c) * 32 + lane];
          const float4 x = *sl, y = o_item(b, c);
          *sl = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
        }
    }
    __syncthreads();
    const bool more = s.next < u1;
    if (more) {  // the next segment's query rows on their way
#pragma unroll
      for (int i = 0; i < kRows; ++i) fetch_query<HD>(p, seg(at_seg ^ 1), warp + i * W, lane, qr[i]);
    }
    // a CTA's first segment uses its slot 0, its last another one: at most two of its segments are parts of groups
    float* mine = p.partials + ((size_t)blockIdx.x * 2 + (s.first ? 0 : 1)) * rec;
    for (int i = threadIdx.x; i < D::kItems; i += 32 * W) {
      const int head = 2 * (i & 3) + ((i >> 5) & 1);
      const int dim = 32 * (i >> 6) + 4 * ((i & 31) >> 2);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int k = 0; k < HW; ++k) {
        const float4 x = red[k * D::kItems + i];
        acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
      }
#pragma unroll
      for (int k = 0; k < W; ++k) top = fmaxf(top, sm_m[k * H + head]);
#pragma unroll
      for (int k = 0; k < W; ++k) sum += sm_l[k * H + head] * part_weight(sm_m[k * H + head], top);
      if (s.parts == 1) {
        write_out(s, head, dim, acc, top, sum);
      } else {
        reinterpret_cast<float4*>(mine)[i] = acc;
        if (dim == 0) {
          mine[H * HD + head] = top;
          mine[H * HD + H + head] = sum;
        }
      }
    }
    if (s.parts > 1) {
      if (n_pending == 0 && threadIdx.x == 0) seg(2) = s;
      ++n_pending;
    }
    if (!more) break;
    at_seg ^= 1;
    __syncthreads();  // the merge buffers, the queries and the new token's stage are free again
  }

  // Groups shared with other CTAs: the last of a group's CTAs to arrive folds its records, in part order.  Left to
  // the end, where the records have long been written and no segment of this CTA waits behind a fold.
  if (n_pending > 0) {
    __syncthreads();
    if (threadIdx.x < (unsigned)n_pending) {
      const Seg& q = seg(threadIdx.x == 0 ? 2 : at_seg);
      sm_flag[threadIdx.x] = atom_add_acq_rel_gpu(&p.counters[q.group_id], 1u) == (uint32_t)q.parts - 1u;
    }
    __syncthreads();
    for (int i = 0; i < n_pending; ++i) {
      if (sm_flag[i] == 0) continue;
      const Seg& q = seg(i == 0 ? 2 : at_seg);
      // part k is CTA c0 + k's: its first segment unless (stream split) its range began before the group, which
      // only the group's first part can
      const int slot0 = aligned || stage_start(q.c0, p.total_units, p.grid) >= q.gb ? 0 : 1;
      auto rec_of = [&](int k) { return p.partials + ((size_t)(q.c0 + k) * 2 + (k == 0 ? slot0 : 0)) * rec; };
      // a thread's items belong to one head; eight records at a time, all of their loads in flight together, and the
      // running state is rescaled per batch
      constexpr int kBatch = 8, kPer = (D::kItems + 32 * W - 1) / (32 * W);
      static_assert((D::kItems % (32 * W) == 0 || kPer == 1) && W % 2 == 0, "items of a thread");
      const int head = 2 * (threadIdx.x & 3) + ((threadIdx.x >> 5) & 1);
      float4 acc[kPer];
#pragma unroll
      for (int n = 0; n < kPer; ++n) acc[n] = make_float4(0.f, 0.f, 0.f, 0.f);
      float top = -INFINITY, sum = 0.f;
      const int parts = threadIdx.x < D::kItems ? q.parts : 0;
      for (int k0 = 0; k0 < parts; k0 += kBatch) {
        float m[kBatch], l[kBatch];
        float4 x[kBatch][kPer];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const bool have = k0 + k < q.parts;
          const float* r = rec_of(have ? k0 + k : 0);
          m[k] = have ? __ldcg(r + H * HD + head) : -INFINITY;
          l[k] = __ldcg(r + H * HD + H + head);
#pragma unroll
          for (int n = 0; n < kPer; ++n) {
            x[k][n] = __ldcg(reinterpret_cast<const float4*>(r) + threadIdx.x + n * 32 * W);
          }
        }
        float all = top;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) all = fmaxf(all, m[k]);
        const float keep = part_weight(top, all);
#pragma unroll
        for (int n = 0; n < kPer; ++n) {
          acc[n].x *= keep; acc[n].y *= keep; acc[n].z *= keep; acc[n].w *= keep;
        }
        sum *= keep;
        top = all;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          if (k0 + k >= q.parts) continue;
          const float e = part_weight(m[k], all);
#pragma unroll
          for (int n = 0; n < kPer; ++n) {
            acc[n].x = fmaf(e, x[k][n].x, acc[n].x);
            acc[n].y = fmaf(e, x[k][n].y, acc[n].y);
            acc[n].z = fmaf(e, x[k][n].z, acc[n].z);
            acc[n].w = fmaf(e, x[k][n].w, acc[n].w);
          }
          sum = fmaf(e, l[k], sum);
        }
      }
#pragma unroll
      for (int n = 0; n < kPer; ++n) {
        const int j = threadIdx.x + n * 32 * W;
        if (j < D::kItems) write_out(q, head, 32 * (j >> 6) + 4 * ((j & 31) >> 2), acc[n], top, sum);
      }
      if (threadIdx.x == 0) p.counters[q.group_id] = 0;
    }
  }
  if (!ok) {
    // copies of this warp may still be in flight: let them land before the CTA leaves
    __syncwarp();
    for (const int issued = *sm_issued; used < issued; ++used) {
      (void)mbar_wait_warp(&bars[slot], phase);
      if (++slot == D::kRing) {
        slot = 0;
        phase ^= 1u;
      }
    }
  }
}

template <int HD>
cudaError_t launch_decode_t(const Kv4DecodeParams& p, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  cudaError_t e = set_smem_limit_once(done, reinterpret_cast<const void*>(kv4_decode_kernel<HD>), Dec<HD>::smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)p.grid);
  cfg.blockDim = dim3(32 * Dec<HD>::kWarps);
  cfg.dynamicSmemBytes = Dec<HD>::smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv4_decode_kernel<HD>, p);
}

// A warp per (layer, kv head, tile), as a programmatic dependent.  These kernels let their own dependents start only
// as they end: an early start's waiting CTAs take the slots of a kernel that fills the GPU once (12.9 us against 6.7
// for 29 MB read back).
cudaError_t launch_rows(void (*kernel)(Kv4RowsParams), const Kv4RowsParams& p, cudaStream_t s) {
  const long long items = kv4_row_items(p);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)((items + kRowWarps - 1) / kRowWarps));
  cfg.blockDim = dim3(32 * kRowWarps);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace

int kv4_decode_ctas_per_sm(int head_dim) { return head_dim == 128 ? Dec<128>::kCtas : Dec<64>::kCtas; }

void plan_kv4_decode(Kv4DecodeParams& p, int head_dim, long long slots) {
  const long long reps = (long long)p.n_layers * p.pool.kv_heads * p.head_blocks;
  int acc = 0, longest = 1;
  for (int i = 0; i < p.n_seqs; ++i) {
    const int n = kv4_units(p.seqs[i].len, head_dim);
    p.seqs[i].unit_begin = acc;
    acc += n + kKv4GroupUnits;
    longest = n > longest ? n : longest;
  }
  p.block_units = acc;
  p.total_units = reps * acc;
  // Aligned split: every group in equal parts of at most `most` units, one part a CTA, all of them resident at once;
  // otherwise the stream split, whose CTAs take equal ranges across groups.  A CTA with one segment saves the merges
  // between segments, an uneven share costs its full length: aligned is taken while its longest part is within an
  // eighth of an equal share.  Measured, aligned against stream: 36 layers x 2 kv heads x 4097 tokens 19.0 against
  // 21.3 us, x 8000 27.7 against 31.2, a ragged batch of 8 12.0 against 15.0; where the rule says stream, 28 layers x
  // 4 kv heads x 6000 38.0 against 34.4, x 32768 172 against 136, 64 ragged sequences 75 against 52.
  auto parts_for = [&](int most) {
    long long c = 0;
    for (int i = 0; i < p.n_seqs; ++i) c += (kv4_units(p.seqs[i].len, head_dim) + most - 1) / most;
    return c * reps;
  };
  const long long ideal = (p.total_units + slots - 1) / slots;
  int lo = 1, hi = longest;
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (parts_for(mid) <= slots) hi = mid; else lo = mid + 1;
  }
  if (parts_for(lo) <= slots && lo <= ideal + ideal / 8) {
    int parts = 0;
    for (int i = 0; i < p.n_seqs; ++i) {
      p.seqs[i].part_begin = parts;
      parts += (kv4_units(p.seqs[i].len, head_dim) + lo - 1) / lo;
    }
    p.block_parts = parts;
    p.grid = (int32_t)(reps * parts);
    return;
  }
  p.block_parts = 0;
  p.grid = (int32_t)(p.total_units < slots ? p.total_units : slots);
}

cudaError_t launch_kv4_decode(const Kv4DecodeParams& p, int head_dim, cudaStream_t s) {
  return head_dim == 128 ? launch_decode_t<128>(p, s) : launch_decode_t<64>(p, s);
}

cudaError_t launch_kv4_append(const Kv4RowsParams& p, int head_dim, cudaStream_t s) {
  if (head_dim == 128) return launch_rows(p.input_f16 ? kv4_append_kernel<128, true> : kv4_append_kernel<128, false>, p, s);
  return launch_rows(p.input_f16 ? kv4_append_kernel<64, true> : kv4_append_kernel<64, false>, p, s);
}

cudaError_t launch_kv4_read(const Kv4RowsParams& p, int head_dim, cudaStream_t s) {
  return launch_rows(head_dim == 128 ? kv4_read_kernel<128> : kv4_read_kernel<64>, p, s);
}

cudaError_t launch_kv4_raw(const Kv4RowsParams& p, int head_dim, bool to_pool, cudaStream_t s) {
  const long long n = (long long)p.n_layers * p.n_tokens * p.pool.kv_heads * (head_dim / 32);
  const unsigned grid = (unsigned)((n + 127) / 128);
  if (head_dim == 128) kv4_raw_kernel<128><<<grid, 128, 0, s>>>(p, to_pool ? 1 : 0);
  else kv4_raw_kernel<64><<<grid, 128, 0, s>>>(p, to_pool ? 1 : 0);
  return cudaGetLastError();
}

}  // namespace te
