// The 8-bit KV pool (include/imba_b200.h, "Cache operators"): geometry, the
// blocks' power-of-two scales and the e4m3 conversions, shared by the append
// and attention kernels.
#pragma once

#include <cuda_fp16.h>

#include "kernels.cuh"

namespace imba {

constexpr int kMinScaleByte = 27;  // 2^-100: keeps ratios of two scales inside fp32

// One layer of a pool in 8 bits.  Offsets are in bytes; a page-layer holds
// the K blocks (H x 16 x d_qk), then the V blocks (H x 8 x d_v x 2).
struct Cache8 {
  uint8_t* data;     // the layer's first K block of page 0
  uint8_t* scales;   // the layer's K scale of head 0, page 0
  int64_t page_stride;
  int64_t scale_stride;  // per page
  int64_t num_pages;
  int64_t v_offset;
  int H;
};

inline int64_t cache8_page_bytes(const imba_cache_desc& c) {
  return (int64_t)c.num_layers * c.num_heads * IMBA_PAGE_TOKENS * (c.attention_dim + c.linear_dim);
}

inline Cache8 cache8_layer(const imba_cache_desc& c, const imba_pool_desc& pool, int layer) {
  Cache8 r;
  const int64_t page = cache8_page_bytes(c);
  r.data = static_cast<uint8_t*>(pool.base) + (int64_t)layer * (page / c.num_layers);
  r.scales = static_cast<uint8_t*>(pool.base) + page * pool.num_pages + (int64_t)layer * 2 * c.num_heads;
  r.page_stride = page;
  r.scale_stride = (int64_t)c.num_layers * 2 * c.num_heads;
  r.num_pages = pool.num_pages;
  r.v_offset = (int64_t)c.num_heads * IMBA_PAGE_TOKENS * c.attention_dim;
  r.H = c.num_heads;
  return r;
}

inline PoolGeom cache_geom(const imba_cache_desc& c, int64_t num_pages) {
  PoolGeom g;
  g.H = c.num_heads;
  g.dqk = c.attention_dim;
  g.dv = c.linear_dim;
  g.v_offset = (int64_t)c.num_heads * IMBA_PAGE_TOKENS * c.attention_dim;
  g.layer_stride = (int64_t)c.num_heads * IMBA_PAGE_TOKENS * (c.attention_dim + c.linear_dim);
  g.page_stride = g.layer_stride * c.num_layers;
  g.num_slots = num_pages * IMBA_PAGE_TOKENS;
  return g;
}

// Head dimensions with an 8-bit kernel.
inline bool cache8_dims_ok(int dqk, int dv) {
  auto ok = [](int d) { return d == 32 || d == 64 || d == 96 || d == 128; };
  return ok(dqk) && ok(dv) && (dqk == dv || (dqk <= 64 && dv <= 64));
}

// Scale byte of a block whose largest magnitude is amax (0 for an empty or
// all-zero block): the smallest exponent e with amax <= 448 2^e, as e + 127.
// amax = 1.m 2^x; 448 = 1.75 2^8, so e = x - 8, one more if 1.m > 1.75.
__device__ __forceinline__ int scale_byte(float amax) {
  const uint32_t u = __float_as_uint(amax);
  if (u == 0) return 0;
  const int b = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return b < kMinScaleByte ? kMinScaleByte : b;
}
// 2^(b - 127); 0 for an empty block.
__device__ __forceinline__ float scale_of(int b) { return __uint_as_float((uint32_t)b << 23); }
// 2^(127 - b) for a scale byte b >= kMinScaleByte (b <= 247: amax is finite).
__device__ __forceinline__ float inv_scale_of(int b) { return __uint_as_float((uint32_t)(254 - b) << 23); }

// Two floats to two e4m3 codes, rounded to nearest even (lo in the low byte).
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two e4m3 codes (low 16 bits) to two f16 values, exact.
__device__ __forceinline__ uint32_t e4m3x2_to_h2(uint32_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
  return r;
}
// Four codes: the first two, and the last two.
__device__ __forceinline__ void e4m3x4_to_h2(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(four));
}
__device__ __forceinline__ float2 e4m3x2_to_f2(uint32_t two) {
  const uint32_t h = e4m3x2_to_h2(two);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Byte offset in a V block ([8][d_v][2]) of a token's dimension e.
__device__ __forceinline__ int v8_off(int tok, int e, int dv) { return ((tok >> 1) * dv + e) * 2 + (tok & 1); }

}  // namespace imba
