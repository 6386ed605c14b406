// Attention over a paged pool in 8 bits: numerics and the join of split
// sequences, shared by the mma.sync kernel (few rows a segment) and the
// tcgen05 kernel (many).
#pragma once

#include "attend8.cuh"

namespace imba {

namespace {

constexpr float kShift = 5.f;
constexpr float kSlack = 4.f;
constexpr int kVWindow = 6;  // 2^(kShift + kSlack + kVWindow) = 2^15 is finite in f16
// A V scale that is further below O's units enters as this one: the weights'
// f16 are zero either way, and no weight that counts is lost in the row's sum,
// which is of the scaled weights.
constexpr int kVLeast = -40;

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_h2(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }

// Scores are kept in log2 without a bias (the factor log2 e joins the
// query's), with one as natural logarithms, where the bias is added as it is;
// `lg` takes them to log2.  A weight is 2^(lg (score - maximum) + kShift), the
// maximum subtracted first: that difference is exact where the weight matters.
// (In one step, lg score + (kShift - lg maximum), the product would be rounded,
// by 64 at a mask of -1e9, and its keys would get weights of 2^64 or none.)  So
// keys that carry any mask, the type's lowest value too, weigh by their
// differences alone.
//
// Running maxima start at the lowest finite value, so that the difference to a
// key that is not seen (-inf) is -inf and not NaN; a row that has seen nothing
// has no weight either, whatever its maximum.
constexpr float kLowest = -3.4028234663852886e38f;

// exp of a difference of running maxima.
__device__ __forceinline__ float weight_of(float a, float b, float lg) { return exp2_approx((a - b) * lg); }

// Four consecutive elements of a row as floats.
template <typename T>
__device__ __forceinline__ void q_load4(const T* p, bool vec, float (&x)[4]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      const float4 f = *reinterpret_cast<const float4*>(p);
      x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
      const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
      x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = to_f(p[i]);
  }
}
template <typename T>
__device__ __forceinline__ void out_store4(T* p, bool vec, const float (&x)[4]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
      __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
      *reinterpret_cast<uint2*>(p) =
          make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = from_f<T>(x[i]);
  }
}

// Rows r0 .. r0 + n - 1 of a split tile joined over its items, by `nthr`
// threads from tid on, kAhead parts in flight.  A part is a row's average over
// its keys, with their maximum and sum, and so is what has been joined: sums of
// values at the upper end of fp32 would run over.  The last item's CTA joins alone
// while others idle, so what it costs is latency: 74 parts of 24 rows of 128
// made a call of 140 us with four in flight, of 131 with eight; the tcgen05
// kernel, short of registers there, is 2 % slower with eight.
template <typename T, int DV, int kAhead>
__device__ __forceinline__ void join_items(const AttendArgs& a, const AttendItem& it, int head, float lg, int r0, int n,
                                           int tid, int nthr) {
  const int H = a.cache.H;
  const size_t first = (size_t)(it.part - it.index) * H + head;
  const int tile_rows = a.shape.tile_rows;
  const AttendRow* rows = a.plan.rows + (size_t)it.tile * tile_rows;
  const bool vec = a.call.out_stride[0] % 4 == 0 && a.call.out_stride[1] % 4 == 0 &&
                   (reinterpret_cast<uintptr_t>(a.call.out) & (4 * sizeof(T) - 1)) == 0;
  for (int i = tid; i < n * (DV / 4); i += nthr) {
    const int r = r0 + i / (DV / 4), e = i % (DV / 4) * 4;
    const AttendRow row = rows[r];
    if (row.row < 0) continue;
    float m = kLowest, l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < it.splits; s0 += kAhead) {
      float2 ml[kAhead];
      float4 o[kAhead];
      float now = m;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const size_t at = (first + (size_t)min(s0 + j, it.splits - 1) * H) * tile_rows + r;
        ml[j] = __ldcg(a.plan.ml + at);
        o[j] = __ldcg(reinterpret_cast<const float4*>(a.plan.o + at * DV + e));
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) now = fmaxf(now, ml[j].x);
      const float was = l * weight_of(m, now, lg);
      l = was;
      m = now;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        ml[j].x = s0 + j < it.splits ? weight_of(ml[j].x, m, lg) * ml[j].y : 0.f;
        l += ml[j].x;
      }
      const float inv = l == 0.f ? 0.f : 1.f / l, f = was * inv;
      x[0] *= f, x[1] *= f, x[2] *= f, x[3] *= f;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const float w = ml[j].x * inv;
        x[0] += w * o[j].x, x[1] += w * o[j].y, x[2] += w * o[j].z, x[3] += w * o[j].w;
      }
    }
    out_store4(static_cast<T*>(a.call.out) + row.row * a.call.out_stride[0] +
                   (int64_t)(head * a.shape.share + row.head) * a.call.out_stride[1] + e,
               vec, x);
  }
}

}  // namespace

}  // namespace imba
