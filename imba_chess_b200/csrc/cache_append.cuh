// Appending keys and values to a paged pool with the rotary position applied
// on the way, and reading rows back (include/imba_b200.h, "Cache operators").
//
// Pair p of a head turns by the angle 2 pi pos f_p, with f_p in turns per
// position held as a 64-bit fraction: pos * f_p mod 2^64 is one wrapping
// integer product, so the fraction of a turn is right to 2^-33 at any
// position and needs no floating-point range reduction.  Its sine and cosine
// are Taylor sums in fp64 over an eighth of a turn, rounded once; products
// and sums of the rotation are fp32, and each stored value is rounded once,
// to the pool's type.
//
// The work is grouped by page (append_plan): the scale of a block of 16
// tokens needs the largest magnitude of all its new tokens, and when it grows
// the block's earlier codes are rounded to it, so one warp owns one block.
// Two shapes of work, told apart on the device by the tokens per page:
//  - dense (documents): a CTA takes one page; the cosines and sines of its
//    tokens are computed once for every head, each warp takes K and V blocks
//    in turn, and loads the next block before it works on the last;
//  - sparse (decode steps: one new token in most pages): two warps take a
//    page, lanes are (head, eight elements), and nothing waits for the CTA.
// Queries do not go to a page: a warp turns a row, in row order.
//
// What bounds it: for documents the bytes (1.2 GB of four documents, 8 heads of
// 128 and 32 query heads, in 254 us, 4.8 TB/s; the rotation and the codes hide
// behind the loads of the next block), for prefixes of many games the pages'
// turns and codes as well (52k tokens of 8 heads of 64, 85 us, 3.1 TB/s; the
// kernel of that size spills 180 bytes a thread at its 80 registers), for a
// decode step the launch (1,024 tokens 4.3 us, one token 2.8).
#pragma once

#include <algorithm>

#include "cache_plan.cuh"

namespace imba {

namespace {

struct Strides {
  int64_t tile, row, head, elem;
  // Row r's first element; rows come in tiles of 16 (a step's staged keys and
  // values lie like a pool's pages), tile = 16 row when they are evenly apart.
  __device__ __forceinline__ int64_t at(int64_t r) const { return (r >> 4) * tile + (r & 15) * row; }
};

struct AppendArgs {
  PlanView plan;
  int n, H, Hq, dqk, dv;
  const void *k, *v, *q;
  void* q_out;
  Strides ks, vs, qs, qo;
  imba_rotary_desc rot;
  const int32_t* slots;
  int32_t* status;
  int page_blocks;  // CTAs that store (the first ones); the others turn queries
  int q_rows;       // rows of a query warp
  int64_t num_slots;
};

// The largest magnitude; a NaN stays one.
__device__ __forceinline__ float most3(float m, float x, float y) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(x), "f"(y));
  return r;
}

// Eight elements of the source type as they are in memory.
template <typename T>
struct Raw8;
template <>
struct Raw8<bf16> {
  uint4 u;
  __device__ __forceinline__ void load(const bf16* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void set(int i, bf16 x) {
    uint32_t* w = &u.x + i / 2;
    const uint32_t h = __bfloat16_as_ushort(x);
    *w = i & 1 ? (*w & 0xffffu) | h << 16 : (*w & 0xffff0000u) | h;
  }
  __device__ __forceinline__ void zero() { u = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  // The largest magnitude, together with `most` (a NaN stays one).
  __device__ __forceinline__ float see(float most) const {
    const uint32_t a = __vmaxu2(__vmaxu2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu),
                                __vmaxu2(u.z & 0x7fff7fffu, u.w & 0x7fff7fffu));
    return most3(most, __uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u));
  }
};
template <>
struct Raw8<float> {
  float4 f[2];
  __device__ __forceinline__ void load(const float* p) {
    f[0] = reinterpret_cast<const float4*>(p)[0];
    f[1] = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void set(int i, float x) { (&f[i / 4].x)[i % 4] = x; }
  __device__ __forceinline__ void zero() { f[0] = f[1] = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    x[0] = f[0].x, x[1] = f[0].y, x[2] = f[0].z, x[3] = f[0].w;
    x[4] = f[1].x, x[5] = f[1].y, x[6] = f[1].z, x[7] = f[1].w;
  }
  __device__ __forceinline__ float see(float most) const {
    most = most3(most3(most, f[0].x, f[0].y), f[0].z, f[0].w);
    return most3(most3(most, f[1].x, f[1].y), f[1].z, f[1].w);
  }
};

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Which elements the pairs of a head are made of.  Pairs past rot_dim / 2
// are neighbours and do not turn.
struct PairMap {
  int half, inter;
  __device__ __forceinline__ int first(int p) const { return p >= half || inter ? 2 * p : p; }
  __device__ __forceinline__ int second(int p) const { return p >= half || inter ? 2 * p + 1 : p + half; }
  // Pairs p0 .. p0 + 7 lie side by side, in a run of sixteen; else, when half
  // is a multiple of eight, in two runs of eight.
  __device__ __forceinline__ bool adjacent(int p0) const { return inter || p0 >= half; }
  __device__ __forceinline__ int lo(int p0) const { return adjacent(p0) ? 2 * p0 : p0; }
  __device__ __forceinline__ int hi(int p0) const { return adjacent(p0) ? 2 * p0 + 8 : p0 + half; }
};

// The rotation, each product and sum rounded on its own.
__device__ __forceinline__ void turn(float2 t, float& x, float& y) {
  const float u = x, v = y;
  x = __fsub_rn(__fmul_rn(u, t.x), __fmul_rn(v, t.y));
  y = __fadd_rn(__fmul_rn(v, t.x), __fmul_rn(u, t.y));
}

// Pairs p0 .. p0 + 7 of a head.  Fast: rows of contiguous elements, 16-byte
// aligned, and a half that is a multiple of eight (the host sees to it).
template <typename T, bool Fast>
struct Pairs {
  Raw8<T> a, b;  // fast and adjacent: the run's first and second half; else first and second elements
  __device__ __forceinline__ void load(const T* head, const Strides& st, const PairMap& m, int p0) {
    if constexpr (Fast) {
      a.load(head + m.lo(p0));
      b.load(head + m.hi(p0));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        a.set(i, head[m.first(p0 + i) * st.elem]);
        b.set(i, head[m.second(p0 + i) * st.elem]);
      }
    }
  }
  __device__ __forceinline__ void zero() {
    a.zero();
    b.zero();
  }
  // The elements turned by cs[p0 ..], in the order of memory of a and b.
  __device__ __forceinline__ void turned(const float2* cs, const PairMap& m, int p0, float (&x)[8], float (&y)[8]) const {
    turned_by(reinterpret_cast<const float4*>(cs + p0), cs, m, p0, x, y);
  }
  // t: the eight pairs' turns, two each (fast).
  template <class Four>
  __device__ __forceinline__ void turned_by(const Four& t, const float2* cs, const PairMap& m, int p0, float (&x)[8],
                                            float (&y)[8]) const {
    a.get(x);
    b.get(y);
    if constexpr (Fast) {
      if (p0 >= m.half) return;  // eight pairs turn, or none does
      if (m.inter) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float4 u = t[i], v = t[2 + i];
          turn(make_float2(u.x, u.y), x[4 * i], x[4 * i + 1]);
          turn(make_float2(u.z, u.w), x[4 * i + 2], x[4 * i + 3]);
          turn(make_float2(v.x, v.y), y[4 * i], y[4 * i + 1]);
          turn(make_float2(v.z, v.w), y[4 * i + 2], y[4 * i + 3]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 u = t[i];
          turn(make_float2(u.x, u.y), x[2 * i], y[2 * i]);
          turn(make_float2(u.z, u.w), x[2 * i + 1], y[2 * i + 1]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (p0 + i < m.half) turn(cs[p0 + i], x[i], y[i]);
    }
  }
  template <typename TO>
  static __device__ __forceinline__ void store(TO* head, const Strides& st, const PairMap& m, int p0,
                                               const float (&x)[8], const float (&y)[8]) {
    if constexpr (Fast) {
      store8(head + m.lo(p0), x);
      store8(head + m.hi(p0), y);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        head[m.first(p0 + i) * st.elem] = from_f<TO>(x[i]);
        head[m.second(p0 + i) * st.elem] = from_f<TO>(y[i]);
      }
    }
  }
};

// Eight dimensions of a value row.
template <typename T, bool Fast>
__device__ __forceinline__ void load_run(Raw8<T>& raw, const T* p, const Strides& st) {
  if constexpr (Fast) {
    raw.load(p);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) raw.set(i, p[i * st.elem]);
  }
}

// (cos, sin) of a 64-bit fraction of a turn.  The nearest quarter is taken
// off exactly; on what is left, |x| <= pi / 4, the Taylor sums to x^11 and
// x^12 are right to 2^-36.
__device__ __forceinline__ float2 cos_sin(uint64_t t) {
  const uint32_t quarter = (uint32_t)((t + (1ull << 61)) >> 62);
  const double x = (double)(int64_t)(t - ((uint64_t)quarter << 62)) * (6.283185307179586476925 / 18446744073709551616.0);
  const double z = x * x;
  double s = fma(z, -1.0 / 39916800, 1.0 / 362880);
  s = fma(z, s, -1.0 / 5040);
  s = fma(z, s, 1.0 / 120);
  s = fma(z, s, -1.0 / 6);
  s = fma(z * x, s, x);
  double c = fma(z, 1.0 / 479001600, -1.0 / 3628800);
  c = fma(z, c, 1.0 / 40320);
  c = fma(z, c, -1.0 / 720);
  c = fma(z, c, 1.0 / 24);
  c = fma(z, c, -0.5);
  c = fma(z, c, 1.0);
  const float fs = (float)s, fc = (float)c;
  const float a = quarter & 1 ? fs : fc, b = quarter & 1 ? fc : fs;
  return make_float2(quarter == 1 || quarter == 2 ? -a : a, quarter & 2 ? -b : b);
}

// What row r turns pair p by.
__device__ __forceinline__ float2 row_turn(const imba_rotary_desc& rot, int64_t r, int p) {
  const int ax = rot.axis ? min(max(rot.axis[p], 0), rot.num_axes - 1) : 0;
  return cos_sin((uint64_t)(int64_t)rot.positions[r * rot.num_axes + ax] * rot.turns[p]);
}

// Every pair of the CTA's tokens (rows[t] < 0: none).
__device__ __forceinline__ void fill_turns(const imba_rotary_desc& rot, const int* rows, float2 (*cs)[kMaxPairs]) {
  const int half = rot.rot_dim / 2;
  for (int t = threadIdx.x / 32; t < kTok; t += kWarps) {
    const int r = rows[t];
    if (r < 0) continue;
    for (int p = threadIdx.x % 32; p < half; p += 32) cs[t][p] = row_turn(rot, r, p);
  }
}

// Lanes of a warp on one row: N lanes of a head, heads side by side.
template <int N>
struct RowLanes {
  static constexpr int kLanes = N <= 2 ? 2 : N <= 4 ? 4 : N <= 8 ? 8 : 16;  // a power of two
  static constexpr int kHeads = 32 / kLanes;
};

// A warp turns rows r0 .. r0 + n - 1 (n <= N; those in the mask `live`) of
// `heads` heads, from src to dst(row).  N rows' turns go to cs[0 .. N - 1].
template <int N, typename T, typename TO, int D, bool Fast, class Dst>
__device__ __forceinline__ void turn_rows(const imba_rotary_desc& rot, int64_t r0, uint32_t live, int heads,
                                          const T* src, const Strides& ss, const Dst& dst, const Strides& ds,
                                          float2 (*cs)[kMaxPairs]) {
  using L = RowLanes<D / 16>;
  constexpr int kAhead = sizeof(T) == 2 ? 4 : 2;  // passes in flight; a pass is kHeads heads of a row
  const int lane = threadIdx.x % 32, l = lane % L::kLanes, p0 = l * 8;
  const PairMap m{rot.rot_dim / 2, rot.interleaved};
  const int groups = (heads + L::kHeads - 1) / L::kHeads, passes = groups * (N == 1 ? 1 : 32 - __clz(live));
  bool filled = false;
  float4 mine[4];  // the turns of this lane's pairs, of a single row (fast)
  for (int j0 = 0; j0 < passes; j0 += kAhead) {
    Pairs<T, Fast> raw[kAhead];
    auto place = [&](int i, int* row, int* h) {
      const int j = j0 + i;
      *row = N == 1 ? 0 : j / groups;
      *h = (j - *row * groups) * L::kHeads + lane / L::kLanes;
      return j < passes && live >> *row & 1 && *h < heads && l < D / 16;
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      int row, h;
      if (place(i, &row, &h)) raw[i].load(src + ss.at(r0 + row) + h * ss.head, ss, m, p0);
    }
    if (!filled) {  // behind the first loads
      __syncwarp();  // the last rows' are done with
#pragma unroll
      for (int row = 0; row < N; ++row)
        if (live >> row & 1)
          for (int p = lane; p < m.half; p += 32) cs[row][p] = row_turn(rot, r0 + row, p);
      __syncwarp();
      if constexpr (N == 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) mine[i] = reinterpret_cast<const float4*>(cs[0] + min(p0, D / 2 - 8))[i];
      }
      filled = true;
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      int row, h;
      if (!place(i, &row, &h)) continue;
      float x[8], y[8];
      if constexpr (N == 1)
        raw[i].turned_by(mine, cs[0], m, p0, x, y);
      else
        raw[i].turned(cs[row], m, p0, x, y);
      Pairs<T, Fast>::store(dst(r0 + row) + h * ds.head, ds, m, p0, x, y);
    }
  }
}

// Any head size: one lane per pair of the row; an odd last element passes.
template <typename T, typename TO>
__device__ __forceinline__ void turn_row_any(const imba_rotary_desc& rot, int64_t r, int heads, int dim, const T* src,
                                             const Strides& ss, TO* dst, const Strides& ds, float2* cs) {
  const PairMap m{rot.rot_dim / 2, rot.interleaved};
  const int lane = threadIdx.x % 32, pairs = (dim + 1) / 2;
  __syncwarp();
  for (int p = lane; p < m.half; p += 32) cs[p] = row_turn(rot, r, p);
  __syncwarp();
  for (int i = lane; i < heads * pairs; i += 32) {
    const int h = i / pairs, p = i % pairs;
    const T* s = src + h * ss.head;
    TO* o = dst + h * ds.head;
    float x = to_f(s[m.first(p) * ss.elem]);
    if (m.second(p) < dim) {
      float y = to_f(s[m.second(p) * ss.elem]);
      if (p < m.half) turn(cs[p], x, y);
      o[m.second(p) * ds.elem] = from_f<TO>(y);
    }
    o[m.first(p) * ds.elem] = from_f<TO>(x);
  }
}

// The first row of a query warp, and which of its rows have a slot in the pool.
__device__ __forceinline__ int64_t query_rows(const AppendArgs& a, uint32_t* live) {
  const int64_t r0 = ((int64_t)(blockIdx.x - a.page_blocks) * kWarps + threadIdx.x / 32) * a.q_rows;
  const int64_t r = r0 + threadIdx.x % 32;
  const int64_t slot = threadIdx.x % 32 < a.q_rows && r < a.n ? a.slots[r] : -1;
  *live = __ballot_sync(0xffffffffu, slot >= 0 && slot < a.num_slots);
  return r0;
}

// The queries of a warp: a row, or with many of them kQueryRows, so that the
// loads of several are in flight at once.
constexpr int kQueryRows = 2 * kTok / kWarps;
template <typename T, int D, bool Fast>
__device__ __forceinline__ void turn_queries(const AppendArgs& a, float2 (*cs)[kMaxPairs]) {
  uint32_t live;
  const int64_t r0 = query_rows(a, &live);
  if (!live) return;
  auto dst = [&](int64_t r) { return static_cast<T*>(a.q_out) + a.qo.at(r); };
  if (a.q_rows == 1)
    turn_rows<1, T, T, D, Fast>(a.rot, r0, live, a.Hq, static_cast<const T*>(a.q), a.qs, dst, a.qo, cs);
  else
    turn_rows<kQueryRows, T, T, D, Fast>(a.rot, r0, live, a.Hq, static_cast<const T*>(a.q), a.qs, dst, a.qo, cs);
}

__device__ __forceinline__ float see(const float (&x)[8], float most) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) most = most3(most, x[i], x[i + 1]);
  return most;
}
// What is not finite becomes zero, and the last half step below 2^128 does
// not round up to it (240 2^120 is the largest stored value).
__device__ __forceinline__ void take_finite(float (&x)[8], bool& bad) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (!isfinite(x[i])) {
      bad = true;
      x[i] = 0.f;
    }
    x[i] = fminf(fmaxf(x[i], -kLargest), kLargest);
  }
}

// 2^(was - now) for the codes of a block whose scale grows; below 2^-126
// every code becomes zero all the same.
__device__ __forceinline__ float shrink(int was, int now) {
  return now - was > 126 ? 0.f : __uint_as_float((uint32_t)(127 - (now - was)) << 23);
}
// Sixteen codes rounded to a larger scale.
__device__ __forceinline__ void rescale16(uint4* p, float f) {
  const uint4 u = *p;
  uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 lo = e4m3x2_to_f2(w[j] & 0xffffu), hi = e4m3x2_to_f2(w[j] >> 16);
    w[j] = to_e4m3x2(lo.x * f, lo.y * f) | to_e4m3x2(hi.x * f, hi.y * f) << 16;
  }
  *p = make_uint4(w[0], w[1], w[2], w[3]);
}

// The block's new scale byte, its earlier codes rounded to it (whole warp).
template <int D>
__device__ __forceinline__ int grow_scale(uint8_t* block, uint8_t* scale, int was, float most, int lane) {
  const int now = max(was, scale_byte(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)))));
  if (now > was) {
    if (was > 0) {
      const float f = shrink(was, now);
#pragma unroll 1
      for (int i = 0; i < D * kTok / 512; ++i) rescale16(reinterpret_cast<uint4*>(block) + i * 32 + lane, f);
    }
    __syncwarp();  // before the new codes
    if (lane == 0) *scale = (uint8_t)now;
  }
  return now;
}

__device__ __forceinline__ uint2 codes8(const float (&x)[8], float f) {
  return make_uint2(to_e4m3x2(x[0] * f, x[1] * f) | to_e4m3x2(x[2] * f, x[3] * f) << 16,
                    to_e4m3x2(x[4] * f, x[5] * f) | to_e4m3x2(x[6] * f, x[7] * f) << 16);
}
// Codes of pairs p0 .. p0 + 7 of a token's K row.
template <bool Fast>
__device__ __forceinline__ void store_k8(uint8_t* o, const PairMap& m, int p0, const float (&x)[8], const float (&y)[8],
                                         float f) {
  if constexpr (Fast) {
    *reinterpret_cast<uint2*>(o + m.lo(p0)) = codes8(x, f);
    *reinterpret_cast<uint2*>(o + m.hi(p0)) = codes8(y, f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t two = to_e4m3x2(x[j] * f, y[j] * f);
      o[m.first(p0 + j)] = (uint8_t)two;
      o[m.second(p0 + j)] = (uint8_t)(two >> 8);
    }
  }
}

// A warp's share of a dense page: the K block of one head.  A lane holds
// eight pairs of every kGroup-th token.
template <typename T, int D, bool Fast>
struct KBlock {
  static constexpr int kLanes = D / 16, kGroup = 32 / kLanes, kPass = (kTok + kGroup - 1) / kGroup;
  Pairs<T, Fast> raw[kPass];
  int was;

  static __device__ __forceinline__ int token(int i) {
    const int lane = threadIdx.x % 32, t = i * kGroup + lane / kLanes;
    return lane / kLanes < kGroup && t < kTok ? t : -1;
  }
  __device__ __forceinline__ void load(const AppendArgs& a, const int* rows, int h, const uint8_t* scale) {
    const PairMap m{a.rot.rot_dim / 2, a.rot.interleaved};
    const int p0 = threadIdx.x % 32 % kLanes * 8;
    was = *scale;
#pragma unroll
    for (int i = 0; i < kPass; ++i) {
      const int t = token(i), r = t < 0 ? -1 : rows[t];
      if (r < 0)
        raw[i].zero();
      else
        raw[i].load(static_cast<const T*>(a.k) + a.ks.at(r) + h * a.ks.head, a.ks, m, p0);
    }
  }
  // The rotation is done twice, for the block's magnitude and for its codes:
  // the rotated values of sixteen tokens would take more registers than the
  // loads of the next block leave.
  __device__ __forceinline__ void put(const AppendArgs& a, const int* rows, float2 (*cs)[kMaxPairs], uint8_t* block,
                                      uint8_t* scale, bool& bad) const {
    const PairMap m{a.rot.rot_dim / 2, a.rot.interleaved};
    const int lane = threadIdx.x % 32, p0 = lane % kLanes * 8;
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < kPass; ++i) {
      const int t = token(i);
      if (t < 0 || rows[t] < 0) continue;
      float x[8], y[8];
      raw[i].turned(cs[t], m, p0, x, y);
      most = see(x, see(y, most));
    }
    const bool odd = __any_sync(0xffffffffu, !(most <= kLargest));
    if (odd) {
      most = 0.f;
#pragma unroll
      for (int i = 0; i < kPass; ++i) {
        const int t = token(i);
        if (t < 0 || rows[t] < 0) continue;
        float x[8], y[8];
        raw[i].turned(cs[t], m, p0, x, y);
        take_finite(x, bad);
        take_finite(y, bad);
        most = see(x, see(y, most));
      }
    }
    __syncwarp();
    const int b = grow_scale<D>(block, scale, was, most, lane);
    const float f = b ? inv_scale_of(b) : 0.f;
#pragma unroll
    for (int i = 0; i < kPass; ++i) {
      const int t = token(i);
      if (t < 0 || rows[t] < 0) continue;
      float x[8], y[8];
      raw[i].turned(cs[t], m, p0, x, y);
      if (odd) {
        take_finite(x, bad);
        take_finite(y, bad);
      }
      store_k8<Fast>(block + t * D, m, p0, x, y, f);
    }
  }
};

// The V block of one head.  A lane holds eight dimensions of a pair of
// tokens: one 16-byte store of [8][d_v][2].
template <typename T, int D, bool Fast>
struct VBlock {
  static constexpr int kLanes = D / 8, kGroup = 32 / kLanes, kPass = (kTok / 2 + kGroup - 1) / kGroup;
  Raw8<T> raw[kPass][2];
  int was;

  static __device__ __forceinline__ int pair(int i) {
    const int lane = threadIdx.x % 32, p = i * kGroup + lane / kLanes;
    return lane / kLanes < kGroup && p < kTok / 2 ? p : -1;
  }
  __device__ __forceinline__ void load(const AppendArgs& a, const int* rows, int h, const uint8_t* scale) {
    const int e = threadIdx.x % 32 % kLanes * 8;
    was = *scale;
#pragma unroll
    for (int i = 0; i < kPass; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int p = pair(i), r = p < 0 ? -1 : rows[2 * p + j];
        if (r < 0)
          raw[i][j].zero();
        else
          load_run<T, Fast>(raw[i][j], static_cast<const T*>(a.v) + a.vs.at(r) + h * a.vs.head + e * a.vs.elem, a.vs);
      }
  }
  __device__ __forceinline__ void put(const AppendArgs& a, const int* rows, uint8_t* block, uint8_t* scale,
                                      bool& bad) const {
    const int lane = threadIdx.x % 32, e = lane % kLanes * 8;
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < kPass; ++i) most = raw[i][0].see(raw[i][1].see(most));
    const bool odd = __any_sync(0xffffffffu, !(most <= kLargest));
    if (odd) {
      most = 0.f;
#pragma unroll
      for (int i = 0; i < kPass; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float x[8];
          raw[i][j].get(x);
          take_finite(x, bad);
          most = see(x, most);
        }
    }
    __syncwarp();
    const int b = grow_scale<D>(block, scale, was, most, lane);
    const float f = b ? inv_scale_of(b) : 0.f;
#pragma unroll
    for (int i = 0; i < kPass; ++i) {
      const int p = pair(i);
      if (p < 0) continue;
      const bool even = rows[2 * p] >= 0, other = rows[2 * p + 1] >= 0;
      if (!even && !other) continue;
      float x[8], y[8];
      raw[i][0].get(x);
      raw[i][1].get(y);
      if (odd) {
        take_finite(x, bad);
        take_finite(y, bad);
      }
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = to_e4m3x2(x[2 * j] * f, y[2 * j] * f) | to_e4m3x2(x[2 * j + 1] * f, y[2 * j + 1] * f) << 16;
      uint4* o = reinterpret_cast<uint4*>(block + v8_off(2 * p, e, D));
      if (!(even && other)) {  // keep the other token's bytes
        const uint4 u = *o;
        const uint32_t keep = even ? 0xff00ff00u : 0x00ff00ffu;
        w[0] = (w[0] & ~keep) | (u.x & keep);
        w[1] = (w[1] & ~keep) | (u.y & keep);
        w[2] = (w[2] & ~keep) | (u.z & keep);
        w[3] = (w[3] & ~keep) | (u.w & keep);
      }
      *o = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
};

// The single new token of a page, offset t, in one head of K or V: the
// codes' scale (kLanes lanes a head; every lane of the warp takes part).
template <int D, int kLanes, int kUsed>
__device__ __forceinline__ int one_scale(uint8_t* block, uint8_t* scale, int was, float most, bool live, bool* again) {
#pragma unroll
  for (int o = 1; o < kLanes; o *= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  const int l = threadIdx.x % kLanes, now = max(was, scale_byte(most));
  *again = live && now > was && was > 0;
  if (*again)
    for (int i = l; i < D * kTok / 16; i += kUsed) rescale16(reinterpret_cast<uint4*>(block) + i, shrink(was, now));
  __syncwarp();
  if (live && now > was && l == 0) *scale = (uint8_t)now;
  return now;
}

// A warp stores the K heads of row r at offset t of a page.
template <typename T, int D, bool Fast>
__device__ __forceinline__ void one_k8(const AppendArgs& a, int64_t r, int t, uint8_t* blocks, uint8_t* scales,
                                       float2* cs, bool& bad) {
  using L = RowLanes<D / 16>;
  const int lane = threadIdx.x % 32, l = lane % L::kLanes, p0 = l * 8;
  const PairMap m{a.rot.rot_dim / 2, a.rot.interleaved};
  bool filled = false;
  for (int h0 = 0; h0 < a.H; h0 += L::kHeads) {
    const int h = h0 + lane / L::kLanes;
    const bool live = h < a.H && l < D / 16;
    uint8_t *block = blocks + (int64_t)h * kTok * D, *scale = scales + h;
    Pairs<T, Fast> raw;
    raw.zero();
    int was = 0;
    if (live) {
      was = *scale;
      raw.load(static_cast<const T*>(a.k) + a.ks.at(r) + h * a.ks.head, a.ks, m, p0);
    }
    if (!filled) {
      __syncwarp();
      for (int p = lane; p < m.half; p += 32) cs[p] = row_turn(a.rot, r, p);
      __syncwarp();
      filled = true;
    }
    float x[8], y[8];
    raw.turned(cs, m, min(p0, D / 2 - 8), x, y);
    float most = see(x, see(y, 0.f));
    if (!(most <= kLargest)) {
      take_finite(x, bad);
      take_finite(y, bad);
      most = see(x, see(y, 0.f));
    }
    __syncwarp();
    bool again;
    const int now = one_scale<D, L::kLanes, D / 16>(block, scale, was, most, live, &again);
    if (live) store_k8<Fast>(block + t * D, m, p0, x, y, now ? inv_scale_of(now) : 0.f);
  }
}

// The same for V, with the neighbour's bytes of the pair kept.
template <typename T, int D, bool Fast>
__device__ __forceinline__ void one_v8(const AppendArgs& a, int64_t r, int t, uint8_t* blocks, uint8_t* scales,
                                       bool& bad) {
  using L = RowLanes<D / 8>;
  constexpr int kAhead = 2;
  const int lane = threadIdx.x % 32, l = lane % L::kLanes;
  for (int h0 = 0; h0 < a.H; h0 += kAhead * L::kHeads) {
    Raw8<T> raw[kAhead];
    uint4 old[kAhead];
    int was[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int h = h0 + i * L::kHeads + lane / L::kLanes;
      raw[i].zero();
      was[i] = 0;
      if (h < a.H && l < D / 8) {
        was[i] = scales[h];
        load_run<T, Fast>(raw[i], static_cast<const T*>(a.v) + a.vs.at(r) + h * a.vs.head + l * 8 * a.vs.elem, a.vs);
        old[i] = *reinterpret_cast<const uint4*>(blocks + (int64_t)h * kTok * D + v8_off(t & ~1, l * 8, D));
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int h = h0 + i * L::kHeads + lane / L::kLanes;
      const bool live = h < a.H && l < D / 8;
      uint8_t* block = blocks + (int64_t)h * kTok * D;
      float x[8];
      raw[i].get(x);
      float most = raw[i].see(0.f);
      if (!(most <= kLargest)) {
        take_finite(x, bad);
        most = see(x, 0.f);
      }
      __syncwarp();
      bool again;
      const int now = one_scale<D, L::kLanes, D / 8>(block, scales + h, was[i], most, live, &again);
      if (!live) continue;
      const float f = now ? inv_scale_of(now) : 0.f;
      uint4* o = reinterpret_cast<uint4*>(block + v8_off(t & ~1, l * 8, D));
      if (again) old[i] = *o;
      const int up = (t & 1) * 8;
      const uint32_t keep = t & 1 ? 0x00ff00ffu : 0xff00ff00u;
      auto spread = [&](float lo, float hi) {  // the codes of two dimensions at the token's place of each pair
        const uint32_t two = to_e4m3x2(lo * f, hi * f);
        return ((two & 0xffu) | (two & 0xff00u) << 8) << up;
      };
      *o = make_uint4(spread(x[0], x[1]) | (old[i].x & keep), spread(x[2], x[3]) | (old[i].y & keep),
                      spread(x[4], x[5]) | (old[i].z & keep), spread(x[6], x[7]) | (old[i].w & keep));
    }
  }
}

constexpr int kSparse = kWarps / 2;  // pages of a CTA in the sparse shape

// A block's registers decide how many CTAs an SM holds: bf16 blocks of 64
// dimensions take 3, wider ones and fp32 ones of 64 take 2, wider fp32 ones 1.
constexpr int append_ctas(int bytes, int d) { return bytes * d <= 128 ? 3 : bytes * d <= 256 ? 2 : 1; }

template <typename T, int DQK, int DV, bool Fast>
__global__ void __launch_bounds__(kThreads, append_ctas(sizeof(T), DQK > DV ? DQK : DV))
    append8_kernel(AppendArgs a, Cache8 c) {
  __shared__ int rows[3][kTok];
  __shared__ __align__(16) float2 cs[2][kTok][kMaxPairs];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if ((int)blockIdx.x >= a.page_blocks) {
    turn_queries<T, DQK, Fast>(a, cs[0] + warp * kQueryRows);
    return;
  }
  const int count = *a.plan.count + 1;
  const int first = blockIdx.x, step = a.page_blocks;
  bool bad = false;

  auto page_of = [&](int at) {  // -1: a plan of another pool
    const int page = a.plan.keys[at];
    return page < c.num_pages ? page : -1;
  };
  // One page by the whole CTA, its rows in rows[now], K's first blocks loaded
  // in k and their turns to be put in cs[side].  A warp takes K and V of
  // every kWarps-th head in turn, each block's loads before the work on the
  // last; `ahead` runs behind the first loads, and what it puts in the other
  // buffers is there for `next`, which runs before the last V block's work.
  auto dense = [&](int page, int now, int side, KBlock<T, DQK, Fast>& k, auto&& ahead, auto&& next) {
    uint8_t *kb = c.data + page * c.page_stride, *vb = kb + c.v_offset, *scales = c.scales + page * c.scale_stride;
    VBlock<T, DV, Fast> v;
    int h = warp;
    if (h < a.H) v.load(a, rows[now], h, scales + a.H + h);
    ahead();
    fill_turns(a.rot, rows[now], cs[side]);
    __syncthreads();
    for (; h < a.H; h += kWarps) {
      k.put(a, rows[now], cs[side], kb + (int64_t)h * kTok * DQK, scales + h, bad);
      const bool more = h + kWarps < a.H;
      if (more)
        k.load(a, rows[now], h + kWarps, scales + h + kWarps);
      else
        next();
      v.put(a, rows[now], vb + (int64_t)h * kTok * DV, scales + a.H + h, bad);
      if (more) v.load(a, rows[now], h + kWarps, scales + a.H + h + kWarps);
    }
    if (warp >= a.H) next();
  };

  if (2 * (int64_t)count <= a.n) {
    // Dense.  Three buffers of rows and two of turns: while the slowest warp is
    // at one page's, the fastest has come to write the rows after the next and
    // the turns of the next.
    int e = first, now = 0, side = 0, page = -1;
    if (e >= count) return;
    {
      const int at = a.plan.list[e];
      page = page_of(at);
      if (threadIdx.x < kTok) rows[0][threadIdx.x] = page < 0 ? -1 : a.plan.rows[(size_t)at * kTok + threadIdx.x];
    }
    __syncthreads();
    KBlock<T, DQK, Fast> k;
    auto load_k = [&](int buf, int pg) {
      if (warp < a.H) k.load(a, rows[buf], warp, c.scales + max(pg, 0) * c.scale_stride + warp);
    };
    load_k(0, page);
    for (; e < count; e += step) {
      const int after = now == 2 ? 0 : now + 1;
      int next_page = -1;
      auto ahead = [&] {
        if (e + step < count) {
          const int at = a.plan.list[e + step];
          next_page = page_of(at);
          if (threadIdx.x < kTok)
            rows[after][threadIdx.x] = next_page < 0 ? -1 : a.plan.rows[(size_t)at * kTok + threadIdx.x];
        }
      };
      auto next = [&] {
        if (e + step < count) load_k(after, next_page);
      };
      dense(max(page, 0), now, side, k, ahead, next);  // (no rows of a page of another pool)
      page = next_page;
      now = after;
      side ^= 1;
    }
  } else {
    for (int e0 = first * kSparse; e0 < count; e0 += step * kSparse) {
      const int e = e0 + warp / 2;
      int page = -1, at = 0, r = -1, tok = 0, live = 0;
      if (e < count) {
        at = a.plan.list[e];
        page = a.plan.keys[at];
        if (page >= c.num_pages) page = -1;
        const int mine = lane < kTok ? a.plan.rows[(size_t)at * kTok + lane] : -1;
        const uint32_t set = __ballot_sync(0xffffffffu, mine >= 0);
        live = page < 0 ? 0 : __popc(set);
        tok = __ffs(set) - 1;
        r = __shfl_sync(0xffffffffu, mine, max(tok, 0));
      }
      if (live == 1) {  // one of the page's warps takes K, the other V
        uint8_t *kb = c.data + page * c.page_stride, *scales = c.scales + page * c.scale_stride;
        if (warp % 2 == 0)
          one_k8<T, DQK, Fast>(a, r, tok, kb, scales, cs[0][warp], bad);
        else
          one_v8<T, DV, Fast>(a, r, tok, kb + c.v_offset, scales + a.H, bad);
      }
      // Pages with several new tokens, one after the other.
      if (__syncthreads_or(live > 1)) {
        for (int i = 0; i < kSparse; ++i) {
          if (warp == 2 * i && lane < kTok) rows[0][lane] = live > 1 ? a.plan.rows[(size_t)at * kTok + lane] : -1;
          if (warp == 2 * i && lane == 0) rows[1][0] = live > 1 ? page : -1;
          __syncthreads();
          const int now = rows[1][0];
          if (now >= 0) {
            KBlock<T, DQK, Fast> k;
            if (warp < a.H) k.load(a, rows[0], warp, c.scales + now * c.scale_stride + warp);
            dense(now, 0, 0, k, [] {}, [] {});
          }
          __syncthreads();
        }
      }
    }
  }
  if (bad) report(a.status, IMBA_ERR_RANGE);
}

// Pools in full precision: no scale, so a warp takes a token.  D: d_qk, or 0
// for any head sizes and alignments.
template <typename T, typename TP, int D>
__global__ void __launch_bounds__(kThreads) append_kernel(AppendArgs a, PoolGeom g, TP* pool, int layer) {
  __shared__ __align__(16) float2 cs[kWarps * kQueryRows][kMaxPairs];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if ((int)blockIdx.x >= a.page_blocks) {
    if constexpr (D > 0) {
      turn_queries<T, D, true>(a, cs + warp * kQueryRows);
    } else {
      uint32_t live;
      const int64_t r0 = query_rows(a, &live);
      for (; live; live &= live - 1) {
        const int64_t r = r0 + __ffs(live) - 1;
        turn_row_any<T, T>(a.rot, r, a.Hq, a.dqk, static_cast<const T*>(a.q) + a.qs.at(r), a.qs,
                           static_cast<T*>(a.q_out) + a.qo.at(r), a.qo, cs[warp * kQueryRows]);
      }
    }
    return;
  }
  const int count = *a.plan.count + 1;
  const Strides ks{0, 0, (int64_t)kTok * g.dqk, 1};
  const int64_t step = (int64_t)a.page_blocks * kWarps;
  for (int64_t u = (int64_t)blockIdx.x * kWarps + warp; u < (int64_t)count * kTok; u += step) {
    const int at = a.plan.list[u / kTok];
    const int r = a.plan.rows[(size_t)at * kTok + u % kTok];
    const int64_t slot = (int64_t)a.plan.keys[at] * kTok + u % kTok;
    if (r < 0 || slot < 0 || slot >= g.num_slots) continue;  // the latter: a plan of another pool
    const T* k = static_cast<const T*>(a.k) + a.ks.at(r);
    const T* v = static_cast<const T*>(a.v) + a.vs.at(r);
    TP *ko = pool + g.k_off(slot, layer, 0), *vo = pool + g.v_off(slot, layer, 0);
    if constexpr (D > 0) {
      const int runs = g.dv / 8;
      for (int i = lane; i < a.H * runs; i += 32) {
        const int h = i / runs, e = i % runs * 8;
        Raw8<T> raw;
        float x[8];
        raw.load(v + h * a.vs.head + e);
        raw.get(x);
        store8(vo + (int64_t)h * kTok * g.dv + e, x);
      }
      turn_rows<1, T, TP, D, true>(a.rot, r, 1, a.H, static_cast<const T*>(a.k), a.ks,
                                   [&](int64_t) { return ko; }, ks, cs + warp);
    } else {
      turn_row_any<T, TP>(a.rot, r, a.H, g.dqk, k, a.ks, ko, ks, cs[warp]);
      for (int i = lane; i < a.H * g.dv; i += 32)
        vo[(int64_t)(i / g.dv) * kTok * g.dv + i % g.dv] =
            from_f<TP>(to_f(v[i / g.dv * a.vs.head + i % g.dv * a.vs.elem]));
    }
  }
}

// Strides of a source, and whether its rows are contiguous and 16-byte aligned.
template <typename T>
bool take_strides(const int64_t (&s)[3], const void* base, int64_t tile, Strides* out) {
  *out = Strides{tile ? tile : 16 * s[0], s[0], s[1], s[2]};
  constexpr int64_t e = 16 / sizeof(T);
  return s[2] == 1 && out->tile % e == 0 && s[0] % e == 0 && s[1] % e == 0 && (reinterpret_cast<uintptr_t>(base) & 15) == 0;
}

template <typename T, int DQK, int DV>
cudaError_t launch_append8(dim3 grid, const AppendArgs& a, const Cache8& l, bool fast, cudaStream_t s) {
  return fast ? launch_pdl(append8_kernel<T, DQK, DV, true>, grid, dim3(kThreads), 0, s, a, l)
              : launch_pdl(append8_kernel<T, DQK, DV, false>, grid, dim3(kThreads), 0, s, a, l);
}

template <typename T, typename TP>
cudaError_t launch_append_full(dim3 grid, const AppendArgs& a, const PoolGeom& g, void* pool, int layer, bool fast,
                               cudaStream_t s) {
  TP* p = static_cast<TP*>(pool);
  if (fast && g.dv % 8 == 0) {
    if (g.dqk == 32) return launch_pdl(append_kernel<T, TP, 32>, grid, dim3(kThreads), 0, s, a, g, p, layer);
    if (g.dqk == 64) return launch_pdl(append_kernel<T, TP, 64>, grid, dim3(kThreads), 0, s, a, g, p, layer);
    if (g.dqk == 96) return launch_pdl(append_kernel<T, TP, 96>, grid, dim3(kThreads), 0, s, a, g, p, layer);
    if (g.dqk == 128) return launch_pdl(append_kernel<T, TP, 128>, grid, dim3(kThreads), 0, s, a, g, p, layer);
  }
  return launch_pdl(append_kernel<T, TP, 0>, grid, dim3(kThreads), 0, s, a, g, p, layer);
}

}  // namespace

template <typename T>
imba_status_t launch_append(const imba_cache_desc& c, const imba_pool_desc& pool, const imba_append_desc& d,
                            void* plan, cudaStream_t s, int64_t k_tile, int64_t v_tile) {
  AppendArgs a;
  a.plan = plan_view(plan, d.num_rows);
  a.n = d.num_rows;
  a.H = c.num_heads;
  a.Hq = d.q ? d.num_q_heads : 0;
  a.dqk = c.attention_dim;
  a.dv = c.linear_dim;
  a.k = d.k, a.v = d.v, a.q = d.q, a.q_out = d.q_out;
  // Fast: runs of eight elements by 16-byte accesses.  A rotation whose halves
  // are no multiple of eight cuts runs in two, and rows that are not contiguous
  // or aligned have none: these go by single elements (8 heads of 64 as fast
  // rows, 52k tokens 85 us; 120k tokens of 2 + 16 heads of 64, 58 of 64 elements
  // rotated, 588 us for 585 MB, a sixth of the rate).
  bool fast = d.rotary.rot_dim % 16 == 0;
  fast &= take_strides<T>(d.k_stride, d.k, k_tile, &a.ks);
  fast &= take_strides<T>(d.v_stride, d.v, v_tile, &a.vs);
  const bool q_fast = take_strides<T>(d.q_stride, d.q, 0, &a.qs);
  const bool o_fast = take_strides<T>(d.q_out_stride, d.q_out, 0, &a.qo);
  fast &= !d.q || (q_fast && o_fast);
  a.rot = d.rotary;
  a.slots = d.slots;
  a.status = d.status;
  a.num_slots = pool.num_pages * kTok;
  // A row of few heads is one or two passes of a warp: several rows then keep
  // its loads in flight (52k rows of 8 heads of 64 84 us with four, 98 with one;
  // rows of 32 heads of 128 274 and 250), if the SMs stay full.
  a.q_rows = d.num_rows >= 148 * 2 * kWarps * kQueryRows && a.Hq * c.attention_dim <= 1024 ? kQueryRows : 1;
  const int64_t q_blocks = a.Hq ? (d.num_rows + kWarps * a.q_rows - 1) / (kWarps * a.q_rows) : 0;
  cudaError_t e = cudaErrorInvalidValue;
  if (c.dtype == IMBA_DTYPE_E4M3) {
    // A page a CTA with two tokens or more in it on average, else kSparse
    // (1,024 games' tokens, one a page: 12.2 us by CTA, 4.3 by warps; 1,024
    // prefixes of up to 300 tokens 85 and 89, four documents 253 and 249);
    // as many CTAs as there is room for, which go from page to page
    const int ctas = append_ctas(sizeof(T), std::max(c.attention_dim, c.linear_dim));
    a.page_blocks = (int)std::min<int64_t>((d.num_rows + 1) / 2, 148 * ctas);
    const dim3 grid((unsigned)(q_blocks + a.page_blocks));
    const Cache8 l = cache8_layer(c, pool, d.layer);
#define IMBA_APPEND8(DQK, DV) \
  if (c.attention_dim == DQK && c.linear_dim == DV) e = launch_append8<T, DQK, DV>(grid, a, l, fast, s);
    IMBA_APPEND8(32, 32)
    IMBA_APPEND8(64, 64)
    IMBA_APPEND8(32, 64)
    IMBA_APPEND8(64, 32)
    IMBA_APPEND8(96, 96)
    IMBA_APPEND8(128, 128)
#undef IMBA_APPEND8
  } else {
    const PoolGeom g = cache_geom(c, pool.num_pages);
    a.page_blocks = (int)std::min<int64_t>(d.num_rows, 148 * 8);
    const dim3 grid((unsigned)(q_blocks + a.page_blocks));
    e = c.dtype == IMBA_DTYPE_BF16 ? launch_append_full<T, bf16>(grid, a, g, pool.base, d.layer, fast, s)
                                   : launch_append_full<T, float>(grid, a, g, pool.base, d.layer, fast, s);
  }
  return e == cudaSuccess ? IMBA_OK : IMBA_ERR_CUDA;
}

}  // namespace imba
