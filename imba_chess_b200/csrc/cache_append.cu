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
#include <algorithm>

#include "cache8.cuh"

namespace imba {

namespace {

constexpr int kTok = IMBA_PAGE_TOKENS;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxPairs = 64;  // of a head: d_qk <= 128
constexpr int kMaxAxes = 8;
constexpr float kLargest = 3.19014718988379809496e38f;  // 1.875 2^127

// Plan layout (int32 words): [0] number of pages, then from word 64 the hash
// table's keys [cap], the rows of each key's page [cap][16], and the list of
// occupied table positions [num_rows].
constexpr int kPlanHead = 64;
inline int plan_cap(int32_t n) {
  int cap = 64;
  while (cap < 2 * (int64_t)n) cap *= 2;
  return cap;
}
struct PlanView {
  int* count;
  int* keys;
  int* rows;
  int* list;
  int cap;
};
inline PlanView plan_view(void* plan, int32_t n) {
  PlanView v;
  v.cap = plan_cap(n);
  v.count = static_cast<int*>(plan);
  v.keys = v.count + kPlanHead;
  v.rows = v.keys + v.cap;
  v.list = v.rows + (size_t)v.cap * kTok;
  return v;
}

// Enters every row into its page's list.  Keys, rows and the count start at
// -1 (one memset), so the count is the number of pages less one.
__global__ void append_plan_kernel(PlanView pv, int n, const int32_t* __restrict__ slots, int64_t num_slots,
                                   int32_t* status) {
  pdl_wait();
  pdl_trigger();
  const int r = blockIdx.x * blockDim.x + threadIdx.x;
  if (r >= n) return;
  const int64_t slot = slots[r];
  if (slot < 0 || slot >= num_slots) {
    if (slot != -1) report(status, IMBA_ERR_RANGE);
    return;
  }
  const int page = (int)(slot / kTok);
  uint32_t at = (uint32_t)page * 0x9e3779b1u;
  at = (at ^ (at >> 15)) & (uint32_t)(pv.cap - 1);
  for (int probe = 0; probe < pv.cap; ++probe) {  // at most n <= cap / 2 keys: an empty place is always found
    const int was = atomicCAS(pv.keys + at, -1, page);
    if (was == -1) pv.list[atomicAdd(pv.count, 1) + 1] = (int)at;
    if (was == -1 || was == page) {
      atomicMax(pv.rows + (size_t)at * kTok + slot % kTok, r);  // the last row of a slot is the one stored
      return;
    }
    at = (at + 1) & (uint32_t)(pv.cap - 1);
  }
}

struct Strides {
  int64_t row, head, elem;
  int vec;  // rows of contiguous elements, aligned for 4-element accesses
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
  int q_blocks;  // CTAs that turn queries (the first ones), a warp a row
  int64_t num_slots;
};

// Four elements of the source type as they are in memory.
template <typename T>
struct Raw4;
template <>
struct Raw4<bf16> {
  uint2 u;
  __device__ __forceinline__ void load(const bf16* p) { u = *reinterpret_cast<const uint2*>(p); }
  __device__ __forceinline__ void load(const bf16* const (&p)[4]) {
    u.x = (uint32_t)__bfloat16_as_ushort(*p[0]) | (uint32_t)__bfloat16_as_ushort(*p[1]) << 16;
    u.y = (uint32_t)__bfloat16_as_ushort(*p[2]) | (uint32_t)__bfloat16_as_ushort(*p[3]) << 16;
  }
  __device__ __forceinline__ void zero() { u = make_uint2(0, 0); }
  __device__ __forceinline__ void get(float (&x)[4]) const {
    x[0] = __uint_as_float(u.x << 16), x[1] = __uint_as_float(u.x & 0xffff0000u);
    x[2] = __uint_as_float(u.y << 16), x[3] = __uint_as_float(u.y & 0xffff0000u);
  }
};
template <>
struct Raw4<float> {
  float4 f;
  __device__ __forceinline__ void load(const float* p) { f = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ void load(const float* const (&p)[4]) { f = make_float4(*p[0], *p[1], *p[2], *p[3]); }
  __device__ __forceinline__ void zero() { f = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void get(float (&x)[4]) const { x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w; }
};

template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&x)[4]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
    __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
  }
}

// Which elements the pairs of a head are made of.  Pairs past rot_dim / 2
// are neighbours and do not turn.
struct PairMap {
  int half, inter;
  __device__ __forceinline__ int first(int p) const { return p >= half || inter ? 2 * p : p; }
  __device__ __forceinline__ int second(int p) const { return p >= half || inter ? 2 * p + 1 : p + half; }
  // Four pairs p0 .. p0 + 3 are two runs of four elements, from lo(p0) and
  // hi(p0), when half is a multiple of four.
  __device__ __forceinline__ bool runs() const { return (half & 3) == 0; }
  __device__ __forceinline__ bool adjacent(int p0) const { return inter || p0 >= half; }
  __device__ __forceinline__ int lo(int p0) const { return adjacent(p0) ? 2 * p0 : p0; }
  __device__ __forceinline__ int hi(int p0) const { return adjacent(p0) ? 2 * p0 + 4 : p0 + half; }
};

// Pairs p0 .. p0 + 3 of a head (runs of four), or its elements e0 .. e0 + 7.
template <typename T>
struct Eight {
  Raw4<T> a, b;
  __device__ __forceinline__ void load_pairs(const T* head, const Strides& st, const PairMap& m, int p0) {
    if (st.vec && m.runs()) {
      a.load(head + m.lo(p0));
      b.load(head + m.hi(p0));
      return;
    }
    const T *p[4], *q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // in the order that get_pairs() takes them apart
      if (m.runs() && m.adjacent(p0)) {
        p[i] = head + (2 * p0 + i) * st.elem;
        q[i] = head + (2 * p0 + 4 + i) * st.elem;
      } else {
        p[i] = head + m.first(p0 + i) * st.elem;
        q[i] = head + m.second(p0 + i) * st.elem;
      }
    }
    a.load(p);
    b.load(q);
  }
  __device__ __forceinline__ void get_pairs(const PairMap& m, int p0, float (&x)[4], float (&y)[4]) const {
    if (m.runs() && m.adjacent(p0)) {
      float u[4], v[4];
      a.get(u);
      b.get(v);
      x[0] = u[0], y[0] = u[1], x[1] = u[2], y[1] = u[3];
      x[2] = v[0], y[2] = v[1], x[3] = v[2], y[3] = v[3];
    } else {
      a.get(x);
      b.get(y);
    }
  }
  __device__ __forceinline__ void load_run(const T* p, const Strides& st) {
    if (st.vec) {
      a.load(p);
      b.load(p + 4);
      return;
    }
    const T *s[4], *t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[i] = p + i * st.elem;
      t[i] = p + (4 + i) * st.elem;
    }
    a.load(s);
    b.load(t);
  }
  __device__ __forceinline__ void zero() {
    a.zero();
    b.zero();
  }
};

// The rotation, each product and sum rounded on its own.
__device__ __forceinline__ void turn(float2 t, float& x, float& y) {
  const float u = x, v = y;
  x = __fsub_rn(__fmul_rn(u, t.x), __fmul_rn(v, t.y));
  y = __fadd_rn(__fmul_rn(v, t.x), __fmul_rn(u, t.y));
}
__device__ __forceinline__ void turn4(const float2* cs, int half, int p0, float (&x)[4], float (&y)[4]) {
  if (p0 + 3 < half) {
    const float4 t0 = *reinterpret_cast<const float4*>(cs + p0), t1 = *reinterpret_cast<const float4*>(cs + p0 + 2);
    turn(make_float2(t0.x, t0.y), x[0], y[0]);
    turn(make_float2(t0.z, t0.w), x[1], y[1]);
    turn(make_float2(t1.x, t1.y), x[2], y[2]);
    turn(make_float2(t1.z, t1.w), x[3], y[3]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (p0 + i < half) turn(cs[p0 + i], x[i], y[i]);
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
__device__ __forceinline__ void fill_turns(const imba_rotary_desc& rot, const int* rows, int ntok,
                                           float2 (*cs)[kMaxPairs]) {
  const int half = rot.rot_dim / 2;
  for (int t = threadIdx.x / 32; t < ntok; t += kWarps) {
    const int r = rows[t];
    if (r < 0) continue;
    for (int p = threadIdx.x % 32; p < half; p += 32) cs[t][p] = row_turn(rot, r, p);
  }
}

// Lanes of a warp on one row: kLanes lanes of a head (eight elements each),
// heads side by side.
template <int D>
struct RowLanes {
  static constexpr int kLanes = D == 96 ? 16 : D / 8;  // a power of two; of 16 lanes 12 are in use
  static constexpr int kHeads = 32 / kLanes;
};

// Queries: a warp turns row `r`.
template <typename T, int D>
__device__ __forceinline__ void turn_query_row(const AppendArgs& a, int64_t r, float2* cs) {
  using L = RowLanes<D>;
  constexpr int kAhead = 4;
  const int lane = threadIdx.x % 32, l = lane % L::kLanes, p0 = l * 4;
  const PairMap m{a.rot.rot_dim / 2, a.rot.interleaved};
  const T* src = static_cast<const T*>(a.q) + r * a.qs.row;
  T* dst = static_cast<T*>(a.q_out) + r * a.qo.row;
  bool turned = false;
  for (int h0 = 0; h0 < a.Hq; h0 += kAhead * L::kHeads) {
    Eight<T> raw[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int h = h0 + i * L::kHeads + lane / L::kLanes;
      if (h < a.Hq && l < D / 8) raw[i].load_pairs(src + h * a.qs.head, a.qs, m, p0);
    }
    if (!turned) {  // behind the first loads
      for (int p = lane; p < m.half; p += 32) cs[p] = row_turn(a.rot, r, p);
      __syncwarp();
      turned = true;
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int h = h0 + i * L::kHeads + lane / L::kLanes;
      if (h >= a.Hq || l >= D / 8) continue;
      T* o = dst + h * a.qo.head;
      float x[4], y[4];
      raw[i].get_pairs(m, p0, x, y);
      turn4(cs, m.half, p0, x, y);
      if (a.qo.vec && m.runs()) {
        if (m.adjacent(p0)) {
          const float u[4] = {x[0], y[0], x[1], y[1]}, v[4] = {x[2], y[2], x[3], y[3]};
          store4(o + 2 * p0, u);
          store4(o + 2 * p0 + 4, v);
        } else {
          store4(o + p0, x);
          store4(o + p0 + m.half, y);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          o[m.first(p0 + j) * a.qo.elem] = from_f<T>(x[j]);
          o[m.second(p0 + j) * a.qo.elem] = from_f<T>(y[j]);
        }
      }
    }
  }
}

// Any head size: one lane per pair of the row.
template <typename T>
__device__ __forceinline__ void turn_query_row_any(const AppendArgs& a, int64_t r, float2* cs) {
  const PairMap m{a.rot.rot_dim / 2, a.rot.interleaved};
  const int lane = threadIdx.x % 32, pairs = a.dqk / 2;
  for (int p = lane; p < m.half; p += 32) cs[p] = row_turn(a.rot, r, p);
  __syncwarp();
  const T* src = static_cast<const T*>(a.q) + r * a.qs.row;
  T* dst = static_cast<T*>(a.q_out) + r * a.qo.row;
  for (int i = lane; i < a.Hq * pairs; i += 32) {
    const int h = i / pairs, p = i % pairs;
    const T* s = src + h * a.qs.head;
    T* o = dst + h * a.qo.head;
    float x = to_f(s[m.first(p) * a.qs.elem]), y = to_f(s[m.second(p) * a.qs.elem]);
    if (p < m.half) turn(cs[p], x, y);
    o[m.first(p) * a.qo.elem] = from_f<T>(x);
    o[m.second(p) * a.qo.elem] = from_f<T>(y);
  }
}

// The row of a query warp; -1: past the end, padding or outside the pool.
__device__ __forceinline__ int64_t query_row(const AppendArgs& a) {
  const int64_t r = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32;
  if (r >= a.n) return -1;
  const int64_t slot = a.slots[r];
  return slot >= 0 && slot < a.num_slots ? r : -1;
}

// Largest magnitude as bits (a NaN's are above infinity's).
__device__ __forceinline__ void see(const float (&x)[4], uint32_t& most) {
#pragma unroll
  for (int i = 0; i < 4; ++i) most = max(most, __float_as_uint(x[i]) & 0x7fffffffu);
}
// What is not finite becomes zero, and the last half step below 2^128 does
// not round up to it (240 2^120 is the largest stored value).
__device__ __forceinline__ void take_finite(float (&x)[4], uint32_t& most, bool& bad) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (!isfinite(x[i])) {
      bad = true;
      x[i] = 0.f;
    }
    x[i] = fminf(fmaxf(x[i], -kLargest), kLargest);
  }
  see(x, most);
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
__device__ __forceinline__ int grow_scale(uint8_t* block, uint8_t* scale, int was, uint32_t most, int lane) {
  const int now = max(was, scale_byte(__uint_as_float(__reduce_max_sync(0xffffffffu, most))));
  if (now > was) {
    if (was > 0) {
      const float f = shrink(was, now);
#pragma unroll
      for (int i = 0; i < D * kTok / 512; ++i) rescale16(reinterpret_cast<uint4*>(block) + i * 32 + lane, f);
    }
    __syncwarp();  // before the new codes
    if (lane == 0) *scale = (uint8_t)now;
  }
  return now;
}

__device__ __forceinline__ uint32_t codes4(const float (&x)[4], float f) {
  return to_e4m3x2(x[0] * f, x[1] * f) | to_e4m3x2(x[2] * f, x[3] * f) << 16;
}

// Codes of pairs p0 .. p0 + 3 of a token's K row.
__device__ __forceinline__ void store_k8(uint8_t* o, const PairMap& m, int p0, const float (&x)[4], const float (&y)[4],
                                         float f) {
  if (m.runs()) {
    if (m.adjacent(p0)) {
      const float u[4] = {x[0], y[0], x[1], y[1]}, v[4] = {x[2], y[2], x[3], y[3]};
      *reinterpret_cast<uint2*>(o + 2 * p0) = make_uint2(codes4(u, f), codes4(v, f));
    } else {
      *reinterpret_cast<uint32_t*>(o + p0) = codes4(x, f);
      *reinterpret_cast<uint32_t*>(o + p0 + m.half) = codes4(y, f);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t two = to_e4m3x2(x[j] * f, y[j] * f);
    o[m.first(p0 + j)] = (uint8_t)two;
    o[m.second(p0 + j)] = (uint8_t)(two >> 8);
  }
}

// A warp's share of a dense page: the block of one head.  K: a lane holds
// four pairs of every kGroup-th token.  V: eight dimensions of consecutive
// tokens, so that a pair of tokens is one 16-byte store of [8][d_v][2].
template <typename T, int D, bool IsV>
struct Block {
  static constexpr int kLanes = D / 8, kGroup = 32 / kLanes, kPass = kTok / kGroup;
  Eight<T> raw[kPass];
  int was;

  static __device__ __forceinline__ int tok(int g, int i) { return IsV ? g * kPass + i : i * kGroup + g; }

  __device__ __forceinline__ void load(const AppendArgs& a, const int* rows, int h, const uint8_t* scale) {
    const int lane = threadIdx.x % 32, g = lane / kLanes, e = lane % kLanes;
    const Strides& st = IsV ? a.vs : a.ks;
    const PairMap m{a.rot.rot_dim / 2, a.rot.interleaved};
    was = *scale;
#pragma unroll
    for (int i = 0; i < kPass; ++i) {
      const int r = g < kGroup ? rows[tok(g, i)] : -1;
      if (r < 0) {
        raw[i].zero();
        continue;
      }
      const T* p = static_cast<const T*>(IsV ? a.v : a.k) + r * st.row + h * st.head;
      if (IsV)
        raw[i].load_run(p + e * 8 * st.elem, st);
      else
        raw[i].load_pairs(p, st, m, e * 4);
    }
  }

  __device__ __forceinline__ void put(const AppendArgs& a, const int* rows, float2 (*cs)[kMaxPairs], uint8_t* block,
                                      uint8_t* scale, bool& bad) const {
    const int lane = threadIdx.x % 32, g = lane / kLanes, e = lane % kLanes, p0 = e * 4;
    const PairMap m{a.rot.rot_dim / 2, a.rot.interleaved};
    float x[kPass][4], y[kPass][4];
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < kPass; ++i) {
      if (IsV) {
        raw[i].a.get(x[i]);
        raw[i].b.get(y[i]);
      } else {
        raw[i].get_pairs(m, p0, x[i], y[i]);
        if ((g < kGroup ? rows[tok(g, i)] : -1) >= 0) turn4(cs[tok(g, i)], m.half, p0, x[i], y[i]);
      }
      see(x[i], most);
      see(y[i], most);
    }
    if (most > __float_as_uint(kLargest)) {
      most = 0;
#pragma unroll
      for (int i = 0; i < kPass; ++i) {
        take_finite(x[i], most, bad);
        take_finite(y[i], most, bad);
      }
    }
    __syncwarp();
    const int b = grow_scale<D>(block, scale, was, most, lane);
    const float f = b ? inv_scale_of(b) : 0.f;
    if constexpr (!IsV) {
#pragma unroll
      for (int i = 0; i < kPass; ++i) {
        const int t = tok(g, i);
        if ((g < kGroup ? rows[t] : -1) >= 0) store_k8(block + t * D, m, p0, x[i], y[i], f);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPass; i += 2) {
        if (g >= kGroup) continue;
        const int t = tok(g, i);
        const bool even = rows[t] >= 0, odd = rows[t + 1] >= 0;
        if (!even && !odd) continue;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          w[j] = to_e4m3x2(x[i][2 * j] * f, x[i + 1][2 * j] * f) |
                 to_e4m3x2(x[i][2 * j + 1] * f, x[i + 1][2 * j + 1] * f) << 16;
          w[2 + j] = to_e4m3x2(y[i][2 * j] * f, y[i + 1][2 * j] * f) |
                     to_e4m3x2(y[i][2 * j + 1] * f, y[i + 1][2 * j + 1] * f) << 16;
        }
        uint4* o = reinterpret_cast<uint4*>(block + v8_off(t, e * 8, D));
        if (!(even && odd)) {  // keep the other token's bytes
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
  }
};

// The single new token of a page, row r, offset t: heads h0 .. of K or V.
// Every lane of the warp takes part; kLanes lanes a head.
template <typename T, int D, bool IsV>
struct OneToken {
  using L = RowLanes<D>;
  Eight<T> raw;
  uint4 old;
  int was;
  bool live;

  __device__ __forceinline__ void load(const AppendArgs& a, int64_t r, int t, int h, uint8_t* block,
                                       const uint8_t* scale) {
    const int l = threadIdx.x % L::kLanes;
    const Strides& st = IsV ? a.vs : a.ks;
    const PairMap m{a.rot.rot_dim / 2, a.rot.interleaved};
    live = h < a.H && l < D / 8;
    raw.zero();
    was = 0;
    if (!live) return;
    was = *scale;
    const T* p = static_cast<const T*>(IsV ? a.v : a.k) + r * st.row + h * st.head;
    if (IsV) {
      raw.load_run(p + l * 8 * st.elem, st);
      old = *reinterpret_cast<const uint4*>(block + v8_off(t & ~1, l * 8, D));
    } else {
      raw.load_pairs(p, st, m, l * 4);
    }
  }

  __device__ __forceinline__ void put(const AppendArgs& a, const float2* cs, int t, uint8_t* block, uint8_t* scale,
                                      bool& bad) {
    const int l = threadIdx.x % L::kLanes, p0 = l * 4;
    const PairMap m{a.rot.rot_dim / 2, a.rot.interleaved};
    float x[4], y[4];
    if (IsV) {
      raw.a.get(x);
      raw.b.get(y);
    } else {
      raw.get_pairs(m, p0, x, y);
      if (l < D / 8) turn4(cs, m.half, p0, x, y);
    }
    uint32_t most = 0;
    see(x, most);
    see(y, most);
    if (most > __float_as_uint(kLargest)) {
      most = 0;
      take_finite(x, most, bad);
      take_finite(y, most, bad);
    }
    __syncwarp();
#pragma unroll
    for (int o = 1; o < L::kLanes; o *= 2) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    const int now = max(was, scale_byte(__uint_as_float(most)));
    const bool again = live && now > was && was > 0;
    if (again)
      for (int i = l; i < D * kTok / 16; i += D / 8) rescale16(reinterpret_cast<uint4*>(block) + i, shrink(was, now));
    __syncwarp();
    if (!live) return;
    if (now > was && l == 0) *scale = (uint8_t)now;
    const float f = now ? inv_scale_of(now) : 0.f;
    if constexpr (!IsV) {
      store_k8(block + t * D, m, p0, x, y, f);
    } else {
      uint4* o = reinterpret_cast<uint4*>(block + v8_off(t & ~1, l * 8, D));
      if (again) old = *o;
      const int up = (t & 1) * 8;
      const uint32_t keep = t & 1 ? 0x00ff00ffu : 0xff00ff00u;
      auto spread = [&](float lo, float hi) {  // the codes of two dimensions at the token's place of each pair
        const uint32_t two = to_e4m3x2(lo * f, hi * f);
        return ((two & 0xffu) | (two & 0xff00u) << 8) << up;
      };
      *o = make_uint4(spread(x[0], x[1]) | (old.x & keep), spread(x[2], x[3]) | (old.y & keep),
                      spread(y[0], y[1]) | (old.z & keep), spread(y[2], y[3]) | (old.w & keep));
    }
  }
};

constexpr int kSparse = kWarps / 2;  // pages of a CTA in the sparse shape

template <typename T, int DQK, int DV>
__global__ void __launch_bounds__(kThreads) append8_kernel(AppendArgs a, Cache8 c) {
  __shared__ int rows[2][kTok];
  __shared__ __align__(16) float2 cs[kTok][kMaxPairs];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if ((int)blockIdx.x < a.q_blocks) {
    const int64_t r = query_row(a);
    if (r >= 0) turn_query_row<T, DQK>(a, r, cs[warp]);
    return;
  }
  const int count = *a.plan.count + 1;
  const int first = blockIdx.x - a.q_blocks, step = gridDim.x - a.q_blocks;
  bool bad = false;
  auto k_block = [&](int page, int h) { return c.data + page * c.page_stride + (int64_t)h * kTok * DQK; };
  auto v_block = [&](int page, int h) { return c.data + page * c.page_stride + c.v_offset + (int64_t)h * kTok * DV; };
  auto scale_at = [&](int page, int i) { return c.scales + page * c.scale_stride + i; };

  // One page by the whole CTA, its rows in `rows[0]`.
  auto dense = [&](int page, auto&& ahead) {
    Block<T, DQK, false> k;
    Block<T, DV, true> v;
    int h = warp;
    if (h < a.H) k.load(a, rows[0], h, scale_at(page, h));
    ahead();
    fill_turns(a.rot, rows[0], kTok, cs);
    __syncthreads();
    for (; h < a.H; h += kWarps) {
      v.load(a, rows[0], h, scale_at(page, a.H + h));
      k.put(a, rows[0], cs, k_block(page, h), scale_at(page, h), bad);
      if (h + kWarps < a.H) k.load(a, rows[0], h + kWarps, scale_at(page, h + kWarps));
      v.put(a, rows[0], cs, v_block(page, h), scale_at(page, a.H + h), bad);
    }
    __syncthreads();
  };

  if (2 * (int64_t)count <= a.n) {
    // Dense: the next page's rows are fetched behind this one's first loads.
    int page = -1, r = -1;
    auto fetch = [&](int e) {
      page = -1;
      if (e >= count) return;
      const int at = a.plan.list[e];
      page = a.plan.keys[at];
      if (page >= c.num_pages) page = -1;  // a plan of another pool
      if (threadIdx.x < kTok) r = a.plan.rows[(size_t)at * kTok + threadIdx.x];
    };
    fetch(first);
    for (int e = first; e < count; e += step) {
      const int now = page;
      if (threadIdx.x < kTok) rows[0][threadIdx.x] = now < 0 ? -1 : r;
      __syncthreads();
      if (now >= 0)
        dense(now, [&] { fetch(e + step); });
      else
        fetch(e + step);
    }
  } else {
    using LK = RowLanes<DQK>;
    using LV = RowLanes<DV>;
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
      if (live == 1) {
        bool turned = false;
        for (int h0 = warp % 2; h0 * min(LK::kHeads, LV::kHeads) < a.H; h0 += 2) {
          // K and V of as many heads as the wider of the two takes at once
          constexpr int kStep = LK::kHeads < LV::kHeads ? LK::kHeads : LV::kHeads;
          OneToken<T, DQK, false> k;
          OneToken<T, DV, true> v;
          const int hk = lane / LK::kLanes < kStep ? h0 * kStep + lane / LK::kLanes : a.H;
          const int hv = lane / LV::kLanes < kStep ? h0 * kStep + lane / LV::kLanes : a.H;
          uint8_t *kb = k_block(page, hk), *vb = v_block(page, hv);
          k.load(a, r, tok, hk, kb, scale_at(page, hk));
          v.load(a, r, tok, hv, vb, scale_at(page, a.H + hv));
          if (!turned) {
            for (int p = lane; p < a.rot.rot_dim / 2; p += 32) cs[warp][p] = row_turn(a.rot, r, p);
            __syncwarp();
            turned = true;
          }
          k.put(a, cs[warp], tok, kb, scale_at(page, hk), bad);
          v.put(a, cs[warp], tok, vb, scale_at(page, a.H + hv), bad);
        }
      }
      // Pages with several new tokens, one after the other.
      if (__syncthreads_or(live > 1)) {
        for (int i = 0; i < kSparse; ++i) {
          if (warp == 2 * i && lane < kTok) rows[0][lane] = live > 1 ? a.plan.rows[(size_t)at * kTok + lane] : -1;
          if (warp == 2 * i && lane == 0) rows[1][0] = live > 1 ? page : -1;
          __syncthreads();
          const int now = rows[1][0];
          if (now >= 0)
            dense(now, [] {});
          else
            __syncthreads();
        }
      }
    }
  }
  if (bad) report(a.status, IMBA_ERR_RANGE);
}

// Pools in full precision: no scale, so every element is on its own.
template <typename T, typename TP>
__global__ void __launch_bounds__(kThreads) append_kernel(AppendArgs a, PoolGeom g, TP* pool, int layer) {
  __shared__ int rows[kTok];
  __shared__ float2 cs[kTok][kMaxPairs];
  pdl_wait();
  pdl_trigger();
  if ((int)blockIdx.x < a.q_blocks) {
    const int64_t r = query_row(a);
    if (r >= 0) turn_query_row_any<T>(a, r, cs[threadIdx.x / 32]);
    return;
  }
  const PairMap m{a.rot.rot_dim / 2, a.rot.interleaved};
  const int count = *a.plan.count + 1;
  const int pairs = (g.dqk + 1) / 2;
  for (int e = blockIdx.x - a.q_blocks; e < count; e += gridDim.x - a.q_blocks) {
    const int at = a.plan.list[e];
    const int64_t slot0 = (int64_t)a.plan.keys[at] * kTok;
    if (slot0 < 0 || slot0 >= g.num_slots) continue;  // a plan of another pool
    if (threadIdx.x < kTok) rows[threadIdx.x] = a.plan.rows[(size_t)at * kTok + threadIdx.x];
    __syncthreads();
    fill_turns(a.rot, rows, kTok, cs);
    __syncthreads();
    for (int t = 0; t < kTok; ++t) {
      const int r = rows[t];
      if (r < 0) continue;
      for (int i = threadIdx.x; i < a.H * pairs; i += kThreads) {
        const int h = i / pairs, p = i % pairs;
        const T* s = static_cast<const T*>(a.k) + r * a.ks.row + h * a.ks.head;
        TP* o = pool + g.k_off(slot0 + t, layer, h);
        float x = to_f(s[m.first(p) * a.ks.elem]);
        if (m.second(p) >= g.dqk) {  // the odd last element
          o[m.first(p)] = from_f<TP>(x);
          continue;
        }
        float y = to_f(s[m.second(p) * a.ks.elem]);
        if (p < m.half) turn(cs[t][p], x, y);
        o[m.first(p)] = from_f<TP>(x);
        o[m.second(p)] = from_f<TP>(y);
      }
      for (int i = threadIdx.x; i < a.H * g.dv; i += kThreads) {
        const int h = i / g.dv, el = i % g.dv;
        pool[g.v_off(slot0 + t, layer, h) + el] =
            from_f<TP>(to_f(static_cast<const T*>(a.v)[r * a.vs.row + h * a.vs.head + el * a.vs.elem]));
      }
    }
    __syncthreads();
  }
}

// Rows read back.  One CTA per row.
template <typename TO>
__global__ void read8_kernel(Cache8 c, int dqk, int dv, int n, const int32_t* __restrict__ slots, TO* k, TO* v,
                             int32_t* status) {
  pdl_wait();
  pdl_trigger();
  const int r = blockIdx.x;
  const int64_t slot = slots[r];
  if (slot < 0 || slot / kTok >= c.num_pages) {
    if (threadIdx.x == 0) report(status, IMBA_ERR_RANGE);
    return;
  }
  const int t = (int)(slot % kTok);
  const uint8_t* data = c.data + slot / kTok * c.page_stride;
  const uint8_t* scales = c.scales + slot / kTok * c.scale_stride;
  for (int i = threadIdx.x; i < c.H * (dqk + dv); i += blockDim.x) {
    const bool isv = i >= c.H * dqk;
    const int j = isv ? i - c.H * dqk : i, d = isv ? dv : dqk, h = j / d, e = j % d;
    const uint8_t code = isv ? data[c.v_offset + (int64_t)h * kTok * dv + v8_off(t, e, dv)]
                             : data[((int64_t)h * kTok + t) * dqk + e];
    const float x = e4m3x2_to_f2(code).x * scale_of(scales[isv ? c.H + h : h]);
    (isv ? v : k)[(int64_t)r * c.H * d + j] = from_f<TO>(x);
  }
}

template <typename T>
void fill_strides(const int64_t (&s)[3], const void* base, Strides* out) {
  out->row = s[0];
  out->head = s[1];
  out->elem = s[2];
  const uintptr_t align = 4 * sizeof(T) - 1;
  out->vec = s[2] == 1 && s[0] % 4 == 0 && s[1] % 4 == 0 && (reinterpret_cast<uintptr_t>(base) & align) == 0;
}

template <typename T>
imba_status_t launch_append(const imba_cache_desc& c, const imba_pool_desc& pool, const imba_append_desc& d,
                            void* plan, cudaStream_t s) {
  AppendArgs a;
  a.plan = plan_view(plan, d.num_rows);
  a.n = d.num_rows;
  a.H = c.num_heads;
  a.Hq = d.q ? d.num_q_heads : 0;
  a.dqk = c.attention_dim;
  a.dv = c.linear_dim;
  a.k = d.k, a.v = d.v, a.q = d.q, a.q_out = d.q_out;
  fill_strides<T>(d.k_stride, d.k, &a.ks);
  fill_strides<T>(d.v_stride, d.v, &a.vs);
  fill_strides<T>(d.q_stride, d.q, &a.qs);
  fill_strides<T>(d.q_out_stride, d.q_out, &a.qo);
  a.rot = d.rotary;
  a.slots = d.slots;
  a.status = d.status;
  a.num_slots = pool.num_pages * kTok;
  a.q_blocks = a.Hq ? (d.num_rows + kWarps - 1) / kWarps : 0;
  // a page a CTA with two tokens or more in it on average, else kSparse
  const int64_t pages = std::min<int64_t>((d.num_rows + 1) / 2, 148 * 4);
  const dim3 grid((unsigned)(a.q_blocks + pages));
  cudaError_t e = cudaErrorInvalidValue;
  if (c.dtype == IMBA_DTYPE_E4M3) {
    const Cache8 l = cache8_layer(c, pool, d.layer);
#define IMBA_APPEND8(DQK, DV)                               \
  if (c.attention_dim == DQK && c.linear_dim == DV)         \
    e = launch_pdl(append8_kernel<T, DQK, DV>, grid, dim3(kThreads), 0, s, a, l);
    IMBA_APPEND8(32, 32)
    IMBA_APPEND8(64, 64)
    IMBA_APPEND8(32, 64)
    IMBA_APPEND8(64, 32)
    IMBA_APPEND8(96, 96)
    IMBA_APPEND8(128, 128)
#undef IMBA_APPEND8
  } else {
    const PoolGeom g = cache_geom(c, pool.num_pages);
    e = c.dtype == IMBA_DTYPE_BF16
            ? launch_pdl(append_kernel<T, bf16>, grid, dim3(kThreads), 0, s, a, g, static_cast<bf16*>(pool.base), d.layer)
            : launch_pdl(append_kernel<T, float>, grid, dim3(kThreads), 0, s, a, g, static_cast<float*>(pool.base),
                         d.layer);
  }
  return e == cudaSuccess ? IMBA_OK : IMBA_ERR_CUDA;
}

}  // namespace

imba_status_t validate_cache(const imba_cache_desc* c) {
  if (!c) return IMBA_ERR_ARG;
  if (c->num_layers <= 0 || c->num_heads <= 0 || c->attention_dim <= 0 || c->linear_dim <= 0) return IMBA_ERR_ARG;
  if (c->dtype < IMBA_DTYPE_F32 || c->dtype > IMBA_DTYPE_E4M3) return IMBA_ERR_ARG;
  if (c->attention_dim > 128 || c->linear_dim > 128 || c->num_heads > 1024 || c->num_layers > 1024)
    return IMBA_ERR_UNSUPPORTED;
  // (a page's bytes in 8 bits are a 32-bit factor of the kernels' addresses)
  if (c->dtype == IMBA_DTYPE_E4M3 &&
      (!cache8_dims_ok(c->attention_dim, c->linear_dim) || cache8_page_bytes(*c) > UINT32_MAX))
    return IMBA_ERR_UNSUPPORTED;
  return IMBA_OK;
}

imba_status_t validate_pool(const imba_pool_desc* pool) {
  if (!pool || !pool->base || pool->num_pages <= 0) return IMBA_ERR_ARG;
  if (reinterpret_cast<uintptr_t>(pool->base) & 255) return IMBA_ERR_ARG;
  if (pool->num_pages > (int64_t)INT32_MAX / IMBA_PAGE_TOKENS) return IMBA_ERR_RANGE;
  return IMBA_OK;
}

}  // namespace imba

extern "C" {

size_t imba_cache_pool_bytes(const imba_cache_desc* cache, int64_t num_pages) {
  if (imba::validate_cache(cache) != IMBA_OK || num_pages <= 0) return 0;
  const int64_t elems = imba::cache8_page_bytes(*cache);
  if (cache->dtype == IMBA_DTYPE_E4M3)
    return (size_t)((elems + (int64_t)cache->num_layers * 2 * cache->num_heads) * num_pages);
  return (size_t)(elems * num_pages * (cache->dtype == IMBA_DTYPE_BF16 ? 2 : 4));
}

size_t imba_append_plan_bytes(int32_t num_rows) {
  if (num_rows < 0 || num_rows > (1 << 28)) return 0;
  const int64_t cap = imba::plan_cap(num_rows);
  return (size_t)(imba::kPlanHead + cap * (1 + IMBA_PAGE_TOKENS) + num_rows) * sizeof(int32_t);
}

imba_status_t imba_append_plan(const imba_pool_desc* pool, int32_t num_rows, const int32_t* slots, void* plan,
                               size_t plan_bytes, int32_t* status, void* stream) {
  const imba_status_t v = imba::validate_pool(pool);
  if (v != IMBA_OK) return v;
  if (num_rows < 0 || num_rows > (1 << 28)) return IMBA_ERR_ARG;
  if (!plan || (num_rows > 0 && !slots) || (reinterpret_cast<uintptr_t>(plan) & 255)) return IMBA_ERR_ARG;
  if (plan_bytes < imba_append_plan_bytes(num_rows)) return IMBA_ERR_OOM;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const imba::PlanView pv = imba::plan_view(plan, num_rows);
  const size_t clear = (size_t)(imba::kPlanHead + (int64_t)pv.cap * (1 + IMBA_PAGE_TOKENS)) * sizeof(int32_t);
  if (cudaMemsetAsync(plan, 0xff, clear, s) != cudaSuccess) return IMBA_ERR_CUDA;
  if (num_rows == 0) return IMBA_OK;
  const cudaError_t e = imba::launch_pdl(imba::append_plan_kernel, dim3((num_rows + 127) / 128), dim3(128), 0, s, pv,
                                         (int)num_rows, slots, pool->num_pages * IMBA_PAGE_TOKENS, status);
  return e == cudaSuccess ? IMBA_OK : IMBA_ERR_CUDA;
}

imba_status_t imba_kv_append(const imba_cache_desc* cache, const imba_pool_desc* pool, const imba_append_desc* append,
                             const void* plan, size_t plan_bytes, void* stream) {
  imba_status_t v = imba::validate_cache(cache);
  if (v == IMBA_OK) v = imba::validate_pool(pool);
  if (v != IMBA_OK) return v;
  if (!append || append->num_rows < 0) return IMBA_ERR_ARG;
  if (append->layer < 0 || append->layer >= cache->num_layers) return IMBA_ERR_RANGE;
  if (append->src_dtype != IMBA_DTYPE_F32 && append->src_dtype != IMBA_DTYPE_BF16) return IMBA_ERR_ARG;
  if (append->num_rows == 0) return IMBA_OK;
  if (!append->slots || !append->k || !append->v) return IMBA_ERR_ARG;
  if (append->q && (!append->q_out || append->num_q_heads <= 0 || append->num_q_heads > 65536)) return IMBA_ERR_ARG;
  const imba_rotary_desc& r = append->rotary;
  if (r.rot_dim < 0 || r.rot_dim % 2 || r.rot_dim > cache->attention_dim) return IMBA_ERR_ARG;
  if (r.rot_dim > 0 && (!r.turns || !r.positions || r.num_axes < 1 || r.num_axes > imba::kMaxAxes))
    return IMBA_ERR_ARG;
  if (append->q && cache->attention_dim % 2) return IMBA_ERR_UNSUPPORTED;
  if (!plan || (reinterpret_cast<uintptr_t>(plan) & 255)) return IMBA_ERR_ARG;
  if (plan_bytes < imba_append_plan_bytes(append->num_rows)) return IMBA_ERR_OOM;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (append->src_dtype == IMBA_DTYPE_BF16)
    return imba::launch_append<imba::bf16>(*cache, *pool, *append, const_cast<void*>(plan), s);
  return imba::launch_append<float>(*cache, *pool, *append, const_cast<void*>(plan), s);
}

imba_status_t imba_kv_read(const imba_cache_desc* cache, const imba_pool_desc* pool, int32_t layer, int32_t n,
                           const int32_t* slots, int32_t out_dtype, void* k, void* v, int32_t* status, void* stream) {
  imba_status_t st = imba::validate_cache(cache);
  if (st == IMBA_OK) st = imba::validate_pool(pool);
  if (st != IMBA_OK) return st;
  if (layer < 0 || layer >= cache->num_layers) return IMBA_ERR_RANGE;
  if (n < 0) return IMBA_ERR_ARG;
  if (n == 0) return IMBA_OK;
  if (!slots || !k || !v) return IMBA_ERR_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (cache->dtype == IMBA_DTYPE_E4M3) {
    const imba::Cache8 c = imba::cache8_layer(*cache, *pool, layer);
    if (out_dtype == IMBA_DTYPE_BF16)
      e = imba::launch_pdl(imba::read8_kernel<imba::bf16>, dim3(n), dim3(256), 0, s, c, cache->attention_dim,
                           cache->linear_dim, (int)n, slots, static_cast<imba::bf16*>(k), static_cast<imba::bf16*>(v),
                           status);
    else if (out_dtype == IMBA_DTYPE_F32)
      e = imba::launch_pdl(imba::read8_kernel<float>, dim3(n), dim3(256), 0, s, c, cache->attention_dim,
                           cache->linear_dim, (int)n, slots, static_cast<float*>(k), static_cast<float*>(v), status);
    else
      return IMBA_ERR_ARG;
    return e == cudaSuccess ? IMBA_OK : IMBA_ERR_CUDA;
  }
  if (out_dtype != cache->dtype) return IMBA_ERR_ARG;
  const imba::PoolGeom g = imba::cache_geom(*cache, pool->num_pages);
  if (cache->dtype == IMBA_DTYPE_BF16)
    e = imba::launch_kv_copy<imba::bf16>(g, static_cast<imba::bf16*>(pool->base), layer, n, slots,
                                         static_cast<imba::bf16*>(k), static_cast<imba::bf16*>(v), 0, status, s);
  else
    e = imba::launch_kv_copy<float>(g, static_cast<float*>(pool->base), layer, n, slots, static_cast<float*>(k),
                                    static_cast<float*>(v), 0, status, s);
  return e == cudaSuccess ? IMBA_OK : IMBA_ERR_CUDA;
}

}  // extern "C"
