// Appending keys and values to a paged pool with the rotary position applied
// on the way, and reading rows back (include/imba_b200.h, "Cache operators").
//
// Pair p of a head turns by the angle 2 pi pos f_p, with f_p in turns per
// position held as a 64-bit fraction: pos * f_p mod 2^64 is one wrapping
// integer product, so the fraction of a turn is right to 2^-33 at any
// position and no floating-point range reduction is needed.  Products and
// sums are fp32 and each stored value is rounded once, to the pool's type.
//
// The work is grouped by page (append_plan): the scale of a block of 16
// tokens needs the largest magnitude of all its new tokens, and when it grows
// the block's earlier codes are rounded to it, so one warp owns one block.
// A CTA takes one page: the cosines and sines of its new tokens are computed
// once and shared by every head; each warp then takes K or V blocks.  Queries
// do not go to a page and are turned by CTAs of their own, in row order.
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
  int q_rows;      // rows per query CTA
  int q_blocks;    // CTAs that turn queries (the first ones)
  int64_t num_slots;
};

template <typename T>
__device__ __forceinline__ void load4(const T* p, int64_t step, int vec, float (&x)[4]) {
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
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = to_f(p[i * step]);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int64_t step, int vec, const float (&x)[4]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
      __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
      uint2 u;
      u.x = *reinterpret_cast<uint32_t*>(&a);
      u.y = *reinterpret_cast<uint32_t*>(&b);
      *reinterpret_cast<uint2*>(p) = u;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i * step] = from_f<T>(x[i]);
}

// Four consecutive pairs of a head, p0 .. p0 + 3, and the elements they are
// made of.  Pairs past rot_dim / 2 are neighbours and do not turn.
struct PairMap {
  int half, inter;
  __device__ __forceinline__ int first(int p) const {
    return p >= half ? 2 * p : inter ? 2 * p : p;
  }
  __device__ __forceinline__ int second(int p) const { return p >= half ? 2 * p + 1 : inter ? 2 * p + 1 : p + half; }
  // All four pairs lie side by side (a run of eight elements) / as two runs
  // of four: the accesses can be vectors when half is a multiple of 4.
  __device__ __forceinline__ bool runs() const { return (half & 3) == 0; }
  __device__ __forceinline__ bool adjacent(int p0) const { return inter || p0 >= half; }
};

template <typename T>
__device__ __forceinline__ void load_pairs(const T* head, const Strides& st, const PairMap& m, int p0, float (&a)[4],
                                           float (&b)[4]) {
  if (st.vec && m.runs()) {
    float x[4], y[4];
    if (m.adjacent(p0)) {
      load4(head + 2 * p0, 1, 1, x);
      load4(head + 2 * p0 + 4, 1, 1, y);
      a[0] = x[0], b[0] = x[1], a[1] = x[2], b[1] = x[3];
      a[2] = y[0], b[2] = y[1], a[3] = y[2], b[3] = y[3];
    } else {
      load4(head + p0, 1, 1, a);
      load4(head + p0 + m.half, 1, 1, b);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[i] = to_f(head[m.first(p0 + i) * st.elem]);
    b[i] = to_f(head[m.second(p0 + i) * st.elem]);
  }
}
template <typename T>
__device__ __forceinline__ void store_pairs(T* head, const Strides& st, const PairMap& m, int p0, const float (&a)[4],
                                            const float (&b)[4]) {
  if (st.vec && m.runs()) {
    if (m.adjacent(p0)) {
      const float x[4] = {a[0], b[0], a[1], b[1]}, y[4] = {a[2], b[2], a[3], b[3]};
      store4(head + 2 * p0, 1, 1, x);
      store4(head + 2 * p0 + 4, 1, 1, y);
    } else {
      store4(head + p0, 1, 1, a);
      store4(head + p0 + m.half, 1, 1, b);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    head[m.first(p0 + i) * st.elem] = from_f<T>(a[i]);
    head[m.second(p0 + i) * st.elem] = from_f<T>(b[i]);
  }
}

__device__ __forceinline__ void turn4(const float2* cs, int half, int p0, float (&a)[4], float (&b)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (p0 + i < half) {
      const float2 t = cs[p0 + i];
      const float x = a[i], y = b[i];
      a[i] = x * t.x - y * t.y;
      b[i] = y * t.x + x * t.y;
    }
  }
}

// Cosine and sine of every pair of the CTA's tokens (rows[t] < 0: none).
__device__ __forceinline__ void fill_turns(const imba_rotary_desc& rot, const int* rows, int ntok,
                                           float2 (*cs)[kMaxPairs]) {
  const int half = rot.rot_dim / 2;
  for (int t = threadIdx.x / 32; t < ntok; t += kWarps) {
    const int r = rows[t];
    if (r < 0) continue;
    for (int p = threadIdx.x % 32; p < half; p += 32) {
      const int ax = rot.axis ? min(max(rot.axis[p], 0), rot.num_axes - 1) : 0;
      const int64_t pos = rot.positions[(int64_t)r * rot.num_axes + ax];
      const uint64_t turn = (uint64_t)pos * rot.turns[p];
      // the fraction of a turn, in half turns: [-1, 1)
      const float x = (float)(int32_t)(turn >> 32) * 4.656612873077393e-10f;
      float s, c;
      sincospif(x, &s, &c);
      cs[t][p] = make_float2(c, s);
    }
  }
}

// Queries of rows [r0, r0 + q_rows): load, turn, store; a warp takes heads.
template <typename T, int D>
__device__ __forceinline__ void turn_queries(const AppendArgs& a, const int* rows, float2 (*cs)[kMaxPairs]) {
  constexpr int kLanes = D / 8, kGroup = 32 / kLanes, kPass = kTok / kGroup;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int p0 = lane % kLanes * 4, g = lane / kLanes;
  const PairMap m{a.rot.rot_dim / 2, a.rot.interleaved};
  for (int h = warp; h < a.Hq; h += kWarps) {
    float x[kPass][4], y[kPass][4];
#pragma unroll
    for (int i = 0; i < kPass; ++i) {
      const int t = i * kGroup + g;
      const int r = g < kGroup ? rows[t] : -1;
      if (r >= 0)
        load_pairs(static_cast<const T*>(a.q) + r * a.qs.row + h * a.qs.head, a.qs, m, p0, x[i], y[i]);
    }
#pragma unroll
    for (int i = 0; i < kPass; ++i) {
      const int t = i * kGroup + g;
      const int r = g < kGroup ? rows[t] : -1;
      if (r >= 0) {
        turn4(cs[t], m.half, p0, x[i], y[i]);
        store_pairs(static_cast<T*>(a.q_out) + r * a.qo.row + h * a.qo.head, a.qo, m, p0, x[i], y[i]);
      }
    }
  }
}

// Any head size: one thread per four pairs of a row's head.
template <typename T>
__device__ __forceinline__ void turn_queries_any(const AppendArgs& a, const int* rows, int ntok,
                                                 float2 (*cs)[kMaxPairs]) {
  const PairMap m{a.rot.rot_dim / 2, a.rot.interleaved};
  const int pairs = a.dqk / 2;
  for (int i = threadIdx.x; i < ntok * a.Hq * pairs; i += kThreads) {
    const int t = i / (a.Hq * pairs), h = i / pairs % a.Hq, p = i % pairs;
    const int r = rows[t];
    if (r < 0) continue;
    const T* s = static_cast<const T*>(a.q) + r * a.qs.row + h * a.qs.head;
    T* o = static_cast<T*>(a.q_out) + r * a.qo.row + h * a.qo.head;
    float x = to_f(s[m.first(p) * a.qs.elem]), y = to_f(s[m.second(p) * a.qs.elem]);
    if (p < m.half) {
      const float2 cc = cs[t][p];
      const float u = x;
      x = u * cc.x - y * cc.y;
      y = y * cc.x + u * cc.y;
    }
    o[m.first(p) * a.qo.elem] = from_f<T>(x);
    o[m.second(p) * a.qo.elem] = from_f<T>(y);
  }
}

// Rows of a query CTA: row ids, -1 for padding and past the end.
__device__ __forceinline__ void query_rows(const AppendArgs& a, int* rows) {
  if (threadIdx.x < kTok) {
    const int r = blockIdx.x * a.q_rows + threadIdx.x;
    const bool live = threadIdx.x < a.q_rows && r < a.n && a.slots[r] >= 0 && a.slots[r] < a.num_slots;
    rows[threadIdx.x] = live ? r : -1;
  }
}

// A magnitude for the block's scale; what is not finite becomes zero, and
// the last half step below 2^128 does not round up to it (240 2^120 is the
// largest stored value).
__device__ __forceinline__ void take_finite(float (&x)[4], float& amax, bool& bad) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (!(fabsf(x[i]) <= kLargest)) {
      bad |= !isfinite(x[i]);
      x[i] = isfinite(x[i]) ? copysignf(kLargest, x[i]) : 0.f;
    }
    amax = fmaxf(amax, fabsf(x[i]));
  }
}

// The block's new scale byte, its earlier codes rounded to it (whole warp).
template <int D>
__device__ __forceinline__ int grow_scale(uint8_t* block, uint8_t* scale, float amax, int lane) {
  const int was = *scale;
  const int now = max(was, scale_byte(warp_max(amax)));
  if (now > was && was > 0) {
    // 2^(was - now); below 2^-126 every code becomes zero all the same
    const float f = now - was > 126 ? 0.f : __uint_as_float((uint32_t)(127 - (now - was)) << 23);
    uint4* b = reinterpret_cast<uint4*>(block);
#pragma unroll
    for (int i = 0; i < D * kTok / 512; ++i) {
      uint4 u = b[i * 32 + lane];
      uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 lo = e4m3x2_to_f2(w[j] & 0xffffu), hi = e4m3x2_to_f2(w[j] >> 16);
        w[j] = to_e4m3x2(lo.x * f, lo.y * f) | to_e4m3x2(hi.x * f, hi.y * f) << 16;
      }
      b[i * 32 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  __syncwarp();
  if (now != was && lane == 0) *scale = (uint8_t)now;
  return now;
}

__device__ __forceinline__ uint32_t codes4(const float (&x)[4], float f) {
  return to_e4m3x2(x[0] * f, x[1] * f) | to_e4m3x2(x[2] * f, x[3] * f) << 16;
}

template <typename T, int D>
__device__ __forceinline__ void put_k8(const AppendArgs& a, const int* rows, float2 (*cs)[kMaxPairs], int h,
                                       uint8_t* block, uint8_t* scale, bool& bad) {
  constexpr int kLanes = D / 8, kGroup = 32 / kLanes, kPass = kTok / kGroup;
  const int lane = threadIdx.x % 32;
  const int p0 = lane % kLanes * 4, g = lane / kLanes;
  const PairMap m{a.rot.rot_dim / 2, a.rot.interleaved};
  float x[kPass][4], y[kPass][4], amax = 0.f;
#pragma unroll
  for (int i = 0; i < kPass; ++i) {
    const int r = g < kGroup ? rows[i * kGroup + g] : -1;
    if (r >= 0) load_pairs(static_cast<const T*>(a.k) + r * a.ks.row + h * a.ks.head, a.ks, m, p0, x[i], y[i]);
  }
#pragma unroll
  for (int i = 0; i < kPass; ++i) {
    const int t = i * kGroup + g;
    if ((g < kGroup ? rows[t] : -1) >= 0) {
      turn4(cs[t], m.half, p0, x[i], y[i]);
      take_finite(x[i], amax, bad);
      take_finite(y[i], amax, bad);
    }
  }
  const int b = grow_scale<D>(block, scale, amax, lane);
  const float f = b ? inv_scale_of(b) : 0.f;
#pragma unroll
  for (int i = 0; i < kPass; ++i) {
    const int t = i * kGroup + g;
    if ((g < kGroup ? rows[t] : -1) < 0) continue;
    uint8_t* o = block + t * D;
    if (m.runs()) {
      if (m.adjacent(p0)) {
        const float u[4] = {x[i][0], y[i][0], x[i][1], y[i][1]}, v[4] = {x[i][2], y[i][2], x[i][3], y[i][3]};
        *reinterpret_cast<uint2*>(o + 2 * p0) = make_uint2(codes4(u, f), codes4(v, f));
      } else {
        *reinterpret_cast<uint32_t*>(o + p0) = codes4(x[i], f);
        *reinterpret_cast<uint32_t*>(o + p0 + m.half) = codes4(y[i], f);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t two = to_e4m3x2(x[i][j] * f, y[i][j] * f);
        o[m.first(p0 + j)] = (uint8_t)two;
        o[m.second(p0 + j)] = (uint8_t)(two >> 8);
      }
    }
  }
}

// A lane holds eight dimensions of consecutive tokens, so that a pair of
// tokens is one 16-byte store of the block's [8][d_v][2] layout.
template <typename T, int D>
__device__ __forceinline__ void put_v8(const AppendArgs& a, const int* rows, int h, uint8_t* block, uint8_t* scale,
                                       bool& bad) {
  constexpr int kLanes = D / 8, kGroup = 32 / kLanes, kPass = kTok / kGroup;
  const int lane = threadIdx.x % 32;
  const int e0 = lane % kLanes * 8, g = lane / kLanes;
  float x[kPass][4], y[kPass][4], amax = 0.f;
#pragma unroll
  for (int i = 0; i < kPass; ++i) {
    const int r = g < kGroup ? rows[g * kPass + i] : -1;
    if (r >= 0) {
      const T* s = static_cast<const T*>(a.v) + r * a.vs.row + h * a.vs.head + e0 * a.vs.elem;
      load4(s, a.vs.elem, a.vs.vec, x[i]);
      load4(s + 4 * a.vs.elem, a.vs.elem, a.vs.vec, y[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[i][j] = y[i][j] = 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < kPass; ++i) {
    take_finite(x[i], amax, bad);
    take_finite(y[i], amax, bad);
  }
  const int b = grow_scale<D>(block, scale, amax, lane);
  const float f = b ? inv_scale_of(b) : 0.f;
#pragma unroll
  for (int i = 0; i < kPass; i += 2) {
    if (g >= kGroup) continue;
    const int t = g * kPass + i;
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
    uint4* o = reinterpret_cast<uint4*>(block + v8_off(t, e0, D));
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

template <typename T, int DQK, int DV>
__global__ void __launch_bounds__(kThreads) append8_kernel(AppendArgs a, Cache8 c) {
  __shared__ int rows[kTok];
  __shared__ float2 cs[kTok][kMaxPairs];
  pdl_wait();
  pdl_trigger();
  if ((int)blockIdx.x < a.q_blocks) {
    query_rows(a, rows);
    __syncthreads();
    fill_turns(a.rot, rows, a.q_rows, cs);
    __syncthreads();
    turn_queries<T, DQK>(a, rows, cs);
    return;
  }
  const int warp = threadIdx.x / 32;
  const int count = *a.plan.count + 1;
  bool bad = false;
  for (int e = blockIdx.x - a.q_blocks; e < count; e += gridDim.x - a.q_blocks) {
    const int at = a.plan.list[e];
    const int page = a.plan.keys[at];
    if (page < 0 || page >= c.num_pages) continue;  // a plan of another pool
    if (threadIdx.x < kTok) rows[threadIdx.x] = a.plan.rows[(size_t)at * kTok + threadIdx.x];
    __syncthreads();
    fill_turns(a.rot, rows, kTok, cs);
    __syncthreads();
    uint8_t* data = c.data + page * c.page_stride;
    uint8_t* scales = c.scales + page * c.scale_stride;
    for (int i = warp; i < 2 * a.H; i += kWarps) {
      const int h = i >> 1;
      if (i & 1)
        put_v8<T, DV>(a, rows, h, data + c.v_offset + (int64_t)h * kTok * DV, scales + a.H + h, bad);
      else
        put_k8<T, DQK>(a, rows, cs, h, data + (int64_t)h * kTok * DQK, scales + h, bad);
    }
    __syncthreads();
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
    query_rows(a, rows);
    __syncthreads();
    fill_turns(a.rot, rows, a.q_rows, cs);
    __syncthreads();
    turn_queries_any<T>(a, rows, a.q_rows, cs);
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
        if (p < m.half) {
          const float2 cc = cs[t][p];
          const float u = x;
          x = u * cc.x - y * cc.y;
          y = y * cc.x + u * cc.y;
        }
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
  // Queries: 16 rows a CTA share their cosines over the heads; with few rows
  // smaller CTAs fill the device.
  a.q_rows = d.num_rows >= 16 * 148 * 2 ? 16 : 4;
  a.q_blocks = a.Hq ? (d.num_rows + a.q_rows - 1) / a.q_rows : 0;
  const int64_t pages = std::min<int64_t>(d.num_rows, 148 * 8);
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
  if (c->dtype == IMBA_DTYPE_E4M3 && !cache8_dims_ok(c->attention_dim, c->linear_dim)) return IMBA_ERR_UNSUPPORTED;
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
