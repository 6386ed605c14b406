// Attention over a paged pool in 8 bits: the kernel (one translation unit per
// query type includes this file).
//
//   o_r = sum_j w_rj v_j / sum_j w_rj,  w_rj = exp(scale q_r . k_j + bias),
//   j < vis[r] and the row's extra keys; k_j and v_j are e4m3 codes times a
//   power of two of their block.
//
// What bounds it: a decode step reads every code once for a few rows, so HBM
// (and, for short lists, the latency of three dependent loads); the design
// keeps many page loads in flight and spends few instructions per code.
//
// Layout.  One warp takes a head's page of 16 tokens at a time, with
// mma.m16n8k16 on f16 operands and fp32 sums: e4m3 is exact in f16, and the
// blocks' scales multiply scores and weights, not elements.  A contraction
// may run over its dimension in any order as long as both operands agree, so
// the order is chosen for the loads: a lane reads 16 (8 when the head size is
// no multiple of 64) consecutive bytes of a key, four lanes a key, and these
// are its B fragments of the next k-steps as they are; V's pairs of tokens
// are the two halves of a B register, so 16 bytes are eight column tiles'
// fragments.  No shuffle, no transposition, and what a lane loads it alone
// reads, so the cp.async ring in shared memory needs no barrier.
//
// Numerics.  A query row is divided by the power of two of its largest
// element before it becomes f16 (bf16 queries lose nothing above 2^-24 of
// that element; fp32 queries are the sum of two f16 parts, 22 bits).  Weights
// are held relative to a running maximum that is raised when a score passes
// it by 2^kSlack, times 2^kShift so that small ones stay normal in f16 (fp32:
// two parts); V's scale enters as its ratio to a reference exponent that
// follows the blocks (|log2 ratio| <= kVWindow, else the sums so far are
// rescaled, a power of two).  Sums, maxima and weights are fp32.
#pragma once

#include "attend8.cuh"

namespace imba {

namespace {

constexpr float kShift = 5.f;
constexpr float kSlack = 4.f;
constexpr int kVWindow = 6;  // 2^(kShift + kSlack + kVWindow) = 2^15 is finite in f16
constexpr float kLowest = -3.402823466e38f;

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_h2(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }

// (lo, hi) as f16 pairs: the rounded values, and with NP == 2 what is left.
template <int NP>
__device__ __forceinline__ void split_h2(float lo, float hi, uint32_t (&out)[NP]) {
  out[0] = pack_h2(lo, hi);
  if constexpr (NP == 2) {
    const float2 r = unpack_h2(out[0]);
    out[1] = pack_h2(lo - r.x, hi - r.y);
  }
}

template <int B>
__device__ __forceinline__ void cp_async(uint32_t dst, const uint8_t* src) {
  if constexpr (B == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <int B>
__device__ __forceinline__ void lds(uint32_t src, uint32_t (&w)[B / 4]) {
  if constexpr (B == 16)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(src)
                 : "memory");
  else
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(src) : "memory");
}

__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 1);
  return x + __shfl_xor_sync(0xffffffffu, x, 2);
}

// The bias in the log2 domain; a finite bias stays finite, so a row whose
// every key carries the type's lowest value still weighs them alike.
__device__ __forceinline__ float bias_log2(float b) {
  return b == -INFINITY ? b : fmaxf(b * kLog2e, kLowest);
}

// 2^(a - b) for running maxima; 0 for a part that has seen nothing.
__device__ __forceinline__ float weight_of(float a, float b) { return a == -INFINITY ? 0.f : exp2_approx(a - b); }

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

// Sizes that follow from the head dimensions.
template <int DQK, int DV, int MT>
struct Dims {
  static constexpr int VK = DQK % 64 ? 8 : 16, VV = DV % 64 ? 8 : 16;  // bytes of a lane's load
  static constexpr int CK = DQK / 4 / VK, CV = DV / 4 / VV;            // loads per 8 keys / per 4 pairs
  static constexpr int KS = DQK / 16, NT = DV / 8;                     // k-steps of a score, column tiles of O
  static constexpr int ROWS = kTileRows * MT;
  static constexpr int STAGE = IMBA_PAGE_TOKENS * (DQK + DV);  // a warp's page
  static constexpr int MERGE = kUnitWarps * ROWS * (DV * 4 + 8) + ROWS * 4;
};

// The state of a warp's rows: row 16 i + lane / 4 + 8 r of the tile.
template <int MT>
struct RowState {
  float m[MT][2];  // running maximum (log2 domain)
  float l[MT][2];  // sum of weights over this lane's keys
};

// Tile rows joined over the items of a split tile; `nthr` threads from tid on.
template <typename T, int DQK, int DV, int MT>
__device__ __forceinline__ void join_items(const AttendArgs& a, const AttendItem& it, int head, int tid, int nthr) {
  using D = Dims<DQK, DV, MT>;
  const int H = a.cache.H;
  const size_t first = (size_t)(it.part - it.index) * H + head;
  const AttendRow* rows = a.plan.rows + (size_t)it.tile * D::ROWS;
  const bool vec = a.call.out_stride[0] % 4 == 0 && a.call.out_stride[1] % 4 == 0 &&
                   (reinterpret_cast<uintptr_t>(a.call.out) & (4 * sizeof(T) - 1)) == 0;
  for (int i = tid; i < D::ROWS * (DV / 4); i += nthr) {
    const int r = i / (DV / 4), e = i % (DV / 4) * 4;
    const AttendRow row = rows[r];
    if (row.row < 0) continue;
    float m = -INFINITY, l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < it.splits; ++s)
      m = fmaxf(m, __ldcg(a.plan.ml + (first + (size_t)s * H) * D::ROWS + r).x);
    for (int s = 0; s < it.splits; ++s) {
      const size_t at = (first + (size_t)s * H) * D::ROWS + r;
      const float2 ml = __ldcg(a.plan.ml + at);
      const float w = weight_of(ml.x, m);
      const float4 o = __ldcg(reinterpret_cast<const float4*>(a.plan.o + at * DV + e));
      l += w * ml.y;
      x[0] += w * o.x, x[1] += w * o.y, x[2] += w * o.z, x[3] += w * o.w;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] *= inv;
    out_store4(static_cast<T*>(a.call.out) + row.row * a.call.out_stride[0] +
                   (int64_t)(head * a.shape.share + row.head) * a.call.out_stride[1] + e,
               vec, x);
  }
}

template <typename T, int DQK, int DV, int MT, int NW, int STAGES>
__global__ void __launch_bounds__(kUnitWarps * 32, DQK <= 64 && MT == 1 && sizeof(T) == 2 ? 2 : 1)
    attend8_kernel(AttendArgs a) {
  using D = Dims<DQK, DV, MT>;
  constexpr int NP = sizeof(T) == 4 ? 2 : 1;
  extern __shared__ __align__(16) uint8_t smem[];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int sub = NW == 1 ? 0 : warp;
  const int H = a.cache.H;
  const int64_t unit = NW == 1 ? (int64_t)blockIdx.x * kUnitWarps + warp : blockIdx.x;
  const int item_id = (int)(unit / H), head = (int)(unit % H);
  if (item_id >= a.plan.head[0]) return;
  const AttendItem it = a.plan.items[item_id];
  const AttendRow* tile = a.plan.rows + (size_t)it.tile * D::ROWS;

  // This warp's pages: list entries sub, sub + NW, ... of the item, 32 at a
  // time in the lanes (id and the two scale bytes), the next 32 in flight.
  const int npages = it.pages > sub ? (it.pages - sub + NW - 1) / NW : 0;
  const uint8_t* head_k = a.cache.data + (int64_t)head * IMBA_PAGE_TOKENS * DQK;
  const int64_t v_from_k = a.cache.v_offset + (int64_t)head * IMBA_PAGE_TOKENS * (DV - DQK);
  auto page_id = [&](int i) -> int {  // -1: none, -2: outside the pool
    if (i >= npages) return -1;
    const int id = a.rows.group_pages[it.list + sub + i * NW];
    return id >= 0 && id < a.cache.num_pages ? id : -2;
  };
  auto page_scales = [&](int id) -> int {
    if (id < 0) return 0;
    const uint8_t* s = a.cache.scales + id * a.cache.scale_stride + head;
    return s[0] | s[H] << 8;
  };
  int ids = page_id(lane), ids_next = page_id(32 + lane);

  AttendRow rows[MT][2];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int4 u = __ldg(reinterpret_cast<const int4*>(tile + 16 * i + g + 8 * r));
      rows[i][r] = AttendRow{u.x, u.y, u.z, u.w};
    }
  int scs = page_scales(ids), scs_next = page_scales(ids_next);
  if (__any_sync(0xffffffffu, ids == -2 || ids_next == -2) && lane == 0) report(a.rows.status, IMBA_ERR_RANGE);

  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * (STAGES * D::STAGE);
  auto issue = [&](int i, int batch) {  // page i of the warp into its stage; `batch` holds i's page id
    const int id = __shfl_sync(0xffffffffu, batch, i & 31);
    if (i < npages) {
      const uint8_t* k = head_k + max(id, 0) * a.cache.page_stride;
      const uint32_t dst = ring + i % STAGES * D::STAGE;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int c = 0; c < D::CK; ++c)
          cp_async<D::VK>(dst + ((n * D::CK + c) * 32 + lane) * D::VK,
                          k + (n * 8 + g) * DQK + c * 4 * D::VK + t * D::VK);
      const uint8_t* v = k + v_from_k;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int c = 0; c < D::CV; ++c)
          cp_async<D::VV>(dst + IMBA_PAGE_TOKENS * DQK + ((n * D::CV + c) * 32 + lane) * D::VV,
                          v + (n * 4 + t) * 2 * DV + c * 8 * D::VV + g * D::VV);
    }
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) issue(i, ids);

  // Queries: f16 A fragments of each row over its power of two.
  uint32_t qa[MT][NP][D::KS][4];
  float fac[MT][2];
  const bool qvec = a.call.q_stride[0] % 4 == 0 && a.call.q_stride[1] % 4 == 0 &&
                    (reinterpret_cast<uintptr_t>(a.call.q) & (4 * sizeof(T) - 1)) == 0;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const AttendRow& row = rows[i][r];
      const T* q = static_cast<const T*>(a.call.q) + row.row * a.call.q_stride[0] +
                   (int64_t)(head * a.shape.share + row.head) * a.call.q_stride[1];
      float x[D::KS][4], amax = 0.f;
#pragma unroll
      for (int s = 0; s < D::KS; ++s) {
        x[s][0] = x[s][1] = x[s][2] = x[s][3] = 0.f;
        if (row.row >= 0) q_load4(q + s / (D::VK / 4) * 4 * D::VK + t * D::VK + s % (D::VK / 4) * 4, qvec, x[s]);
#pragma unroll
        for (int j = 0; j < 4; ++j) amax = fmaxf(amax, fabsf(x[s][j]));
      }
      amax = quad_max(amax);
      const int ex = (int)(__float_as_uint(amax) >> 23);  // 0 for a zero row, 255 for an infinite one
      const int e = ex == 0 || ex == 255 ? 0 : min(ex - 127, 126);
      const float down = __uint_as_float((uint32_t)(127 - e) << 23);
      fac[i][r] = __uint_as_float((uint32_t)(127 + e) << 23) * a.call.scale * kLog2e;
#pragma unroll
      for (int s = 0; s < D::KS; ++s) {
        uint32_t lo[NP], hi[NP];
        split_h2<NP>(x[s][0] * down, x[s][1] * down, lo);
        split_h2<NP>(x[s][2] * down, x[s][3] * down, hi);
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          qa[i][p][s][r] = lo[p];
          qa[i][p][s][2 + r] = hi[p];
        }
      }
    }

  RowState<MT> st;
  float o[MT][D::NT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    st.m[i][0] = st.m[i][1] = -INFINITY;
    st.l[i][0] = st.l[i][1] = 0.f;
#pragma unroll
    for (int j = 0; j < D::NT; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.f;
  }
  int vref = 0;  // scale byte that O is held in units of; 0: none yet

  for (int i = 0; i < npages; ++i) {
    if (i && (i & 31) == 0) {
      ids = ids_next;
      scs = scs_next;
      ids_next = page_id(i + 32 + lane);
      scs_next = page_scales(ids_next);
      if (__any_sync(0xffffffffu, ids_next == -2) && lane == 0) report(a.rows.status, IMBA_ERR_RANGE);
    }
    const int sc = __shfl_sync(0xffffffffu, scs, i & 31);
    const int id = __shfl_sync(0xffffffffu, ids, i & 31);
    {
      const int ahead = i + STAGES - 1;
      const int batch = (ahead >> 5) == (i >> 5) ? ids : ids_next;
      cp_wait<STAGES - 2>();  // page i has arrived
      issue(ahead, batch);    // into the stage that page i - 1 left
    }
    const uint32_t src = ring + i % STAGES * D::STAGE;
    const int key0 = it.key0 + (sub + i * NW) * IMBA_PAGE_TOKENS;
    const float ks = scale_of(sc & 255);
    const int vb = sc >> 8;

    // Scores of 16 keys.
    float s[MT][2][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < 2; ++n) s[m][n][0] = s[m][n][1] = s[m][n][2] = s[m][n][3] = 0.f;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int c = 0; c < D::CK; ++c) {
        uint32_t w[D::VK / 4];
        lds<D::VK>(src + ((n * D::CK + c) * 32 + lane) * D::VK, w);
#pragma unroll
        for (int j = 0; j < D::VK / 4; ++j) {
          const uint32_t b0 = e4m3x2_to_h2(w[j]), b1 = e4m3x2_to_h2(w[j] >> 16);
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int p = 0; p < NP; ++p) mma_f16(s[m][n], qa[m][p][c * (D::VK / 4) + j], b0, b1);
        }
      }

    // log2-domain scores; the keys a row does not see are -inf.
    const bool whole = id >= 0 && key0 + IMBA_PAGE_TOKENS <= it.minvis;
    bool raise = false;
    float mx[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float f = ks * fac[m][r];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) s[m][n][2 * r + j] *= f;
        if (a.call.bias && rows[m][r].row >= 0) {
          const float* b =
              a.call.bias + (int64_t)(head * a.shape.share + rows[m][r].head) * (2 * a.call.max_pos - 1);
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              s[m][n][2 * r + j] +=
                  bias_log2(__ldg(b + bias_index(key0 + n * 8 + 2 * t + j, rows[m][r].pos, a.call.max_pos)));
        }
        if (!whole) {
          const int vis = id >= 0 ? rows[m][r].vis - key0 : 0;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if (n * 8 + 2 * t + j >= vis) s[m][n][2 * r + j] = -INFINITY;
        }
        mx[m][r] = fmaxf(fmaxf(s[m][0][2 * r], s[m][0][2 * r + 1]), fmaxf(s[m][1][2 * r], s[m][1][2 * r + 1]));
        raise |= mx[m][r] > st.m[m][r] + kSlack;
      }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float now = fmaxf(st.m[m][r], quad_max(mx[m][r]));
          const float w = weight_of(st.m[m][r], now);
          st.m[m][r] = now;
          st.l[m][r] *= w;
#pragma unroll
          for (int j = 0; j < D::NT; ++j) {
            o[m][j][2 * r] *= w;
            o[m][j][2 * r + 1] *= w;
          }
        }
    }
    // V's scale as a ratio to vref.
    float ratio = 1.f;
    if (vb) {
      if (vref == 0) vref = vb;
      if (abs(vb - vref) > kVWindow) {
        const int now = max(vb, vref - 60);
        const float f = vref - now < -126 ? 0.f : __uint_as_float((uint32_t)(127 + vref - now) << 23);
        vref = now;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int j = 0; j < D::NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[m][j][e] *= f;
      }
      ratio = vb - vref < -126 ? 0.f : __uint_as_float((uint32_t)(127 + vb - vref) << 23);
    }
    uint32_t pa[MT][NP][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float ref = st.m[m][r] == -INFINITY ? 0.f : st.m[m][r] - kShift;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float p0 = exp2_approx(s[m][n][2 * r] - ref), p1 = exp2_approx(s[m][n][2 * r + 1] - ref);
          st.l[m][r] += p0 + p1;
          uint32_t h[NP];
          split_h2<NP>(p0 * ratio, p1 * ratio, h);
#pragma unroll
          for (int p = 0; p < NP; ++p) pa[m][p][2 * n + r] = h[p];
        }
      }
#pragma unroll
    for (int c = 0; c < D::CV; ++c) {
      uint32_t w0[D::VV / 4], w1[D::VV / 4];
      lds<D::VV>(src + IMBA_PAGE_TOKENS * DQK + (c * 32 + lane) * D::VV, w0);
      lds<D::VV>(src + IMBA_PAGE_TOKENS * DQK + ((D::CV + c) * 32 + lane) * D::VV, w1);
#pragma unroll
      for (int j = 0; j < D::VV / 2; ++j) {
        const uint32_t b0 = e4m3x2_to_h2(w0[j / 2] >> (16 * (j % 2)));
        const uint32_t b1 = e4m3x2_to_h2(w1[j / 2] >> (16 * (j % 2)));
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int p = 0; p < NP; ++p) mma_f16(o[m][c * (D::VV / 2) + j], pa[m][p], b0, b1);
      }
    }
  }

  // The rows' extra keys, one at a time: four lanes share a row, each with
  // the dimensions that its fragments hold.
  if (a.rows.num_extra > 0 && it.index == 0 && sub == 0) {
    const int64_t slots = a.cache.num_pages * IMBA_PAGE_TOKENS;
    if (vref == 0) vref = 127;
    const float unref = __uint_as_float((uint32_t)(254 - vref) << 23);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const AttendRow row = rows[m][r];
        int e0 = 0, e1 = 0;
        if (row.row >= 0) {
          e0 = a.rows.row_extra_off[row.row];
          e1 = a.rows.row_extra_off[row.row + 1];
          if (e0 < 0 || e1 < e0 || e1 > a.rows.num_extra) {
            report(a.rows.status, IMBA_ERR_RANGE);
            e0 = e1 = 0;
          }
        }
        const int most = __reduce_max_sync(0xffffffffu, e1 - e0);
        for (int x = 0; x < most; ++x) {
          int64_t slot = -1;
          float b = 0.f;
          if (e0 + x < e1) {
            slot = a.rows.extra_slot[e0 + x];
            if (slot < 0 || slot >= slots) {
              report(a.rows.status, IMBA_ERR_RANGE);
              slot = -1;
            }
            if (a.call.bias)
              b = bias_log2(a.call.bias[(int64_t)(head * a.shape.share + row.head) * (2 * a.call.max_pos - 1) +
                                        bias_index(a.rows.extra_pos[e0 + x], row.pos, a.call.max_pos)]);
          }
          const int64_t page = max(slot, (int64_t)0) / IMBA_PAGE_TOKENS;
          const int tok = (int)(max(slot, (int64_t)0) % IMBA_PAGE_TOKENS);
          const int sc = page_scales((int)page);
          const uint8_t* k = head_k + page * a.cache.page_stride;
          float dot = 0.f;
#pragma unroll
          for (int c = 0; c < D::CK; ++c)
#pragma unroll
            for (int j = 0; j < D::VK / 4; ++j) {
              const uint32_t w = *reinterpret_cast<const uint32_t*>(k + tok * DQK + c * 4 * D::VK + t * D::VK + 4 * j);
              const float2 k0 = e4m3x2_to_f2(w), k1 = e4m3x2_to_f2(w >> 16);
#pragma unroll
              for (int p = 0; p < NP; ++p) {
                const float2 q0 = unpack_h2(qa[m][p][c * (D::VK / 4) + j][r]);
                const float2 q1 = unpack_h2(qa[m][p][c * (D::VK / 4) + j][2 + r]);
                dot = fmaf(q0.x, k0.x, fmaf(q0.y, k0.y, fmaf(q1.x, k1.x, fmaf(q1.y, k1.y, dot))));
              }
            }
          dot = quad_sum(dot);
          const float sx = slot < 0 ? -INFINITY : dot * scale_of(sc & 255) * fac[m][r] + b;
          const float now = fmaxf(st.m[m][r], sx);
          const float w = weight_of(st.m[m][r], now);
          const float p = now == -INFINITY && sx == sx ? 0.f : exp2_approx(sx - (now - kShift));
          st.m[m][r] = now;
          st.l[m][r] = st.l[m][r] * w + (t == 0 ? p : 0.f);  // summed over the quad at the end
          const float pv = p * (scale_of(sc >> 8) * unref);
          const uint8_t* v = k + v_from_k;
#pragma unroll
          for (int c = 0; c < D::CV; ++c)
#pragma unroll
            for (int j = 0; j < D::VV / 2; ++j) {
              // column tile c, j: dimensions 4 VV c + VV t + j and that + VV / 2
              const int e = c * 4 * D::VV + t * D::VV + j;
              float* od = o[m][c * (D::VV / 2) + j] + 2 * r;
              od[0] = fmaf(pv, e4m3x2_to_f2(v[v8_off(tok, e, DV)]).x, od[0] * w);
              od[1] = fmaf(pv, e4m3x2_to_f2(v[v8_off(tok, e + D::VV / 2, DV)]).x, od[1] * w);
            }
        }
      }
  }

  // Out: true units, relative to each row's running maximum.
  const float unit_v = vref ? scale_of(vref) : 1.f;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int r = 0; r < 2; ++r) st.l[m][r] = quad_sum(st.l[m][r]);
  const bool ovec = a.call.out_stride[0] % 4 == 0 && a.call.out_stride[1] % 4 == 0 &&
                    (reinterpret_cast<uintptr_t>(a.call.out) & (4 * sizeof(T) - 1)) == 0;

  if constexpr (NW == 1) {
    const size_t part = ((size_t)max(it.part, 0) * H + head) * D::ROWS;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const AttendRow& row = rows[m][r];
        if (row.row < 0) continue;
        const int tr = 16 * m + g + 8 * r;
        const float f = it.part >= 0 ? unit_v : st.l[m][r] == 0.f ? 0.f : unit_v / st.l[m][r];
        if (it.part >= 0 && t == 0) a.plan.ml[part + tr] = make_float2(st.m[m][r], st.l[m][r]);
        T* out = static_cast<T*>(a.call.out) + row.row * a.call.out_stride[0] +
                 (int64_t)(head * a.shape.share + row.head) * a.call.out_stride[1];
#pragma unroll
        for (int c = 0; c < D::CV; ++c)
#pragma unroll
          for (int q = 0; q < D::VV / 4; ++q) {  // dimensions 4 VV c + VV t + 4 q .. + 3
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int d = 4 * q + j;
              x[j] = o[m][c * (D::VV / 2) + d % (D::VV / 2)][2 * r + d / (D::VV / 2)] * f;
            }
            const int e = c * 4 * D::VV + t * D::VV + 4 * q;
            if (it.part >= 0)
              *reinterpret_cast<float4*>(a.plan.o + (part + tr) * DV + e) = make_float4(x[0], x[1], x[2], x[3]);
            else
              out_store4(out + e, ovec, x);
          }
      }
    if (it.part >= 0) {
      __threadfence();
      __syncwarp();
      int* done = a.plan.done + (size_t)it.tile * H + head;
      int n = 0;
      if (lane == 0) n = atomicAdd(done, 1);
      if (__shfl_sync(0xffffffffu, n, 0) == it.splits - 1) {  // the others have finished
        __threadfence();
        if (lane == 0) *done = 0;
        join_items<T, DQK, DV, MT>(a, it, head, lane, 32);
      }
    }
  } else {
    // The warps' parts meet in shared memory (over the ring, which is idle).
    float* so = reinterpret_cast<float*>(smem);                              // [warps][rows][DV]
    float2* sml = reinterpret_cast<float2*>(so + kUnitWarps * D::ROWS * DV);  // [warps][rows]
    int* flag = reinterpret_cast<int*>(sml + kUnitWarps * D::ROWS);
    cp_wait<0>();
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int tr = 16 * m + g + 8 * r;
        if (rows[m][r].row < 0) continue;
        if (t == 0) sml[warp * D::ROWS + tr] = make_float2(st.m[m][r], st.l[m][r]);
        float* dst = so + (warp * D::ROWS + tr) * DV;
#pragma unroll
        for (int c = 0; c < D::CV; ++c)
#pragma unroll
          for (int q = 0; q < D::VV / 4; ++q) {
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int d = 4 * q + j;
              x[j] = o[m][c * (D::VV / 2) + d % (D::VV / 2)][2 * r + d / (D::VV / 2)] * unit_v;
            }
            *reinterpret_cast<float4*>(dst + c * 4 * D::VV + t * D::VV + 4 * q) = make_float4(x[0], x[1], x[2], x[3]);
          }
      }
    __syncthreads();
    const size_t part = ((size_t)max(it.part, 0) * H + head) * D::ROWS;
    for (int i = threadIdx.x; i < D::ROWS * (DV / 4); i += kUnitWarps * 32) {
      const int tr = i / (DV / 4), e = i % (DV / 4) * 4;
      const int4 u = __ldg(reinterpret_cast<const int4*>(tile + tr));
      const AttendRow row{u.x, u.y, u.z, u.w};
      if (row.row < 0) continue;
      float mm = -INFINITY, l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kUnitWarps; ++w) mm = fmaxf(mm, sml[w * D::ROWS + tr].x);
#pragma unroll
      for (int w = 0; w < kUnitWarps; ++w) {
        const float2 ml = sml[w * D::ROWS + tr];
        const float f = weight_of(ml.x, mm);
        const float4 v = *reinterpret_cast<const float4*>(so + (w * D::ROWS + tr) * DV + e);
        l += f * ml.y;
        x[0] += f * v.x, x[1] += f * v.y, x[2] += f * v.z, x[3] += f * v.w;
      }
      if (it.part >= 0) {
        if (e == 0) a.plan.ml[part + tr] = make_float2(mm, l);
        *reinterpret_cast<float4*>(a.plan.o + (part + tr) * DV + e) = make_float4(x[0], x[1], x[2], x[3]);
      } else {
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] *= inv;
        out_store4(static_cast<T*>(a.call.out) + row.row * a.call.out_stride[0] +
                       (int64_t)(head * a.shape.share + row.head) * a.call.out_stride[1] + e,
                   ovec, x);
      }
    }
    if (it.part >= 0) {
      __threadfence();
      __syncthreads();
      int* done = a.plan.done + (size_t)it.tile * H + head;
      if (threadIdx.x == 0) *flag = atomicAdd(done, 1) == it.splits - 1;
      __syncthreads();
      if (*flag) {
        __threadfence();
        if (threadIdx.x == 0) *done = 0;
        join_items<T, DQK, DV, MT>(a, it, head, threadIdx.x, kUnitWarps * 32);
      }
    }
  }
}

template <typename T, int DQK, int DV, int MT, int NW>
cudaError_t launch_one(const AttendArgs& a, cudaStream_t s) {
  using D = Dims<DQK, DV, MT>;
  constexpr int kStages = 4;
  constexpr size_t ring = (size_t)kUnitWarps * kStages * D::STAGE;
  constexpr size_t smem = NW > 1 && D::MERGE > ring ? D::MERGE : ring;
  auto fn = attend8_kernel<T, DQK, DV, MT, NW, kStages>;
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  const int64_t units = (int64_t)a.shape.max_items * a.cache.H;
  const int64_t grid = NW == 1 ? (units + kUnitWarps - 1) / kUnitWarps : units;
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  return launch_pdl(fn, dim3((unsigned)grid), dim3(kUnitWarps * 32), smem, s, a);
}

}  // namespace

template <typename T>
cudaError_t launch_attend8(const imba_cache_desc& c, const AttendArgs& a, cudaStream_t s) {
#define IMBA_ATTEND8(DQK, DV)                                                     \
  if (c.attention_dim == DQK && c.linear_dim == DV)                               \
    return a.shape.warps == 1 ? launch_one<T, DQK, DV, 1, 1>(a, s)                \
                              : launch_one<T, DQK, DV, 1, kUnitWarps>(a, s);
  IMBA_ATTEND8(32, 32)
  IMBA_ATTEND8(64, 64)
  IMBA_ATTEND8(32, 64)
  IMBA_ATTEND8(64, 32)
  IMBA_ATTEND8(96, 96)
  IMBA_ATTEND8(128, 128)
#undef IMBA_ATTEND8
  return cudaErrorInvalidValue;
}

}  // namespace imba
