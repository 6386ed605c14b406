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
// blocks' scales multiply scores and weights, not elements.  The cache is the
// 16-row operand, S' = K Q' and O' = V' P', so that a tile is eight query rows
// and not sixteen: a decode step has few of them, and every instruction but
// the conversions is per row.  The weights pass from the result's layout to the
// operand's by movmatrix.  A step of 1,024 one-token games (8 heads of 64)
// takes 34 us, 1.8 TB/s, of which the chain of dependent loads is the most (and
// 104 bytes a thread of spills at three CTAs' 80 registers); 32 long sequences
// (8 heads of 128, four query heads each) 263 us, 4.9 TB/s.  With the rows as
// the 16-row operand they took 45 and 324.
//
// A contraction may run over its dimension in any order as long as both
// operands agree, so the order is chosen for the loads: a lane reads 16 (8
// when the head size is no multiple of 64) consecutive bytes of a key, four
// lanes a key, and these are its fragments of the next k-steps as they are;
// V's pairs of tokens are the two halves of a register, so 16 bytes are four
// row tiles' fragments.  No shuffle, and what a lane loads it alone reads, so
// the cp.async ring in shared memory needs no barrier.
//
// Numerics.  A query row is divided by the power of two of its largest
// element before it becomes f16 (bf16 queries are exact down to 2^-17 of that
// element and off by 2^-25 of it at most below; fp32 queries are the sum of two
// f16 parts, 22 bits, off by 2^-25 of it at most too).  Weights are held
// relative to a running maximum that is raised when a score passes it by
// 2^kSlack, times 2^kShift so that small ones stay normal in f16 (fp32: two
// parts); one below 2^-30 of the row's largest counts in the sum alone.  V's
// scale enters as its ratio to a reference exponent that follows the blocks
// (|log2 ratio| <= kVWindow, else the sums so far are rescaled, a power of two;
// a block whose scale is below 2^-80 of the largest so far loses precision, and
// counts as zero below 2^-110).  Sums, maxima and weights are fp32.
#pragma once

#include "attend8_common.cuh"

namespace imba {

namespace {

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ int add_sat(int a, int b) {
  int r;
  asm("add.sat.s32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// An 8 x 8 matrix of f16 from a fragment of its rows to one of its columns.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

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

// Over the four lanes of a row's query fragment.
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}
// Over the eight lanes that hold a row's keys.
__device__ __forceinline__ float keys_max(float x) {
#pragma unroll
  for (int o = 4; o < 32; o *= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
__device__ __forceinline__ float keys_sum(float x) {
#pragma unroll
  for (int o = 4; o < 32; o *= 2) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// Sizes that follow from the head dimensions.  RT: groups of eight rows.
template <int DQK, int DV, int RT>
struct Dims {
  static constexpr int VK = DQK % 64 ? 8 : 16, VV = DV % 64 ? 8 : 16;  // bytes of a lane's load
  static constexpr int CK = DQK / 4 / VK, CV = DV / 4 / VV;            // loads per 8 keys / per 4 pairs
  static constexpr int KS = DQK / 16, MV = DV / 16;                    // k-steps of a score, row tiles of O'
  static constexpr int ROWS = kTileRows * RT;
  static constexpr int STAGE = IMBA_PAGE_TOKENS * (DQK + DV);  // a warp's page
  static constexpr int MERGE = kUnitWarps * (ROWS * (DV * 4 + 8) + 4) + 16;
};

// A warp's rows and what they have summed up: lane (g, t) = (lane / 4, lane %
// 4) holds rows 8 i + 2 t + r, i < RT, r < 2, of scores and weights for keys g
// and g + 8, and of O' for dimensions 4 VV c + VV / 2 g + 0 .. VV / 2 - 1.
template <int DQK, int DV, int RT, int NP>
struct Rows {
  using D = Dims<DQK, DV, RT>;
  uint32_t q[RT][NP][D::KS][2];  // row 8 i + g: B fragments
  float fac[RT][2];              // of a raw score, without the block's scale
  int vis[RT][2], pos[RT][2];    // visible tokens; the bias column of a key is its position plus pos, clamped
  const float* bias[RT][2];      // the row's bias (the call has one, or none of them is read)
  float m[RT][2], l[RT][2];      // running maximum, sum over this lane's keys
  float lg, slack;               // from scores to log2; kSlack in scores
  float o[RT][D::MV][4];
  int vref, vmost;               // scale byte that O is held in units of, 0: none yet; the largest so far

  // Sixteen keys' scores (keys g and g + 8; -inf: not seen) to weights times
  // 2^up in place, summed up in l without it.
  __device__ __forceinline__ void weigh(float (&s)[RT][4], float up, float down) {
    bool raise = false;
    float mx[RT][2];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        mx[i][r] = fmaxf(s[i][r], s[i][2 + r]);
        raise |= mx[i][r] - m[i][r] > slack;
      }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float now = fmaxf(m[i][r], keys_max(mx[i][r]));
          const float w = weight_of(m[i][r], now, lg);
          m[i][r] = now;
          l[i][r] *= w;
#pragma unroll
          for (int j = 0; j < D::MV; ++j) {
            o[i][j][r] *= w;
            o[i][j][2 + r] *= w;
          }
        }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        // (never fused with the product that made the score: the maximum is of rounded scores)
        s[i][r] = exp2_approx(fmaf(__fsub_rn(s[i][r], m[i][r]), lg, kShift + up));
        s[i][2 + r] = exp2_approx(fmaf(__fsub_rn(s[i][2 + r], m[i][r]), lg, kShift + up));
        l[i][r] = fmaf(s[i][r] + s[i][2 + r], down, l[i][r]);
      }
  }

  // Lets vref follow a block's V scale byte vb (not 0).  It stays within 2^80
  // of the largest scale, so that no sum overflows in its units.
  __device__ __forceinline__ void follow(int vb) {
    if (vref == 0) vref = vb;
    vmost = max(vmost, vb);
    if (abs(vb - vref) <= kVWindow) return;
    const int now = max(vb, vmost - 80);
    const float f = vref - now < -126 ? 0.f : __uint_as_float((uint32_t)(127 + vref - now) << 23);
    vref = now;
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < D::MV; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][j][e] *= f;
  }
  // A block's weights as B fragments.
  __device__ __forceinline__ void pack(const float (&w)[RT][4], uint32_t (&p)[RT][NP][2]) const {
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      uint32_t lo[NP], hi[NP];
      split_h2<NP>(w[i][0], w[i][1], lo);
      split_h2<NP>(w[i][2], w[i][3], hi);
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        p[i][n][0] = transpose8(lo[n]);
        p[i][n][1] = transpose8(hi[n]);
      }
    }
  }
};

template <typename T, int DQK, int DV, int RT, int NW, int STAGES, int CTAS>
__global__ void __launch_bounds__(kUnitWarps * 32, CTAS) attend8_kernel(AttendArgs a) {
  using D = Dims<DQK, DV, RT>;
  constexpr int NP = sizeof(T) == 4 ? 2 : 1;
  extern __shared__ __align__(16) uint8_t smem[];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int sub = NW == 1 ? 0 : warp;
  const int H = a.cache.H;
  const uint32_t unit = NW == 1 ? blockIdx.x * kUnitWarps + warp : blockIdx.x;
  // (fp32 rows on a plan with tiles of 128 or 24 rows: eight units of 16 a
  // tile, or three of eight)
  const int subs = a.shape.tile_rows / D::ROWS, sub_tile = subs > 1 ? (int)(unit % (uint32_t)subs) : 0;
  const uint32_t whole = subs > 1 ? unit / (uint32_t)subs : unit;
  const int item_id = (int)(whole / (uint32_t)H), head = (int)(whole % (uint32_t)H);
  if (item_id >= a.shape.max_items) return;
  const int items = a.plan.head[0];
  const AttendItem it = a.plan.items[item_id];  // together with the count
  if (item_id >= items) return;
  const int r0 = sub_tile * D::ROWS;
  const int4* tile = reinterpret_cast<const int4*>(a.plan.rows + (size_t)it.tile * a.shape.tile_rows + r0);

  // This warp's pages: list entries sub, sub + NW, ... of the item, 32 at a
  // time in the lanes (id and the two scale bytes), the next 32 in flight.
  const int npages = it.pages > sub ? (it.pages - sub + NW - 1) / NW : 0;
  const uint8_t* head_k = a.cache.data + (int64_t)head * IMBA_PAGE_TOKENS * DQK;
  const uint8_t* lane_k = head_k + g * DQK + t * D::VK;
  const int64_t v_from_k = a.cache.v_offset + (int64_t)head * IMBA_PAGE_TOKENS * (DV - DQK);
  const uint8_t* lane_v = head_k + v_from_k + t * 2 * DV + g * D::VV;
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
  int ids = page_id(lane), ids_next = npages > 32 ? page_id(32 + lane) : -1;

  Rows<DQK, DV, RT, NP> st;
  int4 qrow[RT];  // the rows whose query fragments this lane holds
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    qrow[i] = __ldg(tile + 8 * i + g);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int4 u = __ldg(tile + 8 * i + 2 * t + r);
      st.vis[i][r] = u.y;
      st.pos[i][r] = a.call.max_pos - 1 - u.z;
      st.bias[i][r] = a.call.bias + (int64_t)(head * a.shape.share + u.w) * (2 * a.call.max_pos - 1);
      st.m[i][r] = kLowest;
      st.l[i][r] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < D::MV; ++j) st.o[i][j][0] = st.o[i][j][1] = st.o[i][j][2] = st.o[i][j][3] = 0.f;
  }
  st.vref = st.vmost = 0;
  st.lg = a.call.bias ? kLog2e : 1.f;
  st.slack = a.call.bias ? kSlack / kLog2e : kSlack;
  int scs = page_scales(ids), scs_next = page_scales(ids_next);
  if (__any_sync(0xffffffffu, ids == -2 || ids_next == -2) && lane == 0) report(a.rows.status, IMBA_ERR_RANGE);

  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * (STAGES * D::STAGE);
  auto issue = [&](int i, int batch, uint32_t dst) {  // page i of the warp; `batch` holds its id
    const int id = __shfl_sync(0xffffffffu, batch, i & 31);
    if (i < npages) {
      const uint8_t* k = lane_k + (uint64_t)(uint32_t)max(id, 0) * (uint32_t)a.cache.page_stride;
      const uint8_t* v = lane_v + (uint64_t)(uint32_t)max(id, 0) * (uint32_t)a.cache.page_stride;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int c = 0; c < D::CK; ++c)
          cp_async<D::VK>(dst + (n * D::CK + c) * 32 * D::VK + lane * D::VK, k + n * 8 * DQK + c * 4 * D::VK);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int c = 0; c < D::CV; ++c)
          cp_async<D::VV>(dst + IMBA_PAGE_TOKENS * DQK + (n * D::CV + c) * 32 * D::VV + lane * D::VV,
                          v + n * 8 * DV + c * 8 * D::VV);
    }
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) issue(i, ids, ring + i * D::STAGE);

  // Queries: f16 B fragments of each row over its power of two.
  const bool qvec = a.call.q_stride[0] % 4 == 0 && a.call.q_stride[1] % 4 == 0 &&
                    (reinterpret_cast<uintptr_t>(a.call.q) & (4 * sizeof(T) - 1)) == 0;
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const T* q = static_cast<const T*>(a.call.q) + qrow[i].x * a.call.q_stride[0] +
                 (int64_t)(head * a.shape.share + qrow[i].w) * a.call.q_stride[1];
    float x[D::KS][4], amax = 0.f;
#pragma unroll
    for (int s = 0; s < D::KS; ++s) {
      x[s][0] = x[s][1] = x[s][2] = x[s][3] = 0.f;
      if (qrow[i].x >= 0) q_load4(q + s / (D::VK / 4) * 4 * D::VK + t * D::VK + s % (D::VK / 4) * 4, qvec, x[s]);
    }
#pragma unroll
    for (int s = 0; s < D::KS; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) amax = fmaxf(amax, fabsf(x[s][j]));
    amax = quad_max(amax);
    const int ex = (int)(__float_as_uint(amax) >> 23);  // 0 for a zero row, 255 for an infinite one
    const int e = ex == 0 || ex == 255 ? 0 : min(ex - 127, 126);
    const float down = __uint_as_float((uint32_t)(127 - e) << 23);
    const float f = __uint_as_float((uint32_t)(127 + e) << 23) * (a.call.bias ? a.call.scale : a.call.scale * kLog2e);
    st.fac[i][0] = __shfl_sync(0xffffffffu, f, 8 * t);
    st.fac[i][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
    for (int s = 0; s < D::KS; ++s) {
      uint32_t lo[NP], hi[NP];
      split_h2<NP>(x[s][0] * down, x[s][1] * down, lo);
      split_h2<NP>(x[s][2] * down, x[s][3] * down, hi);
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        st.q[i][p][s][0] = lo[p];
        st.q[i][p][s][1] = hi[p];
      }
    }
  }

  // Bias columns: within [0, last] nothing is clamped.
  const bool biased = a.call.bias != nullptr;
  const int last = 2 * a.call.max_pos - 2;
  bool inside = true;
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      inside &= it.key0 + st.pos[r][e] >= 0 && it.key0 + it.pages * IMBA_PAGE_TOKENS + st.pos[r][e] <= last + 1;
      if (biased) st.bias[r][e] += g;
    }
  inside = __all_sync(0xffffffffu, inside);

  uint32_t from = ring, into = ring + (STAGES - 1) * D::STAGE;
  int key0 = it.key0 + sub * IMBA_PAGE_TOKENS;
  for (int i = 0; i < npages; ++i, key0 += NW * IMBA_PAGE_TOKENS) {
    if (i && (i & 31) == 0) {
      ids = ids_next;
      scs = scs_next;
      ids_next = page_id(i + 32 + lane);
      scs_next = page_scales(ids_next);
      if (__any_sync(0xffffffffu, ids_next == -2) && lane == 0) report(a.rows.status, IMBA_ERR_RANGE);
    }
    const int sc = __shfl_sync(0xffffffffu, scs, i & 31);
    float s[RT][4], add[RT][4];
    if (biased) {
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (inside) {
            const float* at = st.bias[r][e] + (key0 + st.pos[r][e]);
            add[r][e] = __ldg(at);
            add[r][2 + e] = __ldg(at + 8);
          } else {
            const float* at = st.bias[r][e] - g;
            const int col = key0 + g + st.pos[r][e];
            add[r][e] = __ldg(at + min(max(col, 0), last));
            add[r][2 + e] = __ldg(at + min(max(col + 8, 0), last));
          }
        }
    }
    cp_wait<STAGES - 2>();  // page i has arrived
    {
      const int ahead = i + STAGES - 1;  // into the stage that page i - 1 left
      issue(ahead, (ahead ^ i) & 32 ? ids_next : ids, into);
      into = into + D::STAGE == ring + STAGES * D::STAGE ? ring : into + D::STAGE;
    }

#pragma unroll
    for (int r = 0; r < RT; ++r) s[r][0] = s[r][1] = s[r][2] = s[r][3] = 0.f;
#pragma unroll
    for (int c = 0; c < D::CK; ++c) {
      uint32_t w0[D::VK / 4], w1[D::VK / 4];
      lds<D::VK>(from + c * 32 * D::VK + lane * D::VK, w0);
      lds<D::VK>(from + (D::CK + c) * 32 * D::VK + lane * D::VK, w1);
#pragma unroll
      for (int j = 0; j < D::VK / 4; ++j) {
        uint32_t ka[4];
        e4m3x4_to_h2(w0[j], ka[0], ka[2]);
        e4m3x4_to_h2(w1[j], ka[1], ka[3]);
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int p = 0; p < NP; ++p)
            mma_f16(s[r], ka, st.q[r][p][c * (D::VK / 4) + j][0], st.q[r][p][c * (D::VK / 4) + j][1]);
      }
    }
    const float ks = scale_of(sc & 255);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float f = ks * st.fac[r][e];
        s[r][e] *= f;
        s[r][2 + e] *= f;
      }
    if (biased) {
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[r][e] += add[r][e];
    }
    const int id = __shfl_sync(0xffffffffu, ids, i & 31);
    if (key0 + IMBA_PAGE_TOKENS > it.minvis || id < 0) {
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int lim = id < 0 ? 0 : st.vis[r][e] - key0 - g;
          if (lim <= 0) s[r][e] = -INFINITY;
          if (lim <= 8) s[r][2 + e] = -INFINITY;
        }
    }
    // V's scale as its ratio to vref, in the weights' exponent.
    const int vb = sc >> 8;
    if ((uint32_t)(vb - st.vref + kVWindow) > 2 * kVWindow && vb) st.follow(vb);
    const int up = vb ? max(vb - st.vref, kVLeast) : 0;
    st.weigh(s, (float)up, __uint_as_float((uint32_t)(127 - up) << 23));
    uint32_t pb[RT][NP][2];
    st.pack(s, pb);
#pragma unroll
    for (int c = 0; c < D::CV; ++c) {
      uint32_t w0[D::VV / 4], w1[D::VV / 4];
      lds<D::VV>(from + IMBA_PAGE_TOKENS * DQK + c * 32 * D::VV + lane * D::VV, w0);
      lds<D::VV>(from + IMBA_PAGE_TOKENS * DQK + (D::CV + c) * 32 * D::VV + lane * D::VV, w1);
#pragma unroll
      for (int j = 0; j < D::VV / 4; ++j) {
        uint32_t va[4];
        e4m3x4_to_h2(w0[j], va[0], va[1]);
        e4m3x4_to_h2(w1[j], va[2], va[3]);
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int p = 0; p < NP; ++p) mma_f16(st.o[r][c * (D::VV / 4) + j], va, pb[r][p][0], pb[r][p][1]);
      }
    }
    from = from + D::STAGE == ring + STAGES * D::STAGE ? ring : from + D::STAGE;
  }
  if (biased) {
#pragma unroll
    for (int r = 0; r < RT; ++r) st.bias[r][0] -= g, st.bias[r][1] -= g;
  }

  // The rows' extra keys, sixteen of the tile's at a time: each is seen by
  // its own row alone, and has its own block's scales.
  if (a.rows.num_extra > 0 && it.index == 0 && sub == 0) {
    const int64_t slots = a.cache.num_pages * IMBA_PAGE_TOKENS;
    int e0 = 0, n = 0;  // lane = row of the tile
    if (lane < D::ROWS) {
      const int row = __ldg(tile + lane).x;
      if (row >= 0) {
        e0 = a.rows.row_extra_off[row];
        const int e1 = a.rows.row_extra_off[row + 1];
        if (e0 < 0 || e1 < e0 || e1 > a.rows.num_extra)
          report(a.rows.status, IMBA_ERR_RANGE);
        else
          n = e1 - e0;
      }
    }
    int upto = n;  // extras of the rows up to this one
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    const int total = __shfl_sync(0xffffffffu, upto, 31);
    for (int x0 = 0; x0 < total; x0 += 16) {
      // Lane x holds key x0 + x: its row, slot, position and scales.
      int owner = 0, slot = -1, kp = 0, sc = 0;
      {
        const int x = x0 + lane;
#pragma unroll
        for (int step = 16; step; step /= 2) {
          const int y = __shfl_sync(0xffffffffu, upto, owner + step - 1);
          if (y <= x) owner += step;
        }
        const int past = __shfl_sync(0xffffffffu, upto - n, owner & 31);
        const int base = __shfl_sync(0xffffffffu, e0, owner & 31);
        if (lane < 16 && x < total) {
          slot = a.rows.extra_slot[base + x - past];
          kp = a.rows.extra_pos[base + x - past];
          if (slot < 0 || slot >= slots) {
            report(a.rows.status, IMBA_ERR_RANGE);
            slot = -1;
          } else {
            sc = page_scales(slot / IMBA_PAGE_TOKENS);
          }
        }
      }
      int kslot[2], kown[2], kpos[2], vb[2];
      float ks[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        kslot[k] = __shfl_sync(0xffffffffu, slot, g + 8 * k);
        kown[k] = __shfl_sync(0xffffffffu, owner, g + 8 * k);
        kpos[k] = __shfl_sync(0xffffffffu, kp, g + 8 * k);
        const int both = __shfl_sync(0xffffffffu, sc, g + 8 * k);
        ks[k] = scale_of(both & 255);
        vb[k] = both >> 8;
      }
      int vslot[4];  // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
      for (int k = 0; k < 4; ++k) vslot[k] = max(__shfl_sync(0xffffffffu, slot, 2 * t + (k & 1) + 8 * (k >> 1)), 0);
      float s[RT][4];
#pragma unroll
      for (int r = 0; r < RT; ++r) s[r][0] = s[r][1] = s[r][2] = s[r][3] = 0.f;
      const uint8_t* kr[2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        kr[k] = head_k + max(kslot[k], 0) / IMBA_PAGE_TOKENS * a.cache.page_stride +
                max(kslot[k], 0) % IMBA_PAGE_TOKENS * DQK + t * D::VK;
#pragma unroll
      for (int c = 0; c < D::CK; ++c)
#pragma unroll
        for (int j = 0; j < D::VK / 4; ++j) {
          const uint32_t w0 = *reinterpret_cast<const uint32_t*>(kr[0] + c * 4 * D::VK + 4 * j);
          const uint32_t w1 = *reinterpret_cast<const uint32_t*>(kr[1] + c * 4 * D::VK + 4 * j);
          uint32_t ka[4];
          e4m3x4_to_h2(w0, ka[0], ka[2]);
          e4m3x4_to_h2(w1, ka[1], ka[3]);
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int p = 0; p < NP; ++p)
              mma_f16(s[r], ka, st.q[r][p][c * (D::VK / 4) + j][0], st.q[r][p][c * (D::VK / 4) + j][1]);
        }
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int k = e >> 1;
          s[r][e] *= ks[k] * st.fac[r][e & 1];
          if (biased)
            s[r][e] += __ldg(st.bias[r][e & 1] + min(max(add_sat(kpos[k], st.pos[r][e & 1]), 0), last));
          if (kslot[k] < 0 || kown[k] != 8 * r + 2 * t + (e & 1)) s[r][e] = -INFINITY;
        }
      st.weigh(s, 0.f, 1.f);
      // Keys whose V scales are too far apart for one reference take turns.
      bool left[2] = {vb[0] > 0, vb[1] > 0};
      do {
        const int top = __reduce_max_sync(0xffffffffu, max(left[0] ? vb[0] : 0, left[1] ? vb[1] : 0));
        if (top == 0) break;
        st.follow(top);
        float w[RT][4];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const bool now = left[k] && vb[k] > top - kVWindow;
          const float f = now ? __uint_as_float((uint32_t)max(127 + vb[k] - st.vref, 0) << 23) : 0.f;
          left[k] = left[k] && !now;
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            w[r][2 * k] = s[r][2 * k] * f;
            w[r][2 * k + 1] = s[r][2 * k + 1] * f;
          }
        }
        uint32_t pb[RT][NP][2];
        st.pack(w, pb);
#pragma unroll
        for (int c = 0; c < D::CV; ++c) {
          // The two keys' codes of each dimension side by side.
          uint32_t w[2][D::VV / 4];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            uint32_t u[2][D::VV / 4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int sl = vslot[2 * k + e], tok = sl % IMBA_PAGE_TOKENS;
              const uint8_t* v = head_k + v_from_k + sl / IMBA_PAGE_TOKENS * a.cache.page_stride +
                                 v8_off(tok & ~1, c * 4 * D::VV + g * (D::VV / 2), DV);
#pragma unroll
              for (int j = 0; j < D::VV / 4; ++j)
                u[e][j] = *reinterpret_cast<const uint32_t*>(v + 4 * j) >> (8 * (tok & 1)) & 0x00ff00ffu;
            }
#pragma unroll
            for (int j = 0; j < D::VV / 4; ++j) w[k][j] = u[0][j] | u[1][j] << 8;
          }
#pragma unroll
          for (int j = 0; j < D::VV / 4; ++j) {
            uint32_t va[4];
            e4m3x4_to_h2(w[0][j], va[0], va[1]);
            e4m3x4_to_h2(w[1][j], va[2], va[3]);
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
              for (int p = 0; p < NP; ++p) mma_f16(st.o[r][c * (D::VV / 4) + j], va, pb[r][p][0], pb[r][p][1]);
          }
        }
      } while (true);
    }
  }

  // Out: averages in true units.
  const float unit_v = st.vref ? scale_of(st.vref) : 1.f;
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int r = 0; r < 2; ++r) st.l[i][r] = keys_sum(st.l[i][r]);
  const bool ovec = a.call.out_stride[0] % 4 == 0 && a.call.out_stride[1] % 4 == 0 &&
                    (reinterpret_cast<uintptr_t>(a.call.out) & (4 * sizeof(T) - 1)) == 0;
  // Dimensions e .. e + 3 of this lane's row i, r, times f; e = dim(c, q).
  auto four = [&](int i, int r, int c, int q, float f, float (&x)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = st.o[i][c * (D::VV / 4) + (4 * q + j) / 2][2 * (j & 1) + r] * f;
  };
  auto dim = [&](int c, int q) { return c * 4 * D::VV + g * (D::VV / 2) + 4 * q; };

  if constexpr (NW == 1) {
    const size_t part = ((size_t)max(it.part, 0) * H + head) * a.shape.tile_rows + r0;
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int tr = 8 * i + 2 * t + r;
        const int4 row = __ldg(tile + tr);
        if (row.x < 0) continue;
        const float f = st.l[i][r] == 0.f ? 0.f : unit_v / st.l[i][r];
        if (it.part >= 0 && g == 0) a.plan.ml[part + tr] = make_float2(st.m[i][r], st.l[i][r]);
        T* out = static_cast<T*>(a.call.out) + row.x * a.call.out_stride[0] +
                 (int64_t)(head * a.shape.share + row.w) * a.call.out_stride[1];
#pragma unroll
        for (int c = 0; c < D::CV; ++c)
#pragma unroll
          for (int q = 0; q < D::VV / 8; ++q) {
            float x[4];
            four(i, r, c, q, f, x);
            if (it.part >= 0)
              *reinterpret_cast<float4*>(a.plan.o + (part + tr) * DV + dim(c, q)) = make_float4(x[0], x[1], x[2], x[3]);
            else
              out_store4(out + dim(c, q), ovec, x);
          }
      }
    if (it.part >= 0) {
      __threadfence();
      __syncwarp();
      int* done = a.plan.done + ((size_t)it.tile * H + head) * subs + sub_tile;
      int n = 0;
      if (lane == 0) n = atomicAdd(done, 1);
      if (__shfl_sync(0xffffffffu, n, 0) == it.splits - 1) {  // the others have finished
        __threadfence();
        if (lane == 0) *done = 0;
        join_items<T, DV, 8>(a, it, head, st.lg, r0, D::ROWS, lane, 32);
      }
    }
  } else {
    // The warps' parts meet in shared memory (over the ring, which is idle).
    float* so = reinterpret_cast<float*>(smem);                               // [warps][rows][DV], each in its warp's units
    float2* sml = reinterpret_cast<float2*>(so + kUnitWarps * D::ROWS * DV);  // [warps][rows]
    float* sunit = reinterpret_cast<float*>(sml + kUnitWarps * D::ROWS);      // [warps]
    int* flag = reinterpret_cast<int*>(sunit + kUnitWarps);
    cp_wait<0>();
    __syncthreads();
    if (lane == 0) sunit[warp] = unit_v;
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int tr = 8 * i + 2 * t + r;
        if (__ldg(tile + tr).x < 0) continue;
        if (g == 0) sml[warp * D::ROWS + tr] = make_float2(st.m[i][r], st.l[i][r]);
        float* dst = so + (warp * D::ROWS + tr) * DV;
#pragma unroll
        for (int c = 0; c < D::CV; ++c)
#pragma unroll
          for (int q = 0; q < D::VV / 8; ++q) {
            float x[4];
            four(i, r, c, q, 1.f, x);
            *reinterpret_cast<float4*>(dst + dim(c, q)) = make_float4(x[0], x[1], x[2], x[3]);
          }
      }
    __syncthreads();
    const size_t part = ((size_t)max(it.part, 0) * H + head) * a.shape.tile_rows + r0;
    for (int i = threadIdx.x; i < D::ROWS * (DV / 4); i += kUnitWarps * 32) {
      const int tr = i / (DV / 4), e = i % (DV / 4) * 4;
      const int4 row = __ldg(tile + tr);
      if (row.x < 0) continue;
      float mm = kLowest, l = 0.f, f[kUnitWarps], x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kUnitWarps; ++w) mm = fmaxf(mm, sml[w * D::ROWS + tr].x);
#pragma unroll
      for (int w = 0; w < kUnitWarps; ++w) {
        const float2 ml = sml[w * D::ROWS + tr];
        f[w] = weight_of(ml.x, mm, st.lg);
        l += f[w] * ml.y;
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int w = 0; w < kUnitWarps; ++w) {
        const float4 v = *reinterpret_cast<const float4*>(so + (w * D::ROWS + tr) * DV + e);
        const float g = f[w] * inv * sunit[w];
        x[0] += g * v.x, x[1] += g * v.y, x[2] += g * v.z, x[3] += g * v.w;
      }
      if (it.part >= 0) {
        if (e == 0) a.plan.ml[part + tr] = make_float2(mm, l);
        *reinterpret_cast<float4*>(a.plan.o + (part + tr) * DV + e) = make_float4(x[0], x[1], x[2], x[3]);
      } else {
        out_store4(static_cast<T*>(a.call.out) + row.x * a.call.out_stride[0] +
                       (int64_t)(head * a.shape.share + row.w) * a.call.out_stride[1] + e,
                   ovec, x);
      }
    }
    if (it.part >= 0) {
      __threadfence();
      __syncthreads();
      int* done = a.plan.done + ((size_t)it.tile * H + head) * subs + sub_tile;
      if (threadIdx.x == 0) *flag = atomicAdd(done, 1) == it.splits - 1;
      __syncthreads();
      if (*flag) {
        __threadfence();
        if (threadIdx.x == 0) *done = 0;
        join_items<T, DV, 8>(a, it, head, st.lg, r0, D::ROWS, threadIdx.x, kUnitWarps * 32);
      }
    }
  }
}

template <typename T, int DQK, int DV, int RT, int NW>
cudaError_t launch_one(const AttendArgs& a, cudaStream_t s) {
  using D = Dims<DQK, DV, RT>;
  constexpr int kCtas = attend8_ctas(DQK, RT);
  // Two pages of each warp in flight behind the one at work: with three (and a
  // CTA less an SM at head size 128) the long sequences took 292 us, not 264.
  constexpr int kStages = 3;
  constexpr size_t ring = (size_t)kUnitWarps * kStages * D::STAGE;
  constexpr size_t smem = NW > 1 && D::MERGE > ring ? D::MERGE : ring;
  auto fn = attend8_kernel<T, DQK, DV, RT, NW, kStages, kCtas>;
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  const int64_t units = (int64_t)a.shape.max_items * a.cache.H * (a.shape.tile_rows / D::ROWS);
  const int64_t grid = NW == 1 ? (units + kUnitWarps - 1) / kUnitWarps : units;
  if (units > INT32_MAX) return cudaErrorInvalidValue;
  return launch_pdl(fn, dim3((unsigned)grid), dim3(kUnitWarps * 32), smem, s, a);
}

template <typename T, int DQK, int DV, int RT>
cudaError_t launch_rows(const AttendArgs& a, cudaStream_t s) {
  return a.shape.warps == 1 ? launch_one<T, DQK, DV, RT, 1>(a, s) : launch_one<T, DQK, DV, RT, kUnitWarps>(a, s);
}

}  // namespace

// 24 rows of queries as two f16 parts do not fit the registers: fp32 takes
// such a tile as three of eight.
template <typename T>
constexpr int kThree = sizeof(T) == 2 ? 3 : 1;

template <typename T>
cudaError_t launch_attend8(const imba_cache_desc& c, const AttendArgs& a, cudaStream_t s) {
  if (a.shape.rt == kTileGroups && sizeof(T) == 2) return launch_attend8_tile(c, a, s);
#define IMBA_ATTEND8(DQK, DV)                                              \
  if (c.attention_dim == DQK && c.linear_dim == DV) {                      \
    if (a.shape.rt == 1) return launch_rows<T, DQK, DV, 1>(a, s);          \
    if (a.shape.rt == 3) return launch_rows<T, DQK, DV, kThree<T>>(a, s);  \
    return launch_rows<T, DQK, DV, 2>(a, s);                               \
  }
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
