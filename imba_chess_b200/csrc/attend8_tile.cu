// Attention over a paged pool in 8 bits for segments of many rows (prompts
// continued over a cache): tcgen05.
//
// A unit is a tile of 128 query rows (one segment's rows with the query heads
// of one key / value head), that head, and a run of pages.  The products of
// blocks of 64 keys are tcgen05.mma on f16 with fp32 sums in TMEM: S = Q K'
// (M 128, N 64) into one of two buffers, O += P V in 64 columns at a time.
// e4m3 is exact in f16, so four warps turn the pages' codes into f16 tiles in
// shared memory (K by rows of dimensions, V by rows of a token's dimensions,
// an MN-major operand; both with the 128-byte swizzle), one block ahead of the
// products; four warps are the tile's rows, one thread a row: they read S from
// TMEM, weigh it and write P; a lane of the last page warp issues the
// products, S of a block before P V of the one before it, which is what its
// own next block waits for.  Scales stay out of the products: K's
// multiplies a page's scores, V's is in its weights' exponent.
//
// What bounds it: the exponentials and the few instructions a score takes
// besides (16 MUFU lanes an SM and cycle), so two CTAs share an SM and each
// has 64-key blocks: 256 TMEM columns, 80 KB (head size 64).
//
// Numerics as in the mma.sync kernel (attend8_kernel.cuh).  V's scales of a
// block's four pages are held against one reference; where they lie more than
// 2^kSpread apart, the block's P V is done page by page.
#include <algorithm>

#include "attend8_common.cuh"
#include "tc_ptx.cuh"

namespace imba {

namespace {

constexpr int kRows = 128;
constexpr int kKeys = 64;
constexpr int kPages = kKeys / IMBA_PAGE_TOKENS;
constexpr int kTileThreads = 256;  // warps 0-3: rows; 4-7: pages, and 7 the products
constexpr uint32_t kCols = 256;    // TMEM columns: S at 0 and 64, O from 128
constexpr int kSpread = 12;        // with kVWindow on both sides
constexpr uint32_t kPanel = 128;   // bytes of a swizzled row: 64 f16
constexpr uint32_t kKvPanel = kKeys * kPanel, kRowPanel = kRows * kPanel;

// kind::f16, fp32 sums, f16 operands.
constexpr uint32_t idesc_f16(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

template <int D>
struct TileMem {
  static constexpr int kPanels = D / 64;
  static constexpr uint32_t kQ = 0;
  static constexpr uint32_t kP = kQ + kPanels * kRowPanel;
  static constexpr uint32_t kK = kP + kRowPanel;              // two stages
  static constexpr uint32_t kV = kK + 2 * kPanels * kKvPanel;  // two stages
  static constexpr uint32_t kMisc = kV + 2 * kPanels * kKvPanel;
  static constexpr uint32_t kBytes = kMisc + 256;
};

__device__ __forceinline__ void sts16(uint32_t dst, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// A page's scale word: K's byte, V's byte, and whether its tokens exist.
constexpr int kPageHere = 1 << 16;

// How many P V a block takes: one, or one a page.
__device__ __forceinline__ int block_parts(const int (&sc)[kPages]) {
  int top = 0, low = 255;
#pragma unroll
  for (int p = 0; p < kPages; ++p) {
    const int vb = sc[p] >> 8 & 255;
    top = max(top, vb);
    low = min(low, vb ? vb : 255);
  }
  return top - low > kSpread && low < 255 ? kPages : 1;
}

template <int D>
__global__ void __launch_bounds__(kTileThreads, 2) attend8_tile_kernel(const AttendArgs a) {
  using M = TileMem<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + M::kMisc);
  uint64_t* kv_full = bars;        // [2] K and V of a block written (4 page warps)
  uint64_t* kv_empty = bars + 2;   // [2] its products are complete (commit)
  uint64_t* s_full = bars + 4;     // [2] S of a block complete (commit)
  uint64_t* s_empty = bars + 6;    // [2] S read (4 row warps)
  uint64_t* q_full = bars + 8;     // Q written (4 row warps)
  uint64_t* p_full = bars + 9;     // P written (4 row warps)
  uint64_t* pv_done = bars + 10;   // P V complete (commit)
  uint64_t* drain = bars + 11;
  volatile int* scales = reinterpret_cast<int*>(bars + 12);  // [2][kPages]
  int* misc = reinterpret_cast<int*>(bars + 12) + 2 * kPages;  // [0] abort, [1] TMEM, [2] last of a split tile
  volatile int* abort_flag = misc;
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int H = a.cache.H;
  const int item_id = (int)(blockIdx.x / (uint32_t)H), head = (int)(blockIdx.x % (uint32_t)H);
  const int items = a.plan.head[0];
  const AttendItem it = a.plan.items[item_id];
  if (item_id >= items) return;
  const int blocks = (it.pages + kPages - 1) / kPages;

  if (tid == 0) {
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(&kv_full[s], 4);
      tc::mbar_init(&kv_empty[s], 1);
      tc::mbar_init(&s_full[s], 1);
      tc::mbar_init(&s_empty[s], 4);
    }
    tc::mbar_init(q_full, 4);
    tc::mbar_init(p_full, 4);
    tc::mbar_init(pv_done, 1);
    tc::mbar_init(drain, 1);
    misc[0] = 0;
    tc::fence_mbar_init();
  }
  if (warp == 0) {
    tc::tmem_alloc(reinterpret_cast<uint32_t*>(&misc[1]), kCols);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = static_cast<uint32_t>(misc[1]);
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return tc::mbar_wait_park_or_abort(bar, parity, a.rows.status, abort_flag);
  };

  if (warp >= 4) {
    // ---------------- pages: codes to f16 tiles; products ----------------
    // Warp w takes page w of every block; ids and scales 32 blocks at a time.
    const int w = warp - 4;
    const uint8_t* head_k = a.cache.data + (int64_t)head * IMBA_PAGE_TOKENS * D;
    const uint8_t* head_v = a.cache.data + a.cache.v_offset + (int64_t)head * IMBA_PAGE_TOKENS * D;
    constexpr int kLoads = D / 32;  // 16-byte loads of a lane, for K and for V
    int id32 = -1, sc32 = 0;
    auto fetch_ids = [&](int b0) {  // lane: page of block b0 + lane
      const int p = (b0 + lane) * kPages + w;
      id32 = -1;
      sc32 = 0;
      if (p < it.pages) {
        const int id = a.rows.group_pages[it.list + p];
        if (id >= 0 && id < a.cache.num_pages) {
          id32 = id;
          const uint8_t* s = a.cache.scales + id * a.cache.scale_stride + head;
          sc32 = s[0] | s[H] << 8 | kPageHere;
        } else {
          report(a.rows.status, IMBA_ERR_RANGE);
        }
      }
    };
    uint4 kr[kLoads], vr[kLoads];
    int sc = 0;
    auto load = [&](int b) {
      if ((b & 31) == 0) fetch_ids(b);
      const int id = __shfl_sync(0xffffffffu, id32, b & 31);
      sc = __shfl_sync(0xffffffffu, sc32, b & 31);
#pragma unroll
      for (int j = 0; j < kLoads; ++j) kr[j] = vr[j] = make_uint4(0, 0, 0, 0);
      if (id < 0) return;
      const uint64_t off = (uint64_t)(uint32_t)id * (uint32_t)a.cache.page_stride;
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        kr[j] = __ldcg(reinterpret_cast<const uint4*>(head_k + off) + j * 32 + lane);
        vr[j] = __ldcg(reinterpret_cast<const uint4*>(head_v + off) + j * 32 + lane);
      }
    };
    // The products (warp 7, lane 0).
    constexpr uint32_t idS = idesc_f16(kRows, kKeys);
    constexpr uint32_t idPV = idesc_f16(kRows, 64) | tc::kIdescBMajorMN;
    uint32_t pv = 0;  // P V issued
    auto issue_s = [&](int b) {
      const int s = b & 1;
      if (b == 0 && !wait(q_full, 0)) return false;
      if (!wait(&kv_full[s], (b / 2) & 1) || (b >= 2 && !wait(&s_empty[s], (b / 2 - 1) & 1))) return false;
      tc::fence_after_sync();
#pragma unroll
      for (int n = 0; n < M::kPanels; ++n) {
        const uint64_t dQ = tc::smem_desc_k128(sm + M::kQ + n * kRowPanel);
        const uint64_t dK = tc::smem_desc_k128(sm + M::kK + (s * M::kPanels + n) * kKvPanel);
#pragma unroll
        for (int k = 0; k < 4; ++k) tc::umma_f16(tmem + 64 * s, dQ + 2 * k, dK + 2 * k, idS, (n | k) != 0);
      }
      tc::umma_commit(&s_full[s]);
      return true;
    };
    auto issue_pv = [&](int b) {
      int sc4[kPages];
#pragma unroll
      for (int p = 0; p < kPages; ++p) sc4[p] = scales[(b & 1) * kPages + p];
      const int parts = block_parts(sc4);
      const uint64_t dP = tc::smem_desc_k128(sm + M::kP);
      for (int i = 0; i < parts; ++i, ++pv) {
        if (!wait(p_full, pv & 1)) return false;
        tc::fence_after_sync();
#pragma unroll
        for (int n = 0; n < M::kPanels; ++n) {
          const uint64_t dV = tc::smem_desc_k128(sm + M::kV + ((b & 1) * M::kPanels + n) * kKvPanel);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            tc::umma_f16(tmem + 128 + 64 * n, dP + 2 * k, dV + 128 * k, idPV, (pv | k) != 0);
        }
        if (i + 1 == parts) tc::umma_commit(&kv_empty[b & 1]);
        tc::umma_commit(pv_done);
      }
      return true;
    };
    if (blocks > 0) load(0);
    bool ok = true;
    for (int b = 0; b < blocks; ++b) {
      const int s = b & 1;
      if (b >= 2 && !__all_sync(0xffffffffu, wait(&kv_empty[s], (b / 2 - 1) & 1))) break;
      const uint32_t kt = tc::smem_u32(sm + M::kK + s * M::kPanels * kKvPanel);
      const uint32_t vt = tc::smem_u32(sm + M::kV + s * M::kPanels * kKvPanel);
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        // K: a row is D / 16 chunks of sixteen dimensions.
        {
          const int q = j * 32 + lane, row = w * IMBA_PAGE_TOKENS + q / (D / 16), e = q % (D / 16) * 16;
          const uint32_t dst = kt + e / 64 * kKvPanel + row * kPanel, c = (uint32_t)(e % 64 / 8), x = row & 7;
          uint32_t h[8];
          e4m3x4_to_h2(kr[j].x, h[0], h[1]);
          e4m3x4_to_h2(kr[j].y, h[2], h[3]);
          e4m3x4_to_h2(kr[j].z, h[4], h[5]);
          e4m3x4_to_h2(kr[j].w, h[6], h[7]);
          sts16(dst + ((c ^ x) << 4), h[0], h[1], h[2], h[3]);
          sts16(dst + (((c + 1) ^ x) << 4), h[4], h[5], h[6], h[7]);
        }
        // V: a pair of tokens is D / 8 chunks of eight dimensions, token by token.
        {
          const int q = j * 32 + lane, row = w * IMBA_PAGE_TOKENS + 2 * (q / (D / 8)), e = q % (D / 8) * 8;
          const uint32_t dst = vt + e / 64 * kKvPanel + row * kPanel, c = (uint32_t)(e % 64 / 8);
          uint32_t h[4];
          e4m3x4_to_h2(__byte_perm(vr[j].x, vr[j].y, 0x6420), h[0], h[1]);
          e4m3x4_to_h2(__byte_perm(vr[j].z, vr[j].w, 0x6420), h[2], h[3]);
          sts16(dst + ((c ^ (row & 7)) << 4), h[0], h[1], h[2], h[3]);
          e4m3x4_to_h2(__byte_perm(vr[j].x, vr[j].y, 0x7531), h[0], h[1]);
          e4m3x4_to_h2(__byte_perm(vr[j].z, vr[j].w, 0x7531), h[2], h[3]);
          sts16(dst + kPanel + ((c ^ ((row + 1) & 7)) << 4), h[0], h[1], h[2], h[3]);
        }
      }
      if (lane == 0) scales[s * kPages + w] = sc;
      if (b + 1 < blocks) load(b + 1);  // behind the stores, ahead of the next wait
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&kv_full[s]);
      if (w == 3) {
        if (lane == 0) ok = issue_s(b) && (b == 0 || issue_pv(b - 1));
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
      }
    }
    if (w == 3 && lane == 0) {
      if (ok && blocks > 0) issue_pv(blocks - 1);
      // Every product issued here completes before TMEM is freed.
      tc::umma_commit(drain);
      tc::mbar_wait_for(drain, 0, a.rows.status, tc::kWaitNs);
    }
    __syncwarp();
  } else {
    // ---------------- rows: thread = row of the tile ----------------
    const int4 row = __ldg(reinterpret_cast<const int4*>(a.plan.rows + (size_t)it.tile * kRows) + tid);
    const uint32_t tl = tmem + ((uint32_t)(32 * warp) << 16);  // this warp's TMEM lanes
    const uint32_t sw = (uint32_t)(tid & 7);
    const bool biased = a.call.bias != nullptr;
    const float lg = biased ? kLog2e : 1.f, slack = biased ? kSlack / kLog2e : kSlack;
    const int vis = row.y - it.key0;  // of the item's keys
    const float* bias = a.call.bias + (int64_t)(head * a.shape.share + row.w) * (2 * a.call.max_pos - 1);
    const int col0 = it.key0 - row.z + a.call.max_pos - 1, last = 2 * a.call.max_pos - 2;
    // The query over its power of two, as f16.
    float fac;
    {
      const bf16* q = static_cast<const bf16*>(a.call.q) + row.x * a.call.q_stride[0] +
                      (int64_t)(head * a.shape.share + row.w) * a.call.q_stride[1];
      const bool vec = a.call.q_stride[0] % 4 == 0 && a.call.q_stride[1] % 4 == 0 &&
                       (reinterpret_cast<uintptr_t>(a.call.q) & 7) == 0;
      float amax = 0.f;
#pragma unroll 4
      for (int e = 0; e < D; e += 4) {
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        if (row.x >= 0) q_load4(q + e, vec, x);
#pragma unroll
        for (int j = 0; j < 4; ++j) amax = fmaxf(amax, fabsf(x[j]));
      }
      const int ex = (int)(__float_as_uint(amax) >> 23);
      const int e2 = ex == 0 || ex == 255 ? 0 : min(ex - 127, 126);
      // a negative scale turns the query, so that the factor is not negative
      const float down = copysignf(__uint_as_float((uint32_t)(127 - e2) << 23), a.call.scale);
      fac = __uint_as_float((uint32_t)(127 + e2) << 23) * fabsf(a.call.scale) * (biased ? 1.f : kLog2e);
      const uint32_t qt = tc::smem_u32(sm + M::kQ) + tid * kPanel;
#pragma unroll 4
      for (int e = 0; e < D; e += 8) {
        float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
        if (row.x >= 0) {
          q_load4(q + e, vec, x);
          q_load4(q + e + 4, vec, y);
        }
        sts16(qt + e / 64 * kRowPanel + (((uint32_t)(e % 64 / 8) ^ sw) << 4), pack_h2(x[0] * down, x[1] * down),
              pack_h2(x[2] * down, x[3] * down), pack_h2(y[0] * down, y[1] * down), pack_h2(y[2] * down, y[3] * down));
      }
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(q_full);
    }

    const uint32_t pt = tc::smem_u32(sm + M::kP) + tid * kPanel;
    float m = -INFINITY, l = 0.f, ref = 0.f;
    int vref = 0, vmost = 0;
    uint32_t pv = 0;  // P written
    bool ok = true;
    // O times f, once the last P V is complete.
    auto rescale = [&](float f) {
      if (pv == 0) return true;
      if (!__all_sync(0xffffffffu, wait(pv_done, (pv - 1) & 1))) return false;
      tc::fence_after_sync();
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        float o[32];
        tc::tmem_ld32(tl + 128 + c, o);
#pragma unroll
        for (int j = 0; j < 32; ++j) o[j] *= f;
        tc::tmem_st32(tl + 128 + c, o);
      }
      tc::fence_before_sync();
      return true;
    };
    // O's units to V scale byte vb, as near as 2^80 of the largest so far lets
    // them be (the same for all rows); what O is to be multiplied by.
    auto set_units = [&](int vb) -> float {
      vmost = max(vmost, vb);
      const int now = max(vb, vmost - 80), by = vref ? vref - now : 0;
      vref = now;
      return by < -126 ? 0.f : __uint_as_float((uint32_t)(127 + by) << 23);
    };
    for (int b = 0; b < blocks; ++b) {
      const int s = b & 1;
      if (!__all_sync(0xffffffffu, wait(&s_full[s], (b / 2) & 1))) {
        ok = false;
        break;
      }
      tc::fence_after_sync();
      float x[kKeys];
      {
        uint32_t r[4][16];
#pragma unroll
        for (int p = 0; p < kPages; ++p) tc::tmem_ld16_async(tl + 64 * s + 16 * p, r[p]);
        tc::tmem_wait_ld();
#pragma unroll
        for (int p = 0; p < kPages; ++p)
#pragma unroll
          for (int j = 0; j < 16; ++j) x[16 * p + j] = __uint_as_float(r[p][j]);
      }
      int sc[kPages];
      bool here = true;
      int top = 0;
#pragma unroll
      for (int p = 0; p < kPages; ++p) {
        sc[p] = scales[s * kPages + p];
        here &= (sc[p] & kPageHere) != 0;
        top = max(top, sc[p] >> 8 & 255);
      }
      const int parts = block_parts(sc);
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&s_empty[s]);

      // Scores: x stays raw, with a factor a page, where nothing is added or hidden.
      float f[kPages], mx = -INFINITY;
#pragma unroll
      for (int p = 0; p < kPages; ++p) f[p] = scale_of(sc[p] & 255) * fac;
      const bool plain = here && !biased && it.key0 + (b + 1) * kKeys <= it.minvis;
      if (plain) {
#pragma unroll
        for (int p = 0; p < kPages; ++p) {
          float t = x[16 * p];
#pragma unroll
          for (int j = 1; j < 16; ++j) t = fmaxf(t, x[16 * p + j]);
          mx = fmaxf(mx, t * f[p]);
        }
      } else {
        const int nv = vis - b * kKeys;
#pragma unroll
        for (int p = 0; p < kPages; ++p) {
          const bool on = (sc[p] & kPageHere) != 0;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float y = x[16 * p + j] * f[p];
            if (biased) y += take_bias(__ldg(bias + min(max(col0 + b * kKeys + 16 * p + j, 0), last)));
            y = on && 16 * p + j < nv ? y : -INFINITY;
            x[16 * p + j] = y;
            mx = fmaxf(mx, y);
          }
          f[p] = 1.f;
        }
      }
      float grow = 1.f;
      if (__any_sync(0xffffffffu, mx > m + slack)) {
        const float now = fmaxf(m, mx);
        grow = weight_of(m, now, lg);
        m = now;
        ref = now == -INFINITY ? 0.f : fmaf(-now, lg, kShift);
        l *= grow;
      }
      if (parts == 1 && top) {
        int low = 255;
#pragma unroll
        for (int p = 0; p < kPages; ++p) low = min(low, sc[p] >> 8 & 255 ? sc[p] >> 8 & 255 : 255);
        // the middle of the block's scales: both ends stay inside the window
        if (vref == 0 || top - vref > kVWindow || vref - low > kVWindow) grow *= set_units((top + low) / 2);
      }
      if (__any_sync(0xffffffffu, grow != 1.f) && !rescale(grow)) {
        ok = false;
        break;
      }
      // Weights, four pages of sixteen, as f16 pairs.
      uint32_t w[kKeys / 2];
#pragma unroll
      for (int p = 0; p < kPages; ++p) {
        const int vb = sc[p] >> 8 & 255;
        const int up = parts == 1 && vb ? min(max(vb - vref, -126), kVWindow) : 0;
        const float from = ref + (float)up, by = f[p] * lg;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          const float e0 = exp2_approx(fmaf(x[16 * p + j], by, from));
          const float e1 = exp2_approx(fmaf(x[16 * p + j + 1], by, from));
          sum += e0 + e1;
          w[8 * p + j / 2] = pack_h2(e0, e1);
        }
        l = fmaf(sum, __uint_as_float((uint32_t)(127 - up) << 23), l);
      }
      for (int i = 0; i < parts && ok; ++i) {
        bool mine = true;
        if (parts > 1) {  // page i alone, in units of its own scale
          int vb = 0;
#pragma unroll
          for (int p = 0; p < kPages; ++p) vb = p == i ? sc[p] >> 8 & 255 : vb;
          if (vb) {
            const float g = set_units(vb);
            if (g != 1.f && !rescale(g)) {
              ok = false;
              break;
            }
          }
          mine = vb == vref;  // (else far below the largest scale, or zeros)
        }
        if (pv > 0 && !__all_sync(0xffffffffu, wait(pv_done, (pv - 1) & 1))) {  // P is free
          ok = false;
          break;
        }
#pragma unroll
        for (int c = 0; c < kKeys / 8; ++c) {
          const bool on = parts == 1 || (mine && c / 2 == i);
          uint32_t u[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) u[j] = on ? w[4 * c + j] : 0u;
          sts16(pt + (((uint32_t)c ^ sw) << 4), u[0], u[1], u[2], u[3]);
        }
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(p_full);
        ++pv;
      }
      if (!ok) break;
    }
    if (ok && pv > 0) ok = __all_sync(0xffffffffu, wait(pv_done, (pv - 1) & 1));
    tc::fence_after_sync();
    const size_t part = ((size_t)max(it.part, 0) * H + head) * kRows + tid;
    const float unit_v = vref ? scale_of(vref) : 1.f;
    const float f = it.part >= 0 ? unit_v : l == 0.f ? 0.f : unit_v / l;
    const bool ovec = a.call.out_stride[0] % 4 == 0 && a.call.out_stride[1] % 4 == 0 &&
                      (reinterpret_cast<uintptr_t>(a.call.out) & 7) == 0;
    bf16* out = static_cast<bf16*>(a.call.out) + row.x * a.call.out_stride[0] +
                (int64_t)(head * a.shape.share + row.w) * a.call.out_stride[1];
    if (ok) {
      if (it.part >= 0 && row.x >= 0) a.plan.ml[part] = make_float2(m, l);
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        float o[32];
        if (pv > 0) {
          tc::tmem_ld32(tl + 128 + c, o);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = 0.f;
        }
        if (row.x >= 0) {
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float y[4] = {o[j] * f, o[j + 1] * f, o[j + 2] * f, o[j + 3] * f};
            if (it.part >= 0)
              *reinterpret_cast<float4*>(a.plan.o + part * D + c + j) = make_float4(y[0], y[1], y[2], y[3]);
            else
              out_store4(out + c + j, ovec, y);
          }
        }
      }
    }
    if (it.part >= 0) {  // (after a wait that ran out too: the counter is left as it was found)
      __threadfence();
      asm volatile("bar.sync 1, 128;" ::: "memory");
      int* done = a.plan.done + (size_t)it.tile * H + head;
      if (tid == 0) misc[2] = atomicAdd(done, 1) == it.splits - 1;
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (misc[2]) {
        __threadfence();
        if (tid == 0) *done = 0;
        join_items<bf16, D>(a, it, head, lg, 0, kRows, tid, kRows);
      }
    }
    tc::fence_before_sync();
  }
  __syncthreads();
  if (warp == 0) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, kCols);
  }
}

template <int D>
cudaError_t launch_tile(const AttendArgs& a, cudaStream_t s) {
  constexpr size_t smem = TileMem<D>::kBytes + 1024;
  auto fn = attend8_tile_kernel<D>;
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  const int64_t units = (int64_t)a.shape.max_items * a.cache.H;
  if (units > INT32_MAX) return cudaErrorInvalidValue;
  return launch_pdl(fn, dim3((unsigned)units), dim3(kTileThreads), smem, s, a);
}

}  // namespace

cudaError_t launch_attend8_tile(const imba_cache_desc& c, const AttendArgs& a, cudaStream_t s) {
  if (a.shape.tile_rows != kRows) return cudaErrorInvalidValue;
  return c.attention_dim == 64 ? launch_tile<64>(a, s) : launch_tile<128>(a, s);
}

}  // namespace imba
