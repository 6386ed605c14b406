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
// products; eight warps are the tile's rows, two threads a row, each with half
// of a block's keys: they read S from TMEM, agree on the row's maximum, weigh
// and write P; a lane of the last page warp issues the products: P V of a
// block, S of the block after next (whose tiles are ready: three stages), and
// its warp then turns its page of the block that P V makes room for.  Scales
// stay out of the products: K's multiplies a page's scores, V's is in its
// weights' exponent.
//
// What bounds it: the chain of a block, S to maxima to weights to P to P V
// (some 4,000 cycles a block of a CTA), so two CTAs share an SM (64-key blocks,
// 256 TMEM columns, 82 KB and, spilling 72 bytes, 80 registers at head size 64).
// 4 x 512 rows of 16 heads of 64 over 2k to 8k tokens take 179 us, 0.2 PFLOP/s;
// with one thread a row and all 64 keys 215, two stages of K and V 205, a
// fourth page warp apart from the products' lane 194, and tiles of 16 rows by
// mma.sync 280.
//
// Numerics as in the mma.sync kernel (attend8_kernel.cuh), but that scores
// without a bias become weights in one fused step while the row's maximum is
// within kNear: the rounding of kShift - maximum puts them off by 2^-8 of a unit
// of log2 at most there, all keys of a maximum alike.  V's scales of a block's
// four pages are held against one reference; where they lie more than 2^kSpread
// apart, the block's P V is done page by page.
#include <algorithm>

#include "attend8_common.cuh"
#include "tc_ptx.cuh"

namespace imba {

namespace {

constexpr int kRows = 128;
constexpr int kKeys = 64;
constexpr int kPages = kKeys / IMBA_PAGE_TOKENS;
constexpr int kTileThreads = 384;  // warps 0-7: rows; 8-11: pages, and 11 the products
constexpr int kRowWarps = 8;
constexpr int kHalf = kKeys / 2;   // keys of a row thread
constexpr uint32_t kCols = 256;    // TMEM columns: S at 0 and 64, O from 128
constexpr int kStages = 3;         // blocks of K and V
constexpr int kSpread = 12;        // with kVWindow on both sides
constexpr float kNear = 65536.f;   // largest maximum of the fused step
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
  static constexpr uint32_t kK = kP + kRowPanel;                     // kStages
  static constexpr uint32_t kV = kK + kStages * kPanels * kKvPanel;  // kStages
  static constexpr uint32_t kMisc = kV + kStages * kPanels * kKvPanel;
  static constexpr uint32_t kInfo = kMisc + 256;
  static constexpr uint32_t kMax = kInfo + 512;  // [2 blocks][2 halves][128] row maxima, and at last sums
  static constexpr uint32_t kFac = kMax + 4 * kRows * 4;  // [128] factors of the rows' scores
  static constexpr uint32_t kBytes = kFac + kRows * 4;
};


__device__ __forceinline__ void sts16(uint32_t dst, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Two floats in a register pair, and their sums and products.
__device__ __forceinline__ uint64_t pack_f2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpack_f2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// What the rows have to know of a block, written by a page warp beside its
// tiles.  V's units (the scale byte that O is held in units of) follow the
// blocks' scales and are the same for every row, so they are kept there.
struct BlockInfo {
  float ks[kPages];    // K's scales
  float up[kPages];    // log2 of V's scales in units of O
  float down[kPages];  // 2^-up
  float turn[kPages];  // with parts: what O is multiplied by before each page's P V
  float grow;          // without: what O is multiplied by
  int here;            // every page exists
  int parts;           // P V of the block: 1, or one a page
  int on;              // with parts: the pages that are not far below the largest scale (bits)
  float unit;          // O's units after the block
  int pages;           // the pages that exist (bits)
};

static_assert(kStages * sizeof(BlockInfo) <= 512, "BlockInfo's place in shared memory");

// The scale byte that O is held in units of.
struct Units {
  int vref = 0, vmost = 0;
  // To byte vb, as near as 2^80 of the largest so far lets it be (no sum then
  // overflows); what O is multiplied by.
  __device__ __forceinline__ float set(int vb) {
    vmost = max(vmost, vb);
    const int now = max(vb, vmost - 80), by = vref ? vref - now : 0;
    vref = now;
    return by < -126 ? 0.f : __uint_as_float((uint32_t)(127 + by) << 23);
  }
  // The next block, its pages' scale bytes K | V << 8 (-1: no page).
  __device__ __forceinline__ void next(const int (&sc)[kPages], BlockInfo& o) {
    int top = 0, low = 255;
    o.pages = 0;
#pragma unroll
    for (int p = 0; p < kPages; ++p) {
      const int vb = sc[p] < 0 ? 0 : sc[p] >> 8;
      o.ks[p] = sc[p] < 0 ? 0.f : scale_of(sc[p] & 255);
      o.pages |= (sc[p] >= 0) << p;
      top = max(top, vb);
      low = min(low, vb ? vb : 255);
      o.up[p] = 0.f;
      o.down[p] = o.turn[p] = 1.f;
    }
    o.here = o.pages == (1 << kPages) - 1;
    o.parts = top - low > kSpread ? kPages : 1;  // (top 0: low is 255)
    o.on = 0;
    o.grow = 1.f;
    if (o.parts == 1) {
      // the middle of the block's scales: both ends stay inside the window
      if (top && (vref == 0 || top - vref > kVWindow || vref - low > kVWindow)) o.grow = set((top + low) / 2);
#pragma unroll
      for (int p = 0; p < kPages; ++p) {
        const int vb = sc[p] < 0 ? 0 : sc[p] >> 8;
        const int up = vb ? min(max(vb - vref, kVLeast), kVWindow) : 0;
        o.up[p] = (float)up;
        o.down[p] = __uint_as_float((uint32_t)(127 - up) << 23);
      }
    } else {
#pragma unroll
      for (int p = 0; p < kPages; ++p) {
        const int vb = sc[p] < 0 ? 0 : sc[p] >> 8;
        if (vb) o.turn[p] = set(vb);
        o.on |= (vb != 0 && vb == vref) << p;
      }
    }
    o.unit = vref ? scale_of(vref) : 1.f;
  }
};

template <int D>
__global__ void __launch_bounds__(kTileThreads, D == 64 ? 2 : 1) attend8_tile_kernel(const AttendArgs a) {
  using M = TileMem<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + M::kMisc);
  uint64_t* kv_full = bars;        // [kStages] K and V of a block written (4 page warps)
  uint64_t* kv_empty = bars + 3;   // [kStages] its products are complete (commit)
  uint64_t* s_full = bars + 6;     // [2] S of a block complete (commit)
  uint64_t* s_empty = bars + 8;    // [2] S read (8 row warps)
  uint64_t* q_full = bars + 10;    // Q written (8 row warps)
  uint64_t* p_full = bars + 11;    // P written (8 row warps)
  uint64_t* pv_done = bars + 12;   // P V complete (commit)
  uint64_t* drain = bars + 13;
  int* misc = reinterpret_cast<int*>(bars + 14);  // [0] abort, [1] TMEM, [2] last of a split tile
  BlockInfo* infos = reinterpret_cast<BlockInfo*>(sm + M::kInfo);  // [kStages]
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
    for (int s = 0; s < kStages; ++s) {
      tc::mbar_init(&kv_full[s], 4);
      tc::mbar_init(&kv_empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(&s_full[s], 1);
      tc::mbar_init(&s_empty[s], kRowWarps);
    }
    tc::mbar_init(q_full, kRowWarps);
    tc::mbar_init(p_full, kRowWarps);
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
  auto wait_ns = [&](uint64_t* bar, uint32_t parity, uint32_t ns) {
    return tc::mbar_wait_sleep_or_abort(bar, parity, a.rows.status, abort_flag, ns);
  };
  auto wait = [&](uint64_t* bar, uint32_t parity) { return wait_ns(bar, parity, 32); };

  if (warp >= kRowWarps) {
    // ---------------- pages: codes to f16 tiles; products ----------------
    // Warp w takes page w of every block; ids and scales 32 blocks at a time.
    const int w = warp - kRowWarps;
    const uint8_t* head_k = a.cache.data + (int64_t)head * IMBA_PAGE_TOKENS * D;
    const uint8_t* head_v = a.cache.data + a.cache.v_offset + (int64_t)head * IMBA_PAGE_TOKENS * D;
    constexpr int kLoads = D / 32;  // 16-byte loads of a lane, for K and for V
    int id32 = -1;
    int sc32[kPages];  // the first page warp: scale bytes of the block's pages, -1 for none
    Units units;
    auto page_at = [&](int p) {
      const int id = p < it.pages ? a.rows.group_pages[it.list + p] : -1;
      if (p < it.pages && (id < 0 || id >= a.cache.num_pages)) {
        report(a.rows.status, IMBA_ERR_RANGE);
        return -1;
      }
      return id;
    };
    auto fetch_ids = [&](int b0) {  // lane: block b0 + lane
      if (w == 0) {
        int id[kPages];
#pragma unroll
        for (int p = 0; p < kPages; ++p) id[p] = page_at((b0 + lane) * kPages + p);
        id32 = id[0];
#pragma unroll
        for (int p = 0; p < kPages; ++p) {
          const uint8_t* s = a.cache.scales + max(id[p], 0) * a.cache.scale_stride + head;
          sc32[p] = id[p] < 0 ? -1 : s[0] | s[H] << 8;
        }
      } else {
        id32 = page_at((b0 + lane) * kPages + w);
      }
    };
    uint4 kr[kLoads], vr[kLoads];
    auto load = [&](int b) {
      const int id = __shfl_sync(0xffffffffu, id32, b & 31);
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
    // The products (warp 11, lane 0).
    constexpr uint32_t idS = idesc_f16(kRows, kKeys);
    constexpr uint32_t idPV = idesc_f16(kRows, 64) | tc::kIdescBMajorMN;
    uint32_t pv = 0;  // P V issued
    auto issue_s = [&](int b) {
      const int s = b & 1, kv = b % kStages;
      if (b == 0 && !wait(q_full, 0)) return false;
      if (!wait(&kv_full[kv], (b / kStages) & 1) || (b >= 2 && !wait(&s_empty[s], (b / 2 - 1) & 1))) return false;
      tc::fence_after_sync();
#pragma unroll
      for (int n = 0; n < M::kPanels; ++n) {
        const uint64_t dQ = tc::smem_desc_k128(sm + M::kQ + n * kRowPanel);
        const uint64_t dK = tc::smem_desc_k128(sm + M::kK + (kv * M::kPanels + n) * kKvPanel);
#pragma unroll
        for (int k = 0; k < 4; ++k) tc::umma_f16(tmem + 64 * s, dQ + 2 * k, dK + 2 * k, idS, (n | k) != 0);
      }
      tc::umma_commit(&s_full[s]);
      return true;
    };
    auto issue_pv = [&](int b) {
      const int kv = b % kStages;
      const int parts = *reinterpret_cast<volatile int*>(&infos[kv].parts);
      const uint64_t dP = tc::smem_desc_k128(sm + M::kP);
      for (int i = 0; i < parts; ++i, ++pv) {
        if (!wait(p_full, pv & 1)) return false;
        tc::fence_after_sync();
#pragma unroll
        for (int n = 0; n < M::kPanels; ++n) {
          const uint64_t dV = tc::smem_desc_k128(sm + M::kV + (kv * M::kPanels + n) * kKvPanel);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            tc::umma_f16(tmem + 128 + 64 * n, dP + 2 * k, dV + 128 * k, idPV, (pv | k) != 0);
        }
        if (i + 1 == parts) tc::umma_commit(&kv_empty[kv]);
        tc::umma_commit(pv_done);
      }
      return true;
    };
    fetch_ids(0);
    if (blocks > 0) load(0);
    bool ok = true;
    for (int b = 0; b < blocks; ++b) {
      const int s = b % kStages;
      // Block b's stage is free when P V of block b - 3 is complete; the warp of
      // the products issues those, and S of the block before this, first.
      if (w == 3 && b >= kStages) {
        if (lane == 0) ok = issue_pv(b - kStages) && issue_s(b - 1);
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
      }
      if (b >= kStages && !__all_sync(0xffffffffu, wait_ns(&kv_empty[s], (b / kStages - 1) & 1, w == 3 ? 32 : 200)))
        break;
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
      if (w == 0) {
        int sc[kPages];
#pragma unroll
        for (int p = 0; p < kPages; ++p) sc[p] = __shfl_sync(0xffffffffu, sc32[p], b & 31);
        BlockInfo info;
        units.next(sc, info);
        if (lane == 0) infos[s] = info;
      }
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&kv_full[s]);
      if (b + 1 < blocks) {  // (not before the fence, which would wait for it)
        if (((b + 1) & 31) == 0) fetch_ids(b + 1);
        load(b + 1);
      }
      if (w == 3 && b < kStages - 1) {  // the first two S
        if (lane == 0) ok = issue_s(b);
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
      }
    }
    if (w == 3 && lane == 0) {
      // What the loop has left: P V of the last three blocks, S of the last.
      for (int b = max(blocks - kStages, 0); ok && b < blocks; ++b)
        ok = issue_pv(b) && (b + 2 >= blocks || b + 2 < kStages - 1 || issue_s(b + 2));
      // Every product issued here completes before TMEM is freed.
      tc::umma_commit(drain);
      tc::mbar_wait_for(drain, 0, a.rows.status, tc::kWaitNs);
    }
    __syncwarp();
  } else {
    // ---------------- rows ----------------
    // Warps w and w + 4 share the rows of TMEM lanes 32 w: thread (row, half).
    const int half = warp / 4, trow = tid % kRows;
    const int4 row = __ldg(reinterpret_cast<const int4*>(a.plan.rows + (size_t)it.tile * kRows) + trow);
    const uint32_t tl = tmem + ((uint32_t)(32 * (warp % 4)) << 16);  // this warp's TMEM lanes
    const uint32_t sw = (uint32_t)(trow & 7);
    const bool biased = a.call.bias != nullptr;
    const float lg = biased ? kLog2e : 1.f, slack = biased ? kSlack / kLog2e : kSlack;
    const int vis = row.y - it.key0 - half * kHalf;  // of the item's keys, from this thread's first
    const float* bias = a.call.bias + (int64_t)(head * a.shape.share + row.w) * (2 * a.call.max_pos - 1);
    const int col0 = it.key0 + half * kHalf - row.z + a.call.max_pos - 1, last = 2 * a.call.max_pos - 2;
    volatile float* maxima = reinterpret_cast<float*>(sm + M::kMax);
    auto pair_sync = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + warp % 4) : "memory"); };
    // The queries over their powers of two, as f16: a warp takes sixteen rows,
    // lanes are (row, eight elements).
    {
      constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes, kPasses = kRows / kRowWarps / kAtOnce;
      const int e = lane % kLanes * 8;
      const bool vec = a.call.q_stride[0] % 8 == 0 && a.call.q_stride[1] % 8 == 0 &&
                       (reinterpret_cast<uintptr_t>(a.call.q) & 15) == 0;
      uint4 raw[kPasses];
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        const int r = warp * (kRows / kRowWarps) + i * kAtOnce + lane / kLanes;
        const int4 to = __ldg(reinterpret_cast<const int4*>(a.plan.rows + (size_t)it.tile * kRows) + r);
        raw[i] = make_uint4(0, 0, 0, 0);
        if (to.x < 0) continue;
        const bf16* q = static_cast<const bf16*>(a.call.q) + to.x * a.call.q_stride[0] +
                        (int64_t)(head * a.shape.share + to.w) * a.call.q_stride[1] + e;
        if (vec) {
          raw[i] = *reinterpret_cast<const uint4*>(q);
        } else {
          uint32_t u[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            u[j] = (uint32_t)__bfloat16_as_ushort(q[2 * j]) | (uint32_t)__bfloat16_as_ushort(q[2 * j + 1]) << 16;
          raw[i] = make_uint4(u[0], u[1], u[2], u[3]);
        }
      }
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        const int r = warp * (kRows / kRowWarps) + i * kAtOnce + lane / kLanes;
        const uint32_t u[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        float x[8], amax = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[2 * j] = __uint_as_float(u[j] << 16);
          x[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
          amax = fmaxf(amax, fmaxf(fabsf(x[2 * j]), fabsf(x[2 * j + 1])));
        }
#pragma unroll
        for (int o = 1; o < kLanes; o *= 2) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        const int ex = (int)(__float_as_uint(amax) >> 23);
        const int e2 = ex == 0 || ex == 255 ? 0 : min(ex - 127, 126);
        // a negative scale turns the query, so that the factor is not negative
        const float down = copysignf(__uint_as_float((uint32_t)(127 - e2) << 23), a.call.scale);
        if (lane % kLanes == 0)
          reinterpret_cast<float*>(sm + M::kFac)[r] =
              __uint_as_float((uint32_t)(127 + e2) << 23) * fabsf(a.call.scale) * (biased ? 1.f : kLog2e);
        sts16(tc::smem_u32(sm + M::kQ) + e / 64 * kRowPanel + r * kPanel + (((uint32_t)(e % 64 / 8) ^ (uint32_t)(r & 7)) << 4),
              pack_h2(x[0] * down, x[1] * down), pack_h2(x[2] * down, x[3] * down), pack_h2(x[4] * down, x[5] * down),
              pack_h2(x[6] * down, x[7] * down));
      }
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(q_full);
      asm volatile("bar.sync 5, 256;" ::: "memory");
    }
    const float fac = reinterpret_cast<const float*>(sm + M::kFac)[trow];

    const uint32_t pt = tc::smem_u32(sm + M::kP) + trow * kPanel;
    float m = kLowest, l = 0.f, ref = kShift;  // ref: kShift, the maximum to be subtracted apart, or with it
    float unit = 1.f;  // O's
    uint32_t pv = 0;   // P written
    bool ok = true;
    // O (this thread's half of its columns) times f, once the last P V is complete.
    auto rescale = [&](float f) {
      if (pv == 0) return true;
      if (!__all_sync(0xffffffffu, wait(pv_done, (pv - 1) & 1))) return false;
      tc::fence_after_sync();
#pragma unroll
      for (int c = 0; c < D / 2; c += 32) {
        float o[32];
        tc::tmem_ld32(tl + 128 + half * (D / 2) + c, o);
#pragma unroll
        for (int j = 0; j < 32; ++j) o[j] *= f;
        tc::tmem_st32(tl + 128 + half * (D / 2) + c, o);
      }
      tc::fence_before_sync();
      return true;
    };
    uint32_t at[4];  // this thread's chunks of P
#pragma unroll
    for (int c = 0; c < 4; ++c) at[c] = pt + (((uint32_t)(4 * half + c) ^ sw) << 4);
    for (int b = 0; b < blocks; ++b) {
      const int s = b & 1;
      // After a wait that ran out a warp only meets its partner, block by block.
      ok = ok && __all_sync(0xffffffffu, wait(&s_full[s], (b / 2) & 1));
      if (!ok) {
        pair_sync();
        continue;
      }
      tc::fence_after_sync();
      float x[kHalf];
      {
        uint32_t r[2][16];
        tc::tmem_ld16_async(tl + 64 * s + kHalf * half, r[0]);
        tc::tmem_ld16_async(tl + 64 * s + kHalf * half + 16, r[1]);
        tc::tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < kHalf; ++j) x[j] = __uint_as_float(r[j / 16][j % 16]);
      }
      const BlockInfo& info = infos[b % kStages];
      const float2 ks = *reinterpret_cast<const float2*>(info.ks + 2 * half);
      const float2 up = *reinterpret_cast<const float2*>(info.up + 2 * half);
      const float2 down = *reinterpret_cast<const float2*>(info.down + 2 * half);
      const float turned = info.grow;
      const int here = info.here, parts = info.parts;
      unit = info.unit;
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&s_empty[s]);

      // Scores: x stays raw, with a factor a page, where nothing is added or hidden.
      float f[2] = {ks.x * fac, ks.y * fac};
      float mx = -INFINITY;
      if (here && !biased && it.key0 + (b + 1) * kKeys <= it.minvis) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          float t = fmaxf(x[16 * p], x[16 * p + 1]);
#pragma unroll
          for (int j = 2; j < 16; j += 2) t = max3(t, x[16 * p + j], x[16 * p + j + 1]);
          mx = fmaxf(mx, t * f[p]);
        }
      } else {
        const int nv = vis - b * kKeys;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const int n = info.pages >> (2 * half + p) & 1 ? nv : 0;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float y = x[16 * p + j] * f[p];
            if (biased) y += __ldg(bias + min(max(col0 + b * kKeys + 16 * p + j, 0), last));
            y = 16 * p + j < n ? y : -INFINITY;
            x[16 * p + j] = y;
            mx = fmaxf(mx, y);
          }
          f[p] = 1.f;
        }
      }
      // The row's maximum over both halves.
      maxima[(s * 2 + half) * kRows + trow] = mx;
      pair_sync();
      mx = fmaxf(mx, maxima[(s * 2 + 1 - half) * kRows + trow]);
      if (__any_sync(0xffffffffu, mx - m > slack) || turned != 1.f) {
        const float now = fmaxf(m, mx), w = weight_of(m, now, lg);
        m = now;
        ref = biased || !(fabsf(now) <= kNear) ? kShift : kShift - now;
        l *= w;
        if (!rescale(w * turned)) {
          ok = false;
          continue;
        }
      }
      if (ref == kShift) {  // (scores rounded as the maximum was, which a fused product would not be)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
#pragma unroll
          for (int j = 0; j < 16; ++j) x[16 * p + j] = __fsub_rn(__fmul_rn(x[16 * p + j], f[p]), m);
          f[p] = 1.f;
        }
      }
      // Weights, two pages of sixteen, as f16 pairs.
      uint32_t w[kHalf / 2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const float from = ref + (p ? up.y : up.x), by = f[p] * lg;
        const uint64_t from2 = pack_f2(from, from), by2 = pack_f2(by, by);
        uint64_t sum = 0;
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          const float2 z = unpack_f2(fma_f2(pack_f2(x[16 * p + j], x[16 * p + j + 1]), by2, from2));
          const float e0 = exp2_approx(z.x), e1 = exp2_approx(z.y);
          sum = add_f2(sum, pack_f2(e0, e1));
          w[8 * p + j / 2] = pack_h2(e0, e1);
        }
        const float2 both = unpack_f2(sum);
        l = fmaf(both.x + both.y, p ? down.y : down.x, l);
      }
      for (int i = 0; i < parts; ++i) {
        bool all = true;
        if (parts > 1) {  // page i alone, in units of its own scale
          const float turn = info.turn[i];
          if (turn != 1.f && !rescale(turn)) {
            ok = false;
            break;
          }
          all = false;
        }
        if (pv > 0 && !__all_sync(0xffffffffu, wait(pv_done, (pv - 1) & 1))) {  // P is free
          ok = false;
          break;
        }
        if (all) {
#pragma unroll
          for (int c = 0; c < 4; ++c) sts16(at[c], w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const bool on = 2 * half + c / 2 == i && (info.on >> i & 1);
            sts16(at[c], on ? w[4 * c] : 0, on ? w[4 * c + 1] : 0, on ? w[4 * c + 2] : 0, on ? w[4 * c + 3] : 0);
          }
        }
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(p_full);
        ++pv;
      }
    }
    if (ok && pv > 0) ok = __all_sync(0xffffffffu, wait(pv_done, (pv - 1) & 1));
    tc::fence_after_sync();
    asm volatile("bar.sync 5, 256;" ::: "memory");  // all rows' maxima have been read
    maxima[half * kRows + trow] = l;
    asm volatile("bar.sync 5, 256;" ::: "memory");
    l += maxima[(1 - half) * kRows + trow];
    const size_t part = ((size_t)max(it.part, 0) * H + head) * kRows + trow;
    const float f = l == 0.f ? 0.f : unit / l;
    const bool ovec = a.call.out_stride[0] % 4 == 0 && a.call.out_stride[1] % 4 == 0 &&
                      (reinterpret_cast<uintptr_t>(a.call.out) & 7) == 0;
    bf16* out = static_cast<bf16*>(a.call.out) + row.x * a.call.out_stride[0] +
                (int64_t)(head * a.shape.share + row.w) * a.call.out_stride[1];
    if (ok) {
      if (it.part >= 0 && row.x >= 0 && half == 0) a.plan.ml[part] = make_float2(m, l);
#pragma unroll
      for (int c = half * (D / 2); c < (half + 1) * (D / 2); c += 32) {
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
      asm volatile("bar.sync 5, 256;" ::: "memory");
      int* done = a.plan.done + ((size_t)it.tile * H + head) * 8;
      if (tid == 0) misc[2] = atomicAdd(done, 1) == it.splits - 1;
      asm volatile("bar.sync 5, 256;" ::: "memory");
      if (misc[2]) {
        __threadfence();
        if (tid == 0) *done = 0;
        join_items<bf16, D, 4>(a, it, head, lg, 0, kRows, tid, 2 * kRows);
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
