// Attention over a pool in 8 bits: the plan pass and the C entry points.
//
// The plan is made once per step and read by every layer: one CTA lays the
// segments' rows out in tiles, finds each tile's visible pages and cuts long
// page lists into items of about the same size, so that a few long sequences
// still fill the device; a second kernel resolves and checks the tiles' rows.
// Nothing about a step's lengths is needed on the host.
#include <algorithm>

#include "attend8.cuh"

namespace imba {

namespace {

constexpr int kPlanThreads = 1024;

inline size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// Exclusive sum over the CTA's threads; the total in *total.
template <typename I>
__device__ __forceinline__ I block_scan(I v, I* warp_sums, I* total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  I x = v;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const I y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    I w = lane < kPlanThreads / 32 ? warp_sums[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const I y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  const I before = (warp ? warp_sums[warp - 1] : 0) + x - v;
  *total = warp_sums[kPlanThreads / 32 - 1];
  __syncthreads();
  return before;
}

// Rows of segment s: [off, off + n) of the row order; n = 0 when malformed.
__device__ __forceinline__ void segment(const imba_attend_desc& r, int s, int* off, int* n) {
  const int o = r.seg_row_off[s];
  int k = r.seg_nrows ? r.seg_nrows[s] : r.seg_row_off[s + 1] - o;
  if (o < 0 || k < 0 || k > r.num_rows - o) {
    report(r.status, IMBA_ERR_RANGE);
    k = 0;
  }
  *off = o;
  *n = k;
}

// First entry and length of a segment's page list.
__device__ __forceinline__ void page_list(const imba_attend_desc& r, int s, int* first, int* count) {
  const int g = r.seg_group ? r.seg_group[s] : s;
  int a = 0, b = 0;
  if (g >= 0 && g < r.num_groups) {
    a = r.group_page_off[g];
    b = r.group_page_off[g + 1];
  } else {
    report(r.status, IMBA_ERR_RANGE);
  }
  if (a < 0 || b < a || b > r.num_group_pages) {
    report(r.status, IMBA_ERR_RANGE);
    a = b = 0;
  }
  *first = a;
  *count = b - a;
}

__device__ __forceinline__ int row_at(const imba_attend_desc& r, int i) {
  int row = r.row_perm ? r.row_perm[i] : i;
  if (row < 0 || row >= r.num_rows) {
    report(r.status, IMBA_ERR_RANGE);
    row = -1;
  }
  return row;
}

__device__ __forceinline__ int visible(const imba_attend_desc& r, int row, int cap) {
  const int v = r.row_vis[row];
  if (v < 0 || v > cap) report(r.status, IMBA_ERR_RANGE);
  return min(max(v, 0), cap);
}

// Items of a tile at most.  What a tile of p pages in n parts waits for is a
// part's pages, p / n, and the join by one CTA, n times the tile's rows: n in
// proportion to the root of p, and fewer for more rows.  One sequence of one
// head of 64, up to 16, 32, 64, 128 parts and this rule's: 4 rows over 20,000
// tokens 12.7, 10.3, 11.6, 15.4 us, over 131,000 48, 28, 22, 21; 20 rows over
// 131,000 54, 35, 28, 32; 256 rows over 20,000 54, 59, 88, 165.
__device__ __forceinline__ int most_parts(int pages, int rt) {
  return (int)ceilf(sqrtf(4.f * (float)pages / (float)(3 + rt)));
}

__global__ void __launch_bounds__(kPlanThreads) attend_items_kernel(imba_attend_desc r, AttendShape sh, AttendPlan p,
                                                                    int H) {
  __shared__ int warp_sums[32];
  __shared__ long long tile_sums[32];
  __shared__ unsigned long long all_pages;
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x;
  if (tid == 0) all_pages = 0;
  // Tiles of each segment, counted in 64 bits: segments that overlap can ask
  // for more rows than there are, each of them for all.
  long long asked = 0;
  for (int s0 = 0; s0 < r.num_segs; s0 += kPlanThreads) {
    const int s = s0 + tid;
    int off = 0, n = 0;
    long long t = 0, sum;
    if (s < r.num_segs) {
      segment(r, s, &off, &n);
      t = ((int64_t)n * sh.share + sh.tile_rows - 1) / sh.tile_rows;
    }
    const long long before = block_scan(t, tile_sums, &sum);
    if (s < r.num_segs) p.tile_off[s] = (int)min(asked + before, (long long)sh.max_tiles);
    asked += sum;
  }
  if (asked > sh.max_tiles && tid == 0) report(r.status, IMBA_ERR_RANGE);
  const int ntiles = (int)min(asked, (long long)sh.max_tiles);
  if (tid == 0) p.tile_off[r.num_segs] = ntiles;
  __syncthreads();
  // Their rows and visible pages.
  unsigned long long mine = 0;
  for (int t = tid; t < ntiles; t += kPlanThreads) {
    int lo = 0, hi = r.num_segs;  // the last segment that starts at or before tile t
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (p.tile_off[mid] <= t) lo = mid; else hi = mid;
    }
    int off, n, first, count;
    segment(r, lo, &off, &n);
    page_list(r, lo, &first, &count);
    const int f0 = (t - p.tile_off[lo]) * sh.tile_rows;
    const int nf = max(0, min(sh.tile_rows, n * sh.share - f0));
    int vmax = 0, vmin = 0x7fffffff;
    for (int i = f0 / sh.share; i * sh.share < f0 + nf; ++i) {
      const int row = row_at(r, off + i);
      const int v = row < 0 ? 0 : visible(r, row, count * IMBA_PAGE_TOKENS);
      vmax = max(vmax, v);
      vmin = min(vmin, v);
    }
    const int pages = (vmax + IMBA_PAGE_TOKENS - 1) / IMBA_PAGE_TOKENS;
    p.tiles[2 * t] = make_int4(lo, f0, nf, pages);
    p.tiles[2 * t + 1] = make_int4(off, first, count, vmin);
    mine += pages;
    for (int h = 0; h < 8 * H; ++h) p.done[(size_t)t * 8 * H + h] = 0;
  }
  if (mine) atomicAdd(&all_pages, mine);
  __syncthreads();
  // Pages per item: aim at shape.target items over all tiles.
  const unsigned long long total = all_pages;
  const int per = (int)max((unsigned long long)sh.min_pages, (total + sh.target - 1) / sh.target);
  int nitems = 0, nparts = 0;
  for (int t0 = 0; t0 < ntiles; t0 += kPlanThreads) {
    const int t = t0 + tid;
    int4 a = make_int4(0, 0, 0, 0), b = a;
    int n = 0, sum;
    if (t < ntiles) {
      a = p.tiles[2 * t];
      b = p.tiles[2 * t + 1];
      n = (a.w + per - 1) / per;
      // a single wave is not passed by a few items (152 units on 148 SMs: 488 us
      // against 313 for 256 rows, 4 heads of 128 and 131,000 tokens)
      if (sh.waves == 1) n = min(n, (int)((unsigned long long)a.w * sh.target / max(total, 1ull)));
      n = max(1, min(n, most_parts(a.w, sh.rt)));
    }
    const int at = nitems + block_scan(n, warp_sums, &sum);
    nitems += sum;
    const int pt = nparts + block_scan(n > 1 ? n : 0, warp_sums, &sum);
    nparts += sum;
    for (int i = 0; i < n; ++i) {
      const int p0 = (int)((int64_t)a.w * i / n), p1 = (int)((int64_t)a.w * (i + 1) / n);
      if (at + i >= sh.max_items) break;
      p.items[at + i] = AttendItem{t, b.y + p0, p1 - p0, p0 * IMBA_PAGE_TOKENS, n > 1 ? pt + i : -1, n, b.w, i};
    }
  }
  if (tid == 0) p.head[0] = min(nitems, sh.max_items);
}

__global__ void attend_rows_kernel(imba_attend_desc r, AttendShape sh, AttendPlan p) {
  pdl_wait();
  pdl_trigger();
  const int ntiles = p.tile_off[r.num_segs];
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < (int64_t)ntiles * sh.tile_rows;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int t = (int)(i / sh.tile_rows), m = (int)(i % sh.tile_rows);
    const int4 a = p.tiles[2 * t], b = p.tiles[2 * t + 1];
    AttendRow o{-1, 0, 0, 0};
    if (m < a.z) {
      const int f = a.y + m;
      o.row = row_at(r, b.x + f / sh.share);
      if (o.row >= 0) {
        o.vis = visible(r, o.row, b.z * IMBA_PAGE_TOKENS);
        o.pos = r.positions ? max(r.positions[o.row], -kMostPos) : 0;
        o.head = f % sh.share;
      }
    }
    p.rows[i] = o;
  }
}

}  // namespace

namespace {

// Rows a segment (with its shared heads), on average over the step, from which
// the tcgen05 kernel's tiles of 128 are better than tiles of 16 by mma.sync.  A
// model's steps cut their groups into chunks of 64 rows, so theirs stay below.
// (8 heads of 64, segments of 2k to 12k tokens: 64 rows 99 us against 91, 96
// rows 98 against 119, 256 rows 160 against 248; heads of 128: 64 rows 180
// against 139, 96 rows 181 against 191, 256 rows 283 against 422; segments of
// up to 600 tokens turn at about the same numbers of rows.)
constexpr int64_t kTileFrom = 80;

// Head sizes of that kernel.
bool tile_dims(const imba_cache_desc& c) { return c.attention_dim == c.linear_dim && c.attention_dim % 64 == 0; }

// The shape with tiles of 8 rt rows and `warps` warps a unit.
AttendShape shape_of(const imba_cache_desc& c, const imba_attend_desc& r, int rt, int warps, int64_t most) {
  AttendShape sh;
  sh.share = r.num_q_heads / c.num_heads;
  sh.rt = rt;
  sh.tile_rows = kTileRows * rt;
  const int64_t flat = (int64_t)r.num_rows * sh.share;
  const int64_t tiles = r.num_segs ? (flat + sh.tile_rows - 1) / sh.tile_rows + r.num_segs : 0;
  sh.max_tiles = (int)std::min<int64_t>(tiles, INT32_MAX);
  sh.warps = warps;
  sh.min_pages = warps == 1 ? 16 : 8;
  // About four CTAs' worth of units for each that is resident (two of the
  // tcgen05 kernel's, whose parts are large), but no more than 32 units a tile
  // and head where that leaves one wave at least, since a tile's parts are
  // joined by one CTA: one sequence of 131,000 tokens (20 rows, 8 heads of 128)
  // takes 80 us as one wave and 131 as four, 32 long sequences 318 and 260.
  // (A wave of few heads can be more parts; most_parts bounds those.)
  const int ctas = std::min(attend8_ctas(c.attention_dim, rt), 2);
  const int64_t few = std::max<int64_t>((flat + sh.tile_rows - 1) / sh.tile_rows, r.num_segs) * c.num_heads * 32;
  const int waves = sh.waves = (int)std::min<int64_t>(rt == kTileGroups ? 2 : 4, std::max<int64_t>(1, few / (148 * ctas)));
  sh.target = (int)std::min<int64_t>(most, std::max(1, 148 * ctas * waves * (kUnitWarps / warps) / c.num_heads));
  const int64_t by_len = (int64_t)sh.max_tiles * ((r.num_group_pages + sh.min_pages - 1) / sh.min_pages);
  const int64_t cut = std::min<int64_t>(by_len, sh.target);  // full-size items; each tile may add one smaller
  sh.max_items = (int)std::min<int64_t>(sh.max_tiles + cut, INT32_MAX / 4);
  sh.max_parts = (int)std::min<int64_t>(2 * cut, INT32_MAX / 4);
  return sh;
}

}  // namespace

AttendShape attend_shape(const imba_cache_desc& c, const imba_attend_desc& r, int64_t most) {
  const int64_t flat = (int64_t)r.num_rows * (r.num_q_heads / c.num_heads);
  // Rows of a tile by what a segment has on average: the fewest groups that
  // hold it (the games' step, one row a segment: 44 us with one group, 48 with
  // two; waves of siblings: 54 with one, 43 with two).
  const int64_t per_seg = r.num_segs ? (flat + r.num_segs - 1) / r.num_segs : 0;
  if (r.num_extra == 0 && tile_dims(c) && per_seg >= kTileFrom) return shape_of(c, r, kTileGroups, kUnitWarps, most);
  // Three groups only where they save a tile of two (20 rows a segment, bf16,
  // 131,000 tokens, 8 heads of 128: 79 us against 157; 512 segments of up to
  // 600 tokens, 4 heads of 64: 79 against 80; with 33 to 60 rows a segment,
  // the waves of siblings, 52 against 46).
  const int rt = per_seg <= 8 ? 1 : per_seg <= 16 || per_seg > 24 ? 2 : 3;
  // One warp per unit when there are enough units to fill the device and the
  // page lists are short on average; else the CTA's warps share a unit.
  // (1,024 one-token games of up to 300 tokens: 44 us against 90; the waves of
  // siblings 52 against 145.)
  const int64_t avg = r.num_groups ? r.num_group_pages / r.num_groups : 0;
  const int64_t busy = std::max<int64_t>(flat / (kTileRows * rt), r.num_segs) * c.num_heads;
  return shape_of(c, r, rt, busy >= 148 * 8 && avg <= 32 ? 1 : kUnitWarps, most);
}

size_t attend_step_bytes(const imba_cache_desc& c, int32_t rows) {
  imba_attend_desc r = {};
  r.num_rows = r.num_groups = rows;
  r.num_group_pages = kMostPages;
  r.num_q_heads = c.num_heads;
  size_t most = 0;
  // What attend_shape gives such a step: a tile size comes with segments of
  // more rows than `past` on average, so there are (rows - 1) / past at most,
  // and every part of a plan grows with their number.
  auto add = [&](int rt, int warps, int past) {
    r.num_segs = past ? (rows - 1) / past : rows;
    if (r.num_segs > 0)
      most = std::max(most, attend_plan_view(c, r, shape_of(c, r, rt, warps, attend_step_most(rows)), nullptr).bytes);
  };
  for (int warps : {1, kUnitWarps}) {
    add(1, warps, 0);
    add(2, warps, 8);
    add(3, warps, 16);
  }
  if (tile_dims(c)) add(kTileGroups, kUnitWarps, kTileFrom - 1);
  return most;
}

AttendPlan attend_plan_view(const imba_cache_desc& c, const imba_attend_desc& r, const AttendShape& sh, void* base) {
  AttendPlan p;
  size_t off = 0;
  char* b = static_cast<char*>(base);
  auto take = [&](size_t bytes) -> void* {
    void* q = b ? b + off : nullptr;
    off += up256(bytes);
    return q;
  };
  p.head = static_cast<int*>(take(256));
  p.tile_off = static_cast<int*>(take(((size_t)r.num_segs + 1) * sizeof(int)));
  p.tiles = static_cast<int4*>(take((size_t)sh.max_tiles * 2 * sizeof(int4)));
  p.items = static_cast<AttendItem*>(take((size_t)sh.max_items * sizeof(AttendItem)));
  p.rows = static_cast<AttendRow*>(take((size_t)sh.max_tiles * sh.tile_rows * sizeof(AttendRow)));
  p.done = static_cast<int*>(take((size_t)sh.max_tiles * c.num_heads * 8 * sizeof(int)));
  p.ml = static_cast<float2*>(take((size_t)sh.max_parts * c.num_heads * sh.tile_rows * sizeof(float2)));
  p.o = static_cast<float*>(take((size_t)sh.max_parts * c.num_heads * sh.tile_rows * c.linear_dim * sizeof(float)));
  p.bytes = off;
  return p;
}

cudaError_t launch_attend_plan(const imba_cache_desc& c, const imba_attend_desc& r, const AttendShape& sh,
                               const AttendPlan& p, cudaStream_t s) {
  const cudaError_t e =
      launch_pdl(attend_items_kernel, dim3(1), dim3(kPlanThreads), 0, s, r, sh, p, (int)c.num_heads);
  if (e != cudaSuccess) return e;
  const int64_t blocks = ((int64_t)sh.max_tiles * sh.tile_rows + 255) / 256;
  return launch_pdl(attend_rows_kernel, dim3((unsigned)std::min<int64_t>(blocks, 148 * 8)), dim3(256), 0, s, r, sh, p);
}

namespace {

imba_status_t validate_rows(const imba_cache_desc* c, const imba_attend_desc* r) {
  const imba_status_t v = validate_cache(c);
  if (v != IMBA_OK) return v;
  if (c->dtype != IMBA_DTYPE_E4M3) return IMBA_ERR_UNSUPPORTED;
  if (!r || r->num_rows < 0 || r->num_segs < 0 || r->num_groups < 0 || r->num_group_pages < 0 || r->num_extra < 0)
    return IMBA_ERR_ARG;
  if (r->num_q_heads <= 0 || r->num_q_heads % c->num_heads) return IMBA_ERR_ARG;
  if (r->num_group_pages > kMostPages || r->num_extra > kMostExtra) return IMBA_ERR_RANGE;
  if ((int64_t)r->num_rows * (r->num_q_heads / c->num_heads) > (1 << 28) || r->num_segs > (1 << 28))
    return IMBA_ERR_UNSUPPORTED;
  if (!r->seg_group && r->num_segs > r->num_groups) return IMBA_ERR_ARG;
  return IMBA_OK;
}

}  // namespace

}  // namespace imba

extern "C" {

size_t imba_attend_plan_bytes(const imba_cache_desc* cache, const imba_attend_desc* rows) {
  if (imba::validate_rows(cache, rows) != IMBA_OK) return 0;
  return imba::attend_plan_view(*cache, *rows, imba::attend_shape(*cache, *rows), nullptr).bytes;
}

static imba_status_t attend_check(const imba_cache_desc* cache, const imba_pool_desc* pool,
                                  const imba_attend_desc* rows, void* plan, size_t plan_bytes) {
  imba_status_t v = imba::validate_rows(cache, rows);
  if (v == IMBA_OK) v = imba::validate_pool(pool);
  if (v != IMBA_OK) return v;
  if (rows->num_rows && rows->num_segs) {
    if (!rows->seg_row_off || !rows->row_vis || !rows->group_page_off) return IMBA_ERR_ARG;
    if (rows->num_group_pages > 0 && !rows->group_pages) return IMBA_ERR_ARG;
    if (rows->num_extra > 0 && (!rows->row_extra_off || !rows->extra_slot || !rows->extra_pos)) return IMBA_ERR_ARG;
  }
  if (!plan || (reinterpret_cast<uintptr_t>(plan) & 255)) return IMBA_ERR_ARG;
  if (plan_bytes < imba_attend_plan_bytes(cache, rows)) return IMBA_ERR_OOM;
  return IMBA_OK;
}

imba_status_t imba_attend_plan(const imba_cache_desc* cache, const imba_pool_desc* pool, const imba_attend_desc* rows,
                               void* plan, size_t plan_bytes, void* stream) {
  const imba_status_t v = attend_check(cache, pool, rows, plan, plan_bytes);
  if (v != IMBA_OK) return v;
  if (rows->num_rows == 0 || rows->num_segs == 0) return IMBA_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const imba::AttendShape sh = imba::attend_shape(*cache, *rows);
  const imba::AttendPlan p = imba::attend_plan_view(*cache, *rows, sh, plan);
  return imba::launch_attend_plan(*cache, *rows, sh, p, s) == cudaSuccess ? IMBA_OK : IMBA_ERR_CUDA;
}

imba_status_t imba_attend(const imba_cache_desc* cache, const imba_pool_desc* pool, const imba_attend_desc* rows,
                          const imba_attend_args* args, void* plan, size_t plan_bytes, void* stream) {
  const imba_status_t v = attend_check(cache, pool, rows, plan, plan_bytes);
  if (v != IMBA_OK) return v;
  if (!args) return IMBA_ERR_ARG;
  if (args->layer < 0 || args->layer >= cache->num_layers) return IMBA_ERR_RANGE;
  if (args->dtype != IMBA_DTYPE_F32 && args->dtype != IMBA_DTYPE_BF16) return IMBA_ERR_ARG;
  if (args->bias && args->max_pos > imba::kMostPos) return IMBA_ERR_UNSUPPORTED;
  if (rows->num_rows == 0 || rows->num_segs == 0) return IMBA_OK;
  if (!args->q || !args->out) return IMBA_ERR_ARG;
  if (args->bias && (args->max_pos <= 0 || !rows->positions)) return IMBA_ERR_ARG;
  imba::AttendArgs a;
  a.cache = imba::cache8_layer(*cache, *pool, args->layer);
  a.shape = imba::attend_shape(*cache, *rows);
  a.plan = imba::attend_plan_view(*cache, *rows, a.shape, plan);
  a.rows = *rows;
  a.call = *args;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = args->dtype == IMBA_DTYPE_BF16 ? imba::launch_attend8<imba::bf16>(*cache, a, s)
                                                       : imba::launch_attend8<float>(*cache, a, s);
  return e == cudaSuccess ? IMBA_OK : IMBA_ERR_CUDA;
}

}  // extern "C"
