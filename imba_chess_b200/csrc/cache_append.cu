// Appending to paged pools: the plan pass, rows read back, and the C entry
// points (the kernels are in cache_append.cuh).
#include <algorithm>

#include "cache_plan.cuh"

namespace imba {

namespace {

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

}  // namespace

cudaError_t launch_append_plan(int64_t num_slots, int32_t num_rows, const int32_t* slots, void* plan, int32_t* status,
                               cudaStream_t s) {
  const PlanView pv = plan_view(plan, num_rows);
  const size_t clear = (size_t)(kPlanHead + (int64_t)pv.cap * (1 + kTok)) * sizeof(int32_t);
  const cudaError_t e = cudaMemsetAsync(plan, 0xff, clear, s);
  if (e != cudaSuccess || num_rows == 0) return e;
  return launch_pdl(append_plan_kernel, dim3((num_rows + 127) / 128), dim3(128), 0, s, pv, (int)num_rows, slots,
                    num_slots, status);
}

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
  if (imba::validate_cache(cache) != IMBA_OK || num_pages <= 0 || num_pages > INT32_MAX / IMBA_PAGE_TOKENS) return 0;
  const int64_t elems = imba::cache8_page_bytes(*cache);
  if (cache->dtype == IMBA_DTYPE_E4M3)
    return (size_t)((elems + (int64_t)cache->num_layers * 2 * cache->num_heads) * num_pages);
  return (size_t)(elems * num_pages * (cache->dtype == IMBA_DTYPE_BF16 ? 2 : 4));
}

size_t imba_append_plan_bytes(int32_t num_rows) {
  if (num_rows < 0 || num_rows > imba::kMostRows) return 0;
  const int64_t cap = imba::plan_cap(num_rows);
  return (size_t)(imba::kPlanHead + cap * (1 + IMBA_PAGE_TOKENS) + num_rows) * sizeof(int32_t);
}

imba_status_t imba_append_plan(const imba_pool_desc* pool, int32_t num_rows, const int32_t* slots, void* plan,
                               size_t plan_bytes, int32_t* status, void* stream) {
  const imba_status_t v = imba::validate_pool(pool);
  if (v != IMBA_OK) return v;
  if (num_rows < 0 || num_rows > imba::kMostRows) return IMBA_ERR_ARG;
  if (!plan || (num_rows > 0 && !slots) || (reinterpret_cast<uintptr_t>(plan) & 255)) return IMBA_ERR_ARG;
  if (plan_bytes < imba_append_plan_bytes(num_rows)) return IMBA_ERR_OOM;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      imba::launch_append_plan(pool->num_pages * IMBA_PAGE_TOKENS, num_rows, slots, plan, status, s);
  return e == cudaSuccess ? IMBA_OK : IMBA_ERR_CUDA;
}

imba_status_t imba_kv_append(const imba_cache_desc* cache, const imba_pool_desc* pool, const imba_append_desc* append,
                             const void* plan, size_t plan_bytes, void* stream) {
  imba_status_t v = imba::validate_cache(cache);
  if (v == IMBA_OK) v = imba::validate_pool(pool);
  if (v != IMBA_OK) return v;
  if (!append || append->num_rows < 0 || append->num_rows > imba::kMostRows) return IMBA_ERR_ARG;
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
