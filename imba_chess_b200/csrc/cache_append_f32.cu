// Appending to paged pools, fp32 sources.
#include "cache_append.cuh"

namespace imba {
template imba_status_t launch_append<float>(const imba_cache_desc&, const imba_pool_desc&, const imba_append_desc&, void*,
                                           cudaStream_t, int64_t, int64_t);
}
