// Appending to paged pools, bf16 sources.
#include "cache_append.cuh"

namespace imba {
template imba_status_t launch_append<bf16>(const imba_cache_desc&, const imba_pool_desc&, const imba_append_desc&, void*,
                                          cudaStream_t, int64_t, int64_t);
}
