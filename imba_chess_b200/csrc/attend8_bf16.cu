// Attention over a paged pool in 8 bits, bf16 queries.
#include "attend8_kernel.cuh"

namespace imba {
template cudaError_t launch_attend8<bf16>(const imba_cache_desc&, const AttendArgs&, cudaStream_t);
}
