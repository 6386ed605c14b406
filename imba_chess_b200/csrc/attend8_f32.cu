// Attention over a paged pool in 8 bits, fp32 queries.
#include "attend8_kernel.cuh"

namespace imba {
template cudaError_t launch_attend8<float>(const imba_cache_desc&, const AttendArgs&, cudaStream_t);
}
