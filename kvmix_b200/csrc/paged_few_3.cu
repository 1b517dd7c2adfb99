// Kernel of few query rows, keys of 3 bits.
#include "paged_few.cuh"

namespace kvq {
int paged_few_3(const PagedArgs &p, cudaStream_t st) { return launch_few<3>(p, st); }
}  // namespace kvq
