// Kernel of few query rows, keys of 4 bits.
#include "paged_few.cuh"

namespace kvq {
int paged_few_4(const PagedArgs &p, cudaStream_t st) { return launch_few<4>(p, st); }
}  // namespace kvq
