// Kernel of few query rows, differential attention, keys of 2 bits.
#include "paged_few.cuh"

namespace kvq {
int paged_diff_few_2(const PagedArgs &p, cudaStream_t st) { return launch_few<2, true>(p, st); }
}  // namespace kvq
