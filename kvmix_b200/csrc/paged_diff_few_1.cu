// Kernel of few query rows, differential attention, keys of 1 bit.
#include "paged_few.cuh"

namespace kvq {
int paged_diff_few_1(const PagedArgs &p, cudaStream_t st) { return launch_few<1, true>(p, st); }
}  // namespace kvq
