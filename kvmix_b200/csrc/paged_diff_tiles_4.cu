// Kernel of tiles, differential attention, keys of 4 bits.
#include "paged_tiles.cuh"

namespace kvq {
int paged_diff_tiles_4(const PagedArgs &p, int max_tiles, cudaStream_t st) {
    return launch_tiles<4, true>(p, max_tiles, p.a.softcap > 0.f || p.a.slopes || !(p.a.softmax_scale > 0.f), st);
}
}  // namespace kvq
