// Kernel of tiles, keys of 2 bits.
#include "paged_tiles.cuh"

namespace kvq {
int paged_tiles_2(const PagedArgs &p, int max_tiles, cudaStream_t st) {
    return launch_tiles<2>(p, max_tiles, p.a.softcap > 0.f || p.a.slopes || !(p.a.softmax_scale > 0.f), st);
}
}  // namespace kvq
