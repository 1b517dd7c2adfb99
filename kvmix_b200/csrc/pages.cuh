// What the kernels of the paged cache share: the geometry of a page and a look at its bookkeeping.
#pragma once
#include "common.cuh"

namespace kvq {

constexpr int kPage = KVQ_PAGE_TOKENS;
constexpr int kPageHalf = kPage * kHeadDim;                       // elements of one head's keys (or values) of a page

int count_launch();                                               // check_launch() of a kernel of the paged cache (api.cu)

__host__ __device__ constexpr int page_words(int bits) { return bits == 3 ? 12 : 4 * bits; }               // per 128 elements
__host__ __device__ constexpr int page_groups(int bits, int group) { return bits == 3 ? 12 : 128 / group; }

__device__ __forceinline__ int pages_of(int tokens) { return (tokens + kPage - 1) / kPage; }

// Whether a call had to be refused: none changes the cache then.  A wait of the attention that gave up, and tokens that page_write left out, concern
// their own call alone; were the writes behind it left out, tokens that are counted already would be missing in later layers.
__device__ __forceinline__ bool refused(const kvq_page_book &b) { return b.count[2] & ~(KVQ_PAGES_STALLED | KVQ_PAGES_NOT_WRITTEN); }

// Every size that a kernel's index arithmetic relies on.
inline int check_book(const kvq_page_book *b) {
    if (!b || !b->table || !b->length || !b->packed || !b->refs || !b->free_ids || !b->count) return KVQ_ERR_NULL;
    if (b->slots <= 0 || b->max_pages <= 0 || b->max_pages > (1 << 23) || b->n_packed < 0 || b->n_fp16 < 0) return KVQ_ERR_SHAPE;
    if ((int64_t)b->n_packed + b->n_fp16 > (1 << 30)) return KVQ_ERR_SHAPE;
    if (b->slots > 1 << 20) return KVQ_ERR_UNSUPPORTED;           // a bit each in shared memory
    return KVQ_OK;
}
inline int check_layer(const kvq_page_layer *l) {
    if (!l) return KVQ_ERR_NULL;
    if (l->Hkv <= 0 || l->n_packed < 0 || l->n_fp16 < 0) return KVQ_ERR_SHAPE;
    if (l->k_bits < 1 || l->k_bits > 4 || l->v_bits < 1 || l->v_bits > 4) return KVQ_ERR_BITS;
    if (l->group != 32 && l->group != 64 && l->group != 128) return KVQ_ERR_UNSUPPORTED;
    if (l->n_packed && (!l->kcode || !l->kscale || !l->kmn || !l->vcode || !l->vscale || !l->vmn)) return KVQ_ERR_NULL;
    if (l->n_fp16 && (!l->kfull || !l->vfull)) return KVQ_ERR_NULL;
    const void *all[] = {l->kcode, l->kscale, l->kmn, l->kfull, l->vcode, l->vscale, l->vmn, l->vfull};
    for (const void *p : all)
        if (reinterpret_cast<uintptr_t>(p) % 16) return KVQ_ERR_ALIGN;
    return KVQ_OK;
}

// The sequence whose new tokens hold token u: the last i with q_start[i] <= u (q_start ascends, q_start[0] <= u < q_start[n]).
__device__ __forceinline__ int sequence_of(const int32_t *q_start, int n, int u) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (q_start[mid] <= u) lo = mid;
        else hi = mid;
    }
    return lo;
}

}  // namespace kvq
