// What the two attention kernels of the paged cache share: which positions a query sees, how a raw score becomes the exponent of
// its weight, bounded waits for bulk copies, packed fields as fp16.
#pragma once
#include "attn_mma_common.cuh"
#include "pages.cuh"

namespace kvq {

constexpr float kLog2e = 1.4426950408889634f;

// Sequences with at most so many rows -- (query head of the kv head, new token) pairs -- go to the kernel of few rows, the others to the
// kernel of tiles.
constexpr int kFewRows = 8;

struct PagedArgs {
    kvq_page_book b;
    kvq_page_layer l;
    kvq_paged_attn_args a;
    int rep, k_groups, v_groups;      // query heads of a kv head; groups of a page's row
    int splits, few_rows;             // few_rows: sequences with at most so many rows are the other kernel's
    float cap_in;                     // softmax_scale / softcap
    int64_t part_rows;                // rows of a split's partial sums: those of q, or kFewRows of every (sequence, kv head)
    bool part_compact;                // the latter
    float *part_out;                  // [splits][part_rows][128], unnormalised
    float *part_ml;                   // [splits][part_rows][2]: the exponents' reference (log2), the weights' sum
};

// Sequence i as every thread sees it: its row of the table, length, packed pages, where its new tokens are.  Numbers that would lead
// outside anything are made harmless.
struct PagedSeq {
    int row, length, packed, q0, n_new, prefix;
    const int32_t *table;
};
__device__ __forceinline__ void new_tokens(const PagedArgs &p, int i, int &q0, int &n_new) {
    q0 = min(max(p.a.q_start[i], 0), p.a.tokens);
    n_new = min(max(p.a.q_start[i + 1], 0), p.a.tokens) - q0;
}
__device__ __forceinline__ PagedSeq paged_seq(const PagedArgs &p, int i) {
    PagedSeq s;
    s.row = p.a.rows[i];
    const bool ok = s.row >= 0 && s.row < p.b.slots;
    const int row = ok ? s.row : 0;
    s.length = ok ? min(max(p.b.length[row], 0), p.b.max_pages * kPage) : 0;
    s.packed = ok ? p.b.packed[row] : 0;
    s.table = p.b.table + (int64_t)row * p.b.max_pages;
    new_tokens(p, i, s.q0, s.n_new);
    s.prefix = p.a.prefix ? p.a.prefix[i] : 0;
    return s;
}
// [lo, hi) of the positions that new token u (of n_new) sees
__device__ __forceinline__ void paged_bounds(const PagedArgs &p, const PagedSeq &s, int u, int &pos, int &lo, int &hi) {
    pos = s.length - s.n_new + u;
    lo = p.a.first ? max(p.a.first[s.q0 + u], 0) : 0;
    if (p.a.window > 0) lo = max(lo, pos + 1 - p.a.window);
    hi = p.a.causal ? min(max(pos + 1, s.prefix), s.length) : s.length;
    if (pos < 0) hi = lo;                                         // more new tokens than the sequence has
}

// A CTA of the kernel of few rows: as many query rows as the columns of an MMA hold with all groups (keys twice, as hi and lo, in one or two
// sets of columns); CTAs of an SM.
struct FewShape { int rows, row_blocks, key_sets, ctas; };
inline FewShape few_shape(const kvq_page_layer &l, int rep, int max_new) {
    const int64_t most = (int64_t)max_new * rep;
    const int rows = most < kFewRows ? (int)most : kFewRows, ng = kHeadDim / l.group;
    FewShape f = {kFewRows, 1, 1, l.k_bits == 3 || l.v_bits == 3 ? 3 : 4};
    if (l.v_bits != 3) f.rows = 8 / ng;
    if (l.k_bits != 3) {
        if (rows <= 4 / ng) f.rows = 4 / ng;
        else { f.rows = 8 / ng; f.key_sets = 2; f.ctas = 3; }
    } else if (f.rows > rows) {
        f.rows = rows < 1 ? 1 : rows;
    }
    f.row_blocks = (rows + f.rows - 1) / f.rows;
    return f;
}

// 2^x for x <= some tens, one instruction; denormal results flush to zero.
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// cap * tanh(x), x = score / softcap.  Where |x| <= 0.75: tanh(x) / x as a polynomial in x * x, minimax in relative error (5.7e-7, by a Remez
// exchange), so that a score keeps its own precision under any cap; beyond: 1 - 2 / (exp(2 x) + 1), whose error of some 2^-23 is
// small against a tanh of 0.63 and more (of a score of 1 under a cap of 1e5 it would be 0.01).  A NaN stays one.
constexpr float kCapSmall = 0.75f;
__device__ __forceinline__ constexpr float cap_poly(int i) {
    constexpr float C[5] = {0.999999435f, -0.333282515f, 0.132589832f, -0.0500563026f, 0.0129296324f};
    return C[i];
}
__device__ __forceinline__ float cap_small(float x, float cap) {
    const float t = x * x;
    float r = cap_poly(4);
#pragma unroll
    for (int i = 3; i >= 0; --i) r = fmaf(r, t, cap_poly(i));
    return x * r * cap;
}
__device__ __forceinline__ float cap_score(float x, float cap) {
    const float large = cap - 2.f * cap * rcp_approx(exp2_approx(x * (2.f * kLog2e)) + 1.f);
    return fabsf(x) <= kCapSmall ? cap_small(x, cap) : large;
}

// ---------------------------------------------------------------------------------------------
// mbarriers.  A wait gives up after two seconds, sets a bit of the status and lets the kernel end.
__device__ __forceinline__ unsigned long long global_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ void mbar_init(uint32_t bar, int count) { asm volatile("mbarrier.init.shared.b64 [%0], %1;\n" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared.b64 _, [%0];\n" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok;
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, int32_t *status) {
    if (mbar_try(bar, parity)) return true;
    const unsigned long long end = global_ns() + 2000000000ull;
    do {
        for (int i = 0; i < 64; ++i)
            if (mbar_try(bar, parity)) return true;
    } while (global_ns() < end);
    atomicOr(status, KVQ_PAGES_STALLED);
    return false;
}
// 16-byte aligned both ways, a multiple of 16 bytes
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// Factor of a partial sum with reference m (log2) and weights' sum l under the common reference: 0 for one that saw nothing; NaN stays.
__device__ __forceinline__ float part_factor(float m, float l, float common) { return l == 0.f ? 0.f : m == -INFINITY ? 1.f : exp2_approx(m - common); }

}  // namespace kvq
