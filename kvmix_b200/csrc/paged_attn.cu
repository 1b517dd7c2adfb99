// kvq_paged_attn: checks, the plan of a call, its launches.
#include "paged_attn.cuh"

#include <cfloat>
#include <cmath>

namespace kvq {

int paged_few_1(const PagedArgs &p, cudaStream_t st);                            // paged_few_1.cu ..
int paged_few_2(const PagedArgs &p, cudaStream_t st);
int paged_few_3(const PagedArgs &p, cudaStream_t st);
int paged_few_4(const PagedArgs &p, cudaStream_t st);
int paged_tiles_1(const PagedArgs &p, int max_tiles, cudaStream_t st);           // paged_tiles_1.cu ..
int paged_tiles_2(const PagedArgs &p, int max_tiles, cudaStream_t st);
int paged_tiles_3(const PagedArgs &p, int max_tiles, cudaStream_t st);
int paged_tiles_4(const PagedArgs &p, int max_tiles, cudaStream_t st);

static int paged_few(const PagedArgs &p, cudaStream_t st) {
    switch (p.l.k_bits) {
        case 1: return paged_few_1(p, st);
        case 2: return paged_few_2(p, st);
        case 3: return paged_few_3(p, st);
        default: return paged_few_4(p, st);
    }
}
static int paged_tiles(const PagedArgs &p, int max_tiles, cudaStream_t st) {
    switch (p.l.k_bits) {
        case 1: return paged_tiles_1(p, max_tiles, st);
        case 2: return paged_tiles_2(p, max_tiles, st);
        case 3: return paged_tiles_3(p, max_tiles, st);
        default: return paged_tiles_4(p, max_tiles, st);
    }
}

// Partial sums of the splits -> outputs, in the splits' order: a row a warp.  `few`: rows of the kernel of few rows, kFewRows places for every (sequence,
// kv head); else rows of q, of which those that the kernel of tiles had are joined.
__global__ void __launch_bounds__(256) paged_merge_kernel(const __grid_constant__ PagedArgs p, int few) {
    const int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const int64_t step = p.part_rows;
    int64_t row;
    int u, h;
    if (few) {
        const int r = (int)(at % kFewRows), head = (int)(at / kFewRows % p.l.Hkv);
        const int64_t i = at / kFewRows / p.l.Hkv;
        if (i >= p.a.n) return;
        const PagedSeq s = paged_seq(p, (int)i);
        if (s.n_new * p.rep > kFewRows || r >= s.n_new * p.rep) return;
        u = s.q0 + r / p.rep;
        h = head * p.rep + r % p.rep;
        row = p.part_compact ? at : (int64_t)u * p.a.nh + h;
    } else {
        const int64_t q = at / p.a.nh;
        if (q >= p.a.tokens || q < p.a.q_start[0] || q >= p.a.q_start[p.a.n]) return;
        u = (int)q;
        h = (int)(at - q * p.a.nh);
        row = at;
        if (p.few_rows) {
            const PagedSeq s = paged_seq(p, sequence_of(p.a.q_start, p.a.n, u));
            if (s.n_new * p.rep <= p.few_rows) return;
        }
    }
    float m = -INFINITY, l = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = lane; i < p.splits; i += 32) m = fmaxf(m, p.part_ml[2 * (i * step + row)]);
    m = warp_max(m);
    for (int base = 0; base < p.splits; base += 8) {              // eight splits' loads under way at once: one by one each waits for L2
        float2 ml[8];
        float4 x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int64_t at_i = (int64_t)min(base + k, p.splits - 1) * step + row;
            ml[k] = *reinterpret_cast<const float2 *>(p.part_ml + 2 * at_i);
            x[k] = *reinterpret_cast<const float4 *>(p.part_out + at_i * 128 + 4 * lane);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float f = base + k < p.splits ? part_factor(ml[k].x, ml[k].y, m) : 0.f;
            if (f != 0.f) { l += f * ml[k].y; v.x += f * x[k].x; v.y += f * x[k].y; v.z += f * x[k].z; v.w += f * x[k].w; }
        }
    }
    __half *out = static_cast<__half *>(p.a.out) + (int64_t)u * p.a.o_sT + (int64_t)h * p.a.o_sH + 4 * lane;
    auto put = [&](int c, float x) { out[c] = __float2half_rn(l == 0.f ? 0.f : x / l); };
    put(0, v.x);
    put(1, v.y);
    put(2, v.z);
    put(3, v.w);
}

static int paged_merge(const PagedArgs &p, int few, cudaStream_t st) {
    const int64_t rows = few ? (int64_t)p.a.n * p.l.Hkv * kFewRows : (int64_t)p.a.tokens * p.a.nh, grid = (rows + 7) / 8;
    if (grid > 2147483647LL) return KVQ_ERR_UNSUPPORTED;
    paged_merge_kernel<<<(unsigned)grid, 256, 0, st>>>(p, few);
    return count_launch();
}

// How a call is cut.  Either kernel may cut the pages of a sequence into splits, whose partial sums meet in a second launch.
struct PagedPlan {
    bool few, tiles;                  // which kernels are launched
    int few_rows;                     // sequences with more rows are the kernel of tiles'
    int few_splits, tile_splits, max_tiles;
};

static PagedPlan paged_plan(const kvq_page_layer &l, int n, int tokens, int nh, int max_new, int max_tokens, int max_chunks) {
    PagedPlan r = {};
    const int rep = nh / l.Hkv;
    const int64_t most = (int64_t)max_new * rep;
    r.tiles = most > kFewRows;
    // every sequence has its max_new tokens, or it is the only one: nothing for the kernel of few rows in a call that needs the other
    r.few = rep <= kFewRows && (!r.tiles || (n > 1 && tokens < (int64_t)n * max_new));
    r.few_rows = r.few ? kFewRows : 0;
    const int pages = (max_tokens + kPage - 1) / kPage;
    // Kernel of few rows: the splits that take the fewest rounds of pages (four warps a CTA), over all waves of CTAs; a CTA's beginning and
    // end count two rounds, the launch that joins the splits another two.
    const FewShape f = few_shape(l, rep, max_new);
    const int64_t pairs = (int64_t)n * l.Hkv * f.row_blocks, slots = 148 * f.ctas;
    double best = 1e30;
    r.few_splits = 1;
    for (int s = 1; r.few && s <= 128 && (s == 1 || s <= pages / 2); ++s) {
        const double w = (double)(pairs * s) / slots, waves = w <= 1 ? 1 : w < 4 ? (double)((pairs * s + slots - 1) / slots) : w + 0.5;
        const int rounds = ((pages + s - 1) / s + 3) / 4;
        const double cost = waves * (rounds + 2) + (s > 1 ? 2 : 0);
        if (cost < best) { best = cost; r.few_splits = s; }
    }
    int64_t tiles = ((int64_t)tokens * rep) / 256 + (r.few && max_chunks < n ? max_chunks : n);     // without the other kernel every sequence is one of chunks
    if (n == 1) tiles = ((int64_t)tokens * rep + 255) / 256;
    r.max_tiles = (int)(tiles < INT32_MAX ? tiles : INT32_MAX);
    // Kernel of tiles: one CTA to an SM, a page a round (some 1.8 us); a CTA's beginning and end count four pages, joining the splits moves
    // their partial sums twice.  Only for a clear gain: max_tokens may be far from what a window or documents leave to see (two chunks of 701 over 8k
    // tokens in documents of 2731: 84 us whole, 103 and 33 to join in four splits).
    const int64_t ctas = tiles * l.Hkv;
    best = 1e30;
    r.tile_splits = 1;
    for (int s = 1; r.tiles && s <= 64 && (s == 1 || s <= pages / 4); ++s) {
        const int64_t waves = (ctas * s + 147) / 148;
        const double joined = s > 1 ? 1.5 + (double)s * tokens * nh * 1040 / 5e6 / 1.8 : 0;
        const double cost = (double)waves * ((pages + s - 1) / s + 4) + joined;
        if (cost < 0.85 * best) { best = cost; r.tile_splits = s; }
    }
    return r;
}

// Partial sums of the kernel of few rows lie by rows of q, and beside chunks by kFewRows places of every (sequence, kv head) where those are fewer: a place in
// every split for the rows of a chunk of 32768 tokens of 32 heads beside a token with 13 splits took 7 GB.
static bool few_compact(const PagedPlan &r, int n, int Hkv, int tokens, int nh) {
    return r.tiles && (int64_t)n * Hkv * kFewRows < (int64_t)tokens * nh;
}
static int64_t few_part_rows(const PagedPlan &r, int n, int Hkv, int tokens, int nh) {
    return few_compact(r, n, Hkv, tokens, nh) ? (int64_t)n * Hkv * kFewRows : (int64_t)tokens * nh;
}
// Both kernels' partial sums, one after the other in the same place; in whole splits of all rows of q, two at least.
static uint64_t paged_bytes(const PagedPlan &r, int n, int Hkv, int tokens, int nh) {
    const int64_t all = (int64_t)tokens * nh, few = r.few && r.few_splits > 1 ? r.few_splits * few_part_rows(r, n, Hkv, tokens, nh) : 0,
                  tiles = r.tiles && r.tile_splits > 1 ? r.tile_splits * all : 0, most = few > tiles ? few : tiles, units = (most + all - 1) / all;
    return (uint64_t)(most == 0 ? 0 : units < 2 ? 2 : units) * all * (kHeadDim + 2) * 4;
}

}  // namespace kvq

extern "C" uint64_t kvq_paged_attn_workspace_bytes(const kvq_page_layer *l, int32_t n, int32_t tokens, int32_t nh, int32_t max_new, int32_t max_tokens,
                                                   int32_t max_chunks) {
    using namespace kvq;
    if (check_layer(l) || n <= 0 || tokens <= 0 || nh <= 0 || nh % l->Hkv || max_new <= 0 || max_tokens <= 0 || max_chunks < 0) return 0;
    return paged_bytes(paged_plan(*l, n, tokens, nh, max_new, max_tokens, max_chunks), n, l->Hkv, tokens, nh);
}

extern "C" int kvq_paged_attn(const kvq_page_book *b, const kvq_page_layer *l, const kvq_paged_attn_args *a, kvq_stream_t stream) {
    using namespace kvq;
    if (const int rc = check_book(b)) return rc;
    if (const int rc = check_layer(l)) return rc;
    if (!a) return KVQ_ERR_NULL;
    if (a->n < 0 || a->tokens < 0 || a->nh <= 0 || a->window < 0) return KVQ_ERR_SHAPE;
    if (a->nh % l->Hkv) return KVQ_ERR_HEADS;
    if (a->n == 0 || a->tokens == 0) return KVQ_OK;
    if (a->max_new <= 0 || a->max_tokens <= 0 || a->max_chunks < 0) return KVQ_ERR_SHAPE;
    if (!a->q || !a->out || !a->q_start || !a->rows) return KVQ_ERR_NULL;
    if (!(a->softcap >= 0.f) || !(fabsf(a->softmax_scale) <= FLT_MAX)) return KVQ_ERR_SHAPE;
    const PagedPlan r = paged_plan(*l, a->n, a->tokens, a->nh, a->max_new, a->max_tokens, a->max_chunks);
    const uint64_t need = paged_bytes(r, a->n, l->Hkv, a->tokens, a->nh);
    if (need && (!a->workspace || a->workspace_bytes < need)) return KVQ_ERR_WORKSPACE;
    if (need && reinterpret_cast<uintptr_t>(a->workspace) % 16) return KVQ_ERR_ALIGN;
    PagedArgs p = {};
    p.b = *b;
    p.l = *l;
    p.a = *a;
    p.rep = a->nh / l->Hkv;
    p.k_groups = page_groups(l->k_bits, l->group);
    p.v_groups = page_groups(l->v_bits, l->group);
    p.few_rows = r.few_rows;
    // A cap that no score comes near is none (its square is beyond 1 / fp32's rounding for every score up to 1e26), and one below 1e-30 leaves nothing of
    // them; what is between keeps products and quotients of caps and scales in fp32's range.
    if (p.a.softcap >= 1e30f) p.a.softcap = 0.f;
    if (p.a.softcap > 0.f) {
        p.a.softcap = fmaxf(p.a.softcap, 1e-30f);
        p.cap_in = fminf(fmaxf(a->softmax_scale / p.a.softcap, -1e30f), 1e30f);
    }
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    p.part_out = static_cast<float *>(a->workspace);
    if (r.few) {
        p.splits = r.few_splits;
        p.part_rows = few_part_rows(r, a->n, l->Hkv, a->tokens, a->nh);
        p.part_compact = few_compact(r, a->n, l->Hkv, a->tokens, a->nh);
        p.part_ml = p.part_out + p.splits * p.part_rows * kHeadDim;
        if (const int rc = paged_few(p, st)) return rc;
        if (p.splits > 1)
            if (const int rc = paged_merge(p, 1, st)) return rc;
    }
    if (r.tiles) {
        p.splits = r.tile_splits;
        p.part_rows = (int64_t)a->tokens * a->nh;
        p.part_ml = p.part_out + p.splits * p.part_rows * kHeadDim;
        if (const int rc = paged_tiles(p, r.max_tiles, st)) return rc;
        if (p.splits > 1)
            if (const int rc = paged_merge(p, 0, st)) return rc;
    }
    return KVQ_OK;
}
