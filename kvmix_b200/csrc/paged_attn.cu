// kvq_paged_attn and kvq_paged_diff_attn: checks, the plan of a call, its launches.
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
int paged_diff_few_1(const PagedArgs &p, cudaStream_t st);                       // paged_diff_few_1.cu ..
int paged_diff_few_2(const PagedArgs &p, cudaStream_t st);
int paged_diff_few_3(const PagedArgs &p, cudaStream_t st);
int paged_diff_few_4(const PagedArgs &p, cudaStream_t st);
int paged_diff_tiles_1(const PagedArgs &p, int max_tiles, cudaStream_t st);      // paged_diff_tiles_1.cu ..
int paged_diff_tiles_2(const PagedArgs &p, int max_tiles, cudaStream_t st);
int paged_diff_tiles_3(const PagedArgs &p, int max_tiles, cudaStream_t st);
int paged_diff_tiles_4(const PagedArgs &p, int max_tiles, cudaStream_t st);

static int paged_few(const PagedArgs &p, cudaStream_t st) {
    if (p.lambdas) {
        switch (p.l.k_bits) {
            case 1: return paged_diff_few_1(p, st);
            case 2: return paged_diff_few_2(p, st);
            case 3: return paged_diff_few_3(p, st);
            default: return paged_diff_few_4(p, st);
        }
    }
    switch (p.l.k_bits) {
        case 1: return paged_few_1(p, st);
        case 2: return paged_few_2(p, st);
        case 3: return paged_few_3(p, st);
        default: return paged_few_4(p, st);
    }
}
static int paged_tiles(const PagedArgs &p, int max_tiles, cudaStream_t st) {
    if (p.lambdas) {
        switch (p.l.k_bits) {
            case 1: return paged_diff_tiles_1(p, max_tiles, st);
            case 2: return paged_diff_tiles_2(p, max_tiles, st);
            case 3: return paged_diff_tiles_3(p, max_tiles, st);
            default: return paged_diff_tiles_4(p, max_tiles, st);
        }
    }
    switch (p.l.k_bits) {
        case 1: return paged_tiles_1(p, max_tiles, st);
        case 2: return paged_tiles_2(p, max_tiles, st);
        case 3: return paged_tiles_3(p, max_tiles, st);
        default: return paged_tiles_4(p, max_tiles, st);
    }
}

// Partial sums of the splits -> outputs, in the splits' order: a row a warp, or a head's two rows.  `few`: rows of the kernel of few rows, kFewRows places
// for every (sequence, kv head); else, where some tiles are cut alone, the rows of their CTAs; else rows of q, of which those that the kernel of tiles had are joined.
template <bool DIFF>
__global__ void __launch_bounds__(256) paged_merge_kernel(const __grid_constant__ PagedArgs p, int few) {
    const int64_t at = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * (DIFF ? 2 : 1);
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
    } else if (DIFF && p.n_whole > 0) {
        const int hs = p.n_whole + (int)(at >> 8), head = hs % p.l.Hkv;
        int tile = p.max_tiles - 1 - hs / p.l.Hkv, i = 0, q0 = 0, n_new = 0;         // as the kernel of tiles counts them
        for (; i < p.a.n; ++i) {
            new_tokens(p, i, q0, n_new);
            const int rows = max(0, n_new) * p.rep, tiles = rows > p.few_rows ? (rows + 255) / 256 : 0;
            if (tile < tiles) break;
            tile -= tiles;
        }
        const int r = tile * 256 + (int)(at & 255);
        if (i == p.a.n || tile < 0 || r >= n_new * p.rep) return;
        u = q0 + r / p.rep;
        h = head * p.rep + r % p.rep;
        row = at;
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
    auto join = [&](int64_t row, float &l) {
        float m = -INFINITY;
        l = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i = lane; i < p.splits; i += 32) m = fmaxf(m, p.part_ml[2 * (i * step + row)]);
        m = warp_max(m);
        for (int base = 0; base < p.splits; base += 8) {          // eight splits' loads under way at once: one by one each waits for L2
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
        return v;
    };
    float l;
    float4 v = join(row, l);
    if constexpr (DIFF) {
        float l2;
        float4 w = join(row + 1, l2);
        h >>= 1;
        const float lambda = p.lambdas[h];
        auto one = [&](float a, float b) { return diff_of(l == 0.f ? 0.f : a / l, l2 == 0.f ? 0.f : b / l2, lambda); };
        v = make_float4(one(v.x, w.x), one(v.y, w.y), one(v.z, w.z), one(v.w, w.w));
        if (p.norm_weight) {
            const float by = diff_norm(p, warp_sum(v.x * v.x + v.y * v.y + (v.z * v.z + v.w * v.w)));
            const float *weight = p.norm_weight + 4 * lane;
            v = make_float4(v.x * (by * weight[0]), v.y * (by * weight[1]), v.z * (by * weight[2]), v.w * (by * weight[3]));
        }
        l = 1.f;
    }
    __half *out = static_cast<__half *>(p.a.out) + (int64_t)u * p.a.o_sT + (int64_t)h * p.a.o_sH + 4 * lane;
    auto put = [&](int c, float x) { out[c] = __float2half_rn(l == 0.f ? 0.f : x / l); };
    put(0, v.x);
    put(1, v.y);
    put(2, v.z);
    put(3, v.w);
}

static int paged_merge(const PagedArgs &p, int few, cudaStream_t st) {
    const int64_t rows = few ? (int64_t)p.a.n * p.l.Hkv * kFewRows : p.part_rows, grid = (rows + 7) / 8;
    if (grid > 2147483647LL) return KVQ_ERR_UNSUPPORTED;
    if (p.lambdas) paged_merge_kernel<true><<<(unsigned)((grid + 1) / 2), 256, 0, st>>>(p, few);
    else paged_merge_kernel<false><<<(unsigned)grid, 256, 0, st>>>(p, few);
    return count_launch();
}

// How a call is cut.  Either kernel may cut the pages of a sequence into splits, whose partial sums meet in a second launch.
struct PagedPlan {
    bool few, tiles;                  // which kernels are launched
    int few_rows;                     // sequences with more rows are the kernel of tiles'
    int few_splits, tile_splits, max_tiles;
    FewShape shape;                   // of the kernel of few rows, differential attention
    int n_whole;                      // tiles that are not cut beside others that are (PagedArgs), differential attention
};

// Bytes of `rows` partial sums: whole splits of all rows of q are asked for, two at least.
static uint64_t part_bytes(int64_t rows, int64_t all) {
    const int64_t units = (rows + all - 1) / all;
    return (uint64_t)(rows == 0 ? 0 : units < 2 ? 2 : units) * all * (kHeadDim + 2) * 4;
}
constexpr uint64_t kMostCutBytes = 1 << 29;

static PagedPlan paged_plan(const kvq_page_layer &l, int n, int tokens, int nh, int max_new, int max_tokens, int max_chunks, bool diff) {
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
    auto splits = [&](const FewShape &f, double round, double &least) {
        const int64_t pairs = (int64_t)n * l.Hkv * f.row_blocks, slots = 148 * f.ctas;
        int r = 1;
        least = 1e30;
        for (int s = 1; s <= 128 && (s == 1 || s <= pages / 2); ++s) {
            const double w = (double)(pairs * s) / slots, waves = w <= 1 ? 1 : w < 4 ? (double)((pairs * s + slots - 1) / slots) : w + 0.5;
            const int rounds = ((pages + s - 1) / s + 3) / 4;
            const double cost = waves * (rounds * round + 2) + (s > 1 ? 2 : 0);
            if (cost < least) { least = cost; r = s; }
        }
        return r;
    };
    double best;
    r.few_splits = 1;
    if (r.few && !diff) r.few_splits = splits(few_shape(l, rep, max_new), 1, best);
    // Differential attention: fewer rows to a CTA while that leaves SMs to do them (one token over 777 tokens, 8 heads of 4: 18 us by two rows, 37 by eight), else as
    // many as the columns hold, what a page costs beside its rows being as much as five rows.
    double least = 1e30;
    for (int most = 2; r.few && diff && most <= kFewRows; most *= 2) {
        const FewShape f = diff_shape(l, rep, max_new, most);
        const int s = splits(f, 0.7 * (1 + f.rows / 5.0), best);
        if (best < 0.97 * least) { least = best; r.few_splits = s; r.shape = f; }
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
    // Differential attention: what is left of a last round of CTAs may be cut alone, where tiles are alike because what is new is little (a chunk of 2048 over
    // 32k tokens, 512 tiles of 148 at a time: 2021 us whole, 1777 with the last 68 halved), unless the sums take more than kMostCutBytes: calls of many rounds
    // gain the least.
    if (diff && r.tiles && r.tile_splits == 1 && n <= kMostCutSequences && ctas > 148 && ctas < INT32_MAX && (int64_t)max_new * 4 <= max_tokens) {
        const int rest = (int)(ctas % 148);
        double least = 0.96 * (double)((ctas + 147) / 148);
        for (int s = 2; rest && s <= 8 && s <= pages / 4; ++s) {
            if (part_bytes((int64_t)s * rest * 256, (int64_t)tokens * nh) > kMostCutBytes) break;
            const double cost = (double)(ctas / 148) + (double)((rest * s + 147) / 148) * (pages / (double)s + 4) / (pages + 4) + (1.5 + (double)s * rest * 256 * 1040 / 5e6 / 1.8) / (pages + 4);
            if (cost < least) { least = cost; r.tile_splits = s; r.n_whole = (int)ctas - rest; }
        }
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
// Rows of a split of the kernel of tiles: where only some tiles are cut, those of their CTAs in the order of CTAs, else those of q.
static int64_t tile_part_rows(const PagedPlan &r, int Hkv, int tokens, int nh) {
    return r.n_whole > 0 ? ((int64_t)r.max_tiles * Hkv - r.n_whole) * 256 : (int64_t)tokens * nh;
}
// Both kernels' partial sums, one after the other in the same place.
static uint64_t paged_bytes(const PagedPlan &r, int n, int Hkv, int tokens, int nh) {
    const int64_t few = r.few && r.few_splits > 1 ? r.few_splits * few_part_rows(r, n, Hkv, tokens, nh) : 0,
                  tiles = r.tiles && r.tile_splits > 1 ? r.tile_splits * tile_part_rows(r, Hkv, tokens, nh) : 0;
    return part_bytes(few > tiles ? few : tiles, (int64_t)tokens * nh);
}

}  // namespace kvq

extern "C" uint64_t kvq_paged_attn_workspace_bytes(const kvq_page_layer *l, int32_t n, int32_t tokens, int32_t nh, int32_t max_new, int32_t max_tokens,
                                                   int32_t max_chunks) {
    using namespace kvq;
    if (check_layer(l) || n <= 0 || tokens <= 0 || nh <= 0 || nh % l->Hkv || max_new <= 0 || max_tokens <= 0 || max_chunks < 0) return 0;
    return paged_bytes(paged_plan(*l, n, tokens, nh, max_new, max_tokens, max_chunks, false), n, l->Hkv, tokens, nh);
}

extern "C" uint64_t kvq_paged_diff_attn_workspace_bytes(const kvq_page_layer *l, int32_t n, int32_t tokens, int32_t nh, int32_t max_new, int32_t max_tokens,
                                                        int32_t max_chunks) {
    using namespace kvq;
    if (check_layer(l) || n <= 0 || tokens <= 0 || nh <= 0 || nh > INT32_MAX / 2 || nh % l->Hkv || max_new <= 0 || max_tokens <= 0 || max_chunks < 0) return 0;
    return paged_bytes(paged_plan(*l, n, tokens, 2 * nh, max_new, max_tokens, max_chunks, true), n, l->Hkv, tokens, 2 * nh);
}

namespace kvq {

// a->nh counts heads; two rows each where `diff` is given
static int attend(const kvq_page_book *b, const kvq_page_layer *l, const kvq_paged_attn_args *a, const kvq_paged_diff_args *diff, kvq_stream_t stream) {
    if (const int rc = check_book(b)) return rc;
    if (const int rc = check_layer(l)) return rc;
    if (!a) return KVQ_ERR_NULL;
    if (a->n < 0 || a->tokens < 0 || a->nh <= 0 || a->window < 0) return KVQ_ERR_SHAPE;
    if (a->nh % l->Hkv) return KVQ_ERR_HEADS;
    if (diff && a->nh > INT32_MAX / 2) return KVQ_ERR_UNSUPPORTED;
    const int nh = diff ? 2 * a->nh : a->nh;
    if (a->n == 0 || a->tokens == 0) return KVQ_OK;
    if (a->max_new <= 0 || a->max_tokens <= 0 || a->max_chunks < 0) return KVQ_ERR_SHAPE;
    if (!a->q || !a->out || !a->q_start || !a->rows) return KVQ_ERR_NULL;
    if (!(a->softcap >= 0.f) || !(fabsf(a->softmax_scale) <= FLT_MAX)) return KVQ_ERR_SHAPE;
    const PagedPlan r = paged_plan(*l, a->n, a->tokens, nh, a->max_new, a->max_tokens, a->max_chunks, diff);
    const uint64_t need = paged_bytes(r, a->n, l->Hkv, a->tokens, nh);
    if (need && (!a->workspace || a->workspace_bytes < need)) return KVQ_ERR_WORKSPACE;
    if (need && reinterpret_cast<uintptr_t>(a->workspace) % 16) return KVQ_ERR_ALIGN;
    PagedArgs p = {};
    p.b = *b;
    p.l = *l;
    p.a = *a;
    p.a.nh = nh;
    p.rep = nh / l->Hkv;
    if (diff) {
        p.lambdas = diff->lambdas;
        p.norm_weight = diff->norm_weight;
        p.norm_eps = diff->norm_eps;
        p.few_shape = r.shape;
    }
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
        p.part_rows = few_part_rows(r, a->n, l->Hkv, a->tokens, nh);
        p.part_compact = few_compact(r, a->n, l->Hkv, a->tokens, nh);
        p.part_ml = p.part_out + p.splits * p.part_rows * kHeadDim;
        if (const int rc = paged_few(p, st)) return rc;
        if (p.splits > 1)
            if (const int rc = paged_merge(p, 1, st)) return rc;
    }
    if (r.tiles) {
        p.splits = r.tile_splits;
        p.max_tiles = r.max_tiles;
        p.n_whole = r.n_whole;
        p.part_rows = tile_part_rows(r, l->Hkv, a->tokens, nh);
        p.part_ml = p.part_out + p.splits * p.part_rows * kHeadDim;
        if (const int rc = paged_tiles(p, r.max_tiles, st)) return rc;
        if (p.splits > 1)
            if (const int rc = paged_merge(p, 0, st)) return rc;
    }
    return KVQ_OK;
}

}  // namespace kvq

extern "C" int kvq_paged_attn(const kvq_page_book *b, const kvq_page_layer *l, const kvq_paged_attn_args *a, kvq_stream_t stream) {
    return kvq::attend(b, l, a, nullptr, stream);
}

extern "C" int kvq_paged_diff_attn(const kvq_page_book *b, const kvq_page_layer *l, const kvq_paged_diff_args *a, kvq_stream_t stream) {
    using namespace kvq;
    if (!a) return KVQ_ERR_NULL;
    if (a->a.n > 0 && a->a.tokens > 0 && !a->lambdas) return KVQ_ERR_NULL;
    if (a->norm_weight && !(a->norm_eps >= 0.f && a->norm_eps <= FLT_MAX)) return KVQ_ERR_SHAPE;
    return attend(b, l, &a->a, a, stream);
}
