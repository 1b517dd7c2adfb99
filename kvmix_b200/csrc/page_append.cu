// New tokens into their pages with the position rotation applied on the way, and their queries rotated beside them.
#include "pages.cuh"
#include "quant_core.cuh"

#include <cuda_bf16.h>

namespace kvq {

// A thread takes 16 channels of a (token, head) row -- eight and their eight partners, or 16 that are not rotated -- of one row after the other: queries, keys
// and values of its token, 32 rows of a CTA at a time, or those of several tokens where a token has fewer (AppendShape), so that no index takes a
// division.  The first rows are asked for before anything else; meanwhile a thread a token looks up where its keys go, a chain of four dependent loads.  Angles
// are read anew for every row, from L1: kept in registers they cost a CTA of four an SM.  Rows that are not 16-byte aligned (a slice of a fused projection at
// an odd offset) are read element by element and take twice as long (two prompts of 8k, cold: 209 us against 111); those instances of 2-byte types spill 112 to 136 bytes.  Bound: bytes in long calls (two prompts of 8k, 32 and 2 x 16 heads: 101 us,
// 5.4 TB/s; 118 with divisions and rows in fours), that chain in short ones (64 tokens: 4.9 us).
constexpr int kAppendThreads = 256, kAppendRows = kAppendThreads / 8;      // eight threads a row
constexpr int kAppendTokens = 128;                                         // of a CTA

// rows: of a token at a time, a power of two; turns: for all its rows; passes: times that many tokens
struct AppendShape { int rows_log2, turns, passes; };

template <typename T> struct Sixteen { uint4 v[sizeof(T) * 16 / 16]; };    // two runs of eight channels

template <typename T, bool VEC>
__device__ __forceinline__ void load8(uint4 *to, const T *from) {
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) to[i] = reinterpret_cast<const uint4 *>(from)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) reinterpret_cast<T *>(to)[i] = from[i];
    }
}
template <typename T> __device__ __forceinline__ float number(T x);
template <> __device__ __forceinline__ float number(float x) { return x; }
template <> __device__ __forceinline__ float number(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float number(__nv_bfloat16 x) { return __bfloat162float(x); }

template <bool VEC>
__device__ __forceinline__ void store8(__half *to, const float *x) {
    alignas(16) __half2 y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    if constexpr (VEC) {
        *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(y);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) to[i] = reinterpret_cast<const __half *>(y)[i];
    }
}
template <bool VEC>
__device__ __forceinline__ void angles8(float *to, const float *from) {
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < 2; ++i) reinterpret_cast<float4 *>(to)[i] = reinterpret_cast<const float4 *>(from)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) to[i] = from[i];
    }
}

template <typename T, bool VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kAppendThreads, sizeof(T) == 4 ? 3 : 4) page_append_kernel(const kvq_page_book b, const kvq_page_layer l, const __grid_constant__ kvq_page_append_args a, const AppendShape shape) {
    constexpr int BATCH = 2;                                      // rows under way
    __shared__ int s_page[kAppendTokens], s_slot[kAppendTokens], s_angle[kAppendTokens];
    __shared__ int s_start[1025];
    if (refused(b)) return;
    const int heads = a.nh + 2 * l.Hkv, tid = threadIdx.x, i = tid & 7, slot = tid >> 3, rows = 1 << shape.rows_log2, tokens_at_once = kAppendRows >> shape.rows_log2;
    const int of_pass = slot >> shape.rows_log2, row0 = slot & (rows - 1), token0 = blockIdx.x * tokens_at_once * shape.passes;
    // this thread's channels: `lo` and seven more, `hi` and seven more; rotated by angles `angle` and seven more, or not (-1)
    const int size = kHeadDim / a.parts, part = i / (8 / a.parts), c = i % (8 / a.parts);
    int lo, hi, angle = -1;
    if (INTERLEAVED) {
        lo = 16 * i;
        hi = lo + 8;
        if (16 * c < 2 * a.angles) angle = 8 * c;
    } else if (8 * c < a.angles) {
        lo = part * size + 8 * c;
        hi = lo + a.angles;
        angle = 8 * c;
    } else {
        lo = part * size + 16 * c;                                // 2 angles + 16 (c - angles / 8)
        hi = lo + 8;
    }
    alignas(16) Sixteen<T> x[BATCH];
    const int steps = shape.turns * shape.passes;
    struct Place { int pass, row; };                              // of a step
    auto next = [&](Place &at) {
        at.row += rows;
        if (at.row >= shape.turns << shape.rows_log2) {
            at.row = row0;
            ++at.pass;
        }
    };
    auto load = [&](Sixteen<T> &to, Place at, int token) {
        const T *from = at.row < a.nh ? static_cast<const T *>(a.q) + token * a.q_sT + at.row * a.q_sH
                        : at.row < a.nh + l.Hkv ? static_cast<const T *>(a.k) + token * a.k_sT + (at.row - a.nh) * a.k_sH
                                                : static_cast<const T *>(a.v) + token * a.v_sT + (at.row - a.nh - l.Hkv) * a.v_sH;
        load8<T, VEC>(to.v, from + lo);
        load8<T, VEC>(to.v + sizeof(T) / 2, from + hi);
    };
    auto token_of = [&](int pass) { return token0 + pass * tokens_at_once + of_pass; };
    Place at = {0, row0};
    auto load_batch = [&](int s) {
        Place p = at;
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const int token = token_of(p.pass);
            if (s + k < steps && token < a.tokens && p.row < heads) load(x[k], p, token);
            next(p);
        }
    };
    load_batch(0);
    const bool few = a.n <= 1024;
    if (few) {
        for (int k = tid; k <= a.n; k += kAppendThreads) s_start[k] = a.q_start[k];
        __syncthreads();
    }
    const int32_t *start = few ? s_start : a.q_start;
    if (tid < min(tokens_at_once * shape.passes, a.tokens - token0)) {
        const int u = token0 + tid;
        int page = -1, place = 0, angle_row = -1;
        if (u >= start[0] && u < start[a.n]) {
            const int s = sequence_of(start, a.n, u), row = a.rows[s];
            if (row >= 0 && row < b.slots) {
                const int pos = length_of(b, row) - max(start[s + 1], 0) + u;
                angle_row = a.positions ? a.positions[u] : pos;
                if (angle_row < 0 || angle_row >= a.angle_rows) {
                    angle_row = -1;
                    atomicOr(&b.count[2], KVQ_PAGES_NO_ANGLE);
                } else {
                    const int j = pos / kPage, id = pos >= 0 && j < b.max_pages && j >= b.packed[row] ? b.table[(int64_t)row * b.max_pages + j] : -1;
                    place = pos % kPage;
                    if (inside(id, min(l.n_fp16, b.n_fp16)) && b.refs[b.n_packed + id] <= 1) page = id;
                    else atomicOr(&b.count[2], KVQ_PAGES_NOT_WRITTEN);                                // a page that others hold too stays as it is
                }
            }
        }
        s_page[tid] = page;
        s_slot[tid] = place;
        s_angle[tid] = angle_row;
    }
    __syncthreads();
    for (int s = 0; s < steps; s += BATCH) {
        if (s) load_batch(s);
#pragma unroll
        for (int k = 0; k < BATCH; ++k, next(at)) {
            const int token = token_of(at.pass);
            if (s + k >= steps || token >= a.tokens || at.row >= heads) continue;
            const int page = s_page[token - token0], angle_row = s_angle[token - token0];
            const bool query = at.row < a.nh, value = at.row >= a.nh + l.Hkv;
            if (angle_row < 0 || (!query && page < 0)) continue;
            float y[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] = number<T>(reinterpret_cast<const T *>(x[k].v)[e]);
            if (!value && angle >= 0) {
                float cs[8], sn[8];
                angles8<VEC>(cs, a.cos + angle_row * a.c_sT + angle);
                angles8<VEC>(sn, a.sin + angle_row * a.s_sT + angle);
#pragma unroll
                for (int e = 0; e < 8; e += 2) {                  // two pairs at a time
                    const int i0 = INTERLEAVED ? 2 * e : e, i1 = INTERLEAVED ? 2 * e + 2 : e + 1, j0 = INTERLEAVED ? 2 * e + 1 : 8 + e, j1 = INTERLEAVED ? 2 * e + 3 : 9 + e;
                    const unsigned long long u = f32x2(y[i0], y[i1]), w = f32x2(y[j0], y[j1]), c2 = f32x2(cs[e], cs[e + 1]), s2 = f32x2(sn[e], sn[e + 1]);
                    const float2 p = f32x2_split(fma_f32x2(u, c2, mul_f32x2(w, f32x2(-sn[e], -sn[e + 1])))), q = f32x2_split(fma_f32x2(w, c2, mul_f32x2(u, s2)));
                    y[i0] = p.x;
                    y[i1] = p.y;
                    y[j0] = q.x;
                    y[j1] = q.y;
                }
            }
            if (query) {
                __half *to = static_cast<__half *>(a.q_out) + token * a.o_sT + at.row * a.o_sH;
                store8<VEC>(to + lo, y);
                store8<VEC>(to + hi, y + 8);
            } else {
                const int h = at.row - a.nh - (value ? l.Hkv : 0);
                __half *to = static_cast<__half *>(value ? l.vfull : l.kfull) + (((int64_t)page * l.Hkv + h) * kPage + s_slot[token - token0]) * kHeadDim;
                store8<true>(to + lo, y);
                store8<true>(to + hi, y + 8);
            }
        }
    }
}

// As many rows of a token at a time as leave the fewest places empty (48 rows: three turns of 16 for two tokens at once).  Four tokens a place where that leaves
// eight CTAs an SM (the two prompts: 112 us with one, 101 with four, 108 with eight).
static AppendShape append_shape(int heads, int tokens) {
    AppendShape r = {5, (heads + 31) / 32, 1};
    for (int k = 4; k >= 1; --k)
        if ((heads + (1 << k) - 1 >> k) << k < r.turns << r.rows_log2) r = {k, heads + (1 << k) - 1 >> k, 1};
    while (r.passes < 4 && tokens / ((kAppendRows >> r.rows_log2) * r.passes * 2) >= 148 * 8 && (kAppendRows >> r.rows_log2) * r.passes * 2 <= kAppendTokens) r.passes *= 2;
    return r;
}

template <typename T>
static int launch_append(const kvq_page_book &b, const kvq_page_layer &l, const kvq_page_append_args &a, cudaStream_t st) {
    constexpr int E = 16 / sizeof(T);
    auto rows16 = [](const void *p, int64_t t, int64_t h, int e) { return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && t % e == 0 && h % e == 0); };
    const bool vec = rows16(a.k, a.k_sT, a.k_sH, E) && rows16(a.v, a.v_sT, a.v_sH, E) && rows16(a.q, a.q_sT, a.q_sH, E) && rows16(a.q_out, a.o_sT, a.o_sH, 8) &&
                     rows16(a.cos, a.c_sT, 0, 4) && rows16(a.sin, a.s_sT, 0, 4);
    const AppendShape shape = append_shape(a.nh + 2 * l.Hkv, a.tokens);
    const int each = (kAppendRows >> shape.rows_log2) * shape.passes, grid = (int)(((int64_t)a.tokens + each - 1) / each);
    if (vec) {
        if (a.interleaved) page_append_kernel<T, true, true><<<grid, kAppendThreads, 0, st>>>(b, l, a, shape);
        else page_append_kernel<T, true, false><<<grid, kAppendThreads, 0, st>>>(b, l, a, shape);
    } else {
        if (a.interleaved) page_append_kernel<T, false, true><<<grid, kAppendThreads, 0, st>>>(b, l, a, shape);
        else page_append_kernel<T, false, false><<<grid, kAppendThreads, 0, st>>>(b, l, a, shape);
    }
    return count_launch();
}

}  // namespace kvq

extern "C" int kvq_page_append(const kvq_page_book *b, const kvq_page_layer *l, const kvq_page_append_args *a, kvq_stream_t stream) {
    using namespace kvq;
    if (const int rc = check_book(b)) return rc;
    if (const int rc = check_layer(l)) return rc;
    if (!a) return KVQ_ERR_NULL;
    if (a->n < 0 || a->tokens < 0 || a->nh < 0 || a->angle_rows < 0 || a->angles <= 0) return KVQ_ERR_SHAPE;
    if ((a->parts != 1 && a->parts != 2) || a->angles % 8 || a->angles > 64 / a->parts || a->type < KVQ_F16 || a->type > KVQ_F32) return KVQ_ERR_UNSUPPORTED;
    if (a->nh > (1 << 20) || l->Hkv > (1 << 20)) return KVQ_ERR_UNSUPPORTED;
    if (a->n == 0 || a->tokens == 0) return KVQ_OK;
    if (!a->k || !a->v || !a->cos || !a->sin || !a->q_start || !a->rows || (a->nh && (!a->q || !a->q_out))) return KVQ_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(a->cos) % 4 || reinterpret_cast<uintptr_t>(a->sin) % 4) return KVQ_ERR_ALIGN;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (a->type == KVQ_F32) return launch_append<float>(*b, *l, *a, st);
    if (a->type == KVQ_BF16) return launch_append<__nv_bfloat16>(*b, *l, *a, st);
    return launch_append<__half>(*b, *l, *a, st);
}
