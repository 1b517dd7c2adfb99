// New tokens into their pages with the position rotation applied on the way, and their queries rotated beside them.
#include "pages.cuh"

#include <cuda_bf16.h>

namespace kvq {

// A thread takes 16 channels of a (token, head) row -- eight and their eight partners, or 16 that are not rotated -- of R rows, queries,
// keys and values behind one another, so that a CTA's rows are those of a few tokens in a run.  The rows are asked for first; meanwhile a thread a token
// looks up where its keys go, a chain of four dependent loads.  Bound: bytes in long calls, that chain in short ones.
constexpr int kAppendThreads = 256, kAppendRows = kAppendThreads / 8;      // eight threads a row

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

template <typename T, bool VEC, int R>
__global__ void __launch_bounds__(kAppendThreads) page_append_kernel(const kvq_page_book b, const kvq_page_layer l, const __grid_constant__ kvq_page_append_args a) {
    constexpr int kMost = kAppendRows * R + 1;                    // tokens that a CTA's rows can belong to
    __shared__ int s_page[kMost], s_slot[kMost], s_angle[kMost];
    __shared__ int s_start[1025];
    if (refused(b)) return;
    const int heads = a.nh + 2 * l.Hkv, tid = threadIdx.x, i = tid & 7;
    const int64_t row0 = (int64_t)blockIdx.x * (kAppendRows * R);
    const int token0 = (int)(row0 / heads), in_token = (int)(row0 - (int64_t)token0 * heads);
    // this thread's channels: `lo` and seven more, `hi` and seven more; rotated by angles `angle` and seven more, or not (-1)
    const int size = kHeadDim / a.parts, part = i / (8 / a.parts), c = i % (8 / a.parts);
    int lo, hi, angle = -1;
    if (a.interleaved) {
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
    alignas(16) Sixteen<T> x[R];
    int token[R], head[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int at = in_token + r * kAppendRows + (tid >> 3);
        token[r] = token0 + at / heads;
        head[r] = at % heads;
        if (token[r] >= a.tokens) continue;
        const T *from = head[r] < a.nh ? static_cast<const T *>(a.q) + token[r] * a.q_sT + head[r] * a.q_sH
                        : head[r] < a.nh + l.Hkv ? static_cast<const T *>(a.k) + token[r] * a.k_sT + (head[r] - a.nh) * a.k_sH
                                                 : static_cast<const T *>(a.v) + token[r] * a.v_sT + (head[r] - a.nh - l.Hkv) * a.v_sH;
        load8<T, VEC>(x[r].v, from + lo);
        load8<T, VEC>(x[r].v + sizeof(T) / 2, from + hi);
    }
    const bool few = a.n <= 1024;
    if (few) {
        for (int k = tid; k <= a.n; k += kAppendThreads) s_start[k] = a.q_start[k];
        __syncthreads();
    }
    const int32_t *start = few ? s_start : a.q_start;
    const int most = min((in_token + kAppendRows * R - 1) / heads + 1, a.tokens - token0);         // of the CTA's tokens
    for (int k = tid; k < most; k += kAppendThreads) {
        const int u = token0 + k;
        int page = -1, slot = 0, at = -1;
        if (u >= start[0] && u < start[a.n]) {
            const int s = sequence_of(start, a.n, u), row = a.rows[s];
            if (row >= 0 && row < b.slots) {
                const int pos = length_of(b, row) - max(start[s + 1], 0) + u;
                at = a.positions ? a.positions[u] : pos;
                if (at < 0 || at >= a.angle_rows) {
                    at = -1;
                    atomicOr(&b.count[2], KVQ_PAGES_NO_ANGLE);
                } else {
                    const int j = pos / kPage, id = pos >= 0 && j < b.max_pages && j >= b.packed[row] ? b.table[(int64_t)row * b.max_pages + j] : -1;
                    slot = pos % kPage;
                    if (inside(id, min(l.n_fp16, b.n_fp16)) && b.refs[b.n_packed + id] <= 1) page = id;
                    else atomicOr(&b.count[2], KVQ_PAGES_NOT_WRITTEN);                                // a page that others hold too stays as it is
                }
            }
        }
        s_page[k] = page;
        s_slot[k] = slot;
        s_angle[k] = at;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (token[r] >= a.tokens) continue;
        const int k = token[r] - token0, page = s_page[k], at = s_angle[k];
        const bool query = head[r] < a.nh, value = head[r] >= a.nh + l.Hkv;
        if (at < 0 || (!query && page < 0)) continue;
        float y[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) y[e] = number<T>(reinterpret_cast<const T *>(x[r].v)[e]);
        if (!value && angle >= 0) {
            float cs[8], sn[8];
            angles8<VEC>(cs, a.cos + at * a.c_sT + angle);
            angles8<VEC>(sn, a.sin + at * a.s_sT + angle);
            auto turn = [&](float &p, float &q, int e) {
                const float u = p, w = q;
                p = u * cs[e] - w * sn[e];
                q = w * cs[e] + u * sn[e];
            };
            if (a.interleaved) {
#pragma unroll
                for (int e = 0; e < 8; ++e) turn(y[2 * e], y[2 * e + 1], e);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) turn(y[e], y[8 + e], e);
            }
        }
        if (query) {
            __half *to = static_cast<__half *>(a.q_out) + token[r] * a.o_sT + head[r] * a.o_sH;
            store8<VEC>(to + lo, y);
            store8<VEC>(to + hi, y + 8);
        } else {
            const int h = head[r] - a.nh - (value ? l.Hkv : 0);
            __half *to = static_cast<__half *>(value ? l.vfull : l.kfull) + (((int64_t)page * l.Hkv + h) * kPage + s_slot[k]) * kHeadDim;
            store8<true>(to + lo, y);
            store8<true>(to + hi, y + 8);
        }
    }
}

template <typename T>
static int launch_append(const kvq_page_book &b, const kvq_page_layer &l, const kvq_page_append_args &a, cudaStream_t st) {
    constexpr int E = 16 / sizeof(T);
    auto rows16 = [](const void *p, int64_t t, int64_t h, int e) { return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && t % e == 0 && h % e == 0); };
    const bool vec = rows16(a.k, a.k_sT, a.k_sH, E) && rows16(a.v, a.v_sT, a.v_sH, E) && rows16(a.q, a.q_sT, a.q_sH, E) && rows16(a.q_out, a.o_sT, a.o_sH, 8) &&
                     rows16(a.cos, a.c_sT, 0, 4) && rows16(a.sin, a.s_sT, 0, 4);
    const int64_t rows = (int64_t)a.tokens * (a.nh + 2 * l.Hkv);
    auto ctas = [&](int r) { return (rows + kAppendRows * r - 1) / (kAppendRows * r); };
    // a row a thread while that leaves the GPU room
    const bool one = ctas(1) <= 148 * 8;
    const int64_t grid = ctas(one ? 1 : 4);
    if (grid > 2147483647LL) return KVQ_ERR_UNSUPPORTED;
    if (vec) {
        if (one) page_append_kernel<T, true, 1><<<(unsigned)grid, kAppendThreads, 0, st>>>(b, l, a);
        else page_append_kernel<T, true, 4><<<(unsigned)grid, kAppendThreads, 0, st>>>(b, l, a);
    } else {
        if (one) page_append_kernel<T, false, 1><<<(unsigned)grid, kAppendThreads, 0, st>>>(b, l, a);
        else page_append_kernel<T, false, 4><<<(unsigned)grid, kAppendThreads, 0, st>>>(b, l, a);
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
