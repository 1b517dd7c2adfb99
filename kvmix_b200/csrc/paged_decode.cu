// Attention of few query rows of a kv head (a new token of a group of query heads) over a paged cache.
#include "paged_attn.cuh"

namespace kvq {

// A CTA of four warps takes one (sequence, kv head, split of its pages); a warp takes every fourth page by itself -- scores, online
// softmax, values -- so nothing in the loop waits for another warp.
//   scores   S[token][row] = K[token][channel] q[row][channel]: mma m16n8k16 with 16 tokens as rows and up to eight query rows as
//            columns
//   values   O[channel][row] = V^T[channel][token] p[row][token]: the same with 16 channels as rows
// In both the packed axis runs along the MMA's rows and the contraction across words, so that the two elements of an operand register
// come from the same place of two words.  Words arrive by bulk copies, 32 contraction rows (codes, scales, minima) a stage, in the warp's own ring; fp16
// pages go straight to registers.
constexpr int kFewWarps = 4;
constexpr int kStageRows = 32;
constexpr int kMaxStages = 8;
constexpr int kPStride = 136;                                     // halves between rows of weights: 2-way conflicts at most

template <int BITS> struct FewGeom {
    static constexpr int W = page_words(BITS);
    static constexpr int TILES = BITS == 3 ? 11 : 8;              // accumulator tiles of 128 packed elements
};

// Which of a page's 128 elements accumulator (tile m, half e) of lane group g stands for: element 16g + f(2m + e) where a lane group owns 16
// neighbours, in the order that puts the four a lane needs for a k-step side by side; 3 bits: field m of word g + 8e (none beyond the end).
template <int BITS> __device__ __forceinline__ int few_element(int g, int m, int e) {
    if constexpr (BITS == 3) {
        const int w = g + 8 * e, i = 11 * w + m;
        return w < 12 && i < kPage ? i : -1;
    } else {
        const int s = 2 * m + e;
        return 16 * g + (s & 3) * 4 + (s >> 2);
    }
}

// acc[tile] += A(16 contraction rows starting at `row` of the stage) * B.  Contraction rows of lane t: row + t + 4j.
template <int BITS>
__device__ __forceinline__ void few_packed_step(float (&acc)[FewGeom<BITS>::TILES][4], uint32_t codes, uint32_t scale, uint32_t mn, int groups, int g_log2,
                                                int row, int g, int t, uint32_t b0, uint32_t b1) {
    constexpr int W = FewGeom<BITS>::W;
    if constexpr (BITS == 3) {
        uint32_t w[2][4];
        __half2 sc[2][2], lo[2][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int word = min(g + 8 * e, 11);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[e][j] = lds32(codes + ((row + t + 4 * j) * W + word) * 4);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r0 = ((row + t + 8 * j) * 12 + word) * 2, r1 = r0 + 4 * 12 * 2;
                sc[e][j] = as_h2(lds16(scale + r0) | lds16(scale + r1) << 16);
                lo[e][j] = as_h2(lds16(mn + r0) | lds16(mn + r1) << 16);
            }
        }
#pragma unroll
        for (int m = 0; m < 11; ++m) {
            uint32_t a[4];
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t x = (m < 10 ? (w[e][2 * j] >> (3 * m)) & 7u : w[e][2 * j] >> 30) | ((m < 10 ? (w[e][2 * j + 1] >> (3 * m)) & 7u : w[e][2 * j + 1] >> 30) << 16);
                    a[e + 2 * j] = as_u32(__hfma2(__hsub2(as_h2(x | 0x64006400u), as_h2(0x64006400u)), sc[e][j], lo[e][j]));
                }
            mma16816(acc[m], a[0], a[1], a[2], a[3], b0, b1);
        }
    } else {
        using F = HalfFields<BITS>;
        const int grp = (16 * g) >> g_log2;
        __half2 sc[2], lo[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r0 = ((row + t + 8 * j) * groups + grp) * 2, r1 = r0 + 4 * groups * 2;
            sc[j] = as_h2(lds16(scale + r0) | lds16(scale + r1) << 16);
            lo[j] = as_h2(lds16(mn + r0) | lds16(mn + r1) << 16);
        }
        // the 16 elements of the lane group are BITS halves of words, x[h][j]: half h of rows t + 8j and t + 8j + 4
        uint32_t x[BITS][2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t at = codes + (row + t + 8 * j) * W * 4;
            if constexpr (BITS == 1) {
                x[0][j] = prmt(lds32(at + (g >> 1) * 4), lds32(at + 4 * W * 4 + (g >> 1) * 4), g & 1 ? 0x7632 : 0x5410);
            } else {
#pragma unroll
                for (int h = 0; h < BITS / 2; ++h) {
                    const uint32_t u = lds32(at + (g * (BITS / 2) + h) * 4), v = lds32(at + 4 * W * 4 + (g * (BITS / 2) + h) * 4);
                    x[2 * h][j] = prmt(u, v, 0x5410);
                    x[2 * h + 1][j] = prmt(u, v, 0x7632);
                }
            }
        }
#pragma unroll
        for (int m = 0; m < 8; ++m) {
            uint32_t a[4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int s = 2 * m + e, i = (s & 3) * 4 + (s >> 2);
#pragma unroll
                for (int j = 0; j < 2; ++j) a[e + 2 * j] = as_u32(__hfma2(F::code(x[i / F::N][j], i % F::N), sc[j], lo[j]));
            }
            mma16816(acc[m], a[0], a[1], a[2], a[3], b0, b1);
        }
    }
}

struct FewState {
    float m[2], l[2];                                             // of columns 2t, 2t + 1: reference (log2 units) and this lane's part of the sum
};

template <int KB, int VB>
__global__ void __launch_bounds__(kFewWarps * 32, KB == 3 || VB == 3 ? 3 : 4) paged_few_kernel(const __grid_constant__ PagedArgs p, int stages, int stage_bytes) {
    extern __shared__ __align__(128) char smem[];
    const int warp = uniform_warp(), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x % p.splits, hs = blockIdx.x / p.splits, head = hs % p.l.Hkv, i = hs / p.l.Hkv;
    const PagedSeq s = paged_seq(p, i);
    const int rows = s.n_new * p.rep;
    if (rows <= 0 || rows > kFewRows) return;

    // shared memory of the CTA: q rows, then per warp: weights, barriers, ring; the outputs meet in [warp][8][128] floats over the rings
    __half *s_q = reinterpret_cast<__half *>(smem);               // [8][128], rows beyond the last zero
    char *mine = smem + 2048 + warp * (kFewRows * kPStride * 2 + kMaxStages * 8 + stages * stage_bytes);
    const uint32_t s_p = smem_u32(mine), s_bar = s_p + kFewRows * kPStride * 2, s_ring = s_bar + kMaxStages * 8;
    for (int k = threadIdx.x; k < kFewRows * 16; k += kFewWarps * 32) {
        const int r = k >> 4, c = (k & 15) * 8;
        alignas(16) __half x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = __ushort_as_half(0);
        if (r < rows) {
            const __half *q = static_cast<const __half *>(p.a.q) + (int64_t)(s.q0 + r / p.rep) * p.a.q_sT + (int64_t)(head * p.rep + r % p.rep) * p.a.q_sH + c;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = q[j];
        }
        *reinterpret_cast<uint4 *>(s_q + r * 128 + c) = *reinterpret_cast<const uint4 *>(x);
    }
    if (lane < stages) mbar_init(s_bar + 8 * lane, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    __syncthreads();

    // bounds and bias of this lane's two columns; the pages that any row sees
    int lo[2], hi[2], pos[2], first = INT32_MAX, last = 0;
    float slope[2];
    for (int u = 0; u < s.n_new; ++u) {
        int a, b, c;
        paged_bounds(p, s, u, c, a, b);
        if (a < b) { first = min(first, a); last = max(last, b); }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int r = 2 * t + c;
        lo[c] = hi[c] = pos[c] = 0;
        slope[c] = 0.f;
        if (r < rows) {
            paged_bounds(p, s, r / p.rep, pos[c], lo[c], hi[c]);
            if (p.a.slopes) slope[c] = p.a.slopes[head * p.rep + r % p.rep] * kLog2e;
        }
    }
    const int p_lo = first < last ? first / kPage : 0, p_hi = first < last ? pages_of(last) : 0, per = (p_hi - p_lo + p.splits - 1) / p.splits;
    const int p0 = p_lo + split * per, p1 = min(p_hi, p0 + per), n_mine = max(0, (p1 - p0 - warp + kFewWarps - 1) / kFewWarps);
    // pages newest first: where values are packed in 3 bits the fp16 pages' sums are kept apart, and they come at the beginning
    auto page_at = [&](int k) { return p1 - 1 - (k * kFewWarps + warp); };

    constexpr int KW = FewGeom<KB>::W, VW = FewGeom<VB>::W, KT = FewGeom<KB>::TILES, VT = FewGeom<VB>::TILES;
    const int kg_log2 = KB == 3 ? 0 : 31 - __clz(p.l.group), vg_log2 = VB == 3 ? 0 : 31 - __clz(p.l.group);
    const uint32_t k_sz = kStageRows * p.k_groups * 2, v_sz = kStageRows * p.v_groups * 2;
    constexpr int SPH = kPage / kStageRows;                       // stages of a page's keys, and of its values

    // page numbers, 32 of the warp's pages at a time, one a lane; -1: not there
    int ids = -1, ids_base = 0;
    auto fetch_ids = [&](int base) {
        ids_base = base;
        ids = -1;
        if (base + lane < n_mine) {
            const int page = page_at(base + lane), id = s.table[page];
            if (id >= 0 && id < (page < s.packed ? p.l.n_packed : p.l.n_fp16)) ids = id;
        }
    };
    auto id_of = [&](int k) { return __shfl_sync(0xffffffffu, ids, k - ids_base); };

    // the producer's place: page number `pk` of the warp's, its next stage; ids are those of the consumer's window, so it stops at its end
    int pk = 0, pstage = 0, filled = 0, used = 0;
    auto produce = [&]() {
        while (pk < n_mine && pk < ids_base + 32 && filled - used < stages) {
            const int id = id_of(pk);
            if (page_at(pk) >= s.packed || id < 0) { ++pk; continue; }
            if (lane == 0) {
                const int slot = filled % stages;
                const uint32_t bar = s_bar + 8 * slot, dst = s_ring + slot * stage_bytes;
                const bool values = pstage >= SPH;
                const int64_t row = ((int64_t)id * p.l.Hkv + head) * kPage + (pstage % SPH) * kStageRows;
                const uint32_t cb = kStageRows * 4 * (values ? VW : KW), sz = values ? v_sz : k_sz;
                const int groups = values ? p.v_groups : p.k_groups;
                mbar_expect(bar, cb + 2 * sz);
                bulk_load(dst, (values ? p.l.vcode + row * VW : p.l.kcode + row * KW), cb, bar);
                bulk_load(dst + cb, static_cast<const __half *>(values ? p.l.vscale : p.l.kscale) + row * groups, sz, bar);
                bulk_load(dst + cb + sz, static_cast<const __half *>(values ? p.l.vmn : p.l.kmn) + row * groups, sz, bar);
            }
            ++filled;
            if (++pstage == 2 * SPH) { pstage = 0; ++pk; }
        }
    };

    float out[VT][4];
#pragma unroll
    for (int m = 0; m < VT; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) out[m][e] = 0.f;
    FewState st = {{-INFINITY, -INFINITY}, {0.f, 0.f}};
    float aside_m[2] = {-INFINITY, -INFINITY};                    // 3-bit values: reference of the sums put aside, see below
    bool aside = false, ok = true;
    float *s_out = reinterpret_cast<float *>(smem + 2048 + kFewWarps * (kFewRows * kPStride * 2 + kMaxStages * 8 + stages * stage_bytes)) + warp * kFewRows * 128;

    const float two = p.a.softcap > 0.f ? 2.f * kLog2e * p.a.softmax_scale / p.a.softcap : 0.f, cap2 = p.a.softcap * kLog2e, scale2 = p.a.softmax_scale * kLog2e;

    // scores of a page -> weights in s_p, sums and references in st; returns the factors for what is summed already
    auto softmax_page = [&](auto &sc, auto element, int base, float (&alpha)[2]) {
        constexpr int T = sizeof(sc) / sizeof(sc[0]);
        const bool whole = base >= 0 && __all_sync(0xffffffffu, (2 * t >= rows || (lo[0] <= base && hi[0] >= base + kPage)) &&
                                                                    (2 * t + 1 >= rows || (lo[1] <= base && hi[1] >= base + kPage)));
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int m = 0; m < T; ++m)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int el = element(m, e), j = base + el;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float x = sc[m][2 * e + c];
                    x = p.a.softcap > 0.f ? cap_score(x, two, cap2) : x * scale2;
                    if (p.a.slopes) x = fmaf(slope[c], (float)(j - pos[c]), x);
                    if (el < 0 || (!whole && (j < lo[c] || j >= hi[c]))) x = -INFINITY;
                    sc[m][2 * e + c] = x;
                    top[c] = fmaxf(top[c], x);
                }
            }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], o));
            const float ref = fmaxf(st.m[c], top[c]);
            alpha[c] = ref == -INFINITY ? 1.f : exp2_approx(st.m[c] - ref);
            st.m[c] = ref;
            st.l[c] *= alpha[c];
        }
        __syncwarp();                                             // the weights of the page before are read
#pragma unroll
        for (int m = 0; m < T; ++m)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float ref = st.m[c] == -INFINITY ? 0.f : st.m[c];
                const float x = exp2_approx(sc[m][c] - ref), y = exp2_approx(sc[m][2 + c] - ref);
                st.l[c] += x + y;
                const uint32_t h = as_u32(__floats2half2_rn(x, y));
                const int e0 = element(m, 0), e1 = element(m, 1);
                const uint32_t at = s_p + (2 * t + c) * kPStride * 2;
                auto slot = [](int el) { return (el & ~15) + 4 * (el & 3) + ((el & 15) >> 2); };
                if constexpr (T == 8) {
                    asm volatile("st.shared.b32 [%0], %1;\n" ::"r"(at + slot(e0) * 2), "r"(h) : "memory");
                } else {
                    if (e0 >= 0) asm volatile("st.shared.u16 [%0], %1;\n" ::"r"(at + slot(e0) * 2), "h"((unsigned short)(h & 0xffff)) : "memory");
                    if (e1 >= 0) asm volatile("st.shared.u16 [%0], %1;\n" ::"r"(at + slot(e1) * 2), "h"((unsigned short)(h >> 16)) : "memory");
                }
            }
        __syncwarp();
    };
    auto rescale = [&](auto &o, const float (&alpha)[2]) {
        if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
            constexpr int T = sizeof(o) / sizeof(o[0]);
#pragma unroll
            for (int m = 0; m < T; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[m][e] *= alpha[e & 1];
        }
    };
    auto weights = [&](int step, uint32_t &b0, uint32_t &b1) {    // B operand of contraction rows 16 step + t + 4j for query row g
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];\n" : "=r"(b0), "=r"(b1) : "r"(s_p + (g * kPStride + 16 * step + 4 * t) * 2));
    };

    auto fp16_page = [&](int id, int page, auto &o) {
        const int base = page * kPage, there = min(kPage, s.length - base);
        const __half *k = static_cast<const __half *>(p.l.kfull) + ((int64_t)id * p.l.Hkv + head) * kPageHalf;
        const __half *v = static_cast<const __half *>(p.l.vfull) + ((int64_t)id * p.l.Hkv + head) * kPageHalf;
        float sc[8][4];
#pragma unroll
        for (int m = 0; m < 8; ++m) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[m][e] = 0.f;
#pragma unroll
            for (int blk = 0; blk < 4; ++blk) {                   // 32 channels, eight neighbours a lane
                const int r0 = min(few_element<1>(g, m, 0), there - 1), r1 = min(few_element<1>(g, m, 1), there - 1);
                const uint4 x = *reinterpret_cast<const uint4 *>(k + r0 * kHeadDim + 32 * blk + 8 * t);
                const uint4 y = *reinterpret_cast<const uint4 *>(k + r1 * kHeadDim + 32 * blk + 8 * t);
                const uint4 q = *reinterpret_cast<const uint4 *>(s_q + g * 128 + 32 * blk + 8 * t);
                mma16816(sc[m], x.x, y.x, x.y, y.y, q.x, q.y);
                mma16816(sc[m], x.z, y.z, x.w, y.w, q.z, q.w);
            }
        }
        float alpha[2];
        softmax_page(sc, [&](int m, int e) { return few_element<1>(g, m, e); }, base, alpha);
        rescale(o, alpha);
#pragma unroll 1
        for (int step = 0; step < 8; ++step) {
            if (16 * step >= there) break;
            uint32_t x[4][8], b0, b1;
#pragma unroll
            for (int j = 0; j < 4; ++j) {                         // tokens t + 4j, channels 16g .. 16g + 15; nothing behind the last token
                const int r = 16 * step + t + 4 * j;
                uint4 a = make_uint4(0, 0, 0, 0), b = a;
                if (r < there) {
                    a = *reinterpret_cast<const uint4 *>(v + r * kHeadDim + 16 * g);
                    b = *reinterpret_cast<const uint4 *>(v + r * kHeadDim + 16 * g + 8);
                }
                x[j][0] = a.x; x[j][1] = a.y; x[j][2] = a.z; x[j][3] = a.w;
                x[j][4] = b.x; x[j][5] = b.y; x[j][6] = b.z; x[j][7] = b.w;
            }
            weights(step, b0, b1);
#pragma unroll
            for (int m = 0; m < 8; ++m) {
                uint32_t a[4];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int q = 2 * m + e, c = (q & 3) * 4 + (q >> 2);
#pragma unroll
                    for (int j = 0; j < 2; ++j) a[e + 2 * j] = prmt(x[2 * j][c >> 1], x[2 * j + 1][c >> 1], c & 1 ? 0x7632 : 0x5410);
                }
                mma16816(o[m], a[0], a[1], a[2], a[3], b0, b1);
            }
        }
    };
    // `o` of the layout of fp16 pages and of 1, 2 and 4 bits, or of 3 bits, as [row][channel]
    auto each_out = [&](auto &o, auto element, auto f) {
        constexpr int T = sizeof(o) / sizeof(o[0]);
#pragma unroll
        for (int m = 0; m < T; ++m)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int c = element(m, e);
                if (c >= 0) {
                    f(2 * t, c, o[m][2 * e]);
                    f(2 * t + 1, c, o[m][2 * e + 1]);
                }
            }
    };

    int k = 0;
    if (n_mine > 0) fetch_ids(0);
    if constexpr (VB == 3) {
        // fp16 pages sum in the layout of eight tiles; the sums go to shared memory before the packed pages begin
        float o[8][4];
#pragma unroll
        for (int m = 0; m < 8; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[m][e] = 0.f;
        produce();
        for (; k < n_mine && page_at(k) >= s.packed; ++k) {
            if (k == ids_base + 32) { fetch_ids(k); pk = max(pk, k); produce(); }
            const int id = id_of(k);
            if (id >= 0) { fp16_page(id, page_at(k), o); aside = true; }
        }
        each_out(o, [&](int m, int e) { return few_element<1>(g, m, e); }, [&](int r, int c, float v) { s_out[r * 128 + c] = v; });
        aside_m[0] = st.m[0];
        aside_m[1] = st.m[1];
    } else {
        produce();
    }
    for (; k < n_mine; ++k) {
        if (k == ids_base + 32) { fetch_ids(k); produce(); }
        const int id = id_of(k), page = page_at(k);
        if (id < 0) continue;
        if (page >= s.packed) {
            if constexpr (VB != 3) fp16_page(id, page, out);
            continue;
        }
        float sc[KT][4], alpha[2];
#pragma unroll
        for (int m = 0; m < KT; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[m][e] = 0.f;
#pragma unroll 1
        for (int q = 0; q < SPH; ++q) {
            const int slot = used % stages;
            ok = __all_sync(0xffffffffu, mbar_wait(s_bar + 8 * slot, used / stages & 1, &p.b.count[2]));
            if (!ok) break;
            const uint32_t c = s_ring + slot * stage_bytes;
#pragma unroll
            for (int step = 0; step < kStageRows / 16; ++step) {
                const __half *qr = s_q + g * 128 + q * kStageRows + step * 16 + t;
                const uint32_t b0 = as_u32(__halves2half2(qr[0], qr[4])), b1 = as_u32(__halves2half2(qr[8], qr[12]));
                few_packed_step<KB>(sc, c, c + kStageRows * 4 * KW, c + kStageRows * 4 * KW + k_sz, p.k_groups, kg_log2, step * 16, g, t, b0, b1);
            }
            ++used;
            __syncwarp();
            produce();
        }
        if (!ok) break;
        softmax_page(sc, [&](int m, int e) { return few_element<KB>(g, m, e); }, page * kPage, alpha);
        rescale(out, alpha);
#pragma unroll 1
        for (int q = 0; q < SPH; ++q) {
            const int slot = used % stages;
            ok = __all_sync(0xffffffffu, mbar_wait(s_bar + 8 * slot, used / stages & 1, &p.b.count[2]));
            if (!ok) break;
            const uint32_t c = s_ring + slot * stage_bytes;
#pragma unroll
            for (int step = 0; step < kStageRows / 16; ++step) {
                uint32_t b0, b1;
                weights(q * (kStageRows / 16) + step, b0, b1);
                few_packed_step<VB>(out, c, c + kStageRows * 4 * VW, c + kStageRows * 4 * VW + v_sz, p.v_groups, vg_log2, step * 16, g, t, b0, b1);
            }
            ++used;
            __syncwarp();
            produce();
        }
        if (!ok) break;
    }
    if (!ok) {                                                    // give the copies in flight time to land before the memory is given up
        for (; used < filled; ++used) mbar_wait(s_bar + 8 * (used % stages), used / stages & 1, &p.b.count[2]);
    }

    // the warps' parts meet
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) st.l[c] += __shfl_xor_sync(0xffffffffu, st.l[c], o);
    float *s_ml = reinterpret_cast<float *>(mine);                // [8][2], over the warp's weights
    __syncwarp();
    if (g == 0) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            s_ml[2 * (2 * t + c)] = st.m[c];
            s_ml[2 * (2 * t + c) + 1] = st.l[c];
        }
    }
    if constexpr (VB == 3) {
        float f[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) f[c] = aside && aside_m[c] != -INFINITY ? exp2_approx(aside_m[c] - st.m[c]) : 0.f;
        __syncwarp();
        each_out(out, [&](int m, int e) { return few_element<3>(g, m, e); }, [&](int r, int c, float v) { s_out[r * 128 + c] = s_out[r * 128 + c] * f[r & 1] + v; });
    } else {
        each_out(out, [&](int m, int e) { return few_element<1>(g, m, e); }, [&](int r, int c, float v) { s_out[r * 128 + c] = v; });
    }
    __syncthreads();
    const int warp_bytes = kFewRows * kPStride * 2 + kMaxStages * 8 + stages * stage_bytes;
    const float *all_out = reinterpret_cast<const float *>(smem + 2048 + kFewWarps * warp_bytes);
    for (int r = 0; r < rows; ++r) {
        float m = -INFINITY, l = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) m = fmaxf(m, reinterpret_cast<const float *>(smem + 2048 + w * warp_bytes)[2 * r]);
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) {
            const float *ml = reinterpret_cast<const float *>(smem + 2048 + w * warp_bytes) + 2 * r;
            const float f = part_factor(ml[0], ml[1], m);
            l += f * ml[1];
            if (f != 0.f) v += f * all_out[(w * kFewRows + r) * 128 + threadIdx.x];
        }
        const int64_t row = (int64_t)(s.q0 + r / p.rep) * p.a.nh + head * p.rep + r % p.rep;
        if (p.splits == 1) {
            static_cast<__half *>(p.a.out)[(int64_t)(s.q0 + r / p.rep) * p.a.o_sT + (int64_t)(head * p.rep + r % p.rep) * p.a.o_sH + threadIdx.x] =
                __float2half_rn(l == 0.f ? 0.f : v / l);
        } else {
            const int64_t at = (int64_t)split * p.a.tokens * p.a.nh + row;
            p.part_out[at * 128 + threadIdx.x] = v;
            if (threadIdx.x == 0) { p.part_ml[2 * at] = m; p.part_ml[2 * at + 1] = l; }
        }
    }
}

// Partial sums of the splits -> outputs, in the splits' order.  A CTA takes one row of q and head; `few`: rows of the kernel above, else of
// the kernel of tiles.
__global__ void __launch_bounds__(128) paged_merge_kernel(const __grid_constant__ PagedArgs p, int few) {
    const int u = blockIdx.x / p.a.nh, h = blockIdx.x - u * p.a.nh;
    if (u < p.a.q_start[0] || u >= p.a.q_start[p.a.n]) return;
    const PagedSeq s = paged_seq(p, sequence_of(p.a.q_start, p.a.n, u));
    const int rows = s.n_new * p.rep;
    if (few ? rows > kFewRows : rows <= p.few_rows) return;
    const int64_t step = (int64_t)p.a.tokens * p.a.nh, row = (int64_t)u * p.a.nh + h;
    float m = -INFINITY, l = 0.f, v = 0.f;
    for (int i = 0; i < p.splits; ++i) m = fmaxf(m, p.part_ml[2 * (i * step + row)]);
    for (int i = 0; i < p.splits; ++i) {
        const float mi = p.part_ml[2 * (i * step + row)], li = p.part_ml[2 * (i * step + row) + 1], x = p.part_out[(i * step + row) * 128 + threadIdx.x];
        const float f = part_factor(mi, li, m);
        l += f * li;
        if (f != 0.f) v += f * x;
    }
    static_cast<__half *>(p.a.out)[(int64_t)u * p.a.o_sT + (int64_t)h * p.a.o_sH + threadIdx.x] = __float2half_rn(l == 0.f ? 0.f : v / l);
}

template <int KB, int VB>
static int launch_few(const PagedArgs &p, cudaStream_t st) {
    const int k_bytes = kStageRows * (4 * page_words(KB) + 4 * p.k_groups), v_bytes = kStageRows * (4 * page_words(VB) + 4 * p.v_groups);
    const int stage_bytes = (k_bytes > v_bytes ? k_bytes : v_bytes), ctas = KB == 3 || VB == 3 ? 3 : 4;
    // what 227 KB leave each of the CTAs of an SM (1 KB of each is the system's)
    const int fixed = 2048 + kFewWarps * (kFewRows * kPStride * 2 + kMaxStages * 8) + kFewWarps * kFewRows * 128 * 4;
    const int room = (227 * 1024 / ctas - 1024 - fixed) / kFewWarps;
    int stages = room / stage_bytes;
    stages = stages < 2 ? 2 : stages > kMaxStages ? kMaxStages : stages;
    const size_t smem = fixed + (size_t)kFewWarps * stages * stage_bytes;
    const cudaError_t e = cudaFuncSetAttribute(paged_few_kernel<KB, VB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return record_cuda_error(e);
    const int64_t grid = (int64_t)p.a.n * p.l.Hkv * p.splits;
    if (grid > 2147483647LL) return KVQ_ERR_UNSUPPORTED;
    paged_few_kernel<KB, VB><<<(unsigned)grid, kFewWarps * 32, smem, st>>>(p, stages, stage_bytes);
    return check_launch();
}

int paged_few(const PagedArgs &p, cudaStream_t st) {
#define KVQ_V(KB)                                                                                                             \
    switch (p.l.v_bits) {                                                                                                     \
        case 1: return launch_few<KB, 1>(p, st);                                                                              \
        case 2: return launch_few<KB, 2>(p, st);                                                                              \
        case 3: return launch_few<KB, 3>(p, st);                                                                              \
        default: return launch_few<KB, 4>(p, st);                                                                             \
    }
    switch (p.l.k_bits) {
        case 1: KVQ_V(1)
        case 2: KVQ_V(2)
        case 3: KVQ_V(3)
        default: KVQ_V(4)
    }
#undef KVQ_V
}

int paged_merge(const PagedArgs &p, int few, cudaStream_t st) {
    const int64_t grid = (int64_t)p.a.tokens * p.a.nh;
    if (grid > 2147483647LL) return KVQ_ERR_UNSUPPORTED;
    paged_merge_kernel<<<(unsigned)grid, 128, 0, st>>>(p, few);
    return check_launch();
}

}  // namespace kvq
