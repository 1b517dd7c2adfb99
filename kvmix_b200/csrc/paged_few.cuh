// Attention of few query rows of a kv head (a new token of a group of query heads) over a paged cache.
#pragma once
#include "paged_attn.cuh"

namespace kvq {

// A CTA of four warps takes one (sequence, kv head, block of query rows, split of the pages); a warp takes every fourth packed page, and 32
// tokens of every fp16 page, by itself -- scores, online softmax, values -- so nothing in the loop waits for another warp.
//   scores   S[token][column] = K[token][channel] B[channel][column]: mma m16n8k16 with 16 tokens as rows
//   values   O[channel][column] = V^T[channel][token] B[token][column]: the same with 16 channels as rows
// In both the packed axis runs along the MMA's rows and the contraction across words, so that the two elements of an operand register
// come from the same place of two words, and a field of 1, 2 or 4 bits is an operand as it stands: masked in place it is the fp16 subnormal
// code * 2^(position - 24), and the power of two, the same for a whole accumulator, comes off at the end.  Scales go to the other
// operand, whose columns are (group of the packed axis, query row) pairs:
//   keys     B = q * scale of a channel's token group, as a pair hi + lo of two columns: exact to 2^-22 of itself and 2^-25 (the largest of a stage is 2^-6 and
//            more); rounded once it would cost 2^-11 of every term
//   values   B = p * scale of a token's channel group, rounded to fp16 as weights are everywhere; a pair as well where columns are left (one
//            sequence of 1, 2 or 4 rows at groups of 32, 64 or 128: 2.5e-4 of an output's size in place of 3.2e-4, at 2 bits)
// An accumulator row needs the column of its own group only; what the others hold is not read.  Minima times q or p come from one more MMA
// a k-step, whose rows are the groups.  3-bit words are groups of their own, so their fields become fp16 values (code * scale + minimum,
// rounded once) and the columns are query rows.
// Words arrive by bulk copies, 32 to 128 contraction rows (codes, scales, minima) a stage, in the warp's own ring; fp16 pages go straight to
// registers, first, and their sums are put aside in shared memory.
constexpr int kFewWarps = 4;
constexpr int kMaxStages = 8;
constexpr int kPStride = 136;                                     // halves between rows of weights
constexpr float kWeightBits = 7.f;                                // weights are 2^7 p: p * scale keeps away from fp16's smallest numbers

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
// Where element el of a page stands among weights and scores: those of a lane's k-step side by side.
__device__ __forceinline__ int few_slot(int el) { return (el & ~15) + 4 * (el & 3) + ((el & 15) >> 2); }

// Field f of two half words, moved to bit 2 and above (see VHalf: lower ones lose product bits in the tensor core).
template <int BITS> __device__ __forceinline__ uint32_t few_field(uint32_t x, int f) {
    if constexpr (BITS == 4) return (f < 2 ? x << 2 : x >> 6) & (0x003c003cu << (f & 1 ? 4 : 0));
    else if constexpr (BITS == 2) return f < 2 ? (x << 6) & (0x00030003u << (6 + 2 * f)) : f < 5 ? x & (0x00030003u << (2 * f)) : (x >> 6) & (0x00030003u << (2 * f - 6));
    else return f < 4 ? (x << 6) & (0x00010001u << (f + 6)) : f < 10 ? x & (0x00010001u << f) : (x >> 6) & (0x00010001u << (f - 6));
}
// 2^(24 - position) of accumulator (m, e)
template <int BITS> __device__ __forceinline__ float few_power(int m, int e) {
    const int s = 2 * m + e, i = (s & 3) * 4 + (s >> 2);
    return (float)(1 << (24 - VHalf<BITS>::pos(i % (16 / BITS))));
}

// The A registers of a k-step: a(m, r) for tile m, register r.  Contraction rows of lane t: row + t + 4j.
template <int BITS>
struct FewWords {
    uint32_t x[BITS][2];                                          // half h of rows t + 8j and t + 8j + 4
    __device__ __forceinline__ FewWords(uint32_t codes, int row, int g, int t) {
        constexpr int W = page_words(BITS);
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
    }
    __device__ __forceinline__ uint32_t a(int m, int r) const {
        const int s = 2 * m + (r & 1), i = (s & 3) * 4 + (s >> 2), n = 16 / BITS;
        return few_field<BITS>(x[i / n][r >> 1], i % n);
    }
};

// Scales or minima of a lane's four contraction rows, group `grp`, as two pairs.
__device__ __forceinline__ void few_pairs(uint32_t at, int row, int t, int groups, int grp, uint32_t (&v)[2]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t r0 = at + ((row + t + 8 * j) * groups + grp) * 2;
        v[j] = prmt(lds16(r0), lds16(r0 + 8 * groups), 0x5410);
    }
}

// 3 bits: acc[tile] += A * B with A the dequantised values.
__device__ __forceinline__ void few_step3(float (&acc)[11][4], uint32_t codes, uint32_t scale, uint32_t mn, int row, int g, int t, uint32_t b0, uint32_t b1) {
    uint32_t w[2][4];
    uint32_t sc[2][2], lo[2][2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int word = min(g + 8 * e, 11);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[e][j] = lds32(codes + ((row + t + 4 * j) * 12 + word) * 4);
        few_pairs(scale, row, t, 12, word, sc[e]);
        few_pairs(mn, row, t, 12, word, lo[e]);
    }
#pragma unroll
    for (int m = 0; m < 11; ++m) {
        uint32_t a[4];
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                // the field at the same place of two half words, or shifted there
                const uint32_t u = w[e][2 * j], v = w[e][2 * j + 1];
                const uint32_t x = m < 5 ? prmt(u, v, 0x5410) >> (m < 3 ? 0 : 9) : m < 10 ? prmt(u >> 15, v >> 15, 0x5410) >> (m < 8 ? 0 : 9) : prmt(u, v, 0x7632) >> 14;
                const int pos = m < 3 ? 3 * m : m < 5 ? 3 * m - 9 : m < 8 ? 3 * m - 15 : m < 10 ? 3 * m - 24 : 0;
                const uint32_t mask = (m < 10 ? 7u : 3u) << pos, expo = (uint32_t)(25 - pos) << 10;
                uint32_t f;
                asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(f) : "r"(x), "r"(mask * 0x10001u), "r"(expo * 0x10001u));        // (x & mask) | expo
                a[e + 2 * j] = as_u32(__hfma2(__hsub2(as_h2(f), as_h2(expo * 0x10001u)), as_h2(sc[e][j]), as_h2(lo[e][j])));
            }
        mma16816(acc[m], a[0], a[1], a[2], a[3], b0, b1);
    }
}

__device__ __forceinline__ float warp_max_f32(float x) {
    float r;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;\n" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float4 lds_f4(uint32_t at) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ void sts_f4(uint32_t at, float x, float y, float z, float w) {
    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};\n" ::"r"(at), "f"(x), "f"(y), "f"(z), "f"(w) : "memory");
}

// Shared memory of a CTA for blocks of R query rows: q as it is and with a lane's four channels of a k-step side by side, the rows' bounds, and for
// every warp weights, scores, sums put aside, sums of weights, barriers, the ring.
struct FewShared {
    int q, bounds, factor, warps, weights, scores, aside, sums, bars, ring, warp_bytes, total;
    __host__ __device__ FewShared(int R, int stages, int stage_bytes) {
        q = 0;
        bounds = 2 * R * 256;
        factor = bounds + R * 16;
        warps = factor + (R + 1) / 2 * 16;
        weights = 0;
        scores = R * kPStride * 2;
        aside = scores + R * 512;
        sums = aside + R * 512;
        bars = sums + R * 128;
        ring = bars + kMaxStages * 8;
        warp_bytes = ring + stages * stage_bytes;
        total = warps + kFewWarps * warp_bytes;
    }
};

template <int KB, int VB, int CK>
__global__ void __launch_bounds__(kFewWarps * 32, KB == 3 || VB == 3 || CK == 2 ? 3 : 4)
    paged_few_kernel(const __grid_constant__ PagedArgs p, int R, int row_blocks, int stages, int stage_rows, int stage_bytes) {
    extern __shared__ __align__(128) char smem[];
    const FewShared sh(R, stages, stage_bytes);
    const int warp = uniform_warp(), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    int hs = blockIdx.x;
    const int split = hs % p.splits;
    hs /= p.splits;
    const int block = hs % row_blocks;
    hs /= row_blocks;
    const int head = hs % p.l.Hkv, i = hs / p.l.Hkv;
    const PagedSeq s = paged_seq(p, i);
    if (s.n_new * p.rep > kFewRows) return;
    const int row0 = block * R, rows = min(R, s.n_new * p.rep - row0);
    if (rows <= 0) return;

    const uint32_t base = smem_u32(smem), mine = base + sh.warps + warp * sh.warp_bytes;
    const uint32_t s_p = mine + sh.weights, s_s = mine + sh.scores, s_sum = mine + sh.sums, s_bar = mine + sh.bars, s_ring = mine + sh.ring;
    float *s_out = reinterpret_cast<float *>(smem + sh.warps + warp * sh.warp_bytes + sh.aside);                // [R][128]
    __half *s_q = reinterpret_cast<__half *>(smem), *s_qs = s_q + R * 128;
    // q by a power of two below 1, so that no product with a scale leaves fp16
    float2 *s_factor = reinterpret_cast<float2 *>(smem + sh.factor);              // raw scores to log2 units; to caps
    for (int r = warp; r < R; r += kFewWarps) {
        const int row = row0 + r;
        float x[4] = {0.f, 0.f, 0.f, 0.f}, top = 0.f;
        if (r < rows) {
            const __half *q = static_cast<const __half *>(p.a.q) + (int64_t)(s.q0 + row / p.rep) * p.a.q_sT + (int64_t)(head * p.rep + row % p.rep) * p.a.q_sH;
#pragma unroll
            for (int c = 0; c < 4; ++c) { x[c] = __half2float(q[lane + 32 * c]); top = fmaxf(top, fabsf(x[c])); }
        }
        top = warp_max_f32(top);
        const int e = top > 0.f && top < INFINITY ? (__float_as_int(top) >> 23 & 255) - 126 : 0;
        const float down = __int_as_float((127 - e) << 23), up = __int_as_float((127 + e) << 23), scale2 = p.a.softmax_scale * kLog2e;
#pragma unroll
        for (int c = 0; c < 4; ++c) s_q[r * 128 + lane + 32 * c] = s_qs[r * 128 + few_slot(lane + 32 * c)] = __float2half_rn(x[c] * down);
        if (lane == 0) s_factor[r] = make_float2(scale2 * up, p.cap_in * up);
    }
    int4 *s_bounds = reinterpret_cast<int4 *>(smem + sh.bounds);  // lowest position, end, position, slope of a row
    if (threadIdx.x < R) {
        int lo = 0, hi = 0, pos = 0;
        float slope = 0.f;
        const int row = row0 + threadIdx.x;
        if ((int)threadIdx.x < rows) {
            paged_bounds(p, s, row / p.rep, pos, lo, hi);
            if (p.a.slopes) slope = p.a.slopes[head * p.rep + row % p.rep] * kLog2e;
        }
        s_bounds[threadIdx.x] = make_int4(lo, hi, pos, __float_as_int(slope));
    }
    if (lane < stages) mbar_init(s_bar + 8 * lane, 1);
    for (int k = lane; k < R * 32; k += 32) asm volatile("st.shared.b32 [%0], %1;\n" ::"r"(s_sum + 4 * k), "r"(0) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    __syncthreads();

    // the pages that any row sees
    int first = INT32_MAX, last = 0;
    for (int r = 0; r < rows; ++r) {
        const int4 b = s_bounds[r];
        if (b.x < b.y) { first = min(first, b.x); last = max(last, b.y); }
    }
    const int p_lo = first < last ? first / kPage : 0, p_hi = first < last ? pages_of(last) : 0, per = (p_hi - p_lo + p.splits - 1) / p.splits;
    const int p0 = p_lo + split * per, p1 = min(p_hi, p0 + per), p_old = max(p0, min(p1, s.packed));            // [p0, p_old) packed
    const int n_mine = max(0, (p_old - p0 - warp + kFewWarps - 1) / kFewWarps);
    auto page_at = [&](int k) { return p0 + k * kFewWarps + warp; };

    constexpr int KW = page_words(KB), VW = page_words(VB), VT = VB == 3 ? 11 : 8;
    const uint32_t k_cb = stage_rows * 4 * KW, v_cb = stage_rows * 4 * VW, k_sz = stage_rows * p.k_groups * 2, v_sz = stage_rows * p.v_groups * 2;
    const int half_stages = kPage / stage_rows;                   // stages of a page's keys, and of its values
    const int ng_log2 = p.l.group == 128 ? 0 : p.l.group == 64 ? 1 : 2;            // of both sides, where they are not 3 bits
    const int own_group = g >> (3 - ng_log2);                     // of the 16 packed elements that this lane's accumulator rows stand for

    // page numbers, 32 of the warp's pages at a time, one a lane; -1: not there
    int ids = -1, ids_base = 0;
    auto fetch_ids = [&](int at) {
        ids_base = at;
        ids = -1;
        if (at + lane < n_mine) {
            const int id = s.table[page_at(at + lane)];
            if (id >= 0 && id < p.l.n_packed) ids = id;
        }
    };
    auto id_of = [&](int k) { return __shfl_sync(0xffffffffu, ids, k - ids_base); };

    // the producer's place: page number `pk` of the warp's, its next stage; ids are those of the consumer's window, so it stops at its end
    int pk = 0, pstage = 0, fill_slot = 0, in_flight = 0, use_slot = 0;
    uint32_t parity = 0;
    auto produce = [&]() {
        while (pk < n_mine && pk < ids_base + 32 && in_flight < stages) {
            const int id = id_of(pk);
            if (id < 0) { ++pk; continue; }
            if (lane == 0) {
                const uint32_t bar = s_bar + 8 * fill_slot, dst = s_ring + fill_slot * stage_bytes;
                const int64_t at = (int64_t)id * p.l.Hkv + head;
                if (pstage < half_stages) {
                    const int off = pstage * stage_rows * p.k_groups;
                    mbar_expect(bar, k_cb + 2 * k_sz);
                    bulk_load(dst, p.l.kcode + at * (kPage * KW) + pstage * stage_rows * KW, k_cb, bar);
                    bulk_load(dst + k_cb, static_cast<const __half *>(p.l.kscale) + at * (kPage * p.k_groups) + off, k_sz, bar);
                    bulk_load(dst + k_cb + k_sz, static_cast<const __half *>(p.l.kmn) + at * (kPage * p.k_groups) + off, k_sz, bar);
                } else {
                    const int st = pstage - half_stages, off = st * stage_rows * p.v_groups;
                    mbar_expect(bar, v_cb + 2 * v_sz);
                    bulk_load(dst, p.l.vcode + at * (kPage * VW) + st * stage_rows * VW, v_cb, bar);
                    bulk_load(dst + v_cb, static_cast<const __half *>(p.l.vscale) + at * (kPage * p.v_groups) + off, v_sz, bar);
                    bulk_load(dst + v_cb + v_sz, static_cast<const __half *>(p.l.vmn) + at * (kPage * p.v_groups) + off, v_sz, bar);
                }
            }
            if (++fill_slot == stages) fill_slot = 0;
            ++in_flight;
            if (++pstage == 2 * half_stages) { pstage = 0; ++pk; }
        }
    };
    bool ok = true;
    auto stage_ready = [&]() {
        ok = __all_sync(0xffffffffu, mbar_wait(s_bar + 8 * use_slot, parity, &p.b.count[2]));
        return s_ring + use_slot * stage_bytes;
    };
    auto stage_done = [&]() {
        if (++use_slot == stages) { use_slot = 0; parity ^= 1; }
        --in_flight;
        __syncwarp();
        produce();
    };

    const float cap2 = p.a.softcap * kLog2e;
    float ref = -INFINITY, alpha = 1.f;                           // of row `lane`: reference (log2 units), factor of what is summed already

    // Scores of `count` tokens, [row][slot] in s_s -> weights in s_p, sums in s_sum, ref and alpha.  A lane takes four tokens of each row.
    auto softmax_page = [&](int page_base, int count) {
        __syncwarp();
        const int j0 = page_base + 16 * (lane >> 2) + (lane & 3);
        float change = 1.f;
#pragma unroll 1
        for (int r = 0; r < rows; ++r) {
            const float4 raw = lds_f4(s_s + r * 512 + lane * 16);
            const int4 b = s_bounds[r];
            const float2 by_row = s_factor[r];
            const float slope = __int_as_float(b.w);
            float x[4] = {raw.x, raw.y, raw.z, raw.w}, top = -INFINITY;
            const bool whole = b.x <= page_base && b.y >= page_base + kPage && count == kPage;
            const int end = min(b.y, page_base + count);
            if (p.a.softcap > 0.f) {                              // the polynomial alone wherever it will do
                bool small = true;
#pragma unroll
                for (int c = 0; c < 4; ++c) { x[c] *= by_row.y; small = small && fabsf(x[c]) <= kCapSmall; }
                if (__all_sync(0xffffffffu, small)) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) x[c] = cap_small(x[c], cap2);
                } else {
#pragma unroll
                    for (int c = 0; c < 4; ++c) x[c] = cap_score(x[c], cap2);
                }
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c) x[c] *= by_row.x;
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                x[c] = fmaf(slope, (float)(j0 + 4 * c - b.z), x[c]);
                if (!whole && (j0 + 4 * c < b.x || j0 + 4 * c >= end)) x[c] = -INFINITY;
            }
            asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(top) : "f"(x[0]), "f"(x[1]), "f"(x[2]));
            asm("max.NaN.f32 %0, %1, %2;" : "=f"(top) : "f"(top), "f"(x[3]));
            top = warp_max_f32(top);
            const float old = __shfl_sync(0xffffffffu, ref, r), now = fmaxf(old, top), by = now == -INFINITY ? 1.f : exp2_approx(old - now);
            if (lane == r) { ref = now; alpha = by; }
            change = fminf(change, by);
            const float to = (now == -INFINITY ? 0.f : now) - kWeightBits;
            float sum = 0.f;
#pragma unroll
            for (int c = 0; c < 4; ++c) { x[c] = exp2_approx(x[c] - to); sum += x[c]; }
            const uint32_t w0 = as_u32(__floats2half2_rn(x[0], x[1])), w1 = as_u32(__floats2half2_rn(x[2], x[3]));
            asm volatile("st.shared.v2.b32 [%0], {%1, %2};\n" ::"r"(s_p + r * kPStride * 2 + lane * 8), "r"(w0), "r"(w1) : "memory");
            const uint32_t at = s_sum + r * 128 + lane * 4;
            sum = fmaf(__uint_as_float(lds32(at)), by, sum);
            asm volatile("st.shared.f32 [%0], %1;\n" ::"r"(at), "f"(sum) : "memory");
        }
        __syncwarp();
        return change != 1.f;                                     // the same in all lanes
    };
    auto weights = [&](int row, int step, uint32_t &b0, uint32_t &b1) {           // contraction rows 16 step + t + 4j; columns beyond R are not read
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];\n" : "=r"(b0), "=r"(b1) : "r"(s_p + (row * kPStride + 16 * step + 4 * t) * 2));
    };
    // Columns that are query rows: scores of accumulators into s_s, factors of columns 2t, 2t + 1
    auto dense_scores = [&](auto &sc, auto element) {
        constexpr int T = sizeof(sc) / sizeof(sc[0]);
#pragma unroll
        for (int m = 0; m < T; ++m)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int el = element(m, e);
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    if (el >= 0 && 2 * t + c < rows) asm volatile("st.shared.f32 [%0], %1;\n" ::"r"(s_s + (2 * t + c) * 512 + few_slot(el) * 4), "f"(sc[m][2 * e + c]) : "memory");
            }
    };
    auto rescale = [&](auto &o, int r0, int r1) {                 // columns 2t, 2t + 1 belong to rows r0, r1
        constexpr int T = sizeof(o) / sizeof(o[0]);
        const float a0 = __shfl_sync(0xffffffffu, alpha, r0), a1 = __shfl_sync(0xffffffffu, alpha, r1);
#pragma unroll
        for (int m = 0; m < T; ++m) { o[m][0] *= a0; o[m][1] *= a1; o[m][2] *= a0; o[m][3] *= a1; }
    };

    // ---- fp16 pages: tokens 32 warp .. 32 warp + 31 of each
    if (n_mine > 0) fetch_ids(0);
    produce();
    {
        float o[8][4];
#pragma unroll
        for (int m = 0; m < 8; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[m][e] = 0.f;
#pragma unroll 1
        for (int page = p_old; page < p1; ++page) {
            const int id = s.table[page], token0 = page * kPage + 32 * warp, there = min(32, s.length - token0);
            if (id < 0 || id >= p.l.n_fp16 || there <= 0) continue;
            const int64_t at = ((int64_t)id * p.l.Hkv + head) * kPageHalf + 32 * warp * kHeadDim;
            const __half *kp = static_cast<const __half *>(p.l.kfull) + at, *vp = static_cast<const __half *>(p.l.vfull) + at;
            float sc[2][4];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[m][e] = 0.f;
#pragma unroll
                for (int blk = 0; blk < 4; ++blk) {               // 32 channels, eight neighbours a lane; tokens 16m + g, 16m + g + 8
                    const uint4 x = *reinterpret_cast<const uint4 *>(kp + min(16 * m + g, there - 1) * kHeadDim + 32 * blk + 8 * t);
                    const uint4 y = *reinterpret_cast<const uint4 *>(kp + min(16 * m + g + 8, there - 1) * kHeadDim + 32 * blk + 8 * t);
                    const uint4 q = *reinterpret_cast<const uint4 *>(s_q + min(g, R - 1) * 128 + 32 * blk + 8 * t);           // columns beyond R are not read
                    mma16816(sc[m], x.x, y.x, x.y, y.y, q.x, q.y);
                    mma16816(sc[m], x.z, y.z, x.w, y.w, q.z, q.w);
                }
            }
            uint4 x[2][4][2];                                     // tokens 16 step + t + 4j, channels 16g .. 16g + 15; nothing behind the last token
#pragma unroll
            for (int step = 0; step < 2; ++step)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = 16 * step + t + 4 * j;
#pragma unroll
                    for (int h = 0; h < 2; ++h) x[step][j][h] = r < there ? *reinterpret_cast<const uint4 *>(vp + r * kHeadDim + 16 * g + 8 * h) : make_uint4(0, 0, 0, 0);
                }
            dense_scores(sc, [&](int m, int e) { return 16 * m + g + 8 * e; });
            if (softmax_page(token0, 32)) rescale(o, 2 * t, 2 * t + 1);
#pragma unroll
            for (int step = 0; step < 2; ++step) {
                uint32_t b0, b1;
                weights(min(g, R - 1), step, b0, b1);
                auto word = [&](int j, int c) {                   // channels 2c, 2c + 1 of token t + 4j
                    const uint4 &v = x[step][j][c >> 2];
                    return (c & 3) == 0 ? v.x : (c & 3) == 1 ? v.y : (c & 3) == 2 ? v.z : v.w;
                };
#pragma unroll
                for (int m = 0; m < 8; ++m) {
                    uint32_t a[4];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int q = 2 * m + e, c = (q & 3) * 4 + (q >> 2);
#pragma unroll
                        for (int j = 0; j < 2; ++j) a[e + 2 * j] = prmt(word(2 * j, c >> 1), word(2 * j + 1, c >> 1), c & 1 ? 0x7632 : 0x5410);
                    }
                    mma16816(o[m], a[0], a[1], a[2], a[3], b0, b1);
                }
            }
        }
#pragma unroll
        for (int m = 0; m < 8; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (2 * t + (e & 1) < rows) s_out[(2 * t + (e & 1)) * 128 + few_element<1>(g, m, e >> 1)] = o[m][e];
    }
    const float aside_ref = ref;

    // ---- packed pages
    float out[VT][4], out_mn[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int m = 0; m < VT; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) out[m][e] = 0.f;
    // values' columns: group and row of B's column g, and of the accumulators' columns 2t, 2t + 1 (VPAIR: hi and lo of one row)
    constexpr bool VPAIR = KB != 3 && VB != 3 && CK == 1;
    const int vr_log2 = VB == 3 ? 3 : (VPAIR ? 2 : 3) - ng_log2, v_col = VPAIR ? g >> 1 : g, o_col = VPAIR ? t : 2 * t;
    const int v_grp = v_col >> vr_log2, v_row = min(v_col & ((1 << vr_log2) - 1), R - 1), o_row = o_col & ((1 << vr_log2) - 1), o_grp = o_col >> vr_log2;
    const int o_row1 = VPAIR ? o_row : o_row + 1;
    const uint32_t v_lo = VPAIR && (g & 1) ? 0xffffffffu : 0u;
    // p * scale * 2^expo: the power of two starts from the first scales (the largest of them becomes 4 to 8) and follows them where a stage's largest
    // would exceed 256 or stay below 2^-5; the sums so far go along, exactly
    int expo = 32;
    // q * scale * 2^lift: 0 wherever a look at some of a stage's scales finds one of 2^-5 or more.  Below that what the pair hi + lo has under 2^-24 would be
    // lost (5e-3 of a score for 4-bit keys of 1e-4); the largest scale becomes 4 to 8 then, in place, so that usual ones cost the look alone.
    int lift = 0;
#pragma unroll 1
    for (int k = 0; k < n_mine; ++k) {
        if (k == ids_base + 32) { fetch_ids(k); produce(); }
        if (id_of(k) < 0) continue;
        if constexpr (KB == 3) {
            float sc[11][4];
#pragma unroll
            for (int m = 0; m < 11; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[m][e] = 0.f;
#pragma unroll 1
            for (int q = 0; q < half_stages; ++q) {
                const uint32_t c = stage_ready();
                if (!ok) break;
                const __half *qv = s_qs + min(g, R - 1) * 128 + q * stage_rows + 4 * t;
#pragma unroll 1
                for (int row = 0; row < stage_rows; row += 16) {
                    const uint2 b = *reinterpret_cast<const uint2 *>(qv + row);
                    few_step3(sc, c, c + k_cb, c + k_cb + k_sz, row, g, t, b.x, b.y);
                }
                stage_done();
            }
            if (!ok) break;
            dense_scores(sc, [&](int m, int e) { return few_element<3>(g, m, e); });
        } else {
            float sc[CK][8][4], z[CK][4];
            int row[CK], grp[CK];                                 // of B's column g of each set: pairs (hi, lo) of (group, row)
            const int kr_log2 = 1 + CK - ng_log2;                 // log2 of the rows that 4 CK pairs hold
#pragma unroll
            for (int n = 0; n < CK; ++n) {
                const int pair = 4 * n + (g >> 1);
                row[n] = pair & ((1 << kr_log2) - 1);
                grp[n] = pair >> kr_log2;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    z[n][e] = 0.f;
#pragma unroll
                    for (int m = 0; m < 8; ++m) sc[n][m][e] = 0.f;
                }
            }
            const uint32_t lo_mask = g & 1 ? 0xffffffffu : 0u;
#pragma unroll 1
            for (int q = 0; q < half_stages; ++q) {
                const uint32_t c = stage_ready(), c_sc = c + k_cb, c_mn = c_sc + k_sz;
                if (!ok) break;
                const int words = stage_rows * p.k_groups / 2;
                const uint32_t look = lds32(c_sc + 4 * min(lane, words - 1));
                if (lift || !__any_sync(0xffffffffu, max(look & 0xffffu, look >> 16) >= 0x2800u)) {
                    uint32_t m2 = 0;
                    for (int w = lane; w < words; w += 32) m2 = as_u32(__hmax2(as_h2(m2), as_h2(lds32(c_sc + 4 * w))));
                    const int top = (int)(__reduce_max_sync(0xffffffffu, max(m2 & 0xffffu, m2 >> 16)) >> 10 & 31), old = lift;
                    if (top + lift > 15 + 7 || top + lift < 10) lift = min(max(17 - top, 0), 15);
                    for (int w = lane; lift && w < words; w += 32)
                        asm volatile("st.shared.b32 [%0], %1;\n" ::"r"(c_sc + 4 * w), "r"(as_u32(__hmul2(as_h2(lds32(c_sc + 4 * w)), as_h2((uint32_t)(lift + 15) * 0x04000400u)))) : "memory");
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");       // the next copy into this place is the async proxy's
                    __syncwarp();
                    if (lift != old) {
                        const float f = exp2f((float)(lift - old));
#pragma unroll
                        for (int n = 0; n < CK; ++n)
#pragma unroll
                            for (int m = 0; m < 8; ++m)
#pragma unroll
                                for (int e = 0; e < 4; ++e) sc[n][m][e] *= f;
                    }
                }
                const __half *q_at = s_qs + q * stage_rows + 4 * t;
#pragma unroll 1
                for (int at = 0; at < stage_rows; at += 16) {
                    const FewWords<KB> a(c, at, g, t);
                    uint32_t mn[2], b[CK][2];
                    few_pairs(c_mn, at, t, p.k_groups, g & (p.k_groups - 1), mn);              // rows beyond the groups are not read
#pragma unroll
                    for (int n = 0; n < CK; ++n) {
                        const uint2 qv = *reinterpret_cast<const uint2 *>(q_at + row[n] * 128 + at);
                        uint32_t sv[2];
                        few_pairs(c_sc, at, t, p.k_groups, grp[n], sv);
                        b[n][0] = hilo(as_h2(qv.x), as_h2(sv[0]), lo_mask);
                        b[n][1] = hilo(as_h2(qv.y), as_h2(sv[1]), lo_mask);
                        mma16816(z[n], mn[0], 0u, mn[1], 0u, qv.x & ~lo_mask, qv.y & ~lo_mask);
                    }
#pragma unroll
                    for (int m = 0; m < 8; ++m) {
                        const uint32_t a0 = a.a(m, 0), a1 = a.a(m, 1), a2 = a.a(m, 2), a3 = a.a(m, 3);
#pragma unroll
                        for (int n = 0; n < CK; ++n) mma16816(sc[n][m], a0, a1, a2, a3, b[n][0], b[n][1]);
                    }
                }
                stage_done();
            }
            if (!ok) break;
            const float undo = __int_as_float((127 - lift) << 23);
#pragma unroll
            for (int n = 0; n < CK; ++n) {
                const int pair = 4 * n + t, r = pair & ((1 << kr_log2) - 1);
                const float zero = __shfl_sync(0xffffffffu, z[n][0], 4 * own_group + t);
                if (pair >> kr_log2 == own_group && r < rows) {
#pragma unroll
                    for (int m = 0; m < 8; m += 2) {
                        float v[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = fmaf(sc[n][m + (e >> 1)][2 * (e & 1)] + sc[n][m + (e >> 1)][2 * (e & 1) + 1], few_power<KB>(m + (e >> 1), e & 1) * undo, zero);
                        sts_f4(s_s + r * 512 + (16 * g + 2 * m) * 4, v[0], v[1], v[2], v[3]);
                    }
                }
            }
        }
        if (softmax_page(page_at(k) * kPage, kPage)) {
            rescale(out, o_row, o_row1);
            if constexpr (VB != 3) {
                const float a0 = __shfl_sync(0xffffffffu, alpha, o_row), a1 = __shfl_sync(0xffffffffu, alpha, o_row1);
                out_mn[0] *= a0;
                out_mn[1] *= a1;
            }
        }
#pragma unroll 1
        for (int q = 0; q < half_stages; ++q) {
            const uint32_t c = stage_ready(), c_sc = c + v_cb, c_mn = c_sc + v_sz;
            if (!ok) break;
            const int step0 = q * (stage_rows / 16);
            if constexpr (VB == 3) {
#pragma unroll 1
                for (int at = 0; at < stage_rows; at += 16) {
                    uint32_t b0, b1;
                    weights(min(g, R - 1), step0 + at / 16, b0, b1);
                    few_step3(out, c, c_sc, c_mn, at, g, t, b0, b1);
                }
            } else {
                // the exponent of the stage's largest scale: its scales are stage_rows * groups / 32 a lane, two at a time
                uint32_t m2 = 0;
                for (int w = lane; w < stage_rows * p.v_groups / 2; w += 32) m2 = as_u32(__hmax2(as_h2(m2), as_h2(lds32(c_sc + 4 * w))));
                const int top = (int)(__reduce_max_sync(0xffffffffu, max(m2 & 0xffffu, m2 >> 16)) >> 10 & 31);
                if (top + expo > 15 + 7 || (top + expo < 10 && top > 0)) {        // rare: the first stage, and where scales grow or shrink some 2^6 fold
                    const int want = min(max(17 - top, -13), 15);
                    if (want != expo) {
                        const float f = expo == 32 ? 0.f : exp2f((float)(want - expo));
#pragma unroll
                        for (int m = 0; m < 8; ++m)
#pragma unroll
                            for (int e = 0; e < 4; ++e) out[m][e] *= f;
                        expo = want;
                    }
                }
                const __half2 by = as_h2((uint32_t)(expo + 15) * 0x04000400u);
#pragma unroll 1
                for (int at = 0; at < stage_rows; at += 16) {
                    const FewWords<VB> a(c, at, g, t);
                    uint32_t b0, b1, mn[2], sv[2];
                    weights(v_row, step0 + at / 16, b0, b1);
                    few_pairs(c_mn, at, t, p.v_groups, g & (p.v_groups - 1), mn);
                    few_pairs(c_sc, at, t, p.v_groups, v_grp, sv);
                    const __half2 s0 = __hmul2(as_h2(sv[0]), by), s1 = __hmul2(as_h2(sv[1]), by);
                    if constexpr (VPAIR) {
                        mma16816(out_mn, mn[0], 0u, mn[1], 0u, b0 & ~v_lo, b1 & ~v_lo);
                        b0 = hilo(as_h2(b0), s0, v_lo);
                        b1 = hilo(as_h2(b1), s1, v_lo);
                    } else {
                        mma16816(out_mn, mn[0], 0u, mn[1], 0u, b0, b1);
                        b0 = as_u32(__hmul2(as_h2(b0), s0));
                        b1 = as_u32(__hmul2(as_h2(b1), s1));
                    }
#pragma unroll
                    for (int m = 0; m < 8; ++m) mma16816(out[m], a.a(m, 0), a.a(m, 1), a.a(m, 2), a.a(m, 3), b0, b1);
                }
            }
            stage_done();
        }
        if (!ok) break;
    }
    if (!ok)                                                      // copies in flight land before the memory is given up
        for (; in_flight > 0; --in_flight) {
            mbar_wait(s_bar + 8 * use_slot, parity, &p.b.count[2]);
            if (++use_slot == stages) { use_slot = 0; parity ^= 1; }
        }

    // ---- the warps' parts meet: sums put aside and sums of packed pages under the last reference
    const float aside_by = ref == -INFINITY ? 0.f : exp2_approx(aside_ref - ref);         // of row `lane`
    __syncwarp();
    auto add = [&](int r, int c, float v, float by) { s_out[r * 128 + c] = fmaf(s_out[r * 128 + c], by, v); };
    if constexpr (VB == 3) {
        const float f0 = __shfl_sync(0xffffffffu, aside_by, 2 * t), f1 = __shfl_sync(0xffffffffu, aside_by, 2 * t + 1);
#pragma unroll
        for (int m = 0; m < 11; ++m)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int c = few_element<3>(g, m, e);
                if (c >= 0 && 2 * t < rows) add(2 * t, c, out[m][2 * e], f0);
                if (c >= 0 && 2 * t + 1 < rows) add(2 * t + 1, c, out[m][2 * e + 1], f1);
            }
    } else {
        const float f0 = __shfl_sync(0xffffffffu, aside_by, o_row), f1 = __shfl_sync(0xffffffffu, aside_by, o_row1);
        const float z0 = __shfl_sync(0xffffffffu, out_mn[0], 4 * own_group + t), z1 = __shfl_sync(0xffffffffu, out_mn[1], 4 * own_group + t);
        const float undo = expo == 32 ? 0.f : exp2f((float)-expo);
        if (o_grp == own_group) {
#pragma unroll
            for (int m = 0; m < 8; ++m)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int c = few_element<1>(g, m, e);
                    const float f = few_power<VB>(m, e) * undo;
                    if (o_row < rows) add(o_row, c, fmaf(VPAIR ? out[m][2 * e] + out[m][2 * e + 1] : out[m][2 * e], f, z0), f0);
                    if (!VPAIR && o_row1 < rows) add(o_row1, c, fmaf(out[m][2 * e + 1], f, z1), f1);
                }
        }
    }
    __syncwarp();
    // reference and sum of weights of row `lane`, over the first scores
    float l = 0.f;
    if (lane < rows)
        for (int j = 0; j < 32; ++j) l += __uint_as_float(lds32(s_sum + lane * 128 + 4 * j));
    if (lane < rows) asm volatile("st.shared.v2.f32 [%0], {%1, %2};\n" ::"r"(s_s + lane * 8), "f"(ref), "f"(l) : "memory");
    __syncthreads();
    for (int r = 0; r < rows; ++r) {
        float m = -INFINITY, v = 0.f;
        l = 0.f;
        auto part = [&](int w) { return reinterpret_cast<const float *>(smem + sh.warps + w * sh.warp_bytes + sh.scores) + 2 * r; };
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) m = fmaxf(m, part(w)[0]);
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) {
            const float f = part_factor(part(w)[0], part(w)[1], m);
            l += f * part(w)[1];
            if (f != 0.f) v += f * reinterpret_cast<const float *>(smem + sh.warps + w * sh.warp_bytes + sh.aside)[r * 128 + threadIdx.x];
        }
        const int u = s.q0 + (row0 + r) / p.rep, h = head * p.rep + (row0 + r) % p.rep;
        if (p.splits == 1) {
            static_cast<__half *>(p.a.out)[(int64_t)u * p.a.o_sT + (int64_t)h * p.a.o_sH + threadIdx.x] = __float2half_rn(l == 0.f ? 0.f : v / l);
        } else {
            const int64_t at = (int64_t)split * p.part_rows + (p.part_compact ? ((int64_t)i * p.l.Hkv + head) * kFewRows + row0 + r : (int64_t)u * p.a.nh + h);
            p.part_out[at * 128 + threadIdx.x] = v;
            if (threadIdx.x == 0) { p.part_ml[2 * at] = m; p.part_ml[2 * at + 1] = l; }
        }
    }
}

template <int KB, int VB, int CK>
static int launch_few(const PagedArgs &p, int R, int row_blocks, cudaStream_t st) {
    const int k_row = 4 * page_words(KB) + 4 * p.k_groups, v_row = 4 * page_words(VB) + 4 * p.v_groups, row = k_row > v_row ? k_row : v_row;
    const int ctas = KB == 3 || VB == 3 || CK == 2 ? 3 : 4;
    // what 227 KB leave each of the CTAs of an SM (1 KB of each is the system's): two stages at least, of as many rows as that allows (a stage costs some
    // 100 instructions besides its rows)
    const int room = (227 * 1024 / ctas - 1024 - FewShared(R, 0, 0).total) / kFewWarps;
    int stage_rows = kPage;
    while (stage_rows > 32 && 2 * stage_rows * row > room) stage_rows /= 2;
    const int stage_bytes = stage_rows * row;
    int stages = room / stage_bytes;
    stages = stages < 2 ? 2 : stages > kMaxStages ? kMaxStages : stages;
    const size_t smem = FewShared(R, stages, stage_bytes).total;
    const cudaError_t e = cudaFuncSetAttribute(paged_few_kernel<KB, VB, CK>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return record_cuda_error(e);
    const int64_t grid = (int64_t)p.a.n * p.l.Hkv * row_blocks * p.splits;
    if (grid > 2147483647LL) return KVQ_ERR_UNSUPPORTED;
    paged_few_kernel<KB, VB, CK><<<(unsigned)grid, kFewWarps * 32, smem, st>>>(p, R, row_blocks, stages, stage_rows, stage_bytes);
    return count_launch();
}

template <int KB, int VB>
static int launch_few(const PagedArgs &p, cudaStream_t st) {
    const FewShape f = few_shape(p.l, p.rep, p.a.max_new);
    if constexpr (KB != 3)
        if (f.key_sets == 2) return launch_few<KB, VB, 2>(p, f.rows, f.row_blocks, st);
    return launch_few<KB, VB, 1>(p, f.rows, f.row_blocks, st);
}

template <int KB>
static int launch_few(const PagedArgs &p, cudaStream_t st) {
    switch (p.l.v_bits) {
        case 1: return launch_few<KB, 1>(p, st);
        case 2: return launch_few<KB, 2>(p, st);
        case 3: return launch_few<KB, 3>(p, st);
        default: return launch_few<KB, 4>(p, st);
    }
}

}  // namespace kvq
