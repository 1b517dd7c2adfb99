// Attention of many query rows of a kv head (chunks of new tokens, more than 8 query heads a kv head) over a paged cache, on tcgen05.  A source
// file for each width of the keys (paged_tiles_1.cu ..): their instances build side by side.
#pragma once
#include "paged_attn.cuh"
#include "quant_core.cuh"

#include <cuda.h>

namespace kvq {

// A CTA takes 256 rows -- (token, query head of the group) pairs of one sequence and kv head, as two tiles of 128 -- and walks the pages
// that any of them sees.  A page is one step of both products:
//   S = Q K^T   128 x 128 x 128, Q and K in shared memory, S (fp32) in TMEM
//   O += P V    P, the weights as fp16, over S in TMEM; V in shared memory; O (fp32) in TMEM
// Twenty-four warps: four warpgroups of softmax, two per tile, half a row a thread (a row a thread: the same time for plain scores, 221 in place of
// 190 us for four capped chunks of 501 tokens); one that fills the operand buffers; a warp that issues the MMAs and a thread that issues
// copies.  While one tile's scores are worked on, the tensor core multiplies for the other.  TMEM: S0 S1 O0 O1, 128 columns each.
// Bound: a page is 2048 cycles of MMA and as many of the special function unit (one exponential a score) and takes some 3200; under it the
// card runs at its power limit (1.5 to 1.6 GHz).  2048 tokens x 32 heads over 34816: 990 to 1050 TFLOP/s from card to card, 0.61 to 0.64 of the rate measured
// in bursts and 0.73 to 0.77 of the sustained one.  Tried without gain: a part of the exponentials as polynomials (2 to 20 % slower), weights handed over in quarters.
//
// Operand buffers hold 128 rows of 128 fp16 as two halves of 64 (128 bytes a row, 16-byte pieces swizzled by the row's number).  Rows are
// tokens of fp16 pages and of packed values, channels of packed keys: what is contiguous in a row is the contraction axis of fp16 keys (K-major
// operand) and the axis of output columns of everything else (MN-major operand), so that packed words are spread where
// their fields lie side by side and nothing is transposed.
// Packed rows become fp16 as code * scale + minimum with one rounding (2^-11 relative): the tensor core takes no wider operand without
// half its rate.
constexpr int kTileRows = 128, kTileThreads = 768;
constexpr uint32_t kOperandBytes = 32768, kOperandHalf = 16384;
constexpr int kRawBytes = 12288;                                  // the largest packed half of a page: 3 bits, or 4 bits and groups of 32
// shared memory, from a 1024-byte boundary
constexpr uint32_t kOffQ = 0, kOffK = 2 * kOperandBytes, kOffV = kOffK + 2 * kOperandBytes, kOffRaw = kOffV + 2 * kOperandBytes,
                   kOffBar = kOffRaw + 2 * kRawBytes, kOffTop = kOffBar + 256, kTileSmem = kOffTop + 2 * 2 * 2 * kTileRows * 4;      // tops: page, tile, half
// barriers
constexpr int kBarKFull = 1, kBarKFree = 3, kBarVFull = 5, kBarVFree = 7, kBarS = 9, kBarP = 11, kBarO = 13, kBarRaw = 14, kBarRawFree = 16, kBarDrain = 18, kBarTail = 19;

// fp16 pages as rows of 128 channels, for copies of 64 channels x 128 rows that swizzle on the way
struct PagedMaps {
    CUtensorMap k, v;
    int there;                        // whether they are (pools of 2^31 rows and more have none)
};
__device__ __forceinline__ void tile_load(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
// One thread (`lead`) issues an MMA or a commit, but its whole warp walks there with values that are the same in all lanes: operands then
// stand in uniform registers, where these instructions want them.  In a branch of that thread alone each descriptor was moved there
// word by word: a page took 4400 cycles, and 3200 so.
__device__ __forceinline__ void tc_commit(uint32_t bar, uint32_t lead) {
    asm volatile("{\n.reg .pred q;\nsetp.ne.u32 q, %1, 0;\n@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar), "r"(lead) : "memory");
}
// Operand descriptor: swizzle of 128 bytes; `lbo`, `sbo` in bytes (see the layouts above).
__device__ __forceinline__ uint64_t tc_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr & 0x3ffff) >> 4) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(sbo >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// fp16 x fp16 -> fp32, M = N = 128; bit 16: B is MN-major
constexpr uint32_t kIdesc = 1u << 4 | (128u >> 3) << 17 | (128u >> 4) << 24, kIdescMn = kIdesc | 1u << 16;

__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add, uint32_t lead) {
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %4, 0;\nsetp.ne.u32 q, %5, 0;\n@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add), "r"(lead) : "memory");
}
__device__ __forceinline__ void tc_mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add, uint32_t lead) {
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %4, 0;\nsetp.ne.u32 q, %5, 0;\n@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add), "r"(lead) : "memory");
}

#define KVQ_R8(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7])
#define KVQ_W8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])
// 32 or 16 columns of this thread's row
__device__ __forceinline__ void tc_load32(uint32_t (&r)[32], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
                 : KVQ_R8(r, 0), KVQ_R8(r, 8), KVQ_R8(r, 16), KVQ_R8(r, 24) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tc_load16(uint32_t (&r)[16], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n" : KVQ_R8(r, 0), KVQ_R8(r, 8) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tc_store16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(addr), KVQ_W8(r, 0), KVQ_W8(r, 8) : "memory");
}

// Piece c (16 bytes, 0..15) of row r of an operand buffer
__device__ __forceinline__ uint32_t operand_at(uint32_t base, int r, int c) { return base + (c >> 3) * kOperandHalf + r * 128 + (((c & 7) ^ (r & 7)) << 4); }
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// One packed row -> 128 fp16 of an operand row.
template <int BITS, int NG>
__device__ __forceinline__ void unpack_row(uint32_t raw, uint32_t to, int r) {
    constexpr int W = page_words(BITS);
    const uint32_t codes = raw + r * W * 4, scale = raw + kPage * W * 4 + r * NG * 2, mn = scale + kPage * NG * 2;
    uint32_t w[W];
#pragma unroll
    for (int k = 0; k < W; k += 4) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(w[k]), "=r"(w[k + 1]), "=r"(w[k + 2]), "=r"(w[k + 3]) : "r"(codes + 4 * k));
    uint32_t sc[NG], lo[NG];                                      // both halves alike
    uint32_t out[4];
    if constexpr (BITS == 3) {
        // Twelve scales and minima in six wide loads: loads wait in one queue with the exponentials of the other warps, some 40 cycles each.  Words hold eleven fields: neighbours
        // stand at the same place of a word's half and of the half three bits on, and every other word begins in mid-pair.  (2048 tokens over 16k, K3V3: 622 -> 508 us, two
        // maps 1124 -> 844, against a load a scale and a shift and a mask a field.  The other widths have few scales; wide loads there cost as much as they gave.)
        uint32_t x[2][NG / 2];
#pragma unroll
        for (int k = 0; k < NG; k += 2)
            asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];\n" : "=r"(x[k >= NG / 2][k % (NG / 2)]), "=r"(x[k >= NG / 2][k % (NG / 2) + 1]) : "r"((k < NG / 2 ? scale : mn) + 4 * (k % (NG / 2))));
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            sc[k] = prmt(x[0][k / 2], 0, k & 1 ? 0x3232 : 0x1010);
            lo[k] = prmt(x[1][k / 2], 0, k & 1 ? 0x3232 : 0x1010);
        }
#pragma unroll
        for (int i = 0; i < 64; ++i) {
            const int a = 2 * i / 11, b = (2 * i + 1) / 11, f = 2 * i % 11, by = 3 * (f & 1) + (f < 6 ? 0 : 18), at = 3 * f - by, pos = a != b || at == 0 ? 0 : 6;
            const uint32_t pair = a != b ? prmt(w[a] >> 30, w[b], 0x5410) : prmt(w[a] >> by, w[a] >> (by + 3), 0x5410), expo = (uint32_t)(25 - pos) << 10;
            uint32_t v;
            asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(v) : "r"(a == b && at == 12 ? pair >> 6 : pair), "r"((7u << pos) * 0x10001u), "r"(expo * 0x10001u));
            const uint32_t s2 = a == b ? sc[a] : prmt(sc[a], sc[b], 0x5410), l2 = a == b ? lo[a] : prmt(lo[a], lo[b], 0x5410);
            out[i & 3] = as_u32(__hfma2(__hsub2(as_h2(v), as_h2(expo * 0x10001u)), as_h2(s2), as_h2(l2)));
            if ((i & 3) == 3) sts128(operand_at(to, r, i >> 2), out[0], out[1], out[2], out[3]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < NG; ++k) { sc[k] = lds16(scale + 2 * k) * 0x10001u; lo[k] = lds16(mn + 2 * k) * 0x10001u; }
        constexpr int PAIRS = 8 / BITS, DIRECT = (10 - BITS) / (2 * BITS) + 1;      // pairs of neighbours in a half word; in reach without a shift
#pragma unroll
        for (int i = 0; i < 64; ++i) {                            // elements 2i, 2i + 1
            const int half = i / PAIRS, f = i % PAIRS, k = half / 2, g = 2 * i / (kPage / NG);
            const uint32_t x = prmt(w[k], w[k] >> BITS, half & 1 ? 0x7632 : 0x5410);
            const int pos = f < DIRECT ? 2 * BITS * f : 2 * BITS * (f - DIRECT);
            const uint32_t mask = ((1u << BITS) - 1u) << pos, expo = (uint32_t)(25 - pos) << 10;
            uint32_t v;
            asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(v) : "r"(f < DIRECT ? x : x >> (2 * BITS * DIRECT)), "r"(mask * 0x10001u), "r"(expo * 0x10001u));
            out[i & 3] = as_u32(__hfma2(__hsub2(as_h2(v), as_h2(expo * 0x10001u)), as_h2(sc[g]), as_h2(lo[g])));
            if ((i & 3) == 3) sts128(operand_at(to, r, i >> 2), out[0], out[1], out[2], out[3]);
        }
    }
}
template <int BITS>
__device__ __forceinline__ void unpack_row(uint32_t raw, uint32_t to, int r, int groups) {
    if constexpr (BITS == 3) {
        unpack_row<3, 12>(raw, to, r);
    } else {
        if (groups == 1) unpack_row<BITS, 1>(raw, to, r);
        else if (groups == 2) unpack_row<BITS, 2>(raw, to, r);
        else unpack_row<BITS, 4>(raw, to, r);
    }
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// cap_small() of two raw scores in log2 units.  in: raw score -> x; by: tanh -> log2 units, in the coefficients.  (With `in` there too the higher ones,
// in^9 and in^7, left fp32 where scale / softcap is small.)  Seven instructions for both where cap_score() takes some thirty and four turns
// of the special function unit.
struct CapSmall {
    float c[5];
    unsigned long long in2;
    __device__ __forceinline__ CapSmall(float in, float by) : in2(f32x2(in, in)) {
#pragma unroll
        for (int i = 0; i < 5; ++i) c[i] = cap_poly(i) * by;
    }
    __device__ __forceinline__ unsigned long long operator()(unsigned long long raw, float &most) const {       // most: the largest square
        const unsigned long long x = mul_f32x2(raw, in2), t = mul_f32x2(x, x);
        const float2 squares = f32x2_split(t);
        most = max3(most, squares.x, squares.y);
        unsigned long long r = f32x2(c[4], c[4]);
#pragma unroll
        for (int i = 3; i >= 0; --i) r = fma_f32x2(r, t, f32x2(c[i], c[i]));
        return mul_f32x2(x, r);
    }
};

// MODS: scores are capped, biased or scaled by a negative number.  Calls without have an instance of their own: with the code beside it the
// 128 scores of a thread no longer fit its registers (2048 tokens over 32k: 1261 us in place of 1132).
// DIFF: heads are two rows each (PagedArgs); the two tiles are the two maps of the same 128 rows -- (token, query head) pairs --, a map's scores the product of
// half the channels, and the map of the second half hands its part of the output over in shared memory.  A page is as many exponentials as with two tiles of
// rows and three quarters of the products, and takes as long (some 3000 cycles; 59 % of the special function unit, 44 % of the tensor core over fp16 pages).  Softmax threads
// have 96 registers (512 x 96 + 128 x 56 + 128 x 40 is what the CTA was launched with): 1777 -> 1727 us for a chunk of 2048 over 32k tokens.  Half a page a turn, so that
// scores are there before weights are done: 2225 us.
template <int KB, int VB, bool MODS, bool DIFF>
__global__ void __launch_bounds__(kTileThreads, 1) paged_tile_kernel(const __grid_constant__ PagedArgs p, const __grid_constant__ PagedMaps maps, int max_tiles) {
    extern __shared__ __align__(1024) char smem[];
    __shared__ uint32_t s_tmem;
    // where this CTA's rows are: tiles of later tokens first, they see more
    const bool whole = DIFF && (int)blockIdx.x < p.n_whole;
    auto splits = [&]() { return DIFF && whole ? 1 : p.splits; };
    const unsigned cta = blockIdx.x - (DIFF ? p.n_whole : 0);
    const int split = DIFF && whole ? 0 : cta % p.splits, hs = DIFF && whole ? blockIdx.x : cta / p.splits + (DIFF ? p.n_whole : 0), head = hs % p.l.Hkv;
    int tile = max_tiles - 1 - hs / p.l.Hkv, seq = 0;
    auto tiles_of = [&](int i) {
        int q0, n_new;
        new_tokens(p, i, q0, n_new);
        const int rows = max(0, n_new) * p.rep;
        return rows > p.few_rows ? (rows + 2 * kTileRows - 1) / (2 * kTileRows) : 0;
    };
    if (p.a.n <= 8) {
        for (; seq < p.a.n; ++seq) {
            const int tiles = tiles_of(seq);
            if (tile < tiles) break;
            tile -= tiles;
        }
        if (seq == p.a.n) return;
    } else {                                                      // many sequences, one a thread
        __shared__ int s_sum[kTileThreads / 32], s_seq, s_tile;
        if (threadIdx.x == 0) s_seq = -1;
        for (int at = 0; at < p.a.n; at += kTileThreads) {
            const int i = at + threadIdx.x, mine = i < p.a.n ? tiles_of(i) : 0;
            int upto = mine, all = 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, upto, o);
                if ((threadIdx.x & 31) >= o) upto += y;
            }
            if ((threadIdx.x & 31) == 31) s_sum[threadIdx.x >> 5] = upto;
            __syncthreads();
            for (int w = 0; w < kTileThreads / 32; ++w) {
                all += s_sum[w];
                if (w < (int)(threadIdx.x >> 5)) upto += s_sum[w];
            }
            if (tile >= upto - mine && tile < upto) { s_seq = i; s_tile = tile - (upto - mine); }
            __syncthreads();
            if (tile < all) break;
            tile -= all;
        }
        seq = s_seq;
        if (seq < 0) return;
        tile = s_tile;
    }
    int q0, n_new;
    new_tokens(p, seq, q0, n_new);                                // as paged_seq has them, which waits for more loads
    const int rep = DIFF ? p.rep / 2 : p.rep, tile_rows = DIFF ? kTileRows : 2 * kTileRows;
    const int row0 = tile * tile_rows, rows = min(n_new * rep - row0, tile_rows), two_tiles = DIFF || rows > kTileRows;
    const int warp = uniform_warp(), lane = threadIdx.x & 31, wg = warp >> 2;

    const uint32_t base = smem_u32(smem), bars = base + kOffBar;
    // Q, 16 threads a row, asked for before anything that does not have to come first: a row a thread, after the barrier, the same loads took 6 us
    // of a CTA that has some 30 us of pages
    constexpr int kTurns = DIFF ? 3 : 6;
    uint4 qv[kTurns];
    {
        const bool vec = (reinterpret_cast<uintptr_t>(p.a.q) % 16 | p.a.q_sT % 8 | p.a.q_sH % 8) == 0;
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
            const int row = (threadIdx.x >> 4) + 48 * i, idx = row0 + row, u = idx / rep, h = head * rep + (idx - u * rep);
            const __half *q = static_cast<const __half *>(p.a.q) + (int64_t)(q0 + u) * p.a.q_sT + (int64_t)h * p.a.q_sH + 8 * (threadIdx.x & 15);
            qv[i] = make_uint4(0, 0, 0, 0);
            if (row >= rows) continue;
            if (vec) qv[i] = *reinterpret_cast<const uint4 *>(q);
            else {
                alignas(16) __half y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = q[j];
                qv[i] = *reinterpret_cast<const uint4 *>(y);
            }
        }
    }
    const PagedSeq s = paged_seq(p, seq);
    auto bar = [&](int k) { return bars + 8 * k; };
    if (threadIdx.x == 0) {
        for (int k = 0; k < 2; ++k) {
            mbar_init(bar(kBarKFull + k), 1);
            mbar_init(bar(kBarKFree + k), 1);
            mbar_init(bar(kBarVFull + k), 1);
            mbar_init(bar(kBarVFree + k), 1);
            mbar_init(bar(kBarS + k), 1);
            mbar_init(bar(kBarP + k), 256);
            mbar_init(bar(kBarRaw + k), 1);
            mbar_init(bar(kBarRawFree + k), 1);
        }
        for (int k = 0; k < 4; ++k) mbar_init(bar(kBarTail + k), 1);
        mbar_init(bar(kBarO), 1);
        mbar_init(bar(kBarDrain), 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 20) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_u32(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
    }
    // the pages that any row sees: bounds of the first and last tokens hold for those between, unless they are given token by token
    int first = INT32_MAX, last = 0;
    {
        const int u0 = row0 / rep, u1 = (row0 + rows - 1) / rep;
        for (int u = u0 + threadIdx.x; u <= u1; u += kTileThreads) {
            int pos, lo, hi;
            paged_bounds(p, s, u, pos, lo, hi);
            if (lo < hi) { first = min(first, lo); last = max(last, hi); }
        }
        first = (int)__reduce_min_sync(0xffffffffu, (unsigned)first);
        last = (int)__reduce_max_sync(0xffffffffu, (unsigned)last);
        __shared__ int s_first[kTileThreads / 32], s_last[kTileThreads / 32];
        if (lane == 0) { s_first[warp] = first; s_last[warp] = last; }
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
            const int row = (threadIdx.x >> 4) + 48 * i;
            if (row < tile_rows) sts128(operand_at(base + kOffQ + (row >> 7) * kOperandBytes, row & 127, threadIdx.x & 15), qv[i].x, qv[i].y, qv[i].z, qv[i].w);
        }
        fence_async();
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
#pragma unroll
        for (int w = 0; w < kTileThreads / 32; ++w) { first = min(first, s_first[w]); last = max(last, s_last[w]); }
    }
    const uint32_t tmem = s_tmem;
    const int p_lo = first < last ? first / kPage : 0, p_hi = first < last ? pages_of(last) : 0, per = (p_hi - p_lo + splits() - 1) / splits();
    const int p0 = p_lo + split * per, np = max(0, min(p_hi, p0 + per) - p0);
    int32_t *const status = &p.b.count[2];
    auto page_id = [&](int page) {
        const int id = s.table[page];
        return id >= 0 && id < (page < s.packed ? p.l.n_packed : p.l.n_fp16) ? id : -1;
    };

    // Whether a full fp16 page comes by the loader's copies.  The others are filled by the warpgroup that unpacks, at the loader's word: a
    // barrier's parity tells a phase from the one before only, so whoever waits by it has to see every phase, and for the buffers of fp16
    // pages that is the loader.
    auto by_loader = [&](int page, int id) { return maps.there && (page + 1) * kPage <= s.length && id >= 0; };

    if (wg < 4) {
        // ------------------------------------------------------------------ softmax, 64 columns of one row a thread
        if constexpr (DIFF) asm volatile("setmaxnreg.inc.sync.aligned.u32 96;\n");
        else asm volatile("setmaxnreg.inc.sync.aligned.u32 88;\n");
        constexpr int N = 64;
        const int tile_of = wg >> 1, half = wg & 1, r = threadIdx.x & 127, at_row = DIFF ? r : tile_of * kTileRows + r, idx = row0 + at_row, u = idx / rep,
                  h = head * rep + (idx - u * rep);
        const bool mine = at_row < rows;
        if (tile_of == 0 || two_tiles) {
            int pos = 0, lo = 0, hi = 0;
            if (mine) paged_bounds(p, s, u, pos, lo, hi);
            const bool cap = MODS && p.a.softcap > 0.f, bias = MODS && p.a.slopes != nullptr, flip = MODS && !cap && !bias;
            const float scale2 = p.a.softmax_scale * kLog2e, cap2 = p.a.softcap * kLog2e;
            const float slope = bias && mine ? p.a.slopes[h] * kLog2e : 0.f, mul = cap || bias || flip ? 1.f : scale2;
            const uint32_t lanes = (uint32_t)(warp & 3) << 21, t_s = tmem + tile_of * 128 + lanes, t_o = tmem + 256 + tile_of * 128 + half * N + lanes;
            const uint32_t my_top = base + kOffTop + ((tile_of * 2 + half) * kTileRows + r) * 4, other_top = half ? my_top - kTileRows * 4 : my_top + kTileRows * 4;
            auto pair_meets = [&]() { asm volatile("bar.sync %0, 256;\n" ::"r"(2 + tile_of) : "memory"); };
            float m = -INFINITY, l = 0.f;
            bool ok = true;
            for (int it = 0; it < np; ++it) {
                const int page = p0 + it, b0 = page * kPage + half * N;
                const bool there = page_id(page) >= 0;
                ok = __all_sync(0xffffffffu, ok && mbar_wait(bar(kBarS + tile_of), it & 1, status));            // given up: through the barriers to the end
                tc_fence_after();
                uint32_t x[2][32];
#pragma unroll
                for (int c = 0; c < 2; ++c) tc_load32(x[c], t_s + half * N + 32 * c);
                tc_wait_ld();
                auto at = [&](int j) -> uint32_t & { return x[j >> 5][j & 31]; };
                auto pair = [&](int j) { return f32x2(__uint_as_float(at(j)), __uint_as_float(at(j + 1))); };
                auto put = [&](int j, unsigned long long v) {
                    const float2 w = f32x2_split(v);
                    at(j) = __float_as_uint(w.x);
                    at(j + 1) = __float_as_uint(w.y);
                };
                if (cap) {
                    const float small = p.cap_in;
                    // the polynomial for all first; where a square says that one was too large, the scores are read again
                    const CapSmall capped(small, cap2);
                    float most = 0.f;
#pragma unroll
                    for (int j = 0; j < N; j += 2) put(j, capped(pair(j), most));
                    if (!__all_sync(0xffffffffu, most <= kCapSmall * kCapSmall)) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) tc_load32(x[c], t_s + half * N + 32 * c);
                        tc_wait_ld();
#pragma unroll
                        for (int j = 0; j < N; ++j) at(j) = __float_as_uint(cap_score(__uint_as_float(at(j)) * small, cap2));
                    }
                }
                if (bias) {
                    unsigned long long b = f32x2(slope * (float)(b0 - pos), slope * (float)(b0 + 1 - pos));
                    const unsigned long long by = f32x2(cap ? 1.f : scale2, cap ? 1.f : scale2), step = f32x2(2.f * slope, 2.f * slope);
#pragma unroll
                    for (int j = 0; j < N; j += 2) {
                        // eight running sums drift by less than the rounding of a bias this large; started anew every 16 positions
                        if (j && j % 16 == 0) b = f32x2(slope * (float)(b0 + j - pos), slope * (float)(b0 + j + 1 - pos));
                        put(j, fma_f32x2(pair(j), by, b));
                        b = add_f32x2(b, step);
                    }
                } else if (flip) {
#pragma unroll
                    for (int j = 0; j < N; j += 2) put(j, mul_f32x2(pair(j), f32x2(scale2, scale2)));
                }
                if (!__all_sync(0xffffffffu, lo <= b0 && hi >= b0 + N && there)) {
                    const int from = there ? lo - b0 : N, to = there ? hi - b0 : 0;
#pragma unroll
                    for (int j = 0; j < N; ++j)
                        if (j < from || j >= to) at(j) = 0xff800000u;
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < N; j += 2) top[j >> 1 & 3] = max3(top[j >> 1 & 3], __uint_as_float(at(j)), __uint_as_float(at(j + 1)));
                // the other half of the row; two places by turns, so that one meeting a page is enough.  It also stands between the other half's reading
                // of S and the weights that are written over it.
                const float half_best = max3(max3(top[0], top[1], top[2]), top[3], top[3]) * mul;
                const uint32_t turn = (it & 1) * (4 * kTileRows * 4);
                asm volatile("st.shared.f32 [%0], %1;\n" ::"r"(my_top + turn), "f"(half_best) : "memory");
                tc_fence_before();
                pair_meets();
                tc_fence_after();
                const float best = max3(half_best, __uint_as_float(lds32(other_top + turn)), half_best);
                if (best != best) l = best;                       // a score is not a number: neither is the row
                // The reference follows the maximum only when it grows by more than 2^8: weights up to 256 are as exact in fp16, and O is
                // rescaled a few times a row in place of at every page.
                const bool grow = best > m + 8.f;
                if (__any_sync(0xffffffffu, grow)) {
                    const float f = grow ? exp2_approx(m - best) : 1.f;
                    if (grow) m = best;
                    l *= f;
                    if (it > 0) {
#pragma unroll 1
                        for (int c = 0; c < 4; ++c) {
                            uint32_t o[16];
                            tc_load16(o, t_o + 16 * c);
                            tc_wait_ld();
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                            tc_store16(t_o + 16 * c, o);
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.f : m;
                unsigned long long sum[2] = {0ull, 0ull};
                const unsigned long long mul2 = f32x2(mul, mul), ref2 = f32x2(-ref, -ref);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t w[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        float2 v = f32x2_split(fma_f32x2(pair(32 * c + 2 * j), mul2, ref2));
                        v.x = exp2_approx(v.x);
                        v.y = exp2_approx(v.y);
                        sum[j & 1] = add_f32x2(sum[j & 1], f32x2(v.x, v.y));
                        w[j] = as_u32(__floats2half2_rn(v.x, v.y));
                    }
                    tc_store16(t_s + half * 32 + 16 * c, w);
                }
                tc_wait_st();
                tc_fence_before();
                if (ok) mbar_arrive(bar(kBarP + tile_of));
                const float2 both = f32x2_split(add_f32x2(sum[0], sum[1]));
                l += both.x + both.y;
            }
            if (np > 0) ok = __all_sync(0xffffffffu, ok && mbar_wait(bar(kBarO), 0, status));
            tc_fence_after();
            asm volatile("st.shared.f32 [%0], %1;\n" ::"r"(my_top), "f"(l) : "memory");
            pair_meets();
            l = half ? __uint_as_float(lds32(other_top)) + l : l + __uint_as_float(lds32(other_top));
            const float inv = l == 0.f ? 0.f : 1.f / l;
            __half *out = static_cast<__half *>(p.a.out) + (int64_t)(s.q0 + u) * p.a.o_sT + (int64_t)h * p.a.o_sH + half * N;
            const int64_t part = DIFF && p.n_whole > 0 ? split * p.part_rows + (int64_t)(hs - p.n_whole) * 256 + 2 * r + tile_of
                                                       : split * p.part_rows + (int64_t)(s.q0 + u) * p.a.nh + (DIFF ? 2 * h + tile_of : h);
            const bool vec = (reinterpret_cast<uintptr_t>(p.a.out) % 16 | p.a.o_sT % 8 | p.a.o_sH % 8) == 0;
            if (DIFF && splits() == 1) {
                // The operand buffers are free: no copy and no product is under way.  A row's 16-byte pieces are mixed by its number.
                float *const other = reinterpret_cast<float *>(smem + kOffK);
                auto piece = [&](int k) { return reinterpret_cast<float4 *>(other + r * 128) + ((half * (N / 4) + k) ^ (r & 31)); };
                auto column = [&](uint32_t v) { return np == 0 || l == 0.f ? 0.f : __uint_as_float(v) * inv; };
                if (tile_of == 1) {
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        uint32_t o[16];
                        if (np > 0) {
                            tc_load16(o, t_o + 16 * c);
                            tc_wait_ld();
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) *piece(4 * c + j) = make_float4(column(o[4 * j]), column(o[4 * j + 1]), column(o[4 * j + 2]), column(o[4 * j + 3]));
                    }
                }
                asm volatile("bar.sync 4, 512;\n" ::: "memory");
                if (tile_of == 0) {
                    const float lambda = mine ? p.lambdas[h] : 0.f;
                    float y[N], squares = 0.f;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t o[16];
                        if (np > 0) {
                            tc_load16(o, t_o + 16 * c);
                            tc_wait_ld();
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float4 b = *piece(4 * c + j);
                            const float second[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const float v = diff_of(column(o[4 * j + k]), second[k], lambda);
                                y[16 * c + 4 * j + k] = v;
                                squares = fmaf(v, v, squares);
                            }
                        }
                    }
                    if (p.norm_weight) {
                        const uint32_t turn = 4 * kTileRows * 4;  // the place that the sums of weights are not in
                        asm volatile("st.shared.f32 [%0], %1;\n" ::"r"(my_top + turn), "f"(squares) : "memory");
                        pair_meets();
                        const float more = __uint_as_float(lds32(other_top + turn)), by = diff_norm(p, half ? more + squares : squares + more);
#pragma unroll
                        for (int j = 0; j < N; ++j) y[j] *= by * p.norm_weight[half * N + j];
                    }
                    if (mine) {
                        if (vec) {
#pragma unroll
                            for (int j = 0; j < N / 8; ++j) {
                                uint32_t w[4];
#pragma unroll
                                for (int k = 0; k < 4; ++k) w[k] = as_u32(__floats2half2_rn(y[8 * j + 2 * k], y[8 * j + 2 * k + 1]));
                                reinterpret_cast<uint4 *>(out)[j] = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < N; ++j) out[j] = __float2half_rn(y[j]);
                        }
                    }
                }
            } else {
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
                uint32_t o[16];
                __syncwarp();
                if (np > 0) {
                    tc_load16(o, t_o + 16 * c);
                    tc_wait_ld();
                }
                if (!mine) continue;
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (np == 0 || l == 0.f) o[j] = 0;
                if (splits() > 1) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) reinterpret_cast<uint4 *>(p.part_out + part * 128 + half * N + 16 * c)[j] = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
                } else {
                    uint32_t w[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j] = as_u32(__floats2half2_rn(__uint_as_float(o[2 * j]) * inv, __uint_as_float(o[2 * j + 1]) * inv));
                    if (vec) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) reinterpret_cast<uint4 *>(out + 16 * c)[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; ++j) out[16 * c + j] = __ushort_as_half((unsigned short)(w[j >> 1] >> (16 * (j & 1))));
                    }
                }
            }
            }
            if (mine && half == 0 && splits() > 1) {
                p.part_ml[2 * part] = m;
                p.part_ml[2 * part + 1] = l;
            }
            tc_fence_before();
        }
    } else if (wg == 4) {
        // ------------------------------------------------------------------ operands: job 2i is page i's keys, 2i + 1 its values.  Packed
        // ones are unpacked here, and the fp16 page that holds the sequence's end is copied here, with zeros behind the end.
        if constexpr (DIFF) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;\n");
        const int r = threadIdx.x & 127;
        bool ok = true;
        uint32_t tails = 0;
        for (int j = 0; j < 2 * np; ++j) {
            const int page = p0 + (j >> 1);
            const bool packed = page < s.packed;
            const int id = page_id(page);
            if (!packed && by_loader(page, id)) continue;
            const uint32_t to = base + (j & 1 ? kOffV : kOffK) + (j >> 1 & 1) * kOperandBytes, raw = base + kOffRaw + (j & 1) * kRawBytes;
            if (packed) {
                ok = ok && mbar_wait(bar((j & 1 ? kBarVFree : kBarKFree) + (j >> 1 & 1)), (j >> 2 & 1) ^ 1, status);
                ok = ok && mbar_wait(bar(kBarRaw + (j & 1)), j >> 1 & 1, status);
            } else {
                ok = ok && mbar_wait(bar(kBarTail + (j & 3)), tails >> (j & 3) & 1, status);
                tails ^= 1u << (j & 3);
            }
            ok = __all_sync(0xffffffffu, ok);                     // after a wait that gave up: through the barriers to the end, without work
            if (!ok) {
            } else if (packed && id >= 0) {
                if (j & 1) unpack_row<VB>(raw, to, r, p.v_groups);
                else unpack_row<KB>(raw, to, r, p.k_groups);
            } else {
                const __half *src = static_cast<const __half *>(j & 1 ? p.l.vfull : p.l.kfull) + ((int64_t)max(id, 0) * p.l.Hkv + head) * kPageHalf;
                const int there = id >= 0 ? min(kPage, s.length - page * kPage) : 0;      // a page without a number: zeros
#pragma unroll 4
                for (int c = 0; c < 16; ++c) {                    // eight rows of 16 pieces a turn
                    const int row = c * 8 + (r >> 4), piece = r & 15;
                    uint4 x = make_uint4(0, 0, 0, 0);
                    if (row < there) x = *reinterpret_cast<const uint4 *>(src + row * kHeadDim + piece * 8);
                    sts128(operand_at(to, row, piece), x.x, x.y, x.z, x.w);
                }
            }
            fence_async();
            asm volatile("bar.sync 1, 128;\n" ::: "memory");
            if (r == 0 && ok) {
                mbar_arrive(bar((j & 1 ? kBarVFull : kBarKFull) + (j >> 1 & 1)));
                if (packed) mbar_arrive(bar(kBarRawFree + (j & 1)));
            }
        }
    } else {
        // ------------------------------------------------------------------ MMAs
        if constexpr (DIFF) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;\n");
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 48;\n");
        if (warp == 20) {
            uint32_t lead;
            asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(lead));
            auto same = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
            const int n_old = same(max(s.packed, 0) - p0), pages = same(np), tiles = same(two_tiles) ? 2 : 1;            // n_old: pages of packed keys
            const uint32_t tm = (uint32_t)same((int)tmem);
            const uint64_t q_desc = tc_desc(base + kOffQ, 16, 1024), k_desc = tc_desc(base + kOffK, 16, 1024), k_mn = tc_desc(base + kOffK, kOperandHalf, 1024),
                           v_desc = tc_desc(base + kOffV, kOperandHalf, 1024);
            auto wait = [&](int b, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar(b), parity, status)); };
            bool ok = true;
            // the address fields of descriptors count 16 bytes, and no operand's end carries out of them
            auto scores = [&](int it, int w) {                    // S[w] = Q[w] K^T of page `it`; DIFF: of the channels of half w
                constexpr int STEPS = DIFF ? 4 : 8;
                const uint64_t q = q_desc + w * ((DIFF ? kOperandHalf : kOperandBytes) / 16);
                const uint32_t stage = (it & 1) * (kOperandBytes / 16);
                if (it < n_old) {
                    const uint64_t k = k_mn + stage + (DIFF ? w * 512 : 0);
#pragma unroll
                    for (int e = 0; e < STEPS; ++e) tc_mma(tm + w * 128, q + (e >> 2) * (kOperandHalf / 16) + (e & 3) * 2, k + e * 128, kIdescMn, e > 0, lead);
                } else {
                    const uint64_t k = k_desc + stage + (DIFF ? w * (kOperandHalf / 16) : 0);
#pragma unroll
                    for (int e = 0; e < STEPS; ++e)
                        tc_mma(tm + w * 128, q + (e >> 2) * (kOperandHalf / 16) + (e & 3) * 2, k + (e >> 2) * (kOperandHalf / 16) + (e & 3) * 2, kIdesc, e > 0, lead);
                }
                tc_commit(bar(kBarS + w), lead);
            };
            auto values = [&](int it, int w) {                    // O[w] += P[w] V
                const uint64_t v = v_desc + (it & 1) * (kOperandBytes / 16);
#pragma unroll
                for (int e = 0; e < 8; ++e) tc_mma_tmem(tm + 256 + w * 128, tm + w * 128 + e * 8, v + e * 128, kIdescMn, it > 0 || e > 0, lead);
            };
            if (ok && pages > 0) {
                ok = wait(kBarKFull, 0);
                if (ok) {
                    tc_fence_after();
                    for (int w = 0; w < tiles; ++w) scores(0, w);
                    tc_commit(bar(kBarKFree), lead);
                }
            }
            for (int it = 0; ok && it < pages; ++it) {
                ok = wait(kBarVFull + (it & 1), it >> 1 & 1);
                for (int w = 0; ok && w < tiles; ++w) {
                    ok = wait(kBarP + w, it & 1);
                    tc_fence_after();
                    if (ok) values(it, w);
                    if (ok && w == tiles - 1) tc_commit(bar(kBarVFree + (it & 1)), lead);
                    if (ok && it + 1 < pages && w == 0) ok = wait(kBarKFull + (it + 1 & 1), (it + 1) >> 1 & 1);
                    if (ok && it + 1 < pages) scores(it + 1, w);
                }
                if (!ok) break;
                if (it + 1 < pages) tc_commit(bar(kBarKFree + (it + 1 & 1)), lead);
            }
            if (ok && pages > 0) tc_commit(bar(kBarO), lead);
            tc_commit(bar(kBarDrain), lead);                      // whatever was begun is done before the memory is given up
            wait(kBarDrain, 0);
        } else if (warp == 21 && lane == 0) {
            // -------------------------------------------------------------- copies: packed pages as they are, fp16 pages into their operands
            bool ok = true;
            int j = 0, next = np > 0 ? page_id(p0) : -1, id = -1;
            auto landed = [&](int q) { return p0 + (q >> 1) < s.packed ? bar(kBarRaw + (q & 1)) : bar((q & 1 ? kBarVFull : kBarKFull) + (q >> 1 & 1)); };
            for (; ok && j < 2 * np; ++j) {
                const int page = p0 + (j >> 1);
                const bool values = j & 1;
                if (!values) {
                    id = next;
                    if (page + 1 < p0 + np) next = page_id(page + 1);
                }
                const uint32_t full = landed(j);
                if (page < s.packed) {
                    ok = mbar_wait(bar(kBarRawFree + (j & 1)), (j >> 1 & 1) ^ 1, status);
                    if (!ok) break;
                    if (id < 0) { mbar_arrive(full); continue; }
                    const int64_t row = ((int64_t)id * p.l.Hkv + head) * kPage;
                    const int words = values ? page_words(VB) : page_words(KB), groups = values ? p.v_groups : p.k_groups;
                    const uint32_t cb = kPage * words * 4, sz = kPage * groups * 2, dst = base + kOffRaw + (j & 1) * kRawBytes;
                    mbar_expect(full, cb + 2 * sz);
                    bulk_load(dst, (values ? p.l.vcode : p.l.kcode) + row * words, cb, full);
                    bulk_load(dst + cb, static_cast<const __half *>(values ? p.l.vscale : p.l.kscale) + row * groups, sz, full);
                    bulk_load(dst + cb + sz, static_cast<const __half *>(values ? p.l.vmn : p.l.kmn) + row * groups, sz, full);
                } else {
                    ok = mbar_wait(bar((values ? kBarVFree : kBarKFree) + (j >> 1 & 1)), (j >> 2 & 1) ^ 1, status);
                    if (!ok) break;
                    if (!by_loader(page, id)) { mbar_arrive(bar(kBarTail + (j & 3))); continue; }
                    const uint32_t dst = base + (values ? kOffV : kOffK) + (j >> 1 & 1) * kOperandBytes;
                    const int y = (id * p.l.Hkv + head) * kPage;
                    mbar_expect(full, kOperandBytes);
                    tile_load(dst, values ? &maps.v : &maps.k, 0, y, full);
                    tile_load(dst + kOperandHalf, values ? &maps.v : &maps.k, 64, y, full);
                }
            }
            if (!ok)                                              // copies in flight land before the CTA ends
                for (int q = max(0, j - 4); q < j; ++q) mbar_wait(landed(q), p0 + (q >> 1) < s.packed ? q >> 1 & 1 : q >> 2 & 1, status);
        }
        __syncwarp();
    }
    __syncthreads();
    if (warp == 20) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem));
    }
}

// The rows of a pool of fp16 pages as a tensor map.  The encoder is the driver's; the library links the runtime only.
static bool page_map(CUtensorMap *map, void *base, int64_t rows) {
    using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                                CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) f = nullptr;
        return reinterpret_cast<Encode>(f);
    }();
    if (!encode || rows <= 0 || rows >= 1LL << 31) return false;
    const cuuint64_t sizes[2] = {kHeadDim, (cuuint64_t)rows}, strides[1] = {kHeadDim * 2};
    const cuuint32_t box[2] = {64, kPage}, step[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, base, sizes, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int KB, int VB, bool MODS, bool DIFF>
static int launch_tiles(const PagedArgs &p, int max_tiles, cudaStream_t st) {
    const cudaError_t e = cudaFuncSetAttribute(paged_tile_kernel<KB, VB, MODS, DIFF>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kTileSmem);
    if (e != cudaSuccess) return record_cuda_error(e);
    const int64_t grid = p.n_whole + ((int64_t)max_tiles * p.l.Hkv - p.n_whole) * p.splits;
    if (grid > 2147483647LL) return KVQ_ERR_UNSUPPORTED;
    if (grid == 0) return KVQ_OK;
    PagedMaps maps = {};
    const int64_t rows = (int64_t)p.l.n_fp16 * p.l.Hkv * kPage;
    maps.there = page_map(&maps.k, p.l.kfull, rows) && page_map(&maps.v, p.l.vfull, rows);
    paged_tile_kernel<KB, VB, MODS, DIFF><<<(unsigned)grid, kTileThreads, kTileSmem, st>>>(p, maps, max_tiles);
    return count_launch();
}

template <int KB, bool DIFF = false>
static int launch_tiles(const PagedArgs &p, int max_tiles, bool mods, cudaStream_t st) {
    switch (p.l.v_bits) {
        case 1: return mods ? launch_tiles<KB, 1, true, DIFF>(p, max_tiles, st) : launch_tiles<KB, 1, false, DIFF>(p, max_tiles, st);
        case 2: return mods ? launch_tiles<KB, 2, true, DIFF>(p, max_tiles, st) : launch_tiles<KB, 2, false, DIFF>(p, max_tiles, st);
        case 3: return mods ? launch_tiles<KB, 3, true, DIFF>(p, max_tiles, st) : launch_tiles<KB, 3, false, DIFF>(p, max_tiles, st);
        default: return mods ? launch_tiles<KB, 4, true, DIFF>(p, max_tiles, st) : launch_tiles<KB, 4, false, DIFF>(p, max_tiles, st);
    }
}

}  // namespace kvq
