// Beam search's selection: the best continuations of every request over its beams and the vocabulary.
//
//   value(b, t) = score_b + ((logit_bt - top_b) - log sum_t' exp(logit_bt' - top_b)),   the n largest of a request, equal ones by (b, t)
//
// with top_b the largest logit of the beam, which is never added to the logarithm: beside a top of 1e30, or where all logits are the type's lowest number, that
// would be lost, and every token have the probability of one.
// Within a beam the order of the values is the order of the logits, so one pass over a row gives both what it needs: the sum of
// exponentials under a running maximum and the row's n best logits.  A row is cut into up to 32 parts, a CTA each (beam_scan_kernel); a second launch
// joins the parts of each beam, then the beams of each request (beam_join_kernel).
// A candidate within a beam is one 64-bit key, the logit in an order of unsigned numbers above the complement of the token: keys are
// all different, the largest is the best and ties go to the lowest token, in whatever order threads come.
// Sums are fp32 within a thread -- V / (256 parts) terms, each to 2^-22 of itself -- and 64-bit from there: which of two beams goes on may hang on the last bits of
// their sums, and 64 bits add nothing to the error of the terms.
#include "beam_reach.cuh"
#include "quant_core.cuh"

#include <cuda_bf16.h>

namespace kvq {

using u64 = unsigned long long;
constexpr int kScanThreads = 256, kTurn = 16;                     // elements a thread takes at a time
constexpr int kMostBest = KVQ_MOST_BEST, kMostBeams = KVQ_MOST_BEAMS, kMostParts = 32;
constexpr int kKeys = 16 * kMostBest;                             // room for what reaches a part's threshold
constexpr float kLog2 = 1.4426950408889634f;

struct BeamArgs {
    kvq_beam_args a;
    int parts;
    u64 *keys;                        // [rows][parts][n], best first, 0 where there are fewer
    double *sums;                     // [rows][parts]
    float *tops;                      // [rows][parts]
};

__device__ __forceinline__ float beam_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t ordered(float x) {            // unsigned numbers in the order of the floats; -0 is 0
    const uint32_t u = __float_as_uint(x + 0.f);
    return u ^ ((int)u < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t u) { return __uint_as_float(u ^ ((int)u < 0 ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ u64 beam_key(float x, int token) { return (u64)ordered(x) << 32 | (uint32_t)~token; }

template <typename T> __device__ __forceinline__ float as_float(T x);
template <> __device__ __forceinline__ float as_float(float x) { return x; }
template <> __device__ __forceinline__ float as_float(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ void floats(uint4 v, float *x) {
    if constexpr (sizeof(T) == 4) {
        x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
    } else {
        const T *t = reinterpret_cast<const T *>(&v);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = as_float<T>(t[i]);
    }
}

// exp(x - top) of a thread's elements under its own running maximum.  The difference comes first: times log2 e it may lose bits only of itself, whatever
// the logits are added to, and the type's lowest value stays a number.
__device__ __forceinline__ float max3_of(float a, float b, float c) {             // what is not a number is left out
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
struct RunningSum {
    float top = -INFINITY, sum = 0.f;
    __device__ __forceinline__ void add(const float (&v)[kTurn], float now) {          // now: the maximum with these
        const float from = now == -INFINITY ? 0.f : now;
        const u64 by = f32x2(kLog2, kLog2), off = f32x2(-from, -from);
        u64 more[2] = {f32x2(sum * beam_exp2((top - from) * kLog2), 0.f), 0ull};
#pragma unroll
        for (int e = 0; e < kTurn; e += 2) {
            const float2 d = f32x2_split(mul_f32x2(add_f32x2(f32x2(v[e], v[e + 1]), off), by));
            more[e >> 1 & 1] = add_f32x2(more[e >> 1 & 1], f32x2(beam_exp2(d.x), beam_exp2(d.y)));
        }
        const float2 all = f32x2_split(add_f32x2(more[0], more[1]));
        sum = all.x + all.y;
        top = now;
    }
};

// A part of a row, 4096 elements a turn.  The pass over it keeps a thread's sum, its maximum and where that came first, and nothing else.  Of the groups of threads (eight
// lanes, fewer where n is large) the n-th best then has a key that n elements reach at least, and none of the n best is in a thread whose best does not reach
// it: what the others hold -- those of some 1.1 n threads -- is read once more, from L2, and what reaches the threshold goes to shared memory.  Should
// there be no room for all of it (rows that were made for that), the n best of what there was room for give a higher threshold (Reach).
// Which thread has which token follows from the token alone, not from the row's alignment: rows alike have sums alike, to the last bit, and ties between
// beams stay ties.  Rows that are not 16-byte aligned are therefore read element by element (VEC false).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kScanThreads, 4) beam_scan_kernel(const __grid_constant__ BeamArgs p) {
    constexpr int E = 16 / sizeof(T), U = kTurn / E, kStep = U * kScanThreads;         // pieces of 16 bytes a turn
    __shared__ u64 s_key[kKeys], s_best[kScanThreads], s_from;
    __shared__ double s_sum[kScanThreads / 32];
    __shared__ float s_top[kScanThreads / 32];
    __shared__ int s_count, s_threads, s_thread[kScanThreads];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = p.a.n, V = p.a.vocabulary;
    const int part = blockIdx.x % p.parts;
    const int64_t row = blockIdx.x / p.parts;
    const T *x = static_cast<const T *>(p.a.logits) + row * p.a.l_sR;
    const int pieces = V / E + (V % E != 0), lo = (int)((int64_t)pieces * part / p.parts), hi = (int)((int64_t)pieces * (part + 1) / p.parts);
    const int whole = VEC ? min(hi, V / E) : lo;                  // pieces before it are 16 bytes that are all there, aligned
    auto load = [&](int piece) {                                  // elements that are not there: whatever
        uint4 to = make_uint4(0, 0, 0, 0);
        if (piece < whole) {
            to = reinterpret_cast<const uint4 *>(x)[piece];
        } else if (piece < hi) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (piece * (int64_t)E + e < V) reinterpret_cast<T *>(&to)[e] = x[(int64_t)piece * E + e];
        }
        return to;
    };
    auto here = [&](int piece) { return piece < whole ? E : piece < hi ? min(E, V - piece * E) : 0; };

    RunningSum sum;
    int first = INT32_MAX;                                        // the piece in which the maximum came first
    auto turn = [&](int at, const uint4 (&raw)[U], bool full) {
        float v[kTurn], most[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            floats<T>(raw[u], v + u * E);
            if (!full) {
                const int some = here(at + u * kScanThreads + tid);
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (e >= some) v[u * E + e] = -INFINITY;
                if (some && first == INT32_MAX) first = at + u * kScanThreads + tid;           // where there is nothing but -infinity
            }
            most[u] = fmaxf(v[u * E], v[u * E + 1]);
#pragma unroll
            for (int e = 2; e < E; e += 2) most[u] = max3_of(most[u], v[u * E + e], v[u * E + e + 1]);
        }
        float now = sum.top;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (most[u] > now) first = at + u * kScanThreads + tid;
            now = fmaxf(now, most[u]);
        }
        sum.add(v, now);
    };
    const int turns = (whole - lo) / kStep, rest = lo + turns * kStep;                 // turns that are all there
    {
        const uint4 *vec = reinterpret_cast<const uint4 *>(x) + lo + tid;
        uint4 next[2][U];
        auto ask = [&](uint4 (&to)[U], int k) {
            if (k >= turns) return;
#pragma unroll
            for (int u = 0; u < U; ++u) to[u] = vec[k * kStep + u * kScanThreads];
        };
        ask(next[0], 0);
        ask(next[1], 1);
        if (turns > 0) first = lo + tid;
        for (int k = 0; k < turns; k += 2) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (k + h >= turns) break;
                uint4 raw[U];
#pragma unroll
                for (int u = 0; u < U; ++u) raw[u] = next[h][u];
                ask(next[h], k + h + 2);
                turn(lo + (k + h) * kStep, raw, true);
            }
        }
    }
    if (tid == 0) { s_from = 0; s_threads = s_count = 0; }
    for (int at = rest; at < hi; at += kStep) {
        uint4 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = load(at + u * kScanThreads + tid);
        turn(at, raw, false);
    }

    const u64 mine = first == INT32_MAX ? 0 : beam_key(sum.top, first);
    const float all = warp_max(sum.top);
    if (lane == 0) s_top[warp] = all;
    if (n <= 32) {                                                // groups of eight or four lanes
        const int width = n <= 16 ? 8 : 4, groups = kScanThreads / width;
        u64 best = mine;
        for (int o = 1; o < width; o <<= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        if (lane % width == 0) s_best[tid / width] = best;
        __syncthreads();
        const u64 held[2] = {s_best[lane], groups > 32 ? s_best[32 + lane] : 0};
        for (int g = warp; g < groups; g += kScanThreads / 32) {
            const u64 one = s_best[g];
            const int rank = __popc(__ballot_sync(0xffffffffu, held[0] > one)) + __popc(__ballot_sync(0xffffffffu, held[1] > one));
            if (lane == 0 && rank == n - 1 && one) s_from = one;
        }
    } else {                                                      // an eighth of n of every warp's lanes; the least of the warps' thresholds has n above it
        const int want = (n + kScanThreads / 32 - 1) / (kScanThreads / 32);
        u64 nth = 0;
#pragma unroll 8
        for (int g = 0; g < 32; ++g) {
            const u64 one = __shfl_sync(0xffffffffu, mine, g);
            if (__popc(__ballot_sync(0xffffffffu, mine > one)) == want - 1 && one) nth = one;
        }
        if (lane == 0) s_best[warp] = nth;
        __syncthreads();
        if (tid == 0) {
            u64 least = s_best[0];
#pragma unroll
            for (int w = 1; w < kScanThreads / 32; ++w) least = min(least, s_best[w]);
            s_from = least;
        }
    }
    float top = s_top[0];
#pragma unroll
    for (int w = 1; w < kScanThreads / 32; ++w) top = fmaxf(top, s_top[w]);
    double d = sum.sum == 0.f ? 0.0 : (double)sum.sum * (double)beam_exp2((sum.top - top) * kLog2);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    if (lane == 0) s_sum[warp] = d;
    __syncthreads();
    const int64_t out = row * p.parts + part;
    if (tid == kScanThreads - 1) {
        d = 0.0;
#pragma unroll
        for (int w = 0; w < kScanThreads / 32; ++w) d += s_sum[w];
        p.sums[out] = d;
        p.tops[out] = top;
    }
    // keys of pieces here: a token's place behind its piece's
    if (mine && mine >= s_from) s_thread[atomicAdd(&s_threads, 1)] = tid;
    Reach reaches(s_from);
    const float from_x = from_ordered((uint32_t)(reaches.by_piece >> 32));
    bool lost;
    do {
        __syncthreads();
        lost = false;
        const int each = (hi - lo + kScanThreads - 1) / kScanThreads;                  // pieces of a thread
        for (int i = warp; i < s_threads; i += kScanThreads / 32)
            for (int j = lane; j < each; j += 32) {
                const int piece = lo + j * kScanThreads + s_thread[i], some = here(piece);
                const uint4 raw = load(piece);
                float v[E];
                floats<T>(raw, v);
                uint32_t reach = 0;
#pragma unroll
                for (int e = 0; e < E; ++e) reach |= v[e] < from_x ? 0u : 1u << e;     // from_x is no number where everything does
                reach &= (1u << some) - 1u;
                while (reach) {
                    const int e = __ffs(reach) - 1;
                    reach &= reach - 1;
                    float one = v[0];
#pragma unroll
                    for (int k = 1; k < E; ++k) one = k == e ? v[k] : one;
                    const u64 key = beam_key(one, piece * E + e);
                    if (!reaches.takes(beam_key(one, piece), key)) continue;
                    const int place = atomicAdd(&s_count, 1);
                    if (place < kKeys) s_key[place] = key;
                    else lost = true;
                }
            }
        lost = __syncthreads_or(lost);
        const int kept = min(s_count, kKeys);
        for (int i = warp; i < kept; i += kScanThreads / 32) {    // a vote counts those that are better
            const u64 key = s_key[i];
            int rank = 0;
            for (int j = lane; j < (kept + 31) / 32 * 32; j += 32) rank += __popc(__ballot_sync(0xffffffffu, (j < kept ? s_key[j] : 0) > key));
            if (lane == 0 && rank < n) s_best[rank] = key;
        }
        __syncthreads();
        if (lost) {
            reaches.raise(s_best[n - 1]);
            if (tid == 0) s_count = 0;
        } else if (tid < n) {
            p.keys[out * n + tid] = tid < kept ? s_best[tid] : 0;
        }
    } while (lost);
}

// The largest of the lanes' keys; `lane_of`: the first lane that has it.
__device__ __forceinline__ u64 warp_best(u64 key, int &lane_of) {
    const uint32_t high = __reduce_max_sync(0xffffffffu, (uint32_t)(key >> 32));
    const uint32_t low = __reduce_max_sync(0xffffffffu, (uint32_t)(key >> 32) == high ? (uint32_t)key : 0u);
    const u64 best = (u64)high << 32 | low;
    lane_of = __ffs(__ballot_sync(0xffffffffu, key == best)) - 1;
    return best;
}
__device__ __forceinline__ u64 ordered64(double x) {              // as ordered()
    const u64 u = (u64)__double_as_longlong(x + 0.0);
    return u ^ ((long long)u < 0 ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ double from_ordered64(u64 u) { return __longlong_as_double((long long)(u ^ ((long long)u < 0 ? 1ull << 63 : ~0ull))); }

// A beam's largest logit and the logarithm of its sum of exponentials from its parts', a lane each; not finite where the beam offers nothing.
struct BeamBase {
    double score, top, log_sum;
    __device__ __forceinline__ bool alive() const { return isfinite(score) && isfinite(log_sum); }
    __device__ __forceinline__ u64 value(u64 key) const { return ordered64(score + (((double)from_ordered((uint32_t)(key >> 32)) - top) - log_sum)); }
};
__device__ __forceinline__ BeamBase beam_base(const BeamArgs &p, int64_t row, int lane) {
    const float my_top = lane < p.parts ? p.tops[row * p.parts + lane] : -INFINITY, top = warp_max(my_top);
    double sum = lane < p.parts ? p.sums[row * p.parts + lane] : 0.0;
    if (sum != 0.0) sum *= (double)expf(my_top - top);             // 2^-23: as exact as the terms
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return {(double)p.a.scores[row], (double)top, log(sum)};       // no sum, no number or an infinite top: neither is the logarithm finite
}
__device__ __forceinline__ void put_best(const BeamArgs &p, int64_t at, float value, int beam, int token) {
    p.a.out_scores[at] = value;
    p.a.out_beams[at] = beam;
    p.a.out_tokens[at] = token;
}
__device__ __forceinline__ void put_next(const BeamArgs &p, int64_t at, float value, int beam, int token) {
    p.a.next_scores[at] = value;
    p.a.next_beams[at] = beam;
    p.a.next_tokens[at] = token;
}

// A CTA a request: of all its candidates -- beam, part, place in the part's sorted list -- those that reach a bound are counted against each other, 32 by a
// vote.  The bound: the n-th best of the first ceil(n / lists) of every list, or, as beams' scores may lie far apart, what n of one beam or
// list reach: BY_BEAMS, the n-th best of the first ceil(n / parts) of a beam's lists, closer where n is large and longer to find (16 beams, n = 48, 4 parts of 128256
// tokens, both launches: 44 us, and 61 by the lists' last ones; 4 beams, n = 8: 10.2 and 8.9); hardly more than n reach both.  Should there be no room for all that do, the n best of what there was room for give
// a higher one.  What counts here is the chain of dependent instructions (some 300, at eight cycles each): both launches for 4 beams of 32000
// tokens 8.9 us, 11.0 where beams and parts were merged by looking n times which list's head is the best.
constexpr int kJoined = 1024;
template <bool BY_BEAMS>
__global__ void __launch_bounds__(512) beam_join_kernel(const __grid_constant__ BeamArgs p) {
    __shared__ BeamBase s_base[kMostBeams];
    __shared__ u64 s_value[kJoined], s_place[kJoined], s_from, s_full[16];         // ordered values; (beam, token)
    __shared__ uint32_t s_goes[(kMostBest + 31) / 32];
    __shared__ int s_left, s_best[kMostBest];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5, n = p.a.n, K = p.a.beams, list = p.parts * n, all = K * list;
    const u64 *keys = p.keys + (int64_t)blockIdx.x * all;
    const u64 mine_first = tid < all ? keys[tid] : 0;             // asked for early
    const float per_list = 1.f / list;                            // c / list = (c + 0.5) * this for every c here (below 2^22)
    u64 full = 0, unused;
    for (int b = warp; b < K; b += warps) {
        const BeamBase base = beam_base(p, (int64_t)blockIdx.x * K + b, lane);
        if (lane == 0) s_base[b] = base;
        if constexpr (BY_BEAMS) {                                 // 159 of its keys at most
            const int each = (n + p.parts - 1) / p.parts, some = p.parts * each;
            u64 held[5], nth = 0;
#pragma unroll
            for (int k = 0; k < 5; ++k) {
                const int e = 32 * k + lane;
                held[k] = e < some ? keys[b * list + e / each * n + e % each] : 0;
            }
#pragma unroll
            for (int k = 0; k < 5; ++k)
                for (int e = 0; e < min(32, some - 32 * k); ++e) {
                    const u64 one = __shfl_sync(0xffffffffu, held[k], e);
                    int rank = 0;
#pragma unroll
                    for (int h = 0; h < 5; ++h)
                        if (32 * h < some) rank += __popc(__ballot_sync(0xffffffffu, held[h] > one));
                    if (rank == n - 1 && one) nth = one;
                }
            if (nth && base.alive()) full = max(full, base.value(nth));
        }
    }
    if (tid < (kMostBest + 31) / 32) s_goes[tid] = 0;
    if (tid == 0) { s_left = 0; s_from = 0; }
    __syncthreads();
    // candidate c's value, in order, and its place; 0: there is none
    auto candidate = [&](int c, u64 key, u64 &place) -> u64 {
        const int beam = (int)((c + 0.5f) * per_list), i = c - beam * list;
        const bool alive = s_base[beam].alive();
        const int token = alive ? (int)~(uint32_t)key : i;        // a beam that offers nothing: its first tokens, once
        place = (u64)beam << 32 | (uint32_t)token;
        if (alive ? key == 0 : i >= n || i >= p.a.vocabulary) return 0;
        return alive ? s_base[beam].value(key) : ordered64(-INFINITY);
    };
    const int lists = K * p.parts, firsts = (n + lists - 1) / lists, heads = lists * firsts;       // 192 + 128 heads at most (beam_parts)
    for (int h = tid; h < heads; h += blockDim.x) {
        const int c = firsts == 1 ? h * n : h / firsts * n + h % firsts;
        s_value[h] = candidate(c, keys[c], unused);
    }
    int whose;
    if constexpr (!BY_BEAMS) {
        for (int l = tid; l < lists; l += blockDim.x) full = max(full, candidate(l * n + n - 1, keys[l * n + n - 1], unused));
        if (32 * warp < lists) full = warp_best(full, whose);
    }
    if (lane == 0) s_full[warp] = full;
    __syncthreads();
    for (int h = warp; h < heads; h += warps) {
        const u64 one = s_value[h];
        int better = 0, reach = 0;
        for (int j = lane; j < (heads + 31) / 32 * 32; j += 32) {
            const u64 other = j < heads ? s_value[j] : 0;
            better += __popc(__ballot_sync(0xffffffffu, other > one));
            reach += __popc(__ballot_sync(0xffffffffu, j < heads && other >= one));
        }
        if (lane == 0 && better < n && reach >= n) s_from = one;  // several may be the n-th best
    }
    for (int w = 0; w < warps; ++w) full = max(full, s_full[w]);
    __syncthreads();
    u64 from = max(s_from, full), from_place = ~0ull;             // what reaches it: better, or as good and its place not behind
    int left;
    for (;;) {
        bool lost = false;
        for (int c = tid; c < all; c += blockDim.x) {
            u64 place;
            const u64 value = candidate(c, c == tid ? mine_first : keys[c], place);
            if (value == 0 || value < from || (value == from && place > from_place)) continue;
            const int slot = atomicAdd(&s_left, 1);
            if (slot < kJoined) {
                s_value[slot] = value;
                s_place[slot] = place;
            } else {
                lost = true;
            }
        }
        lost = __syncthreads_or(lost);
        left = min(s_left, kJoined);
        for (int m = warp; m < left; m += warps) {
            const u64 v = s_value[m], at = s_place[m];
            int rank = 0;
            for (int j = lane; j < (left + 31) / 32 * 32; j += 32) {
                const u64 other = j < left ? s_value[j] : 0;
                rank += __popc(__ballot_sync(0xffffffffu, other > v));
                if (__popc(__ballot_sync(0xffffffffu, other == v)) > (m >> 5 == j >> 5)) rank += __popc(__ballot_sync(0xffffffffu, other == v && s_place[min(j, left - 1)] < at));
            }
            if (lane == 0 && rank < n) s_best[rank] = m;
        }
        __syncthreads();
        if (!lost) break;
        from = s_value[s_best[n - 1]];
        from_place = s_place[s_best[n - 1]];
        __syncthreads();
        if (tid == 0) s_left = 0;
        __syncthreads();
    }
    const bool chosen = tid < min(n, left);
    const u64 place = chosen ? s_place[s_best[tid]] : 0, value = chosen ? s_value[s_best[tid]] : 0;
    const int beam = (int)(place >> 32), token = (int)(uint32_t)place;
    const float score = (float)from_ordered64(value);
    if (chosen) {
        put_best(p, (int64_t)blockIdx.x * n + tid, score, beam, token);
        bool ends = false;
        for (int e = 0; e < p.a.n_ends; ++e) ends |= p.a.ends[e] == token;
        if (!ends) atomicOr(&s_goes[tid >> 5], 1u << lane);
    }
    __syncthreads();
    int before = 0, going = 0;                                    // those that go on and are better; all
#pragma unroll
    for (int w = 0; w < (kMostBest + 31) / 32; ++w) {
        const uint32_t bits = s_goes[w];
        before += __popc(w < warp ? bits : w == warp ? bits & ((1u << lane) - 1u) : 0u);
        going += __popc(bits);
    }
    if (chosen && (s_goes[warp] >> lane & 1u) && before < K) put_next(p, (int64_t)blockIdx.x * K + before, score, beam, token);
    for (int k = going + tid; k < K; k += blockDim.x) put_next(p, (int64_t)blockIdx.x * K + k, -INFINITY, 0, 0);       // everything else ends
}

// Parts of a row: a part of its own costs some 4 us of beginning and end beside 0.4 us a turn, so one CTA an SM, two where there are six million logits and few are wanted, and four where
// rows are many (32 rows of 128256: 11.8 us in 4 parts, 14.7 in 16; 128 of 32000: 12.0 in one, 13.2 in 2; 128 of 128256: 24.6 in one, 20.6 in 2; 256: 25.4 in 2,
// 28.3 in 4).  1024 keys of a beam at most are joined.
static int beam_parts(const kvq_beam_args &a) {
    const int64_t rows = (int64_t)a.requests * a.beams;
    int64_t parts = (rows > 148 ? 4 * 148 : rows * a.vocabulary >= 6 << 20 && a.n <= 32 ? 2 * 148 : 148) / (rows > 0 ? rows : 1);
    const int64_t most = ((int64_t)a.vocabulary + kScanThreads * kTurn - 1) / (kScanThreads * kTurn);
    if (parts > most) parts = most;
    if (parts > kMostParts) parts = kMostParts;
    if (parts > 1024 / a.n) parts = 1024 / a.n;
    return parts < 1 ? 1 : (int)parts;
}
static int check_beams(const kvq_beam_args *a) {
    if (!a) return KVQ_ERR_NULL;
    if (a->requests < 0 || a->beams <= 0 || a->vocabulary <= 0 || a->n <= 0 || a->n_ends < 0) return KVQ_ERR_SHAPE;
    if (a->beams > kMostBeams || a->n > kMostBest || a->type < 0 || a->type > 2) return KVQ_ERR_UNSUPPORTED;
    const int64_t all = (int64_t)a->beams * a->vocabulary, want = (int64_t)a->beams * (1 + (int64_t)a->n_ends);
    if (a->n > all || a->n < (want < all ? want : all)) return KVQ_ERR_SHAPE;
    if ((int64_t)a->requests * a->beams * kMostParts > 2147483647LL) return KVQ_ERR_UNSUPPORTED;
    return KVQ_OK;
}
static uint64_t beam_bytes(const kvq_beam_args &a) { return (uint64_t)a.requests * a.beams * beam_parts(a) * (8 * a.n + 16); }

}  // namespace kvq

extern "C" uint64_t kvq_beam_select_workspace_bytes(const kvq_beam_args *a) {
    using namespace kvq;
    return check_beams(a) ? 0 : beam_bytes(*a);
}

extern "C" int kvq_beam_select(const kvq_beam_args *a, kvq_stream_t stream) {
    using namespace kvq;
    if (const int rc = check_beams(a)) return rc;
    if (a->requests == 0) return KVQ_OK;
    if (!a->logits || !a->scores || (a->n_ends && !a->ends) || !a->out_scores || !a->out_beams || !a->out_tokens || !a->next_scores || !a->next_beams || !a->next_tokens)
        return KVQ_ERR_NULL;
    if (!a->workspace || a->workspace_bytes < beam_bytes(*a)) return KVQ_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(a->workspace) % 16 || reinterpret_cast<uintptr_t>(a->logits) % (a->type == KVQ_F32 ? 4 : 2)) return KVQ_ERR_ALIGN;
    BeamArgs p = {};
    p.a = *a;
    p.parts = beam_parts(*a);
    const int64_t ctas = (int64_t)a->requests * a->beams * p.parts;
    p.keys = static_cast<u64 *>(a->workspace);
    p.sums = reinterpret_cast<double *>(p.keys + ctas * a->n);
    p.tops = reinterpret_cast<float *>(p.sums + ctas);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const bool vec = reinterpret_cast<uintptr_t>(a->logits) % 16 == 0 && a->l_sR % (a->type == KVQ_F32 ? 4 : 8) == 0;
    auto scan = [&](auto aligned, auto rows) { (vec ? aligned : rows)<<<(unsigned)ctas, kScanThreads, 0, st>>>(p); };
    if (a->type == KVQ_F32) scan(beam_scan_kernel<float, true>, beam_scan_kernel<float, false>);
    else if (a->type == KVQ_BF16) scan(beam_scan_kernel<__nv_bfloat16, true>, beam_scan_kernel<__nv_bfloat16, false>);
    else scan(beam_scan_kernel<__half, true>, beam_scan_kernel<__half, false>);
    if (const int rc = check_launch()) return rc;
    const unsigned threads = a->beams * p.parts * a->n <= 512 ? 256 : 512;
    if (a->n > 16 && p.parts > 1) beam_join_kernel<true><<<(unsigned)a->requests, threads, 0, st>>>(p);
    else beam_join_kernel<false><<<(unsigned)a->requests, threads, 0, st>>>(p);
    return check_launch();
}
