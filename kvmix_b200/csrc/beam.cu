// Beam search's selection: the best continuations of every request over its beams and the vocabulary.
//
//   value(b, t) = score_b + (logit_bt - log sum_t' exp(logit_bt')),   the n largest of a request, equal ones by (b, t)
//
// Within a beam the order of the values is the order of the logits, so one pass over a row gives both what it needs: the sum of
// exponentials under a running maximum and the row's n best logits.  A row is cut into up to 32 parts, a CTA each (beam_scan_kernel); a second launch
// joins the parts of each beam, then the beams of each request (beam_join_kernel).
// A candidate within a beam is one 64-bit key, the logit in an order of unsigned numbers above the complement of the token: keys are
// all different, the largest is the best and ties go to the lowest token, in whatever order threads come.
// Sums are fp32 within a thread (some hundred terms) and 64-bit from there: which of two beams goes on may hang on the last bits of their sums.
#include "common.cuh"

#include <cuda_bf16.h>

namespace kvq {

using u64 = unsigned long long;
constexpr int kScanThreads = 256, kTurn = 16;                     // elements a thread takes at a time
constexpr int kMostBest = KVQ_MOST_BEST, kMostBeams = KVQ_MOST_BEAMS, kMostParts = 32;
constexpr int kKeys = kMostBest * kTurn + 64;                     // of a first turn no more pass: n groups of threads have a key that reaches the threshold
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

// A part of a row.  The first turn's threshold: of the groups of threads (four lanes, or one where n is large) the n-th best has a key that n elements reach.
// Which thread has which token follows from the token alone, not from the row's alignment: rows alike have sums alike, to the last bit, and ties between
// beams stay ties.  Rows that are not 16-byte aligned are therefore read element by element (VEC false).
// What reaches it goes to shared memory, some 1.1 n of the first turn's 4096, and in later turns n a turn; every 48 beyond n, the n best
// of them give the next threshold.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kScanThreads) beam_scan_kernel(const __grid_constant__ BeamArgs p) {
    constexpr int E = 16 / sizeof(T), U = kTurn / E;
    __shared__ u64 s_key[kKeys], s_best[kScanThreads], s_from;
    __shared__ double s_sum[kScanThreads / 32];
    __shared__ float s_top[kScanThreads / 32];
    __shared__ int s_count;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = p.a.n, V = p.a.vocabulary;
    const int part = blockIdx.x % p.parts;
    const int64_t row = blockIdx.x / p.parts;
    const T *x = static_cast<const T *>(p.a.logits) + row * p.a.l_sR;
    const int pieces = V / E + (V % E != 0), lo = (int)((int64_t)pieces * part / p.parts), hi = (int)((int64_t)pieces * (part + 1) / p.parts);
    float top = -INFINITY, sum = 0.f;

    uint4 next[U];
    auto load = [&](int at) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int piece = at + u * kScanThreads + tid;
            if (piece >= hi) continue;
            if (VEC && (piece + 1) * (int64_t)E <= V) {
                next[u] = reinterpret_cast<const uint4 *>(x)[piece];
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (piece * (int64_t)E + e < V) reinterpret_cast<T *>(&next[u])[e] = x[(int64_t)piece * E + e];
            }
        }
    };
    if (tid == 0) { s_count = 0; s_from = 0; }
    auto compact = [&]() {                                        // the n best of what is kept, in order
        const int kept = min(s_count, kKeys);
        for (int i = tid; i < kept; i += kScanThreads) {
            const u64 key = s_key[i];
            int rank = 0;
            for (int j = 0; j < kept; ++j) rank += s_key[j] > key;
            if (rank < n) s_best[rank] = key;
        }
        __syncthreads();
        if (tid < min(kept, n)) s_key[tid] = s_best[tid];
        if (tid == 0) {
            s_count = min(kept, n);
            if (kept >= n) s_from = s_best[n - 1] + 1;
        }
        __syncthreads();
    };
    load(lo);
    for (int at = lo; at == lo || at < hi; at += U * kScanThreads) {
        float v[kTurn], most = -INFINITY;
        uint32_t pending = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int piece = at + u * kScanThreads + tid, there = piece < hi ? (int)min((int64_t)E, V - (int64_t)piece * E) : 0;
            floats<T>(next[u], v + u * E);
            pending |= ((1u << there) - 1u) << (u * E);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (e >= there) v[u * E + e] = -INFINITY;
                most = fmaxf(most, v[u * E + e]);
            }
        }
        load(at + U * kScanThreads);
        const float now = fmaxf(top, most), ref = now == -INFINITY ? 0.f : now;
        float more[2] = {sum * beam_exp2((top - ref) * kLog2), 0.f};
#pragma unroll
        for (int e = 0; e < kTurn; ++e) more[e & 1] += beam_exp2((v[e] - ref) * kLog2);
        sum = more[0] + more[1];
        top = now;
        auto token = [&](int e) { return (at + (e / E) * kScanThreads + tid) * E + e % E; };
        if (at == lo) {
            u64 best = 0;
#pragma unroll
            for (int e = 0; e < kTurn; ++e)
                if (pending >> e & 1) best = max(best, beam_key(v[e], token(e)));
            const bool fours = n <= 32;
            if (fours) {
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
            }
            const int groups = fours ? kScanThreads / 4 : kScanThreads;
            if (!fours || (lane & 3) == 0) s_best[fours ? tid >> 2 : tid] = best;
            __syncthreads();
            if (tid < groups) {
                const u64 mine = s_best[tid];
                int rank = 0;
#pragma unroll 8
                for (int j = 0; j < groups; ++j) rank += s_best[j] > mine;
                if (rank == n - 1 && mine) s_from = mine;
            }
            __syncthreads();
        }
        bool again;
        do {                                                      // more than once where there is no room for all that pass
            const u64 from = s_from;
            bool full = false;
            if (most >= from_ordered((uint32_t)(from >> 32)) || from == 0) {
#pragma unroll
                for (int e = 0; e < kTurn; ++e)
                    if (pending >> e & 1) {
                        const u64 key = beam_key(v[e], token(e));
                        if (key >= from) {
                            const int place = atomicAdd(&s_count, 1);
                            if (place < kKeys) s_key[place] = key;
                            full |= place >= n + 48;
                            if (place < kKeys) pending &= ~(1u << e);
                        } else {
                            pending &= ~(1u << e);
                        }
                    }
            } else {
                pending = 0;
            }
            again = __syncthreads_or(full);
            if (again) {
                compact();
                again = __syncthreads_or(pending != 0);
            }
        } while (again);
    }
    __syncthreads();
    compact();
    const int64_t at = row * p.parts + part;
    if (tid < n) p.keys[at * n + tid] = tid < s_count ? s_key[tid] : 0;
    const float all = warp_max(top);
    if (lane == 0) s_top[warp] = all;
    __syncthreads();
    float best = s_top[0];
#pragma unroll
    for (int w = 1; w < kScanThreads / 32; ++w) best = fmaxf(best, s_top[w]);
    double d = sum == 0.f ? 0.0 : (double)sum * (double)beam_exp2((top - best) * kLog2);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    if (lane == 0) s_sum[warp] = d;
    __syncthreads();
    if (tid == 0) {
        d = 0.0;
        for (int w = 0; w < kScanThreads / 32; ++w) d += s_sum[w];
        p.sums[at] = d;
        p.tops[at] = best;
    }
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

// A CTA a request.  A warp joins a beam's parts: its sum, and the n best of sorted lists, one a lane, by looking n times which head is the best.  Then
// one warp joins the beams alike, two a lane, and lists those that do not end.
__global__ void __launch_bounds__(256) beam_join_kernel(const __grid_constant__ BeamArgs p) {
    extern __shared__ __align__(16) u64 s_join[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, n = p.a.n, K = p.a.beams, parts = p.parts;
    double *s_value = reinterpret_cast<double *>(s_join);         // [K][n]
    int *s_token = reinterpret_cast<int *>(s_value + K * n);      // [K][n]
    u64 *s_list = reinterpret_cast<u64 *>(s_token + (K * n + 1) / 2 * 2) + warp * parts * n;
    for (int b = warp; b < K; b += warps) {
        const int64_t row = (int64_t)blockIdx.x * K + b;
        for (int i = lane; i < parts * n; i += 32) s_list[i] = p.keys[row * parts * n + i];
        const float score = p.a.scores[row], my_top = lane < parts ? p.tops[row * parts + lane] : -INFINITY;
        const float top = warp_max(my_top);
        double sum = lane < parts ? p.sums[row * parts + lane] : 0.0;
        if (sum != 0.0) sum *= exp((double)my_top - (double)top);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const double all = (double)top + log(sum);
        const bool alive = isfinite(all) && isfinite(score);
        __syncwarp();
        int at = 0;
        u64 mine = lane < parts ? s_list[lane * n] : 0;
        for (int i = 0; i < n; ++i) {
            int whose, token = i;
            double value = -INFINITY;
            if (alive) {
                const u64 best = warp_best(mine, whose);
                token = (int)~(uint32_t)best;
                if (best) value = (double)score + ((double)from_ordered((uint32_t)(best >> 32)) - all);
                else token = INT32_MAX;                           // a vocabulary of fewer than n
                if (lane == whose) mine = ++at < n ? s_list[lane * n + at] : 0;
            } else if (i >= p.a.vocabulary) {
                token = INT32_MAX;
            }
            if (lane == 0) { s_value[b * n + i] = value; s_token[b * n + i] = token; }
        }
        __syncwarp();
    }
    __syncthreads();
    if (warp != 0) return;
    const int64_t out = (int64_t)blockIdx.x * n, go = (int64_t)blockIdx.x * K;
    const int end = lane < p.a.n_ends ? p.a.ends[lane] : 0;
    int at[2] = {0, 0}, going = 0;
    // A place of none (a beam's list is at its end) is 0, below the key of -infinity.
    auto key_of = [&](int k) { return 2 * lane + k < K && at[k] < n && s_token[(2 * lane + k) * n + at[k]] != INT32_MAX ? ordered64(s_value[(2 * lane + k) * n + at[k]]) : 0ull; };
    u64 mine[2] = {key_of(0), key_of(1)};
    for (int i = 0; i < n; ++i) {
        int whose;
        const u64 best = warp_best(max(mine[0], mine[1]), whose);
        const bool second = mine[0] != best;
        const int k = __shfl_sync(0xffffffffu, (int)second, whose), place = __shfl_sync(0xffffffffu, second ? at[1] : at[0], whose), b = 2 * whose + k;
        const float value = (float)s_value[b * n + place];
        const int token = s_token[b * n + place];
        if (lane == whose) {
            if (second) { ++at[1]; mine[1] = key_of(1); }
            else { ++at[0]; mine[0] = key_of(0); }
        }
        bool ends = lane < p.a.n_ends && end == token;
        for (int e = lane + 32; e < p.a.n_ends; e += 32) ends |= p.a.ends[e] == token;
        ends = __any_sync(0xffffffffu, ends);
        if (lane == 0) {
            p.a.out_scores[out + i] = value;
            p.a.out_beams[out + i] = b;
            p.a.out_tokens[out + i] = token;
            if (!ends && going < K) {
                p.a.next_scores[go + going] = value;
                p.a.next_beams[go + going] = b;
                p.a.next_tokens[go + going] = token;
            }
        }
        going += !ends;
    }
    for (int i = going + lane; i < K; i += 32) {                  // everything else ends
        p.a.next_scores[go + i] = -INFINITY;
        p.a.next_beams[go + i] = 0;
        p.a.next_tokens[go + i] = 0;
    }
}

// Parts of a row: enough CTAs for all SMs, whole first turns; 1024 keys of a beam at most are joined.
static int beam_parts(const kvq_beam_args &a) {
    const int64_t rows = (int64_t)a.requests * a.beams;
    int64_t parts = (4 * 148 + rows - 1) / rows;
    const int64_t most = (a.vocabulary + kScanThreads * kTurn - 1) / (kScanThreads * kTurn);
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
    const int warps = a->beams < 8 ? a->beams : 8, pairs = a->beams * a->n;
    const size_t smem = (size_t)pairs * 8 + (size_t)(pairs + 1) / 2 * 8 + (size_t)warps * p.parts * a->n * 8;
    const cudaError_t e = cudaFuncSetAttribute(beam_join_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e != cudaSuccess) return record_cuda_error(e);
    beam_join_kernel<<<(unsigned)a->requests, 32 * warps, smem, st>>>(p);
    return check_launch();
}
