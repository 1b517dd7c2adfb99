// The paged cache's bookkeeping (who holds which page), and the kernels that move pages' contents: new tokens in, pages packed, pages
// copied.
//
// A bookkeeping call is one CTA: its work is a few thousand numbers, and prefix sums over rows and pages inside a CTA give every
// page number without an atomic whose order could change them.  It is a chain of some ten dependent looks at L2.
#include "pages.cuh"
#include "quant_tiles.cuh"

namespace kvq {

constexpr int kBookThreads = 1024;
constexpr int kGone = INT32_MIN;                                  // a page whose last reference this call took

struct BookShared {
    int warp[33];
    long long total;
    int before[kBookThreads], need[kBookThreads], row[kBookThreads], from[kBookThreads];
};

// Exclusive prefix sum over the CTA; `total` the sum.
__device__ __forceinline__ int block_scan(BookShared &s, int v, int &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) s.warp[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int w = s.warp[lane], z = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, z, o);
            if (lane >= o) z += y;
        }
        s.warp[lane] = z - w;
        if (lane == 31) s.warp[32] = z;
    }
    __syncthreads();
    const int r = s.warp[warp] + x - v;
    total = s.warp[32];
    __syncthreads();
    return r;
}

__device__ __forceinline__ long long block_sum(BookShared &s, long long v) {
    if (threadIdx.x == 0) s.total = 0;
    __syncthreads();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) atomicAdd(reinterpret_cast<unsigned long long *>(&s.total), (unsigned long long)v);
    __syncthreads();
    return s.total;
}

// The bookkeeping's numbers as they are used: whatever the tensors hold, no index that follows from them leaves a tensor.
__device__ __forceinline__ int length_of(const kvq_page_book &b, int row) { return min(max(b.length[row], 0), b.max_pages * kPage); }
__device__ __forceinline__ int packed_of(const kvq_page_book &b, int row) { return min(max(b.packed[row], 0), pages_of(length_of(b, row))); }
__device__ __forceinline__ int free_packed(const kvq_page_book &b) { return min(max(b.count[0], 0), b.n_packed); }
__device__ __forceinline__ int free_fp16(const kvq_page_book &b) { return min(max(b.count[1], 0), b.n_fp16); }
__device__ __forceinline__ bool inside(int id, int n) { return id >= 0 && id < n; }

extern __shared__ uint32_t s_seen[];                              // a bit for every slot

__device__ __forceinline__ void clear_seen(const kvq_page_book &b) {
    for (int i = threadIdx.x; i < (b.slots + 31) / 32; i += kBookThreads) s_seen[i] = 0;
    __syncthreads();
}
// Whether a row is in the table and has not been named before.
__device__ __forceinline__ bool first_seen(const kvq_page_book &b, int row) {
    return row >= 0 && row < b.slots && !(atomicOr(&s_seen[row >> 5], 1u << (row & 31)) >> (row & 31) & 1u);
}

// One reference less; the last one marks the page.
__device__ __forceinline__ void drop(int32_t *ref) {
    if (atomicSub(ref, 1) == 1) atomicExch(ref, kGone);
}

// The pages of a pool that were marked go on its stack in ascending order.
__device__ __forceinline__ void collect(BookShared &s, int32_t *refs, int32_t *stack, int n, int32_t *n_free) {
    int at = min(max(*n_free, 0), n), total;
    for (int base = 0; base < n; base += 4 * kBookThreads) {
        const int p = base + 4 * threadIdx.x;
        bool gone[4];
        int mine = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            gone[i] = p + i < n && __ldcg(refs + p + i) == kGone;
            mine += gone[i];
        }
        int k = at + block_scan(s, mine, total);
        at += total;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (gone[i]) {
                refs[p + i] = 0;
                if (k < n) stack[k++] = p + i;
            }
    }
    __syncthreads();
    if (threadIdx.x == 0) *n_free = min(at, n);
}

__global__ void __launch_bounds__(kBookThreads) pages_extend_kernel(kvq_page_book b, const int32_t *rows, const int32_t *counts, int n) {
    __shared__ BookShared s;
    if (refused(b)) return;
    clear_seen(b);
    int bad = 0;
    long long want = 0;
    for (int i = threadIdx.x; i < n; i += kBookThreads) {
        const int row = rows[i], c = counts[i];
        if (!first_seen(b, row) || c < 0) { bad |= KVQ_PAGES_BAD_ROWS; continue; }
        const int len = length_of(b, row);
        if ((long long)len + c > (long long)b.max_pages * kPage) { bad |= KVQ_PAGES_TOO_LONG; continue; }
        want += pages_of(len + c) - pages_of(len);
    }
    bad = (__syncthreads_or(bad & KVQ_PAGES_BAD_ROWS) ? KVQ_PAGES_BAD_ROWS : 0) | (__syncthreads_or(bad & KVQ_PAGES_TOO_LONG) ? KVQ_PAGES_TOO_LONG : 0);
    want = block_sum(s, want);
    const int n_free = free_fp16(b);
    if (!bad && want > n_free) bad = KVQ_PAGES_NO_FP16;
    if (bad) {
        if (threadIdx.x == 0) atomicOr(&b.count[2], bad);
        return;
    }
    int at = 0, total;
    for (int base = 0; base < n; base += kBookThreads) {
        const int i = base + threadIdx.x;
        int need = 0, have = 0, row = 0;
        if (i < n) {
            row = rows[i];
            const int len = length_of(b, row), c = counts[i];
            have = pages_of(len);
            need = pages_of(len + c) - have;
            b.length[row] = len + c;
        }
        s.before[threadIdx.x] = at + block_scan(s, need, total);
        s.need[threadIdx.x] = need;
        s.row[threadIdx.x] = row;
        s.from[threadIdx.x] = have;
        __syncthreads();
        for (int r = threadIdx.x >> 5; r < min(kBookThreads, n - base); r += kBookThreads / 32)
            for (int k = threadIdx.x & 31; k < s.need[r]; k += 32) {
                const int id = b.free_ids[b.n_packed + n_free - 1 - s.before[r] - k];
                b.table[(int64_t)s.row[r] * b.max_pages + s.from[r] + k] = id;
                if (inside(id, b.n_fp16)) b.refs[b.n_packed + id] = 1;
            }
        at += total;
        __syncthreads();
    }
    if (threadIdx.x == 0) b.count[1] = n_free - at;
}

__global__ void __launch_bounds__(kBookThreads) pages_free_kernel(kvq_page_book b, const int32_t *rows, int n) {
    __shared__ BookShared s;
    if (refused(b)) return;
    clear_seen(b);
    bool bad = false;
    for (int i = threadIdx.x; i < n; i += kBookThreads) bad |= !first_seen(b, rows[i]);
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) atomicOr(&b.count[2], KVQ_PAGES_BAD_ROWS);
        return;
    }
    for (int r = threadIdx.x >> 5; r < n; r += kBookThreads / 32) {
        const int row = rows[r], packed = b.packed[row], held = min(max(pages_of(length_of(b, row)), packed), b.max_pages);
        int32_t *t = b.table + (int64_t)row * b.max_pages;
        for (int j = threadIdx.x & 31; j < held; j += 32) {
            const int id = t[j];
            if (inside(id, j < packed ? b.n_packed : b.n_fp16)) drop(b.refs + (j < packed ? id : b.n_packed + id));
            t[j] = -1;
        }
        __syncwarp();
        if ((threadIdx.x & 31) == 0) b.length[row] = b.packed[row] = 0;
    }
    __syncthreads();
    collect(s, b.refs, b.free_ids, b.n_packed, &b.count[0]);
    collect(s, b.refs + b.n_packed, b.free_ids + b.n_packed, b.n_fp16, &b.count[1]);
}

__global__ void __launch_bounds__(kBookThreads) pages_settle_kernel(kvq_page_book b, const int32_t *rows, int n, int window, int32_t *moves) {
    __shared__ BookShared s;
    if (threadIdx.x == 0) moves[0] = 0;
    if (refused(b)) return;
    clear_seen(b);
    bool bad = false;
    long long want = 0;
    auto due = [&](int row) { return max(0, max(0, length_of(b, row) - window) / kPage - packed_of(b, row)); };
    for (int i = threadIdx.x; i < n; i += kBookThreads) {
        const int row = rows[i];
        if (first_seen(b, row)) want += due(row);
        else bad = true;
    }
    bad = __syncthreads_or(bad);
    want = block_sum(s, want);
    const int n_free = free_packed(b);
    if (bad || want > n_free) {
        if (threadIdx.x == 0) atomicOr(&b.count[2], bad ? KVQ_PAGES_BAD_ROWS : KVQ_PAGES_NO_PACKED);
        return;
    }
    if (!want) return;
    int at = 0, total;
    for (int base = 0; base < n; base += kBookThreads) {
        const int i = base + threadIdx.x;
        int need = 0, row = 0, from = 0;
        if (i < n) {
            row = rows[i];
            need = due(row);
            from = packed_of(b, row);
            b.packed[row] = from + need;
        }
        s.before[threadIdx.x] = at + block_scan(s, need, total);
        s.need[threadIdx.x] = need;
        s.row[threadIdx.x] = row;
        s.from[threadIdx.x] = from;
        __syncthreads();
        for (int r = threadIdx.x >> 5; r < min(kBookThreads, n - base); r += kBookThreads / 32)
            for (int k = threadIdx.x & 31; k < s.need[r]; k += 32) {
                int32_t *t = b.table + (int64_t)s.row[r] * b.max_pages + s.from[r] + k;
                const int m = s.before[r] + k, to = b.free_ids[n_free - 1 - m], src = *t;
                moves[4 + 2 * m] = src;
                moves[5 + 2 * m] = to;
                *t = to;
                if (inside(to, b.n_packed)) b.refs[to] = 1;
                if (inside(src, b.n_fp16)) drop(b.refs + b.n_packed + src);
            }
        at += total;
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        moves[0] = at;
        b.count[0] = n_free - at;
    }
    collect(s, b.refs + b.n_packed, b.free_ids + b.n_packed, b.n_fp16, &b.count[1]);
}

__global__ void __launch_bounds__(kBookThreads) pages_fork_kernel(kvq_page_book b, const int32_t *parents, const int32_t *children, int n, int32_t *moves) {
    __shared__ BookShared s;
    if (threadIdx.x == 0) moves[0] = 0;
    if (refused(b)) return;
    clear_seen(b);
    bool bad = false;
    for (int i = threadIdx.x; i < n; i += kBookThreads) bad |= !first_seen(b, children[i]);
    if (!__syncthreads_or(bad)) {
        long long want = 0;
        for (int i = threadIdx.x; i < n; i += kBookThreads) {
            const int row = parents[i];
            if (row < 0 || row >= b.slots || (s_seen[row >> 5] >> (row & 31) & 1u) || b.length[children[i]] != 0) bad = true;
            else want += length_of(b, row) % kPage != 0;
        }
        bad = __syncthreads_or(bad);
        want = block_sum(s, want);
        const int n_free = free_fp16(b);
        if (!bad && want <= n_free) {
            int at = 0, total;
            for (int base = 0; base < n; base += kBookThreads) {
                const int i = base + threadIdx.x;
                const int part = i < n && length_of(b, parents[i]) % kPage != 0;
                s.before[threadIdx.x] = at + block_scan(s, part, total);
                __syncthreads();
                for (int r = threadIdx.x >> 5; r < min(kBookThreads, n - base); r += kBookThreads / 32) {
                    const int from = parents[base + r], to = children[base + r], len = length_of(b, from), packed = packed_of(b, from);
                    const int32_t *src = b.table + (int64_t)from * b.max_pages;
                    int32_t *dst = b.table + (int64_t)to * b.max_pages;
                    for (int j = threadIdx.x & 31; j < pages_of(len); j += 32) {
                        int id = src[j];
                        if ((j + 1) * kPage > len) {              // not full: a page of its own
                            const int m = s.before[r], own = b.free_ids[b.n_packed + n_free - 1 - m];
                            const bool both = inside(id, b.n_fp16) && inside(own, b.n_fp16);        // else page 0 onto itself
                            moves[4 + 2 * m] = both ? id : 0;
                            moves[5 + 2 * m] = both ? own : 0;
                            if (inside(own, b.n_fp16)) b.refs[b.n_packed + own] = 1;
                            id = own;
                        } else if (inside(id, j < packed ? b.n_packed : b.n_fp16)) {
                            atomicAdd(b.refs + (j < packed ? id : b.n_packed + id), 1);
                        }
                        dst[j] = id;
                    }
                    if ((threadIdx.x & 31) == 0) {
                        b.length[to] = len;
                        b.packed[to] = packed;
                    }
                }
                at += total;
                __syncthreads();
            }
            if (threadIdx.x == 0) {
                moves[0] = at;
                b.count[1] = n_free - at;
            }
            return;
        }
    } else {
        bad = true;
    }
    if (threadIdx.x == 0) atomicOr(&b.count[2], bad ? KVQ_PAGES_BAD_ROWS : KVQ_PAGES_NO_FP16);
}

// One pool of kvq_pages_compact.  to: the new number of every page beyond the number of live ones; its entries below that hold
// the list of holes meanwhile (there are no more holes than live pages).
__device__ __forceinline__ int close_up(BookShared &s, int32_t *refs, int32_t *stack, int n, int32_t *n_free, int32_t *moves, int32_t *to) {
    int live = 0;
    for (int p = threadIdx.x; p < n; p += kBookThreads) live += refs[p] > 0;
    live = (int)block_sum(s, live);
    int at = 0, total;
    for (int base = 0; base < live; base += kBookThreads) {
        const int p = base + threadIdx.x;
        const bool hole = p < live && refs[p] <= 0;
        const int k = at + block_scan(s, hole, total);
        if (hole) to[k] = p;
        at += total;
    }
    __syncthreads();
    int moved = 0;
    for (int base = live; base < n; base += kBookThreads) {
        const int p = base + threadIdx.x;
        const int held = p < n ? refs[p] : 0;
        const int k = moved + block_scan(s, held > 0, total);
        if (held > 0) {
            const int hole = to[k];
            moves[4 + 2 * k] = p;
            moves[5 + 2 * k] = hole;
            to[p] = hole;
            refs[hole] = held;
            refs[p] = 0;
        }
        moved += total;
    }
    for (int i = threadIdx.x; i < n - live; i += kBookThreads) stack[i] = n - 1 - i;
    if (threadIdx.x == 0) {
        moves[0] = moved;
        *n_free = n - live;
    }
    __syncthreads();
    return live;
}

__global__ void __launch_bounds__(kBookThreads) pages_compact_kernel(kvq_page_book b, int32_t *moves) {
    __shared__ BookShared s;
    int32_t *moves16 = moves + 4 + 2 * (int64_t)b.n_packed, *to = moves16 + 4 + 2 * (int64_t)b.n_fp16;
    if (threadIdx.x == 0) moves[0] = moves16[0] = 0;
    if (refused(b)) return;
    const int live = close_up(s, b.refs, b.free_ids, b.n_packed, &b.count[0], moves, to);
    const int live16 = close_up(s, b.refs + b.n_packed, b.free_ids + b.n_packed, b.n_fp16, &b.count[1], moves16, to + b.n_packed);
    for (int row = threadIdx.x >> 5; row < b.slots; row += kBookThreads / 32) {
        int32_t *t = b.table + (int64_t)row * b.max_pages;
        const int packed = b.packed[row], held = pages_of(length_of(b, row));
        for (int j = threadIdx.x & 31; j < held; j += 32) {
            const int id = t[j];
            if (j < packed ? id >= live && id < b.n_packed : id >= live16 && id < b.n_fp16) t[j] = to[j < packed ? id : b.n_packed + id];
        }
    }
}

// ---------------------------------------------------------------------------------------------
// New tokens into their pages: a thread takes eight channels of one (token, head), keys and values.
template <bool VEC>
__global__ void __launch_bounds__(256) page_write_kernel(const kvq_page_book b, const kvq_page_layer l, const kvq_page_write_args a) {
    if (refused(b)) return;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int c = (int)(i & 15) * 8;
    const int64_t th = i >> 4;
    const int u = (int)(th / l.Hkv), h = (int)(th - (int64_t)u * l.Hkv);
    if (u >= a.tokens || u < a.q_start[0] || u >= a.q_start[a.n]) return;
    // asked for first: they land while the token's place is looked up, four loads one behind the other
    const __half *k = static_cast<const __half *>(a.k) + u * a.k_sT + h * a.k_sH + c, *v = static_cast<const __half *>(a.v) + u * a.v_sT + h * a.v_sH + c;
    uint4 x, y;
    if constexpr (VEC) {
        x = *reinterpret_cast<const uint4 *>(k);
        y = *reinterpret_cast<const uint4 *>(v);
    } else {
        __half *px = reinterpret_cast<__half *>(&x), *py = reinterpret_cast<__half *>(&y);
#pragma unroll
        for (int j = 0; j < 8; ++j) { px[j] = k[j]; py[j] = v[j]; }
    }
    const int s = sequence_of(a.q_start, a.n, u), row = a.rows[s];
    if (row < 0 || row >= b.slots) return;
    const int pos = length_of(b, row) - max(a.q_start[s + 1], 0) + u, page = pos / kPage;
    const int id = pos >= 0 && page < b.max_pages && page >= b.packed[row] ? b.table[(int64_t)row * b.max_pages + page] : -1;
    if (!inside(id, min(l.n_fp16, b.n_fp16)) || b.refs[b.n_packed + id] > 1) {    // a page that others hold too stays as it is
        if (c == 0) atomicOr(&b.count[2], KVQ_PAGES_NOT_WRITTEN);
        return;
    }
    const int64_t to = (((int64_t)id * l.Hkv + h) * kPage + pos % kPage) * kHeadDim + c;
    *reinterpret_cast<uint4 *>(static_cast<__half *>(l.kfull) + to) = x;
    *reinterpret_cast<uint4 *>(static_cast<__half *>(l.vfull) + to) = y;
}

// ---------------------------------------------------------------------------------------------
// Whole pages from one number to another, in pieces of 16 KB.
constexpr int kCopyPiece = 16384;
struct PageTensors {
    kvq_page_tensor t[KVQ_MAX_PAGE_TENSORS];
    int first[KVQ_MAX_PAGE_TENSORS + 1];                          // the tensors' first pieces of a page
    int n;
};

__global__ void __launch_bounds__(256) page_copy_kernel(const __grid_constant__ PageTensors p, const int32_t *moves, int max_moves) {
    const int pieces = p.first[p.n];
    const int64_t units = (int64_t)min(moves[0], max_moves) * pieces;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int m = (int)(u / pieces), piece = (int)(u - (int64_t)m * pieces);
        int lo = 0, hi = p.n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (p.first[mid] <= piece) lo = mid;
            else hi = mid;
        }
        const int64_t bytes = p.t[lo].page_bytes, at = (int64_t)(piece - p.first[lo]) * kCopyPiece;
        char *base = static_cast<char *>(p.t[lo].base) + at;
        const uint4 *src = reinterpret_cast<const uint4 *>(base + (int64_t)moves[4 + 2 * m] * bytes);
        uint4 *dst = reinterpret_cast<uint4 *>(base + (int64_t)moves[5 + 2 * m] * bytes);
        const int n = (int)min((int64_t)kCopyPiece, bytes - at) / 16;
        uint4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if ((int)threadIdx.x + 256 * i < n) x[i] = src[threadIdx.x + 256 * i];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if ((int)threadIdx.x + 256 * i < n) dst[threadIdx.x + 256 * i] = x[i];
    }
}

// ---------------------------------------------------------------------------------------------
// fp16 pages into packed ones, with quant_core's bit-exact arithmetic.  A unit is one head's keys or values of a page, 128 rows of 128
// elements.  Keys go through shared memory: a thread owns two neighbouring channels and 32 tokens of them (3 bits: a word of 11, the last of
// 7), and the parts of a group meet there; words, scales and minima leave from there in one run.  Values: a thread owns 32 channels of a token,
// the parts of a group meet by shuffles.  Loops over words stay rolled: with a thread's words unrolled, tie path included, warps waited for
// instructions (5.6 of 14 cycles per issued one): 448 pages of 8 heads, 4 bits, 84 us rolled, 129 unrolled.
template <int BITS>
struct PackShared {
    static constexpr int W = page_words(BITS), PAD = W + (BITS == 3 ? 1 : 4), GROUPS = BITS == 3 ? 12 : 4;      // rows are read by 16 bytes, but for 3 bits
    __half2 tile[kPage * 64];
    uint32_t code[128 * PAD];
    __half scale[128 * GROUPS], mn[128 * GROUPS];
    __half2 lo[4][64], hi[4][64];
};

template <int BITS>
__device__ __forceinline__ void pack_keys(const __half *x, int32_t *code, __half *scale, __half *mn, int group, PackShared<BITS> &s) {
    constexpr int QMAX = (1 << BITS) - 1, W = page_words(BITS), PAD = PackShared<BITS>::PAD, FPI = fields_per_word(BITS);
    const int pair = threadIdx.x & 63, part = threadIdx.x >> 6, groups = page_groups(BITS, group);
    {
        uint4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = reinterpret_cast<const uint4 *>(x)[threadIdx.x + 256 * i];
#pragma unroll
        for (int i = 0; i < 8; ++i) reinterpret_cast<uint4 *>(s.tile)[threadIdx.x + 256 * i] = v[i];
    }
    __syncthreads();
    const __half2 *t = s.tile + pair;
    auto put = [&](int w, int e, const __half2 (&raw)[FPI], __half2 lo2, __half2 hi2, int n, int group_at, bool first) {
        const float lo = e ? __high2float(lo2) : __low2float(lo2), range = (e ? __high2float(hi2) : __low2float(hi2)) - lo, sc = range / (float)QMAX;
        const int c = 2 * pair + e;
        s.code[c * PAD + w] = quant_word<BITS>([&](int i) { return i < n ? (e ? __high2float(raw[i]) : __low2float(raw[i])) : lo; }, lo, sc, __frcp_rn(sc));
        if (first) {
            s.scale[c * groups + group_at] = __float2half_rn(stored_scale<QMAX>(range, sc, 0));
            s.mn[c * groups + group_at] = __float2half_rn(lo);
        }
    };
    if constexpr (BITS == 3) {
#pragma unroll 1
        for (int w = part; w < 12; w += 4) {
            const int n = min(11, kPage - 11 * w);
            __half2 raw[11], lo2, hi2;
#pragma unroll
            for (int i = 0; i < 11; ++i) raw[i] = t[(11 * w + min(i, n - 1)) * 64];
            lo2 = hi2 = raw[0];
#pragma unroll
            for (int i = 1; i < 11; ++i) { lo2 = __hmin2(lo2, raw[i]); hi2 = __hmax2(hi2, raw[i]); }
            put(w, 0, raw, lo2, hi2, n, w, true);
            put(w, 1, raw, lo2, hi2, n, w, true);
        }
    } else {
        const int span = group / 32, p0 = part / span * span;
        __half2 lo2 = t[part * 32 * 64], hi2 = lo2;
#pragma unroll
        for (int i = 1; i < 32; ++i) { const __half2 v = t[(part * 32 + i) * 64]; lo2 = __hmin2(lo2, v); hi2 = __hmax2(hi2, v); }
        if (span > 1) {
            s.lo[part][pair] = lo2;
            s.hi[part][pair] = hi2;
            __syncthreads();
            for (int p = p0; p < p0 + span; ++p) { lo2 = __hmin2(lo2, s.lo[p][pair]); hi2 = __hmax2(hi2, s.hi[p][pair]); }
        }
#pragma unroll 1
        for (int k = 0; k < BITS; ++k) {
            __half2 raw[FPI];
#pragma unroll
            for (int i = 0; i < FPI; ++i) raw[i] = t[(part * 32 + k * FPI + i) * 64];
            put(part * BITS + k, 0, raw, lo2, hi2, FPI, part / span, part == p0 && k == 0);
            put(part * BITS + k, 1, raw, lo2, hi2, FPI, part / span, part == p0 && k == 0);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 128 * W / 4; i += 256) {
        const int c = 4 * i / W, w = 4 * i % W;                   // W is a multiple of 4
        uint4 v;
        if constexpr (BITS == 3) v = make_uint4(s.code[c * PAD + w], s.code[c * PAD + w + 1], s.code[c * PAD + w + 2], s.code[c * PAD + w + 3]);
        else v = *reinterpret_cast<const uint4 *>(&s.code[c * PAD + w]);
        reinterpret_cast<uint4 *>(code)[i] = v;
    }
    for (int i = threadIdx.x; i < 128 * groups / 8; i += 256) {
        reinterpret_cast<uint4 *>(scale)[i] = reinterpret_cast<const uint4 *>(s.scale)[i];
        reinterpret_cast<uint4 *>(mn)[i] = reinterpret_cast<const uint4 *>(s.mn)[i];
    }
    __syncthreads();
}

template <int BITS>
__device__ __forceinline__ void pack_values(const __half *x, int32_t *code, __half *scale, __half *mn, int group) {
    if constexpr (BITS == 3) {
        QuantDims d = {1, 1, kPage, kHeadDim, 0, 0, kHeadDim, 1, 0, 0, 12, 0, 0, 12, 11, 0};
#pragma unroll 1
        for (int i = threadIdx.x; i < kPage * 12; i += 256) quant_ragged3_word<__half>(x, code, scale, mn, d, i);
    } else {
        const int groups = kHeadDim / group;
        const QuantDims d = {1, 1, kPage, kHeadDim, 0, 0, kHeadDim, 1, 0, 0, 4 * BITS, 0, 0, groups, group, 0};
#pragma unroll 1
        for (int i = threadIdx.x; i < kPage * 4; i += 256)
            quant_contig_unit<BITS, __half, BITS>(x, code, scale, mn, d, group / 32, true, true, 0, 0, i);
    }
}

template <int KB, int VB>
__global__ void __launch_bounds__(256, 3) page_pack_kernel(const kvq_page_layer l, const int32_t *moves, int max_moves) {
    __shared__ __align__(16) PackShared<KB> s;
    const int64_t units = 2LL * min(moves[0], max_moves) * l.Hkv;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const bool values = u & 1;
        const int m = (int)((u >> 1) / l.Hkv), h = (int)((u >> 1) - (int64_t)m * l.Hkv), src = moves[4 + 2 * m], dst = moves[5 + 2 * m];
        if (src < 0 || src >= l.n_fp16 || dst < 0 || dst >= l.n_packed) continue;
        const int64_t from = ((int64_t)src * l.Hkv + h) * kPageHalf, to = ((int64_t)dst * l.Hkv + h) * kPage;
        if (!values) {
            const int64_t z = to * page_groups(KB, l.group);
            pack_keys<KB>(static_cast<const __half *>(l.kfull) + from, l.kcode + to * page_words(KB), static_cast<__half *>(l.kscale) + z,
                          static_cast<__half *>(l.kmn) + z, l.group, s);
        } else {
            const int64_t z = to * page_groups(VB, l.group);
            pack_values<VB>(static_cast<const __half *>(l.vfull) + from, l.vcode + to * page_words(VB), static_cast<__half *>(l.vscale) + z,
                            static_cast<__half *>(l.vmn) + z, l.group);
        }
    }
}

template <int KB>
static void launch_pack(const kvq_page_layer &l, const int32_t *moves, int max_moves, unsigned grid, cudaStream_t st) {
    switch (l.v_bits) {
        case 1: page_pack_kernel<KB, 1><<<grid, 256, 0, st>>>(l, moves, max_moves); break;
        case 2: page_pack_kernel<KB, 2><<<grid, 256, 0, st>>>(l, moves, max_moves); break;
        case 3: page_pack_kernel<KB, 3><<<grid, 256, 0, st>>>(l, moves, max_moves); break;
        default: page_pack_kernel<KB, 4><<<grid, 256, 0, st>>>(l, moves, max_moves); break;
    }
}

static size_t seen_bytes(const kvq_page_book &b) { return (size_t)(b.slots + 31) / 32 * 4; }

template <typename K>
static int book_smem(K kernel, size_t bytes) {                    // 16 KB (131072 slots) beside BookShared need no asking
    if (bytes <= 16384) return KVQ_OK;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    return e == cudaSuccess ? KVQ_OK : record_cuda_error(e);
}

}  // namespace kvq

extern "C" int kvq_pages_extend(const kvq_page_book *b, const int32_t *rows, const int32_t *counts, int32_t n, kvq_stream_t stream) {
    using namespace kvq;
    if (const int rc = check_book(b)) return rc;
    if (n < 0) return KVQ_ERR_SHAPE;
    if (n == 0) return KVQ_OK;
    if (!rows || !counts) return KVQ_ERR_NULL;
    if (const int rc = book_smem(pages_extend_kernel, seen_bytes(*b))) return rc;
    pages_extend_kernel<<<1, kBookThreads, seen_bytes(*b), reinterpret_cast<cudaStream_t>(stream)>>>(*b, rows, counts, n);
    return count_launch();
}

extern "C" int kvq_pages_free(const kvq_page_book *b, const int32_t *rows, int32_t n, kvq_stream_t stream) {
    using namespace kvq;
    if (const int rc = check_book(b)) return rc;
    if (n < 0) return KVQ_ERR_SHAPE;
    if (n == 0) return KVQ_OK;
    if (!rows) return KVQ_ERR_NULL;
    if (const int rc = book_smem(pages_free_kernel, seen_bytes(*b))) return rc;
    pages_free_kernel<<<1, kBookThreads, seen_bytes(*b), reinterpret_cast<cudaStream_t>(stream)>>>(*b, rows, n);
    return count_launch();
}

extern "C" int kvq_pages_settle(const kvq_page_book *b, const int32_t *rows, int32_t n, int32_t window, int32_t *moves, kvq_stream_t stream) {
    using namespace kvq;
    if (const int rc = check_book(b)) return rc;
    if (n < 0 || window < 0) return KVQ_ERR_SHAPE;
    if (!moves || (n && !rows)) return KVQ_ERR_NULL;
    if (const int rc = book_smem(pages_settle_kernel, seen_bytes(*b))) return rc;
    pages_settle_kernel<<<1, kBookThreads, seen_bytes(*b), reinterpret_cast<cudaStream_t>(stream)>>>(*b, rows, n, window, moves);
    return count_launch();
}

extern "C" int kvq_pages_fork(const kvq_page_book *b, const int32_t *parents, const int32_t *children, int32_t n, int32_t *moves, kvq_stream_t stream) {
    using namespace kvq;
    if (const int rc = check_book(b)) return rc;
    if (n < 0) return KVQ_ERR_SHAPE;
    if (!moves || (n && (!parents || !children))) return KVQ_ERR_NULL;
    if (const int rc = book_smem(pages_fork_kernel, seen_bytes(*b))) return rc;
    pages_fork_kernel<<<1, kBookThreads, seen_bytes(*b), reinterpret_cast<cudaStream_t>(stream)>>>(*b, parents, children, n, moves);
    return count_launch();
}

extern "C" int kvq_pages_compact(const kvq_page_book *b, int32_t *moves, kvq_stream_t stream) {
    using namespace kvq;
    if (const int rc = check_book(b)) return rc;
    if (!moves) return KVQ_ERR_NULL;
    pages_compact_kernel<<<1, kBookThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(*b, moves);
    return count_launch();
}

extern "C" int kvq_page_pack(const kvq_page_layer *l, const int32_t *moves, int32_t max_moves, kvq_stream_t stream) {
    using namespace kvq;
    if (const int rc = check_layer(l)) return rc;
    if (!moves) return KVQ_ERR_NULL;
    if (max_moves <= 0 || !l->n_fp16 || !l->n_packed) return KVQ_OK;
    const int64_t units = 2LL * max_moves * l->Hkv;
    const unsigned grid = (unsigned)(units < 148 * 6 - 1 ? units : 148 * 6 - 1);         // odd: every CTA has keys and values in turn
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    switch (l->k_bits) {
        case 1: launch_pack<1>(*l, moves, max_moves, grid, st); break;
        case 2: launch_pack<2>(*l, moves, max_moves, grid, st); break;
        case 3: launch_pack<3>(*l, moves, max_moves, grid, st); break;
        default: launch_pack<4>(*l, moves, max_moves, grid, st); break;
    }
    return count_launch();
}

extern "C" int kvq_page_copy(const kvq_page_tensor *tensors, int32_t n, const int32_t *moves, int32_t max_moves, kvq_stream_t stream) {
    using namespace kvq;
    if (n < 0 || n > KVQ_MAX_PAGE_TENSORS) return KVQ_ERR_SHAPE;
    if (!moves || (n && !tensors)) return KVQ_ERR_NULL;
    PageTensors p = {};
    for (int i = 0; i < n; ++i) {
        if (!tensors[i].base || tensors[i].page_bytes <= 0) continue;         // an empty pool
        if (reinterpret_cast<uintptr_t>(tensors[i].base) % 16 || tensors[i].page_bytes % 16) return KVQ_ERR_ALIGN;
        if (tensors[i].page_bytes > (1LL << 30)) return KVQ_ERR_SHAPE;
        p.t[p.n] = tensors[i];
        p.first[p.n + 1] = p.first[p.n] + (int)((tensors[i].page_bytes + kCopyPiece - 1) / kCopyPiece);
        ++p.n;
    }
    if (!p.n || max_moves <= 0) return KVQ_OK;
    const int64_t units = (int64_t)max_moves * p.first[p.n];
    page_copy_kernel<<<(unsigned)(units < 148 * 8 ? units : 148 * 8), 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(p, moves, max_moves);
    return count_launch();
}

extern "C" int kvq_page_write(const kvq_page_book *b, const kvq_page_layer *l, const kvq_page_write_args *a, kvq_stream_t stream) {
    using namespace kvq;
    if (const int rc = check_book(b)) return rc;
    if (const int rc = check_layer(l)) return rc;
    if (!a) return KVQ_ERR_NULL;
    if (a->n < 0 || a->tokens < 0) return KVQ_ERR_SHAPE;
    if (a->n == 0 || a->tokens == 0) return KVQ_OK;
    if (!a->k || !a->v || !a->q_start || !a->rows) return KVQ_ERR_NULL;
    auto rows16 = [](const void *p, int64_t t, int64_t h) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && t % 8 == 0 && h % 8 == 0; };
    const bool vec = rows16(a->k, a->k_sT, a->k_sH) && rows16(a->v, a->v_sT, a->v_sH);
    const int64_t ctas = ((int64_t)a->tokens * l->Hkv * 16 + 255) / 256;
    if (ctas > 2147483647LL) return KVQ_ERR_UNSUPPORTED;
    (vec ? page_write_kernel<true> : page_write_kernel<false>)<<<(unsigned)ctas, 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(*b, *l, *a);
    return count_launch();
}
