// Which keys the second look at a part of a row takes (beam_scan_kernel).  No CUDA in it: the host tests walk the same loop.
#pragma once

namespace kvq {

#ifdef __CUDACC__
#define KVQ_BOTH __host__ __device__ __forceinline__
#else
#define KVQ_BOTH inline
#endif

// The first threshold is the key of a thread's best, a value and the PIECE that it is in; one that is raised, because there was no room for all that reached
// it, is the n-th best of those that found room, a value and a TOKEN.  The two are not to be compared with each other: numbers of tokens and of pieces may
// coincide.  Keys by token are all different, so that each raised threshold leaves out all but n of those that found room, and there is room again after a
// few.
struct Reach {
    unsigned long long by_piece, by_token = 0;
    bool raised = false;
    KVQ_BOTH explicit Reach(unsigned long long first) : by_piece(first) {}
    KVQ_BOTH bool takes(unsigned long long piece_key, unsigned long long token_key) const { return piece_key >= by_piece && !(raised && token_key < by_token); }
    KVQ_BOTH void raise(unsigned long long to) {
        by_token = to;
        raised = true;
    }
};

}  // namespace kvq
