// The ring of K and V steps in the tile kernel of the long-context attention (attention_long_tc.cu), apart from it so that its protocol can be
// checked on the host.
//
// Item i of K (or V) is filled into a stage of its kind: filler waits for "empty" of the item that had the stage before, fills, completes a phase of
// "full"; the consumers wait for that phase and complete a phase of "empty". A wait names the parity of a phase, which is only unambiguous
// for someone who has seen the phase before it: to one who has not, the phase two before looks complete. K and V therefore have stages of their own, so that every
// phase of a stage is waited for, in order, by each of its consumers and by its filler. (In one ring for both, the issuer of a tile without rows, whom no weights hold
// back, could take the K step before the last V step for that one.)
#pragma once

#include <cstdint>

namespace attn_long {

#ifdef __CUDACC__
#define RLB_BOTH __host__ __device__ __forceinline__
#else
#define RLB_BOTH inline
#endif

template <int K_STAGES, int V_STAGES> struct KvRing {
    static constexpr int K = K_STAGES, V = V_STAGES, STAGES = K + V;
    struct Slot {
        uint32_t stage, parity;   // of the item's phase of "full"; the filler waits for "empty" with the other one,
        bool used;                // if the stage had an item before
    };
    static RLB_BOTH Slot at(bool v, uint32_t i) {
        return v ? Slot{K + i % V, i / V & 1, i >= (uint32_t)V} : Slot{i % K, i / K & 1, i >= (uint32_t)K};
    }
    // What one thread that fills for both kinds fills next, with k and v items of n each filled: K is ahead by a step, as its products are.
    static RLB_BOTH bool next_is_v(int k, int v, int n) { return !(k < n && k <= v + 1); }
};

}  // namespace attn_long
