// Where the pieces that a warp copies one after the other lie in its ring of stages, and which phase of a stage's barrier a copy completes.
// (Plain C++: the arithmetic is tested without a GPU.)
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define LSB_RING_FN __host__ __device__ __forceinline__
#else
#define LSB_RING_FN inline
#endif

// Piece k of a walk of n is issued when piece k - (STAGES - 1) is about to be waited for, the first STAGES - 1 before the walk begins.
template <int STAGES>
struct CopyRing {
    uint32_t used;                                 // pieces of the walks before this one
    LSB_RING_FN int stage(int k) const { return (int)((used + (uint32_t)k) % STAGES); }
    LSB_RING_FN uint32_t parity(int k) const { return (used + (uint32_t)k) / STAGES & 1u; }
    // While piece k is waited for, pieces k up to this one are under way.
    LSB_RING_FN static int issued(int k, int n) { return k + STAGES < n ? k + STAGES : n; }
};
