// The range of 32-bit order keys that a selection by histograms still looks at.
// Plain C++, so that the search's arithmetic is also tested on the host.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define POPKV_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define POPKV_HOST_DEVICE inline
#endif

namespace popkv {

// Keys lo .. hi, both included, in bins of 2^shift() keys, 2^kBits bins at most.  Each step keeps one bin:
// the first leaves at most 2^21 keys, the second 2^10, and the third's bins hold one key each.
struct KeyRange {
    static constexpr int kBits = 11;
    static constexpr int kSteps = 3;
    uint32_t lo, hi;

    POPKV_HOST_DEVICE int shift() const {
        const uint32_t span = hi - lo;
#ifdef __CUDA_ARCH__
        const int bits = 32 - __clz(static_cast<int>(span));
#else
        const int bits = span ? 32 - __builtin_clz(span) : 0;
#endif
        return bits > kBits ? bits - kBits : 0;
    }
    POPKV_HOST_DEVICE bool holds(uint32_t key) const { return key >= lo && key <= hi; }
    POPKV_HOST_DEVICE uint32_t bin(uint32_t key, int shift) const { return (key - lo) >> shift; }
    // Narrows the range to a bin that holds a key.  Distances from lo only: the end of the last bin may lie past
    // 2^32 (the key of NaN is 2^32 - 1).
    POPKV_HOST_DEVICE void keep(uint32_t bin, int shift) {
        lo += bin << shift;
        const uint32_t last = (1u << shift) - 1u;
        if (hi - lo > last) hi = lo + last;
    }
};

}  // namespace popkv
