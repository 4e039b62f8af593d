// What the products of quantised rows share: which rows a tile of the output
// has, and how many of them pass through LDS at a time.  `Args` has the
// products' offsets, m and experts.
#pragma once

#include "layer_math.h"

namespace layer {

// Rows r0 .. r1-1 of the output, one tile of one expert's (expert = experts:
// of none's, which come out as 0).
struct RowTile {
    int expert;
    size_t r0, r1;
};

template <class Args>
__device__ __forceinline__ size_t bound_of(const Args &a, int x) {
    if (!a.offsets) return x <= 0 ? 0 : a.m;
    const int v = a.offsets[x];
    return v < 0 ? 0 : (size_t)v < a.m ? (size_t)v : a.m;
}

// The rows fall into runs: before the first expert, each expert's, behind the
// last.  The wave counts the runs' tiles 64 runs at a time until it reaches
// `tile`; false if there are fewer.
template <class Args>
__device__ __forceinline__ bool find_rows(const Args &a, size_t tile, int height,
                                          RowTile &t) {
    const int lane = threadIdx.x & 63;
    const int runs = a.experts + 2;
    for (int base = 0; base < runs; base += 64) {
        const int x = base + lane - 1;
        size_t lo = 0, hi = 0;
        if (x < a.experts + 1) {
            lo = x < 0 ? 0 : bound_of(a, x);
            hi = x < a.experts ? bound_of(a, x + 1) : a.m;
        }
        const unsigned tiles = hi > lo ? (unsigned)((hi - lo + height - 1) / height) : 0;
        const unsigned sum = (unsigned)running_sum((int)tiles);
        const unsigned long long reach = __ballot(tile < sum);
        if (reach) {
            const int at = __ffsll(reach) - 1;
            // Counts below 2^31, the same for the whole wave.
            const size_t before = __builtin_amdgcn_readlane(sum - tiles, at);
            lo = (unsigned)__builtin_amdgcn_readlane((int)lo, at);
            hi = (unsigned)__builtin_amdgcn_readlane((int)hi, at);
            const int expert = base + at - 1;
            t.expert = expert < 0 ? a.experts : expert;
            t.r0 = lo + (tile - before) * height;
            t.r1 = t.r0 + height < hi ? t.r0 + height : hi;
            return true;
        }
        tile -= __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

typedef __attribute__((address_space(3))) void *LdsPtr;

// The most row tiles, halving from `all`, whose `bytes` each fit into `room`.
constexpr int pass_tiles(int all, int bytes, int room) {
    return all * bytes <= room ? all : pass_tiles(all / 2, bytes, room);
}

}  // namespace layer
