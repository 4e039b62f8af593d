// What the products of quantised rows share: which rows a tile of the output
// has, loads that write LDS themselves, and stores of whole runs.  `Args` has
// the products' offsets, m, n, experts, out and vector.
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

typedef const __attribute__((address_space(1))) void *GlobalPtr;
typedef __attribute__((address_space(3))) void *LdsPtr;

__device__ __forceinline__ void load_to_lds(const void *from, void *to) {
    __builtin_amdgcn_global_load_lds((GlobalPtr)from, (LdsPtr)to, 16, 0, 0);
}

// Waits for the wave's loads and LDS accesses, then for the other waves.
__device__ __forceinline__ void arrive() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
}

// The most row tiles, halving from `all`, whose `bytes` each fit into `room`.
constexpr int pass_tiles(int all, int bytes, int room) {
    return all * bytes <= room ? all : pass_tiles(all / 2, bytes, room);
}

// 16 bytes of columns from n0 on of row r.  Nothing here reads them again:
// stores past the caches (8,192 x 2,048 results, k 1,024: 20.7 us, else 22.4).
template <class T, class Args>
__device__ __forceinline__ void store_run(const Args &a, size_t r, size_t n0, u32x4 run) {
    constexpr int kRun = 16 / sizeof(T);
    T *out = reinterpret_cast<T *>(a.out) + r * a.n + n0;
    if (a.vector) {  // rows hold whole runs
        __builtin_nontemporal_store(run, reinterpret_cast<u32x4 *>(out));
    } else {
        typedef T elems __attribute__((ext_vector_type(kRun)));
        const elems v = __builtin_bit_cast(elems, run);
#pragma unroll
        for (int i = 0; i < kRun; ++i)
            if (n0 + i < a.n) out[i] = v[i];
    }
}

}  // namespace layer
