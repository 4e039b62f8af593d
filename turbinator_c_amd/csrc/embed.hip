// Embeddings (hip_layers.h): lookup with scaling, the order of the tokens by
// entry, and the table's gradient in that order.
//
//   lookup     out[t] = base[t] + scale table[id[t]]
//   order      the tokens sorted by id, equal ids in the order of the tokens;
//              range v = the places of entry v's tokens in it
//   gradient   dtable[v] = scale sum_{t: id[t] = v} dout[t]
//
// The gradient adds up partial sums of the order's places, whose tree the ranges
// and sizes fix, so that it never depends on timing (but on where a range lies
// among the chunks, and on the kernel that the sizes choose); every entry's row
// is written once, dout is read once.
//
// Lookup is bound by memory: 163,840 x 1,024 bf16 of 32,768 entries 92 us (84 at a
// copy's rate).  The gradient of as much, skewed: the order 32 us, five launches
// of which each is mostly its own chain; the sums 86 us for the 470 MB of dout
// and table and 30 to 40 of parts (5.9 TB/s); the joins 15.
#include "layer_math.h"

namespace {

using namespace layer;

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr size_t kMaxCount = 0x7fffffffu, kMaxGrid = 1 << 20;

unsigned grid_of(size_t items, size_t per) {
    const size_t want = (items + per - 1) / per;
    return (unsigned)(want < kMaxGrid ? want : kMaxGrid);
}

// Rows in vectors of B bytes, the last of which ends with the row and repeats
// some of the one before; `lanes` lanes, a power of two, have a vector each.
struct RowShape {
    unsigned width, vectors, pieces, lanes;
};

template <class T, int B>
RowShape shape_of(size_t width) {
    RowShape s;
    s.width = (unsigned)width;
    s.vectors = (unsigned)((width * sizeof(T) + B - 1) / B);
    s.pieces = (s.vectors + 63) / 64;
    s.lanes = 1;
    while (s.lanes < s.vectors && s.lanes < 64) s.lanes *= 2;
    return s;
}

// Vector v's first element.
template <int N>
__device__ __forceinline__ unsigned first_of(const RowShape &s, unsigned v) {
    return (v + 1) * N <= s.width ? v * N : s.width - N;
}

// --------------------------------------------------------------------------
// Lookup

struct LookupArgs {
    const int *ids;
    const char *table, *base;
    char *out;
    size_t table_stride, base_stride, tokens, entries;
    float scale;
    bool stream;  // base past the caches
    RowShape s;
};

template <class T, int B, int LANES>
__global__ __launch_bounds__(kThreads) void lookup_kernel(LookupArgs a) {
    typedef Vec<T, B> X;
    typedef typename X::raw raw;
    const unsigned lanes = LANES ? LANES : a.s.lanes, lane = threadIdx.x & (lanes - 1);
    const unsigned groups = kThreads / lanes;
    unsigned group = threadIdx.x / lanes;
    if (LANES == 64) group = __builtin_amdgcn_readfirstlane(group);
    const size_t items = a.tokens * a.s.pieces, row_bytes = (size_t)a.s.width * sizeof(T);
    for (size_t item = (size_t)blockIdx.x * groups + group; item < items;
         item += (size_t)gridDim.x * groups) {
        const size_t t = a.s.pieces > 1 ? item / a.s.pieces : item;
        const unsigned v = (unsigned)(item - t * a.s.pieces) * lanes + lane;
        if (v >= a.s.vectors) continue;
        const unsigned e = first_of<X::n>(a.s, v);
        const int id = a.ids[t];
        raw out = {};
        if (a.base && a.stream)
            out = stream_in<T, B>(a.base + t * a.base_stride, e);
        else if (a.base)
            out = load_loose<T, B>(a.base + t * a.base_stride, e);
        if (id >= 0 && (size_t)id < a.entries) {
            float x[X::n], y[X::n];
            X::unpack(load_loose<T, B>(a.table + (size_t)id * a.table_stride, e), x);
            X::unpack(out, y);
#pragma unroll
            for (int i = 0; i < X::n; ++i)
                y[i] = a.base ? fmaf(a.scale, x[i], y[i]) : a.scale * x[i];
            out = X::pack(y);
        }
        stream_out<T, B>(a.out + t * row_bytes, e, out);
    }
}

// --------------------------------------------------------------------------
// Order

struct OrderArgs {
    const int *ids, *from;  // from: the order of the pass before, NULL for none
    int *to;
    i32x2 *ranges;
    int *counts;            // [segments][digits + 1]
    size_t tokens, entries, segment;
    unsigned segments;
    int shift, bits, last;  // last: the pass whose order is the result
};

// The entry of a token, `entries` for none.
__device__ __forceinline__ unsigned entry_of(const int *ids, size_t entries, size_t t) {
    const unsigned id = (unsigned)ids[t], none = (unsigned)entries;
    return id < none ? id : none;
}

__global__ __launch_bounds__(kThreads) void clear_kernel(i32x2 *ranges, size_t entries) {
    for (size_t v = (size_t)blockIdx.x * kThreads + threadIdx.x; v < entries;
         v += (size_t)gridDim.x * kThreads)
        ranges[v] = (i32x2){0, 0};
}

// The lanes with the same value of `bits` bits among those that are live.
__device__ __forceinline__ unsigned long long same_lanes(bool live, unsigned value, int bits) {
    unsigned long long same = __ballot(live);
    for (int bit = 0; bit < bits; ++bit) {
        const bool set = value >> bit & 1;
        const unsigned long long all = __ballot(set);
        same &= set ? all : ~all;
    }
    return same;
}

// Few tokens: a token's place is the number of smaller keys and of equal ones
// before it, an entry's range what lies below and up to it.  Each lane has a
// token (or an entry), each wave a share of the keys, which come through scalar
// loads; the shares are added up in LDS.  RANGES: each entry's first token writes
// its range, which takes a second comparison.
constexpr int kRankWaves = 16;

template <bool RANGES>
__global__ __launch_bounds__(64 * kRankWaves) void rank_kernel(OrderArgs a, unsigned token_blocks) {
    __shared__ int parts[kRankWaves][3][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const bool tokens = blockIdx.x < token_blocks;
    const int n = (int)a.tokens, last = tokens ? n : (int)a.entries;
    const int i0 = (tokens ? blockIdx.x : blockIdx.x - token_blocks) * 64, i = i0 + lane;
    const unsigned key = !tokens ? i : i < n ? entry_of(a.ids, a.entries, i) : 0;
    // Smaller keys; those and equal ones; keys in front of the token's.
    int less = 0, most = 0, place = 0;
    for (int j0 = wave * 64; j0 < n; j0 += 64 * kRankWaves) {
        const int j1 = j0 + 64 < n ? j0 + 64 : n;
        // Equal keys count in front of the token's 64, and not among or behind them.
        const unsigned bound = tokens && j0 < i0 ? key + 1 : key;
        int front = 0;
        if (RANGES || !tokens) {
            int below = 0, upto = 0;
#pragma unroll 16
            for (int j = j0; j < j1; ++j) {
                const unsigned o = entry_of(a.ids, a.entries, j);
                below += o < key;
                upto += o <= key;
            }
            less += below;
            most += upto;
            front = j0 < i0 ? upto : below;
        } else {
#pragma unroll 16
            for (int j = j0; j < j1; ++j) front += entry_of(a.ids, a.entries, j) < bound;
        }
        if (tokens && j0 == i0) {
            // Behind the smaller ones, the lanes in front with the same key.
            front += __popcll(same_lanes(true, key, a.bits) & ((1ull << lane) - 1));
        }
        place += front;
    }
    parts[wave][0][lane] = less;
    parts[wave][1][lane] = most;
    parts[wave][2][lane] = place;
    __syncthreads();
    if (wave || i >= last) return;
    for (int w = 1; w < kRankWaves; ++w) {
        less += parts[w][0][lane];
        most += parts[w][1][lane];
        place += parts[w][2][lane];
    }
    const bool known = key < a.entries;
    if (tokens) a.to[place] = known ? i : -1;
    if (!tokens)
        a.ranges[i] = most > less ? (i32x2){less, most} : (i32x2){0, 0};
    else if (RANGES && known && place == less)
        a.ranges[key] = (i32x2){less, most};
}

// Some thousand tokens: the counting sort below in one workgroup, keys and both
// orders in LDS, seven bits or fewer at a time; tokens without an entry have the
// largest key.  Each wave has a run of the order, of four turns at the most.
constexpr int kSmallWaves = 16, kSmallSort = 64 * kSmallWaves, kSmallBits = 7;
constexpr int kSmallTurns = 4;
constexpr size_t kSmallMost = kSmallSort * kSmallTurns;

__global__ __launch_bounds__(kSmallSort) void sort_kernel(OrderArgs a, int passes, bool clear) {
    __shared__ unsigned key[kSmallMost];
    __shared__ unsigned short order[2][kSmallMost];
    __shared__ int next[kSmallWaves][1 << kSmallBits], start[1 << kSmallBits];
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63, n = (int)a.tokens;
    const int digits = 1 << a.bits, run = (n + kSmallSort - 1) / kSmallSort * 64;
    // At most 64 kSmallTurns: n is at most kSmallMost.
    const int c0 = wave * run, c1 = c0 + run < n ? c0 + run : n;
    for (int c = t; c < n; c += kSmallSort) {
        key[c] = entry_of(a.ids, a.entries, c);
        order[0][c] = (unsigned short)c;
    }
    if (clear)
        for (size_t v = t; v < a.entries; v += kSmallSort) a.ranges[v] = (i32x2){0, 0};
    for (int p = 0; p < passes; ++p) {
        const unsigned short *from = order[p & 1];
        unsigned short *to = order[(p + 1) & 1];
        const int shift = p * a.bits;
        for (int i = t; i < kSmallWaves * digits; i += kSmallSort) next[i / digits][i % digits] = 0;
        __syncthreads();
        unsigned token[kSmallTurns], digit[kSmallTurns];
#pragma unroll
        for (int j = 0; j < kSmallTurns; ++j)
            token[j] = c0 + 64 * j + lane < c1 ? from[c0 + 64 * j + lane] : 0;
#pragma unroll
        for (int j = 0; j < kSmallTurns; ++j) {
            digit[j] = key[token[j]] >> shift & (digits - 1);
            if (c0 + 64 * j + lane < c1) atomicAdd(&next[wave][digit[j]], 1);
        }
        __syncthreads();
        if (t < digits) {
            int all = 0;
            for (int w = 0; w < kSmallWaves; ++w) {
                const int count = next[w][t];
                next[w][t] = all;
                all += count;
            }
            start[t] = all;
        }
        __syncthreads();
        if (wave == 0) {
            int below = 0;
            for (int d0 = 0; d0 < digits; d0 += 64) {
                const int d = d0 + lane, count = d < digits ? start[d] : 0;
                const int sum = running_sum(count);
                if (d < digits) start[d] = below + sum - count;
                below += __builtin_amdgcn_readlane(sum, 63);
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kSmallTurns; ++j) {
            if (c0 + 64 * j >= c1) break;
            const bool live = c0 + 64 * j + lane < c1;
            const unsigned d = digit[j];
            const unsigned long long same = same_lanes(live, d, a.bits);
            const int rank = __popcll(same & ((1ull << lane) - 1));
            const int at = next[wave][d] + rank;
            wave_fence();
            if (live && rank == 0) next[wave][d] = at + __popcll(same);
            wave_fence();
            if (live) to[start[d] + at] = (unsigned short)token[j];
        }
        __syncthreads();
    }
    const unsigned short *sorted = order[passes & 1];
    for (int c = t; c < n; c += kSmallSort) {
        const unsigned token = sorted[c], id = key[token];
        const bool known = id < a.entries;
        a.to[c] = known ? (int)token : -1;
        int *range = reinterpret_cast<int *>(a.ranges + id);
        if (known && (c == 0 || key[sorted[c - 1]] != id)) range[0] = c;
        if (known && (c + 1 == n || key[sorted[c + 1]] != id)) range[1] = c + 1;
    }
}

// Many tokens: a stable counting sort by digits, the least first; tokens
// without an entry have a digit of their own behind the others.  A workgroup
// has a segment of the tokens, each of its waves a run of it.  Segments of 512:
// 12,693 tokens to 2,945 x 592 fp16 with their gradient 35.5 us, of 1,024 37.2;
// more than 256 of them make every workgroup add up more counts than it places
// tokens (163,840 tokens: 135 us with 256 at the most, 146 with 320).
constexpr int kSortBits = 9, kSortThreads = 1 << kSortBits, kSortWaves = kSortThreads / 64;
constexpr size_t kSegment = 512, kMaxSegments = 256;

__device__ __forceinline__ unsigned digit_of(const OrderArgs &a, size_t c, int &token) {
    token = a.from ? a.from[c] : (int)c;
    const unsigned id = (unsigned)a.ids[token];
    return id < a.entries ? id >> a.shift & ((1u << a.bits) - 1) : 1u << a.bits;
}

__global__ __launch_bounds__(kSortThreads) void count_kernel(OrderArgs a) {
    extern __shared__ int lds[];
    const int digits = (1 << a.bits) + 1;
    for (int d = threadIdx.x; d < digits; d += kSortThreads) lds[d] = 0;
    __syncthreads();
    const size_t c0 = blockIdx.x * a.segment;
    const size_t c1 = c0 + a.segment < a.tokens ? c0 + a.segment : a.tokens;
    for (size_t c = c0 + threadIdx.x; c < c1; c += kSortThreads) {
        int token;
        atomicAdd(&lds[digit_of(a, c, token)], 1);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += kSortThreads)
        a.counts[(size_t)blockIdx.x * digits + d] = lds[d];
    // A single pass knows the ranges, others look for them in the order.
    if (!a.shift && !a.last)
        for (size_t v = (size_t)blockIdx.x * kSortThreads + threadIdx.x; v < a.entries;
             v += (size_t)gridDim.x * kSortThreads)
            a.ranges[v] = (i32x2){0, 0};
}

// A lane's tokens of one turn and their digits, one past the others behind c1.
constexpr int kBatch = 4, kCounts = 16;
struct Turn {
    int token[kBatch];  // -1 behind c1
    unsigned digit[kBatch];
    __device__ __forceinline__ void tokens(const OrderArgs &a, size_t c, size_t c1) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const size_t at = c + 64 * j;
            token[j] = at >= c1 ? -1 : a.from ? a.from[at] : (int)at;
        }
    }
    __device__ __forceinline__ void keys(const OrderArgs &a) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j) digit[j] = (unsigned)a.ids[token[j] < 0 ? 0 : token[j]];
    }
    __device__ __forceinline__ void digits(const OrderArgs &a) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
            digit[j] = token[j] < 0              ? ~0u
                       : digit[j] < a.entries ? digit[j] >> a.shift & ((1u << a.bits) - 1)
                                              : 1u << a.bits;
    }
    __device__ __forceinline__ void load(const OrderArgs &a, size_t c, size_t c1) {
        tokens(a, c, c1);
        keys(a);
        digits(a);
    }
};

__global__ __launch_bounds__(kSortThreads) void place_kernel(OrderArgs a) {
    extern __shared__ int lds[];
    const int digits = (1 << a.bits) + 1, lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int *start = lds, *next = lds + digits * (1 + wave), *before = lds + digits * (1 + kSortWaves);
    const size_t run = a.segment / kSortWaves, c0 = blockIdx.x * a.segment + wave * run;
    const size_t c1 = c0 + run < a.tokens ? c0 + run : a.tokens;
    Turn now;
    now.tokens(a, c0 + lane, c1);
    for (int i = threadIdx.x; i < digits * (2 + kSortWaves); i += kSortThreads) lds[i] = 0;
    __syncthreads();
    now.keys(a);
    // The last digit needs the counts before only: nothing lies behind it.
    static_assert(kMaxSegments <= kSortThreads);
    int none = 0;
    if (threadIdx.x < blockIdx.x) none = a.counts[(size_t)threadIdx.x * digits + digits - 1];
    // Of the others: all segments' counts, and those of the segments before.  The
    // segments are shared out, and a thread's counts of kCounts are on their way
    // at once.
    const int shares = a.bits < kSortBits ? 1 << (kSortBits - a.bits) : 1;
    for (int i = threadIdx.x; i < shares << a.bits; i += kSortThreads) {
        const int d = i & ((1 << a.bits) - 1);
        int all = 0, front = 0;
        for (unsigned s0 = i >> a.bits; s0 < a.segments; s0 += shares * kCounts) {
            int n[kCounts];
#pragma unroll
            for (int j = 0; j < kCounts; ++j) {
                const unsigned s = s0 + j * shares;
                n[j] = a.counts[(s < a.segments ? s : 0u) * digits + d];
            }
#pragma unroll
            for (int j = 0; j < kCounts; ++j) {
                const unsigned s = s0 + j * shares;
                all += s < a.segments ? n[j] : 0;
                front += s < blockIdx.x ? n[j] : 0;
            }
        }
        atomicAdd(&start[d], all);
        atomicAdd(&before[d], front);
    }
    if (none) atomicAdd(&before[digits - 1], none);
    now.digits(a);
    __syncthreads();
    for (size_t c = c0; c < c1; c += 64 * kBatch) {
        if (c > c0) now.load(a, c + lane, c1);
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
            if (now.digit[j] != ~0u) atomicAdd(&next[now.digit[j]], 1);
    }
    if (wave == 0) {
        int below = 0;
        for (int d0 = 0; d0 < digits; d0 += 64) {
            const int d = d0 + lane, n = d < digits ? start[d] : 0, sum = running_sum(n);
            if (d < digits) start[d] = below + sum - n + before[d];
            if (a.last && !a.shift && blockIdx.x == 0 && (size_t)d < a.entries)
                a.ranges[d] = n ? (i32x2){below + sum - n, below + sum} : (i32x2){0, 0};
            below += __builtin_amdgcn_readlane(sum, 63);
        }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += kSortThreads) {
        int at = start[d];
        for (int w = 0; w < kSortWaves; ++w) {
            const int n = lds[digits * (1 + w) + d];
            lds[digits * (1 + w) + d] = at;
            at += n;
        }
    }
    __syncthreads();
    for (size_t c = c0; c < c1; c += 64 * kBatch) {
        // One turn holds a run of the usual length throughout.
        if (run > 64 * kBatch) now.load(a, c + lane, c1);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            if (c + 64 * j >= c1) break;
            const unsigned d = now.digit[j];
            const bool live = d != ~0u;
            const unsigned long long same = same_lanes(live, d, a.bits + 1);
            const int rank = __popcll(same & ((1ull << lane) - 1));
            int at = 0;
            if (live) at = next[d] + rank;
            wave_fence();
            if (live && rank == 0) next[d] = at + __popcll(same);
            wave_fence();
            if (live) a.to[at] = a.last && d == 1u << a.bits ? -1 : now.token[j];
        }
    }
}

// The ranges from the places where the entry changes.
__global__ __launch_bounds__(kThreads) void range_kernel(OrderArgs a) {
    for (size_t c = (size_t)blockIdx.x * kThreads + threadIdx.x; c < a.tokens;
         c += (size_t)gridDim.x * kThreads) {
        const int token = a.to[c];
        if (token < 0) continue;
        const int id = a.ids[token], front = c ? a.to[c - 1] : -1;
        const int behind = c + 1 < a.tokens ? a.to[c + 1] : -1;
        int *range = reinterpret_cast<int *>(a.ranges + id);
        if (front < 0 || a.ids[front] != id) range[0] = (int)c;
        if (behind < 0 || a.ids[behind] != id) range[1] = (int)c + 1;
    }
}

// --------------------------------------------------------------------------
// Gradient.  An entry with at most kChunk tokens is summed by one group of
// lanes.  Longer ranges are cut where the order's chunks of kChunk places end:
// a chunk has parts of at most two of them, the one that its first place
// belongs to and the one that its last does; the parts are summed side by side
// into the workspace and joined afterwards.

constexpr size_t kChunk = 32;

struct GradArgs {
    const char *dout;
    size_t stride;
    const int *ids, *order;
    const i32x2 *ranges;
    float *dtable, *parts;  // parts: [chunks][2][part_width]
    size_t tokens, entries, part_width, chunks, chunk_blocks;
    float scale;
    RowShape s;
};

// An entry's range, within the order whatever it holds.
__device__ __forceinline__ i32x2 range_of(const GradArgs &a, size_t v) {
    i32x2 r = a.ranges[v];
    r[0] = r[0] < 0 ? 0 : r[0];
    r[1] = (size_t)(r[1] < 0 ? 0 : r[1]) < a.tokens ? r[1] : (int)a.tokens;
    return r;
}

// The entry of a place of the order, -1 for none.
__device__ __forceinline__ long long entry_at(const GradArgs &a, size_t place) {
    const int t = a.order[place];
    if (t < 0 || (size_t)t >= a.tokens) return -1;
    const int id = a.ids[t];
    return id >= 0 && (size_t)id < a.entries ? id : -1;
}

// Adds up element e on of the rows at every `step`th place from b to end of the
// order, four rows at a time and those in pairs, the next places on their way
// meanwhile.  More at a time cost registers, and with them waves whose chains of
// loads (range, places, rows) overlap: 163,840 x 1,024 bf16 to 32,768 entries
// with their order 137 us, and 142 with two, 149 with eight (153 without looking
// ahead); of smaller gradients eight saves up to 8%.
template <class T, int B, bool STREAM>
__device__ __forceinline__ void add_rows(const GradArgs &a, long long b, long long end, int step,
                                         unsigned e, float (&sum)[Vec<T, B>::n]) {
    typedef Vec<T, B> X;
    constexpr int kAhead = 4;
    int token[kAhead];
    auto look = [&](long long first) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            token[i] = first + i * step < end ? a.order[first + i * step] : -1;
    };
    look(b);
    for (; b < end; b += kAhead * step) {
        typename X::raw row[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const char *from = a.dout + (size_t)token[i] * a.stride;
            row[i] = typename X::raw{};
            if (token[i] >= 0 && (size_t)token[i] < a.tokens)
                row[i] = STREAM ? stream_in<T, B>(from, e) : load_loose<T, B>(from, e);
        }
        look(b + kAhead * step);  // on their way with the rows
        float x[kAhead][X::n];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) X::unpack(row[i], x[i]);
#pragma unroll
        for (int half = kAhead / 2; half; half /= 2)
#pragma unroll
            for (int i = 0; i < half; ++i)
#pragma unroll
                for (int j = 0; j < X::n; ++j) x[i][j] += x[i + half][j];
#pragma unroll
        for (int j = 0; j < X::n; ++j) sum[j] += x[0][j];
    }
}

template <int N>
__device__ __forceinline__ void store_floats(float *row, unsigned e, const float (&v)[N],
                                             float scale) {
    constexpr int kPart = N < 4 ? N : 4;
    typedef Vec<float, kPart * 4> F;
#pragma unroll
    for (int p = 0; p < N; p += kPart) {
        float part[kPart];
#pragma unroll
        for (int j = 0; j < kPart; ++j) part[j] = v[p + j] * scale;
        store_loose<float, kPart * 4>(reinterpret_cast<char *>(row), e + p, F::pack(part));
    }
}

// STREAM: dout is read past the caches.
template <class T, int B, int LANES, bool STREAM>
__global__ __launch_bounds__(kThreads) void grad_kernel(GradArgs a) {
    constexpr int N = Vec<T, B>::n;
    const unsigned lanes = LANES ? LANES : a.s.lanes, lane = threadIdx.x & (lanes - 1);
    const unsigned groups = kThreads / lanes;
    unsigned group = threadIdx.x / lanes;
    if (LANES == 64) group = __builtin_amdgcn_readfirstlane(group);
    const bool whole = blockIdx.x >= a.chunk_blocks;
    const size_t block = whole ? blockIdx.x - a.chunk_blocks : blockIdx.x;
    const size_t blocks = whole ? gridDim.x - a.chunk_blocks : a.chunk_blocks;
    const size_t items = (whole ? a.entries : a.chunks) * a.s.pieces;
    for (size_t item = block * groups + group; item < items; item += blocks * groups) {
        const size_t at = a.s.pieces > 1 ? item / a.s.pieces : item;
        const unsigned v = (unsigned)(item - at * a.s.pieces) * lanes + lane;
        if (v >= a.s.vectors) continue;
        const unsigned e = first_of<N>(a.s, v);
        float sum[N] = {};
        if (whole) {
            const i32x2 r = range_of(a, at);
            if (r[1] - r[0] > (int)kChunk) continue;
            add_rows<T, B, STREAM>(a, r[0], r[1], 1, e, sum);
            store_floats<N>(a.dtable + at * a.s.width, e, sum, a.scale);
            continue;
        }
        const size_t c0 = at * kChunk, c1 = c0 + kChunk < a.tokens ? c0 + kChunk : a.tokens;
        const long long head = entry_at(a, c0), tail = entry_at(a, c1 - 1);
        float *part = a.parts + at * 2 * a.part_width;
        if (head >= 0) {
            const i32x2 r = range_of(a, head);
            if (r[1] - r[0] > (int)kChunk) {
                add_rows<T, B, STREAM>(a, (long long)c0, r[1] < (long long)c1 ? r[1] : (long long)c1, 1,
                               e, sum);
                store_floats<N>(part, e, sum, 1.0f);
            }
        }
        if (tail >= 0 && tail != head) {
            const i32x2 r = range_of(a, tail);
            if (r[1] - r[0] > (int)kChunk) {
                float other[N] = {};
                add_rows<T, B, STREAM>(a, r[0] > (long long)c0 ? r[0] : (long long)c0, (long long)c1, 1,
                               e, other);
                store_floats<N>(part + a.part_width, e, other, 1.0f);
            }
        }
    }
}

// Joins the parts of the long ranges: a workgroup has 16 chunks and 64 columns,
// and finds the ranges that start in its chunks, at most one in each.  Those of
// a few parts are added up by 16 lanes each, the others by the workgroup.  More
// threads would shorten a single range's chain (163,840 tokens of one entry,
// 512 wide, with their order 6 of 73 us with 512 threads), but most workgroups
// find little to do (32,768 entries, 1,024 wide: 8 of 153 us more).
constexpr int kJoinThreads = 256, kJoinLanes = 16, kJoinGroups = kJoinThreads / kJoinLanes;
constexpr int kJoinColumns = 4 * kJoinLanes, kJoinChunks = 16, kJoinShort = 8, kJoinAhead = 8;
static_assert(kJoinChunks <= kJoinGroups);

__global__ __launch_bounds__(kJoinThreads) void join_kernel(GradArgs a) {
    __shared__ f32x4 sums[kJoinGroups][kJoinLanes];
    __shared__ int entries[kJoinChunks], slots[kJoinChunks], ends[kJoinChunks];
    const size_t slices = (a.s.width + kJoinColumns - 1) / kJoinColumns;
    const size_t blocks = (a.chunks + kJoinChunks - 1) / kJoinChunks;
    const unsigned lane = threadIdx.x % kJoinLanes, group = threadIdx.x / kJoinLanes;
    for (size_t item = blockIdx.x; item < blocks * slices; item += gridDim.x) {
        const size_t first = item / slices * kJoinChunks;
        const size_t column = item % slices * kJoinColumns + lane * 4;
        if (threadIdx.x < kJoinChunks) {
            const size_t chunk = first + threadIdx.x, c0 = chunk * kChunk;
            entries[threadIdx.x] = -1;
            if (chunk < a.chunks) {
                const size_t c1 = c0 + kChunk < a.tokens ? c0 + kChunk : a.tokens;
                const long long entry = entry_at(a, c1 - 1);
                const i32x2 r = entry < 0 ? (i32x2){0, 0} : range_of(a, entry);
                if (r[1] - r[0] > (int)kChunk && (size_t)r[0] >= c0 && (size_t)r[0] < c1) {
                    entries[threadIdx.x] = (int)entry;
                    // The first chunk's sum is its second one unless the range fills it.
                    slots[threadIdx.x] = (size_t)r[0] > c0;
                    ends[threadIdx.x] = (int)(((size_t)r[1] - 1) / kChunk - chunk) + 1;
                }
            }
        }
        __syncthreads();
        // Sums parts b, b + step, .. of a range that starts in chunk first + i,
        // kJoinAhead of them on their way at once, the last ones too (81,920 tokens to
        // 256 x 128 fp16 with their order 35.5 us, one at a time 37.2; twelve at once cost
        // the large case of the file's head 3 us).
        auto add = [&](int i, int b, int step) {
            f32x4 sum = {0, 0, 0, 0};
            if (column >= a.part_width) return sum;
            const int end = ends[i];
            const float *head = a.parts + (2 * (first + i) + slots[i]) * a.part_width + column;
            const float *part = a.parts + 2 * (first + i) * a.part_width + column;
            auto at = [&](int c) {
                return *reinterpret_cast<const f32x4 *>(
                    c ? part + (size_t)(2 * c) * a.part_width : head);
            };
            int c = b;
            for (; c + (kJoinAhead - 1) * step < end; c += kJoinAhead * step) {
                f32x4 x[kJoinAhead];
#pragma unroll
                for (int j = 0; j < kJoinAhead; ++j) x[j] = at(c + j * step);
#pragma unroll
                for (int j = 0; j < kJoinAhead; ++j) sum += x[j];
            }
            if (c < end) {
                f32x4 x[kJoinAhead];
#pragma unroll
                for (int j = 0; j < kJoinAhead; ++j) x[j] = at(c + j * step < end ? c + j * step : c);
#pragma unroll
                for (int j = 0; j < kJoinAhead; ++j)
                    if (c + j * step < end) sum += x[j];
            }
            return sum;
        };
        auto write = [&](int i, f32x4 sum) {
            float *row = a.dtable + (size_t)entries[i] * a.s.width + column;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (column + j < a.s.width) row[j] = sum[j] * a.scale;
        };
        if (group < kJoinChunks && entries[group] >= 0 && ends[group] <= kJoinShort)
            write(group, add(group, 0, 1));
        for (int i = 0; i < kJoinChunks; ++i) {
            if (entries[i] < 0 || ends[i] <= kJoinShort) continue;
            sums[group][lane] = add(i, group, kJoinGroups);
            __syncthreads();
            for (int half = kJoinGroups / 2; half; half /= 2) {
                if ((int)group < half) sums[group][lane] += sums[group + half][lane];
                __syncthreads();
            }
            if (group == 0) write(i, sums[0][lane]);
        }
        __syncthreads();
    }
}

// Few tokens and entries: a workgroup has an entry's row or a piece of it, its
// groups of lanes every so manieth token; their sums meet in LDS, in pairs.
// One launch instead of two.
constexpr int kSmallThreads = 1024;
constexpr size_t kSmallTokens = 4096, kSmallItems = 4096;

template <class T, int B>
__global__ __launch_bounds__(kSmallThreads) void small_kernel(GradArgs a) {
    constexpr int N = Vec<T, B>::n;
    __shared__ float sums[N][kSmallThreads];
    const unsigned lane = threadIdx.x & (a.s.lanes - 1), group = threadIdx.x / a.s.lanes;
    const unsigned groups = kSmallThreads / a.s.lanes;
    const size_t entry = blockIdx.x / a.s.pieces;
    const unsigned v = (unsigned)(blockIdx.x - entry * a.s.pieces) * a.s.lanes + lane;
    const bool there = v < a.s.vectors;
    const unsigned e = there ? first_of<N>(a.s, v) : 0;
    const i32x2 r = range_of(a, entry);
    float sum[N] = {};
    if (there) add_rows<T, B, false>(a, (long long)r[0] + group, r[1], groups, e, sum);
    const unsigned used = r[1] - r[0] < (int)groups ? r[1] > r[0] ? r[1] - r[0] : 0 : groups;
    unsigned half = 1;
    while (half < used) half *= 2;
    for (half /= 2; half; half /= 2) {
        __syncthreads();
        if (group >= half && group < 2 * half)
#pragma unroll
            for (int i = 0; i < N; ++i) sums[i][threadIdx.x] = sum[i];
        __syncthreads();
        if (group < half)
#pragma unroll
            for (int i = 0; i < N; ++i) sum[i] += sums[i][threadIdx.x + half * a.s.lanes];
    }
    if (group == 0 && there) store_floats<N>(a.dtable + entry * a.s.width, e, sum, a.scale);
}

// --------------------------------------------------------------------------

bool sizes_ok(size_t tokens, size_t entries) {
    return tokens && tokens <= kMaxCount && entries && entries <= TB_HIP_EMBED_MAX_ENTRIES;
}

bool rows_ok(const void *p, size_t stride, int dtype) {
    return p && multiple_of(p, type_size(dtype)) && stride % type_size(dtype) == 0;
}

// Ranking takes tokens^2 comparisons, a workgroup's sort its own chain, sorting by
// launches up to five of them.  Orders on the GPU: 1,024 tokens ranked 4.3 us,
// 2,000 7.5; 3,000 to 4,096 sorted by one workgroup 7 to 9.  With their gradient
// and the launches, one workgroup and by launches: 2,100 tokens to 1,000 entries
// 15.1 and 18.0 us, 4,096 tokens 19.3 and 19.5, 6,000 tokens 36 and 28; 4,096
// ranked take 2 us more than sorted.
constexpr size_t kRankMost = 2048, kRankEntries = 4096;

int log2_up(size_t n) {
    int bits = 0;
    while (size_t(1) << bits < n) ++bits;
    return bits;
}

struct SortShape {
    int low, high;  // bits of the digits, high 0 for a single one
    size_t segment;
    unsigned segments;
};

SortShape sort_shape(size_t tokens, size_t entries) {
    SortShape s;
    const int bits = log2_up(entries);
    s.low = bits <= 10 ? bits : (bits + 1) / 2;
    s.high = bits - s.low;
    s.segment = kSegment;
    const size_t least = (tokens + kMaxSegments - 1) / kMaxSegments;
    if (least > s.segment) s.segment = (least + kSortThreads - 1) / kSortThreads * kSortThreads;
    s.segments = (unsigned)((tokens + s.segment - 1) / s.segment);
    return s;
}

size_t whole16(size_t bytes) { return (bytes + 15) & ~size_t(15); }
size_t count_bytes(const SortShape &s) {
    return whole16(s.segments * ((size_t(1) << s.low) + 1) * sizeof(int));
}

void sort_pass(OrderArgs &a, int shift, int bits, hipStream_t q) {
    a.shift = shift;
    a.bits = bits;
    const size_t row = ((size_t(1) << bits) + 1) * sizeof(int);
    count_kernel<<<a.segments, kSortThreads, row, q>>>(a);
    place_kernel<<<a.segments, kSortThreads, row * (2 + kSortWaves), q>>>(a);
}

size_t chunks_of(size_t tokens) { return (tokens + kChunk - 1) / kChunk; }
size_t part_width(size_t width) { return (width + 3) / 4 * 4; }

template <class T, int B>
void launch_lookup(LookupArgs &a, hipStream_t q) {
    a.s = shape_of<T, B>(a.s.width);
    a.stream = a.tokens * a.s.width * sizeof(T) > kStreamBytes;
    const unsigned grid = grid_of(a.tokens * a.s.pieces, kThreads / a.s.lanes);
    if constexpr (B == 16)
        if (a.s.lanes == 64) {
            lookup_kernel<T, B, 64><<<grid, kThreads, 0, q>>>(a);
            return;
        }
    lookup_kernel<T, B, 0><<<grid, kThreads, 0, q>>>(a);
}

template <class T, int B>
void launch_grad(GradArgs &a, hipStream_t q) {
    a.s = shape_of<T, B>(a.s.width);
    const bool stream = B == 16 && a.tokens * a.s.width * sizeof(T) > kStreamBytes;
    const size_t per = kThreads / a.s.lanes;
    if (a.tokens <= kSmallTokens && a.entries * a.s.pieces <= kSmallItems) {
        const unsigned items = (unsigned)(a.entries * a.s.pieces);
        small_kernel<T, B><<<items, kSmallThreads, 0, q>>>(a);
        return;
    }
    // Chunks that no range is longer than need no joining.
    const bool join = a.tokens > kChunk;
    a.chunk_blocks = join ? grid_of(a.chunks * a.s.pieces, per) : 0;
    const unsigned grid = grid_of(a.entries * a.s.pieces, per) + (unsigned)a.chunk_blocks;
    constexpr int kWide = B == 16 ? 64 : 0;
    constexpr bool kStreams = B == 16;
    auto launch = [&](auto kernel) { kernel<<<grid, kThreads, 0, q>>>(a); };
    if (a.s.lanes == 64)
        stream ? launch(grad_kernel<T, B, kWide, kStreams>)
               : launch(grad_kernel<T, B, kWide, false>);
    else
        stream ? launch(grad_kernel<T, B, 0, kStreams>) : launch(grad_kernel<T, B, 0, false>);
    if (join) {
        const size_t slices = (a.s.width + kJoinColumns - 1) / kJoinColumns;
        const size_t blocks = (a.chunks + kJoinChunks - 1) / kJoinChunks;
        join_kernel<<<grid_of(blocks * slices, 1), kJoinThreads, 0, q>>>(a);
    }
}

// Calls f with a zero of the type and a vector's bytes: rows shorter than a
// vector go by single elements.
template <class F>
void with_type(int dtype, size_t width, F f) {
    const bool whole = width * type_size(dtype) >= 16;
    if (dtype == TB_HIP_F32)
        whole ? f(0.0f, Int<16>()) : f(0.0f, Int<4>());
    else if (dtype == TB_HIP_BF16)
        whole ? f((__bf16)0.0f, Int<16>()) : f((__bf16)0.0f, Int<2>());
    else
        whole ? f((_Float16)0.0f, Int<16>()) : f((_Float16)0.0f, Int<2>());
}

}  // namespace

extern "C" int tb_hip_embed_device(const int *ids, const void *table, size_t table_stride,
                                   const void *base, size_t base_stride, float scale, void *out,
                                   size_t tokens, size_t entries, size_t width, int dtype,
                                   void *stream) {
    if (!ids || !words_ok(ids) || !sizes_ok(tokens, entries) || !width || width > kMaxCount ||
        !known_type(dtype) || !rows_ok(table, table_stride, dtype) || !rows_ok(out, 0, dtype) ||
        (base && !rows_ok(base, base_stride, dtype)))
        return 0;
    LookupArgs a = {};
    a.ids = ids;
    a.table = static_cast<const char *>(table);
    a.table_stride = table_stride;
    a.base = static_cast<const char *>(base);
    a.base_stride = base_stride;
    a.scale = scale;
    a.out = static_cast<char *>(out);
    a.tokens = tokens;
    a.entries = entries;
    a.s.width = (unsigned)width;
    hipStream_t q = reinterpret_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    with_type(dtype, width, [&](auto zero, auto bytes) {
        launch_lookup<decltype(zero), decltype(bytes)::value>(a, q);
    });
    return hipGetLastError() == hipSuccess;
}

extern "C" size_t tb_hip_embed_order_workspace_bytes(size_t tokens, size_t entries) {
    if (!sizes_ok(tokens, entries)) return 0;
    const SortShape s = sort_shape(tokens, entries);
    return count_bytes(s) + whole16(tokens * sizeof(int));
}

extern "C" int tb_hip_embed_order_device(const int *ids, int *order, int *ranges, void *workspace,
                                         size_t tokens, size_t entries, void *stream) {
    if (!ids || !order || !words_ok(ids, order) || !ranges || !multiple_of(ranges, 8) ||
        !workspace || !multiple_of(workspace, 16) || !sizes_ok(tokens, entries))
        return 0;
    OrderArgs a = {};
    a.ids = ids;
    a.to = order;
    a.ranges = reinterpret_cast<i32x2 *>(ranges);
    a.tokens = tokens;
    a.entries = entries;
    hipStream_t q = reinterpret_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    auto clear = [&] {
        clear_kernel<<<grid_of(entries, kThreads), kThreads, 0, q>>>(a.ranges, entries);
    };
    const bool few_entries = entries <= kRankEntries;
    if (tokens <= kRankMost) {
        const unsigned blocks = (unsigned)((tokens + 63) / 64);
        a.bits = log2_up(entries + 1);
        if (few_entries) {
            const unsigned more = (unsigned)((entries + 63) / 64);
            rank_kernel<false><<<blocks + more, 64 * kRankWaves, 0, q>>>(a, blocks);
        } else {
            clear();
            rank_kernel<true><<<blocks, 64 * kRankWaves, 0, q>>>(a, blocks);
        }
        return hipGetLastError() == hipSuccess;
    }
    if (tokens <= kSmallMost) {
        const int bits = log2_up(entries + 1), passes = (bits + kSmallBits - 1) / kSmallBits;
        a.bits = (bits + passes - 1) / passes;
        if (!few_entries) clear();
        sort_kernel<<<1, kSmallSort, 0, q>>>(a, passes, few_entries);
        return hipGetLastError() == hipSuccess;
    }
    const SortShape s = sort_shape(tokens, entries);
    a.counts = static_cast<int *>(workspace);
    a.segment = s.segment;
    a.segments = s.segments;
    if (s.high) {
        int *half = reinterpret_cast<int *>(static_cast<char *>(workspace) + count_bytes(s));
        a.to = half;
        sort_pass(a, 0, s.low, q);
        a.from = half;
        a.to = order;
    }
    a.last = 1;
    sort_pass(a, s.high ? s.low : 0, s.high ? s.high : s.low, q);
    if (s.high) range_kernel<<<grid_of(tokens, kThreads), kThreads, 0, q>>>(a);
    return hipGetLastError() == hipSuccess;
}

extern "C" size_t tb_hip_embed_backward_workspace_bytes(size_t tokens, size_t entries,
                                                        size_t width) {
    if (!sizes_ok(tokens, entries) || !width || width > kMaxCount) return 0;
    return chunks_of(tokens) * 2 * part_width(width) * sizeof(float);
}

extern "C" int tb_hip_embed_backward_device(const void *dout, size_t dout_stride, const int *ids,
                                            const int *order, const int *ranges, float scale,
                                            float *dtable, void *workspace, size_t tokens,
                                            size_t entries, size_t width, int dtype,
                                            void *stream) {
    if (!ids || !order || !ranges || !multiple_of(ranges, 8) || !dtable ||
        !words_ok(ids, order, dtable) || !workspace || !multiple_of(workspace, 16) ||
        !sizes_ok(tokens, entries) || !width || width > kMaxCount || !known_type(dtype) ||
        !rows_ok(dout, dout_stride, dtype))
        return 0;
    GradArgs a = {};
    a.dout = static_cast<const char *>(dout);
    a.stride = dout_stride;
    a.ids = ids;
    a.order = order;
    a.ranges = reinterpret_cast<const i32x2 *>(ranges);
    a.scale = scale;
    a.dtable = dtable;
    a.parts = static_cast<float *>(workspace);
    a.tokens = tokens;
    a.entries = entries;
    a.part_width = part_width(width);
    a.chunks = chunks_of(tokens);
    a.s.width = (unsigned)width;
    hipStream_t q = reinterpret_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    with_type(dtype, width, [&](auto zero, auto bytes) {
        launch_grad<decltype(zero), decltype(bytes)::value>(a, q);
    });
    return hipGetLastError() == hipSuccess;
}
