// Rows in 8-bit integers with a scale each (hip_layers.h): quantisation, the
// values they stand for, and their products, dense or per expert.
//
//   scale  s = max(max |x| / 127, 2^-126), NaN for a row with an Inf or NaN
//   code   x (1 / s), to the nearest integer, ties to even; each of the two
//          steps before is rounded to 32 bits
//   out    = act((sum_k a_k w_k s_a) s_w + bias) row_scale, the sum in 32-bit
//            integers and exact, by v_mfma_i32_16x16x64_i8: lane l holds row
//            l % 16, values 16 (l / 16) .. + 15 of a step of 64
#include "product_tiles.h"
#include "xcd_order.h"

namespace {

using namespace layer;

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr size_t kMaxCount = 0x7fffffffu, kMaxOutputs = size_t(1) << 38;
constexpr size_t kMaxGrid = 1 << 20;
constexpr int kStep = 64, kPad = 128;

__host__ __device__ inline size_t padded(size_t k) { return (k + kPad - 1) / kPad * kPad; }

// --------------------------------------------------------------------------
// Quantisation: a row belongs to one wave or to a workgroup, eight values of a
// lane at a time, kept in registers between the maximum and the codes where
// they fit.

constexpr int kQuantThreads = 256;

struct QuantArgs {
    const char *x;
    size_t stride, rows, kp;
    unsigned char *codes;
    float *scales;
    unsigned k, pieces;  // pieces: kp / 8
};

// Values 8 p .. 8 p + 7 of a row, 0 past its end.
template <class T>
__device__ __forceinline__ void load8(const QuantArgs &a, const char *row, unsigned p,
                                      float (&v)[8]) {
    const unsigned k0 = p * 8;
    if (k0 + 8 <= a.k) {
        typedef Vec<T, 16> X;
#pragma unroll
        for (int i = 0; i < 8 / X::n; ++i) {
            float part[X::n];
            X::unpack(load_loose<T, 16>(row, k0 + i * X::n), part);
#pragma unroll
            for (int j = 0; j < X::n; ++j) v[i * X::n + j] = part[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = k0 + j < a.k ? (float)reinterpret_cast<const T *>(row)[k0 + j] : 0.0f;
    }
}

// Magnitudes order as integers; Inf and NaN lie above all others.
__device__ __forceinline__ unsigned larger(unsigned most, const float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const unsigned m = __builtin_bit_cast(unsigned, v[j]) & 0x7fffffffu;
        most = m > most ? m : most;
    }
    return most;
}

__device__ __forceinline__ u32x2 codes_of(const float (&v)[8], float inverse, bool finite) {
    u32x2 out = {0, 0};
    if (finite)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            out[j / 4] |= ((unsigned)(int)__builtin_rintf(v[j] * inverse) & 255u) << (8 * (j % 4));
    return out;
}

constexpr int kHeld = 4;  // pieces that a lane keeps

// THREADS: a row's, 64 or the workgroup's.
template <class T, int THREADS>
__global__ __launch_bounds__(kQuantThreads) void quantise_kernel(QuantArgs a) {
    __shared__ unsigned wave_most[kQuantThreads / 64];
    constexpr int kRows = kQuantThreads / THREADS;
    const unsigned t = threadIdx.x % THREADS;
    unsigned in = threadIdx.x / THREADS;
    in = __builtin_amdgcn_readfirstlane(in);
    for (size_t r = (size_t)blockIdx.x * kRows + in; r < a.rows; r += (size_t)gridDim.x * kRows) {
        const char *row = a.x + r * a.stride;
        float v[kHeld][8];
        unsigned most = 0;
#pragma unroll
        for (int h = 0; h < kHeld; ++h) {
            const unsigned p = t + h * THREADS;
            if (p < a.pieces) load8<T>(a, row, p, v[h]);
        }
#pragma unroll
        for (int h = 0; h < kHeld; ++h)
            if (t + h * THREADS < a.pieces) most = larger(most, v[h]);
        for (unsigned p = t + kHeld * THREADS; p < a.pieces; p += THREADS) {
            float w[8];
            load8<T>(a, row, p, w);
            most = larger(most, w);
        }
        for (int off = 1; off < 64; off *= 2) {
            const unsigned o = __shfl_xor(most, off);
            most = o > most ? o : most;
        }
        if (THREADS > 64) {
            __syncthreads();
            if ((threadIdx.x & 63) == 0) wave_most[threadIdx.x >> 6] = most;
            __syncthreads();
            for (int w = 0; w < kQuantThreads / 64; ++w)
                most = wave_most[w] > most ? wave_most[w] : most;
        }
        const bool finite = most < 0x7f800000u;
        const float top = __builtin_bit_cast(float, most) / 127.0f, least = 0x1p-126f;
        const float scale = finite ? (top > least ? top : least) : __builtin_nanf("");
        const float inverse = 1.0f / scale;
        u32x2 *codes = reinterpret_cast<u32x2 *>(a.codes + r * a.kp);
#pragma unroll
        for (int h = 0; h < kHeld; ++h) {
            const unsigned p = t + h * THREADS;
            if (p < a.pieces) codes[p] = codes_of(v[h], inverse, finite);
        }
        for (unsigned p = t + kHeld * THREADS; p < a.pieces; p += THREADS) {
            float w[8];
            load8<T>(a, row, p, w);
            codes[p] = codes_of(w, inverse, finite);
        }
        if (t == 0) a.scales[r] = scale;
    }
}

struct ValueArgs {
    const unsigned char *codes;
    const float *scales;
    char *out;
    size_t items, kp;
    unsigned per, k;  // per: pieces of eight values that hold a row's k
};

template <class T>
__global__ __launch_bounds__(kQuantThreads) void values_kernel(ValueArgs a) {
    typedef Vec<T, 16> X;
    for (size_t i = (size_t)blockIdx.x * kQuantThreads + threadIdx.x; i < a.items;
         i += (size_t)gridDim.x * kQuantThreads) {
        const size_t row = i / a.per;
        const unsigned k0 = (unsigned)(i - row * a.per) * 8;
        const float scale = a.scales[row];
        const u32x2 codes = *reinterpret_cast<const u32x2 *>(a.codes + row * a.kp + k0);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = (float)(signed char)(codes[j / 4] >> (8 * (j % 4)) & 255u) * scale;
        char *out = a.out + row * a.k * sizeof(T);
        if (k0 + 8 <= a.k) {
#pragma unroll
            for (int p = 0; p < 8 / X::n; ++p) {
                float part[X::n];
#pragma unroll
                for (int j = 0; j < X::n; ++j) part[j] = v[p * X::n + j];
                store_loose<T, 16>(out, k0 + p * X::n, X::pack(part));
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (k0 + j < a.k) reinterpret_cast<T *>(out)[k0 + j] = (T)v[j];
        }
    }
}

// --------------------------------------------------------------------------
// Products

struct ProductArgs {
    const unsigned char *a_codes, *w_codes;
    const float *a_scales, *w_scales, *bias, *row_scale;
    const int *rows, *offsets;
    char *out;
    size_t a_rows, m, n, kp;
    int experts, vector;
};

__device__ __forceinline__ i32x4 step_of(i32x4 w, i32x4 x, i32x4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x, c, 0, 0, 0);
}

// Few rows: tiles of 16 columns and 16 MT rows, operands straight from memory
// in the instruction's layout, k split over the workgroup's waves in pairs of
// steps (128 bytes of a row) and joined in LDS.  The weights are the first
// operand, so a lane ends with four consecutive columns of one row.
constexpr int kFewWaves = 8;

template <class T, int ACT, int MT>
__global__ __launch_bounds__(64 * kFewWaves) void few_kernel(ProductArgs a) {
    __shared__ i32x4 sums[kFewWaves][MT][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int low = lane & 15, part = lane >> 4;
    const unsigned block = blockIdx.y * gridDim.x + blockIdx.x;
    const unsigned columns = (unsigned)((a.n + 15) / 16), tile = block / columns;
    RowTile rt;
    if (!find_rows(a, tile, 16 * MT, rt)) return;
    const size_t n0 = (size_t)(block - tile * columns) * 16;
    const bool some = rt.expert < a.experts;
    const size_t w_first = some ? rt.expert * a.n : 0;
    const size_t wr = w_first + (n0 + low < a.n ? n0 + low : a.n - 1);
    const unsigned char *wc = a.w_codes + wr * a.kp + part * 16;
    const unsigned char *xc[MT];
    float scale[MT];
    unsigned real = 0;  // a bit for each row tile
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        size_t m = rt.r0 + j * 16 + low;
        m = m < rt.r1 ? m : rt.r1 - 1;
        const long long row = a.rows ? a.rows[m] : (long long)m;
        const bool there = row >= 0 && (size_t)row < a.a_rows;
        real |= (some && there ? 1u : 0u) << j;
        xc[j] = a.a_codes + (there ? row : 0) * a.kp + part * 16;
        scale[j] = a.a_scales[there ? row : 0];
    }
    i32x4 acc[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[j] = (i32x4){0, 0, 0, 0};
    const size_t pairs = some ? a.kp / kPad : 0;
    for (size_t s = wave; s < pairs; s += kFewWaves) {
        const i32x4 w0 = *reinterpret_cast<const i32x4 *>(wc + s * kPad);
        const i32x4 w1 = *reinterpret_cast<const i32x4 *>(wc + s * kPad + kStep);
        i32x4 x0[MT], x1[MT];
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            x0[j] = *reinterpret_cast<const i32x4 *>(xc[j] + s * kPad);
            x1[j] = *reinterpret_cast<const i32x4 *>(xc[j] + s * kPad + kStep);
        }
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[j] = step_of(w0, x0[j], acc[j]);
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[j] = step_of(w1, x1[j], acc[j]);
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) sums[wave][j][lane] = acc[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        if (wave != j % kFewWaves) continue;
        i32x4 sum = sums[0][j][lane];
        for (int w = 1; w < kFewWaves; ++w) sum += sums[w][j][lane];
        const size_t r = rt.r0 + j * 16 + low, c = n0 + part * 4;
        if (r >= rt.r1 || c >= a.n) continue;
        const bool there = real >> j & 1;
        const float row_scale = a.row_scale && there ? a.row_scale[r] : 1.0f;
        T *out = reinterpret_cast<T *>(a.out) + r * a.n + c;
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = 0.0f;
            if (there && c + i < a.n) {
                const size_t at = w_first + c + i;
                const float z = fmaf((float)sum[i] * scale[j], a.w_scales[at],
                                     a.bias ? a.bias[at] : 0.0f);
                v[i] = act_of<kFine<T>, ACT>(z) * row_scale;
            }
        }
        if (c + 4 <= a.n) {
            typedef Vec<T, 4 * sizeof(T)> X;
            store_loose<T, 4 * sizeof(T)>(reinterpret_cast<char *>(out), 0, X::pack(v));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c + i < a.n) out[i] = (T)v[i];
        }
    }
}

// Large products: tiles of BM rows and BN columns, staged through LDS in
// slices of two steps (128 values, 128 bytes a row), two slices in turn.
//
// Codes come by loads that write LDS themselves: a wave's load fills 1 KB,
// eight rows, in lane order.  16-byte piece c of row r lies at slot c ^ (r & 7)
// of its row, so that the rows of an operand read, 128 bytes apart, fall on
// all banks.
//
// Turn s: read step 1 of slice s while multiplying step 0; wait for the loads
// of slice s + 1; barrier: all waves have them, and have read slice s; load
// slice s + 2 over it, and read step 0 of slice s + 1 while multiplying step 1.
template <int MT, int NT>
struct Operands {
    i32x4 x[MT], w[NT];
};

template <int MT, int NT>
__device__ __forceinline__ void multiply(const Operands<MT, NT> &o, i32x4 (&acc)[NT][MT]) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = step_of(o.w[i], o.x[j], acc[i][j]);
}

template <class T, int ACT, int WM, int WN, int MT, int NT>
__global__ __launch_bounds__(64 * WM * WN) void tile_kernel(ProductArgs a) {
    constexpr int BM = 16 * MT * WM, BN = 16 * NT * WN, kWaves = WM * WN, kThreads = 64 * kWaves;
    constexpr int kRows = BM + BN, kLoads = kRows / 8 / kWaves;  // 1 KB a load of a wave
    constexpr int kReads = MT + NT;  // of a step
    static_assert(kRows == kThreads && BM % (kLoads * 8) == 0);
    constexpr int kGroup = 8;  // column tiles that neighbours in time share
    // Two arrays, chosen at compile time: the compiler knows that a read of one
    // need not wait for the loads into the other.
    __shared__ __attribute__((aligned(1024))) unsigned char codes0[kRows * kPad];
    __shared__ __attribute__((aligned(1024))) unsigned char codes1[kRows * kPad];
    // Each row's codes, in pieces of 16 bytes, by the loading wave, lane / 8
    // and load.
    __shared__ __attribute__((aligned(16))) unsigned row_code[kRows];
    __shared__ float scale_of_row[BM], weight_of_row[BM];
    __shared__ __attribute__((aligned(16))) float scale_of[BN], bias_of[BN];
    __shared__ unsigned char real_row[BM];

    const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
    const int low = lane & 15, part = lane >> 4;
    const int wm = wave % WM, wn = wave / WM;
    const unsigned columns = (unsigned)((a.n + BN - 1) / BN), heights = gridDim.x / columns;
    const unsigned at = (unsigned)xcd_contiguous(blockIdx.x, gridDim.x);
    const unsigned band = at / (kGroup * heights), rest = at - band * kGroup * heights;
    const unsigned wide = columns - band * kGroup < kGroup ? columns - band * kGroup : kGroup;
    RowTile rt;
    if (!find_rows(a, rest / wide, BM, rt)) return;
    const size_t n0 = (size_t)(band * kGroup + rest % wide) * BN, m0 = rt.r0;
    const int height = (int)(rt.r1 - rt.r0);
    const size_t w_first = rt.expert < a.experts ? (size_t)rt.expert * a.n : 0;

    if (rt.expert >= a.experts) {
        constexpr int kRun = 16 / sizeof(T), kAcross = BN / kRun;
        const size_t c = n0 + t % kAcross * kRun;
        for (int r = t / kAcross; r < height; r += kThreads / kAcross)
            if (c < a.n) store_run<T>(a, m0 + r, c, (u32x4){0, 0, 0, 0});
        return;
    }
    // The matrix row behind each row of the tile, the output's rows first,
    // counted from the tile's first (from the matrix's where they are
    // gathered; row 0 is read for one that is not there); rows past the tile's
    // end stand in for the last one and are not stored.
    int row;
    if (t >= BM) {
        row = n0 + (t - BM) < a.n ? t - BM : (int)(a.n - 1 - n0);
        scale_of[t - BM] = a.w_scales[w_first + n0 + row];
        bias_of[t - BM] = a.bias ? a.bias[w_first + n0 + row] : 0.0f;
    } else {
        const int in = t < height ? t : height - 1;
        row = a.rows ? a.rows[m0 + in] : in;
        const bool real = !a.rows || (row >= 0 && (size_t)row < a.a_rows);
        row = real ? row : 0;
        real_row[t] = real;
        scale_of_row[t] = a.a_scales[(a.rows ? 0 : m0) + row];
        weight_of_row[t] = a.row_scale ? a.row_scale[m0 + in] : 1.0f;
    }
    const unsigned pieces = (unsigned)(a.kp / 16);
    row_code[(t / (8 * kLoads) * 8 + t % 8) * kLoads + t / 8 % kLoads] = (unsigned)row * pieces;
    __syncthreads();

    i32x4 acc[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = (i32x4){0, 0, 0, 0};

    const int row0 = wave * kLoads * 8;
    const bool w_side = row0 >= BM;
    const size_t first = w_side ? w_first + n0 : a.rows ? 0 : m0;
    const unsigned char *base = (w_side ? a.w_codes : a.a_codes) + first * a.kp;
    unsigned from[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
        from[i] = row_code[(t >> 3) * kLoads + i] + ((lane & 7) ^ (lane >> 3));
    const unsigned slices = (unsigned)(a.kp / kPad);
    auto load = [&](unsigned slice, unsigned char *codes) {
        // Slices behind the last are the last again, and not multiplied.
        const unsigned s = slice < slices ? slice : slices - 1;
        const unsigned char *here = base + (size_t)s * kPad;
        unsigned char *to = codes + row0 * kPad;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) load_to_lds(here + (size_t)from[i] * 16, to + i * 1024);
    };
    const int row_x = wm * MT * 16, row_w = BM + wn * NT * 16;
    const int lane_row = low * kPad, slot = (part ^ (low & 7)) * 16;
    auto read = [&](const unsigned char *codes, int s, Operands<MT, NT> &o) {
        const unsigned char *p = codes + lane_row + (slot ^ (s * kStep));
#pragma unroll
        for (int j = 0; j < MT; ++j)
            o.x[j] = *reinterpret_cast<const i32x4 *>(p + (row_x + j * 16) * kPad);
#pragma unroll
        for (int i = 0; i < NT; ++i)
            o.w[i] = *reinterpret_cast<const i32x4 *>(p + (row_w + i * 16) * kPad);
    };
    Operands<MT, NT> even, odd;
    auto turn = [&](unsigned slice, unsigned char *codes, unsigned char *codes_next) {
        read(codes, 1, odd);
        multiply<MT, NT>(even, acc);
#pragma unroll
        for (int i = 0; i < kReads; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
        }
        arrive();
        load(slice + 2, codes);
        read(codes_next, 0, even);
        multiply<MT, NT>(odd, acc);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        }
#pragma unroll
        for (int i = 0; i < kReads; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    load(0, codes0);
    arrive();
    read(codes0, 0, even);
    load(1, codes1);
    for (unsigned slice = 0; slice < slices; slice += 2) {
        turn(slice, codes0, codes1);
        if (slice + 1 < slices) turn(slice + 1, codes1, codes0);
    }
    arrive();

    // Results through LDS, whose rows leave in runs: kPass rows of the tile at a
    // time, the arrays in turn, so that a pass is read before the next but one
    // is written.  A lane's four columns are one piece; piece c of a wave's row
    // r lies at c ^ 4 r, so that the rows of a write fall on different banks.
    typedef Vec<T, 4 * sizeof(T)> Four;
    constexpr int kPassTiles = pass_tiles(MT, WM * 16 * BN * sizeof(T), sizeof(codes0));
    constexpr int kPass = kPassTiles * WM * 16, kPieces = BN / 4;
    constexpr int kRun = 16 / sizeof(T), kAcross = BN / kRun, kSweep = kThreads / kAcross;
    const int c = t % kAcross * kRun;
    const size_t n1 = n0 + c;
    f32x4 bias[NT], scale[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        bias[i] = *reinterpret_cast<const f32x4 *>(bias_of + (wn * NT + i) * 16 + part * 4);
        scale[i] = *reinterpret_cast<const f32x4 *>(scale_of + (wn * NT + i) * 16 + part * 4);
    }
#pragma unroll
    for (int j0 = 0; j0 < MT; j0 += kPassTiles) {
        unsigned char *results = j0 / kPassTiles % 2 ? codes1 : codes0;
#pragma unroll
        for (int j = 0; j < kPassTiles; ++j) {
            const int in = (wm * MT + j0 + j) * 16 + low, at = (wm * kPassTiles + j) * 16 + low;
            const float row_scale = scale_of_row[in], weight = weight_of_row[in];
            const bool real = real_row[in];
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                float v[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float z = fmaf((float)acc[i][j0 + j][q] * row_scale, scale[i][q],
                                         bias[i][q]);
                    v[q] = act_of<kFine<T>, ACT>(z) * weight;
                    v[q] = real ? v[q] : 0.0f;
                }
                const int piece = ((wn * NT + i) * 4 + part) ^ (low * 4 & (kPieces - 1));
                reinterpret_cast<typename Four::raw *>(results)[at * kPieces + piece] =
                    Four::pack(v);
            }
        }
        __syncthreads();
        if (n1 >= a.n) continue;
#pragma unroll 4
        for (int row = t / kAcross; row < kPass; row += kSweep) {
            const int in = row / (kPassTiles * 16) * (MT * 16) + j0 * 16 + row % (kPassTiles * 16);
            const int piece = c / 4 ^ (row % 16 * 4 & (kPieces - 1));
            const u32x4 run = *reinterpret_cast<const u32x4 *>(
                results + (row * kPieces + piece) * sizeof(typename Four::raw));
            if (in < height) store_run<T>(a, m0 + in, n1, run);
        }
    }
}

// Rows and columns of a workgroup's tile, by shape.
struct TileSize {
    int rows, columns;
};
constexpr TileSize kTiles[] = {{16, 16}, {32, 16}, {64, 16}, {128, 128}, {256, 256}};
enum { kFew1, kFew2, kFew4, kMiddle, kLarge };

size_t tiles_of(const ProductArgs &a, int shape) {
    const TileSize t = kTiles[shape];
    // Every run of rows may end within a tile.
    const size_t high = (a.m + t.rows - 1) / t.rows + (a.offsets ? a.experts + 2 : 0);
    return high * ((a.n + t.columns - 1) / t.columns);
}

// A dimension of a grid holds less than 2^32 threads, 512 to a tile.  More than
// 2^22 tiles of few rows take rows of 2^22 workgroups, the last of which find
// no tile; staged tiles leave narrow products of 2^23 tiles and more to them.
constexpr unsigned kGridRow = 1 << 22;
static_assert(64 * kFewWaves * (size_t)kGridRow < size_t(1) << 32);

int shape_for(const ProductArgs &a) {
    // The staged kernels count a matrix in 32 bits of 16 bytes, from a tile's
    // first row (from the first of all where rows are gathered).
    const size_t reach = 0xffffffffu / (a.kp / 16);
    const bool staged = (!a.rows || a.a_rows <= reach) && tiles_of(a, kMiddle) < 2 * kGridRow;
    const size_t per = a.m / a.experts;
    if (staged && per > 32 && a.m * a.n > (1 << 18)) {
        // Half of the runs of rows end within a tile of their own, about.
        const size_t slices = a.kp / kPad, ends = a.experts / 2;
        const size_t large = ((a.m + 255) / 256 + ends) * ((a.n + 255) / 256);
        const size_t middle = ((a.m + 127) / 128 + ends) * ((a.n + 127) / 128);
        return (large + 255) / 256 * (82 + 24 * slices) <= (middle + 511) / 512 * (39 + 18 * slices)
                   ? kLarge
                   : kMiddle;
    }
    if (per > 32 && tiles_of(a, kFew4) >= 256) return kFew4;
    if (per > 16 && tiles_of(a, kFew2) >= 256) return kFew2;
    return kFew1;
}

template <class T>
void launch_product(const ProductArgs &a, int act, int shape, unsigned tiles, hipStream_t q) {
    const dim3 few = tiles < kGridRow ? dim3(tiles)
                                      : dim3(kGridRow, (tiles + kGridRow - 1) / kGridRow);
    with_act(act, [&](auto which) {
        constexpr int ACT = decltype(which)::value;
        switch (shape) {
            case kFew1: few_kernel<T, ACT, 1><<<few, 64 * kFewWaves, 0, q>>>(a); break;
            case kFew2: few_kernel<T, ACT, 2><<<few, 64 * kFewWaves, 0, q>>>(a); break;
            case kFew4: few_kernel<T, ACT, 4><<<few, 64 * kFewWaves, 0, q>>>(a); break;
            case kMiddle: tile_kernel<T, ACT, 2, 2, 4, 4><<<tiles, 256, 0, q>>>(a); break;
            default: tile_kernel<T, ACT, 2, 4, 8, 4><<<tiles, 512, 0, q>>>(a); break;
        }
    });
}

unsigned grid_of(size_t items, size_t per) {
    const size_t want = (items + per - 1) / per;
    return (unsigned)(want < kMaxGrid ? want : kMaxGrid);
}

template <class T>
void launch_quantise(const QuantArgs &a, hipStream_t q) {
    if (a.pieces <= 64 * kHeld)
        quantise_kernel<T, 64><<<grid_of(a.rows, kQuantThreads / 64), kQuantThreads, 0, q>>>(a);
    else
        quantise_kernel<T, kQuantThreads><<<grid_of(a.rows, 1), kQuantThreads, 0, q>>>(a);
}

bool rows_ok(size_t rows, size_t k, int dtype) {
    return rows && rows <= kMaxCount && k && k <= TB_HIP_INT8_MAX_K && known_type(dtype);
}

}  // namespace

extern "C" size_t tb_hip_int8_padded(size_t k) { return padded(k); }

extern "C" int tb_hip_int8_quantise_device(const void *x, size_t row_stride, void *codes,
                                           float *scales, size_t rows, size_t k, int dtype,
                                           void *stream) {
    if (!x || !codes || !scales || !rows_ok(rows, k, dtype) || !multiple_of(codes, 16) ||
        !multiple_of(scales, 4) || !multiple_of(x, type_size(dtype)) ||
        row_stride % type_size(dtype))
        return 0;
    QuantArgs a = {};
    a.x = static_cast<const char *>(x);
    a.stride = row_stride;
    a.rows = rows;
    a.kp = padded(k);
    a.codes = static_cast<unsigned char *>(codes);
    a.scales = scales;
    a.k = (unsigned)k;
    a.pieces = (unsigned)(a.kp / 8);
    hipStream_t q = reinterpret_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    if (dtype == TB_HIP_F32)
        launch_quantise<float>(a, q);
    else if (dtype == TB_HIP_BF16)
        launch_quantise<__bf16>(a, q);
    else
        launch_quantise<_Float16>(a, q);
    return hipGetLastError() == hipSuccess;
}

extern "C" int tb_hip_int8_values_device(const void *codes, const float *scales, void *values,
                                         size_t rows, size_t k, int dtype, void *stream) {
    if (!codes || !scales || !values || !rows_ok(rows, k, dtype) || !multiple_of(codes, 16) ||
        !multiple_of(scales, 4) || !multiple_of(values, type_size(dtype)))
        return 0;
    ValueArgs a = {};
    a.codes = static_cast<const unsigned char *>(codes);
    a.scales = scales;
    a.out = static_cast<char *>(values);
    a.kp = padded(k);
    a.k = (unsigned)k;
    a.per = (unsigned)((k + 7) / 8);
    a.items = rows * a.per;
    hipStream_t q = reinterpret_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    const unsigned grid = grid_of(a.items, kQuantThreads);
    if (dtype == TB_HIP_F32)
        values_kernel<float><<<grid, kQuantThreads, 0, q>>>(a);
    else if (dtype == TB_HIP_BF16)
        values_kernel<__bf16><<<grid, kQuantThreads, 0, q>>>(a);
    else
        values_kernel<_Float16><<<grid, kQuantThreads, 0, q>>>(a);
    return hipGetLastError() == hipSuccess;
}

extern "C" int tb_hip_int8_product_device(const void *a_codes, const float *a_scales,
                                          size_t a_rows, const int *rows, const void *w_codes,
                                          const float *w_scales, const int *offsets,
                                          const float *bias, const float *row_scale, void *out,
                                          size_t m, size_t n, size_t k, int experts, int act,
                                          int dtype, void *stream) {
    if (!a_codes || !a_scales || !w_codes || !w_scales || !out || !rows_ok(a_rows, k, dtype) ||
        !m || m > kMaxCount || !n || n > kMaxCount || experts < 1 ||
        experts > TB_HIP_ROUTE_MAX_EXPERTS || (experts > 1 && !offsets) ||
        n > kMaxCount / experts || m > kMaxOutputs / n || (!rows && m != a_rows) ||
        !known_act(act) || !multiple_of(a_codes, 16) || !multiple_of(w_codes, 16) ||
        !multiple_of(a_scales, 4) || !multiple_of(w_scales, 4) ||
        !multiple_of(out, type_size(dtype)))
        return 0;
    ProductArgs a = {};
    a.a_codes = static_cast<const unsigned char *>(a_codes);
    a.a_scales = a_scales;
    a.w_codes = static_cast<const unsigned char *>(w_codes);
    a.w_scales = w_scales;
    a.rows = rows;
    a.offsets = offsets;
    a.bias = bias;
    a.row_scale = row_scale;
    a.out = static_cast<char *>(out);
    a.a_rows = a_rows;
    a.m = m;
    a.n = n;
    a.kp = padded(k);
    a.experts = experts;
    a.vector = multiple_of(out, 16) && n * type_size(dtype) % 16 == 0;
    hipStream_t q = reinterpret_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    const int shape = shape_for(a);
    // Below 2^31: 2^30 for 2^38 values in tiles of 16 x 16, and the runs' ends.
    const size_t tiles = tiles_of(a, shape);
    if (dtype == TB_HIP_F32)
        launch_product<float>(a, act, shape, (unsigned)tiles, q);
    else if (dtype == TB_HIP_BF16)
        launch_product<__bf16>(a, act, shape, (unsigned)tiles, q);
    else
        launch_product<_Float16>(a, act, shape, (unsigned)tiles, q);
    return hipGetLastError() == hipSuccess;
}
