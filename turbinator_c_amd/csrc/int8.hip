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
// they fit.  Bound by memory: 40,959 x 1,999 bf16 54 us, the values back 37 us (4.6
// and 6.7 TB/s of what they read and write, the codes in between in the last
// cache); 16,384 x 4,096 bf16 41 us, 4.9 TB/s.

constexpr int kQuantThreads = 256;

struct QuantArgs {
    const char *x;
    size_t stride, rows, kp;
    unsigned char *codes;
    float *scales;
    unsigned k, pieces;  // pieces: kp / 8
};

// Eight values as they are stored.
template <class T>
struct Eight {
    typedef Vec<T, 16> X;
    static constexpr int kParts = 8 / X::n;
    u32x4 part[kParts];

    // Values 8 p .. 8 p + 7 of a row, 0 past its end.
    template <bool STREAM>
    __device__ __forceinline__ void load(const QuantArgs &a, const char *row, unsigned p) {
        const unsigned k0 = p * 8;
        if (k0 + 8 <= a.k) {
#pragma unroll
            for (int i = 0; i < kParts; ++i)
                part[i] = STREAM ? stream_in<T, 16>(row, k0 + i * X::n)
                                 : load_loose<T, 16>(row, k0 + i * X::n);
            return;
        }
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
            typename X::elems v;
#pragma unroll
            for (int j = 0; j < X::n; ++j) {
                const unsigned k = k0 + i * X::n + j;
                v[j] = k < a.k ? reinterpret_cast<const T *>(row)[k] : (T)0.0f;
            }
            part[i] = __builtin_bit_cast(u32x4, v);
        }
    }
    // Magnitudes order as integers, Inf and NaN above all others: the largest
    // of `most` and these, of 16-bit types in both halves.
    __device__ __forceinline__ unsigned most(unsigned most) const {
        typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < kParts; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (sizeof(T) == 4) {
                    const unsigned m = part[i][j] & 0x7fffffffu;
                    most = m > most ? m : most;
                } else {
                    most = __builtin_bit_cast(
                        unsigned,
                        __builtin_elementwise_max(
                            __builtin_bit_cast(u16x2, most),
                            __builtin_bit_cast(u16x2, part[i][j] & 0x7fff7fffu)));
                }
            }
        return most;
    }
    // The codes: adding 1.5 2^23 rounds to an integer, ties to even, and leaves
    // it in the low bits.
    __device__ __forceinline__ u32x2 codes(float inverse) const {
        unsigned q[8];
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
            float v[X::n];
            X::unpack(part[i], v);
#pragma unroll
            for (int j = 0; j < X::n; ++j)
                q[i * X::n + j] = __builtin_bit_cast(unsigned, v[j] * inverse + 12582912.0f);
        }
        u32x2 out;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const unsigned low = __builtin_amdgcn_perm(q[4 * i + 1], q[4 * i], 0x0c0c0400);
            const unsigned high = __builtin_amdgcn_perm(q[4 * i + 3], q[4 * i + 2], 0x0c0c0400);
            out[i] = __builtin_amdgcn_perm(high, low, 0x05040100);
        }
        return out;
    }
};

// The largest of the wave's, as 32-bit floating point's bits.
template <class T>
__device__ __forceinline__ unsigned wave_most(unsigned v) {
    if (sizeof(T) == 2) v = (v & 0xffffu) > v >> 16 ? v & 0xffffu : v >> 16;
    auto step = [&](unsigned o) { v = o > v ? o : v; };
    step(__builtin_amdgcn_update_dpp(0, v, 0x111, 15, 15, false));
    step(__builtin_amdgcn_update_dpp(0, v, 0x112, 15, 15, false));
    step(__builtin_amdgcn_update_dpp(0, v, 0x114, 15, 15, false));
    step(__builtin_amdgcn_update_dpp(0, v, 0x118, 15, 15, false));
    step(__builtin_amdgcn_update_dpp(0, v, 0x142, 10, 15, false));
    step(__builtin_amdgcn_update_dpp(0, v, 0x143, 12, 15, false));
    v = (unsigned)__builtin_amdgcn_readlane((int)v, 63);
    if constexpr (sizeof(T) == 4)
        return v;
    else
        return __builtin_bit_cast(unsigned, (float)__builtin_bit_cast(T, (unsigned short)v));
}

constexpr int kHeld = 4;  // pieces that a lane keeps

// THREADS: a row's, 64 or the workgroup's.  STREAM: the first loads go past the
// caches.
template <class T, int THREADS, bool STREAM>
__global__ __launch_bounds__(kQuantThreads) void quantise_kernel(QuantArgs a) {
    __shared__ unsigned mosts[kQuantThreads / 64];
    constexpr int kRows = kQuantThreads / THREADS;
    const unsigned t = threadIdx.x % THREADS;
    const unsigned in = __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS);
    for (size_t r = (size_t)blockIdx.x * kRows + in; r < a.rows; r += (size_t)gridDim.x * kRows) {
        const char *row = a.x + r * a.stride;
        Eight<T> held[kHeld], other;
        unsigned most = 0;
#pragma unroll
        for (int h = 0; h < kHeld; ++h)
            if (t + h * THREADS < a.pieces) held[h].template load<STREAM>(a, row, t + h * THREADS);
#pragma unroll
        for (int h = 0; h < kHeld; ++h)
            if (t + h * THREADS < a.pieces) most = held[h].most(most);
        for (unsigned p = t + kHeld * THREADS; p < a.pieces; p += THREADS) {
            other.template load<false>(a, row, p);
            most = other.most(most);
        }
        most = wave_most<T>(most);
        if (THREADS > 64) {
            __syncthreads();
            if ((threadIdx.x & 63) == 0) mosts[threadIdx.x >> 6] = most;
            __syncthreads();
            for (int w = 0; w < kQuantThreads / 64; ++w) most = mosts[w] > most ? mosts[w] : most;
        }
        const bool finite = most < 0x7f800000u;
        const float top = __builtin_bit_cast(float, most) / 127.0f, least = 0x1p-126f;
        const float scale = finite ? (top > least ? top : least) : __builtin_nanf("");
        const float inverse = 1.0f / scale;
        u32x2 *codes = reinterpret_cast<u32x2 *>(a.codes + r * a.kp);
        auto write = [&](unsigned p, const Eight<T> &v) {
            codes[p] = finite ? v.codes(inverse) : (u32x2){0, 0};
        };
#pragma unroll
        for (int h = 0; h < kHeld; ++h)
            if (t + h * THREADS < a.pieces) write(t + h * THREADS, held[h]);
        for (unsigned p = t + kHeld * THREADS; p < a.pieces; p += THREADS) {
            other.template load<false>(a, row, p);
            write(p, other);
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
    int experts;
    bool direct;  // results leave from registers
};

__device__ __forceinline__ i32x4 step_of(i32x4 w, i32x4 x, i32x4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x, c, 0, 0, 0);
}

// Few rows: tiles of 16 columns and 16 rows, operands straight from memory in
// the instruction's layout, k split over the workgroup's waves in pairs of steps
// (128 bytes of a row) and joined in LDS.  The weights are the first operand, so
// a lane ends with four consecutive columns of one row.  A wave's loads of four
// pairs are on their way at once.
constexpr int kFewWaves = 8, kAhead = 4;

template <class T, int ACT>
__global__ __launch_bounds__(64 * kFewWaves) void few_kernel(ProductArgs a) {
    __shared__ i32x4 sums[kFewWaves][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int low = lane & 15, part = lane >> 4;
    const unsigned block = blockIdx.y * gridDim.x + blockIdx.x;
    const unsigned columns = (unsigned)((a.n + 15) / 16), tile = block / columns;
    RowTile rt;
    if (!find_rows(a, tile, 16, rt)) return;
    const size_t n0 = (size_t)(block - tile * columns) * 16;
    const bool some = rt.expert < a.experts;
    const size_t w_first = some ? rt.expert * a.n : 0;
    const size_t wr = w_first + (n0 + low < a.n ? n0 + low : a.n - 1);
    const unsigned char *wc = a.w_codes + wr * a.kp + part * 16;
    const size_t m = rt.r0 + low < rt.r1 ? rt.r0 + low : rt.r1 - 1;
    const long long row = a.rows ? a.rows[m] : (long long)m;
    const bool there = row >= 0 && (size_t)row < a.a_rows;
    const unsigned char *xc = a.a_codes + (there ? row : 0) * a.kp + part * 16;
    i32x4 acc = {0, 0, 0, 0};
    const size_t pairs = some ? a.kp / kPad : 0;
    for (size_t s0 = wave; s0 < pairs; s0 += kFewWaves * kAhead) {
        i32x4 w[kAhead][2], x[kAhead][2];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const size_t s = s0 + i * kFewWaves;
            if (s >= pairs) break;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                w[i][h] = *reinterpret_cast<const i32x4 *>(wc + s * kPad + h * kStep);
                x[i][h] = *reinterpret_cast<const i32x4 *>(xc + s * kPad + h * kStep);
            }
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (s0 + i * kFewWaves >= pairs) break;
#pragma unroll
            for (int h = 0; h < 2; ++h) acc = step_of(w[i][h], x[i][h], acc);
        }
    }
    sums[wave][lane] = acc;
    __syncthreads();
    const size_t r = rt.r0 + low, c = n0 + part * 4;
    if (wave || r >= rt.r1 || c >= a.n) return;
    i32x4 sum = sums[0][lane];
    for (int w = 1; w < kFewWaves; ++w) sum += sums[w][lane];
    const bool real = some && there;
    const float scale = a.a_scales[there ? row : 0];
    const float weight = a.row_scale && real ? a.row_scale[r] : 1.0f;
    T *out = reinterpret_cast<T *>(a.out) + r * a.n + c;
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = 0.0f;
        if (real && c + i < a.n) {
            const size_t at = w_first + c + i;
            const float z = fmaf((float)sum[i] * scale, a.w_scales[at], a.bias ? a.bias[at] : 0.0f);
            v[i] = act_of<kFine<T>, ACT>(z) * weight;
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

// 16 bytes of columns from n0 on of row r, past the caches: nothing here reads
// them again (16,384 x 4,096 x 4,096: 232 us, with ordinary stores 250).
template <class T>
__device__ __forceinline__ void store_columns(const ProductArgs &a, size_t r, size_t n0,
                                              u32x4 run) {
    constexpr int kRun = 16 / sizeof(T);
    T *out = reinterpret_cast<T *>(a.out) + r * a.n + n0;
    if (n0 + kRun <= a.n) {
        stream_out<T, 16>(reinterpret_cast<char *>(out), 0, run);
    } else {
        typedef T elems __attribute__((ext_vector_type(kRun)));
        const elems v = __builtin_bit_cast(elems, run);
#pragma unroll
        for (int i = 0; i < kRun; ++i)
            if (n0 + i < a.n) out[i] = v[i];
    }
}

// 16 bytes of each lane to 1 KB of LDS from `to` on.  In assembly, because the
// compiler, which follows such loads in LDS, waits for all of them before it
// reads any LDS behind a loop's start, the ones just issued too: the waits are
// arrive_but's.  The place in LDS stands in m0, as an operand: the compiler
// writes it and knows what it holds; the pause behind that write is needed.
__device__ __forceinline__ void fetch(const void *from, unsigned to) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"{m0}"(to), "v"(from) : "memory");
}

// Waits for all but the wave's last `COUNT` loads and for its LDS accesses, then
// for the other waves.
template <int COUNT>
__device__ __forceinline__ void arrive_but() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt((COUNT & 15) | (COUNT >> 4) << 14 | 0x0070);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
}

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

// The column of a wave's that row `low` of column tile i's operand is.  Of 16-bit
// results a lane ends with 16 bytes of consecutive columns in two tiles, the four
// lanes of a row with 64 bytes; where rows start on 64 bytes they leave from
// registers (8,192 tokens to 2 of 8 experts, 2,048 x 1,024, with quantisation: 61
// us, through LDS 64), else through LDS (12,000 x 1,500 x 700: 30 us, from
// registers 37), as 32-bit results do (8,000 x 2,048 x 1,000: 35 us, from
// registers 40).  spread_of: where the swizzle puts a column's codes, for such
// reads.
template <class T>
__device__ __forceinline__ int column_of(int i, int low) {
    if (sizeof(T) == 4) return 16 * i + low;
    return 32 * (i / 2) + 8 * (low / 4) + 4 * (i % 2) + low % 4;
}
template <class T>
__device__ __forceinline__ int spread_of(int row) {
    if (sizeof(T) == 4) return row & 7;
    return (row & 3) | (row >> 3 & 1) << 2;
}

// Staged tiles of BM rows and BN columns: slices of two steps (128 values, 128
// bytes a row) through STAGES buffers in LDS.
//
// Codes come by loads that write LDS themselves: a wave's load fills 1 KB,
// eight rows, in lane order.  16-byte piece c of row r lies at slot c ^ (r & 7)
// of its row (of a column: c ^ spread_of it), so that the rows of an operand
// read, 128 bytes apart, fall on all banks.
//
// Turn s: wait for the loads of slice s + 1; barrier: all waves have them, and
// have read slice s; then a step's products at a time, in NT groups, among them
// the loads of slice s + STAGES over slice s and the reads of the next step.
// The loads go early where the next turn waits for them (two buffers), else over
// the whole turn; all of them in a row would hold up the wave's products.
//
// m 16,384, n 4,096, k 4,096: 212 to 241 us by the card, 2.3 to 2.6 POPS; the
// instruction does 4.0 from registers, at 1.9 GHz.  By counters the matrix units
// are busy in 64% of the cycles (55% with GELU, 72% at k 8,192), at 1.95 GHz (1.76
// at k 8,192, of 2.4).  Between k 4,096 and 8,192, in the loop alone, they are in
// 81%: of the 53 us of a round of 256 tiles the products take 34, the loop's waits
// for loads, LDS and barriers 8, start and stores 11; GELU adds 8.  Tried and not
// faster: slices of one step in four buffers, three buffers under tiles of 128
// rows, rows touched ahead to have them in the L2.
template <class T, int ACT, int WM, int WN, int MT, int NT, int STAGES>
__global__ __launch_bounds__(64 * WM * WN) void tile_kernel(ProductArgs a) {
    constexpr int BM = 16 * MT * WM, BN = 16 * NT * WN, kWaves = WM * WN, kThreads = 64 * kWaves;
    constexpr int kRows = BM + BN, kLoads = kRows / 8 / kWaves;  // 1 KB a load of a wave
    constexpr int kReads = MT + NT;  // of a step
    static_assert(kRows <= kThreads && kRows % (8 * kWaves) == 0);
    constexpr int kGroup = 8;  // column tiles that neighbours in time share
    constexpr unsigned kStage = kRows * kPad;
    __shared__ __attribute__((aligned(1024))) unsigned char codes[STAGES * kStage];
    // Where each row's codes begin, in pieces of 16 bytes.
    __shared__ unsigned row_code[kRows];
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

    if (rt.expert >= a.experts) {
        constexpr int kRun = 16 / sizeof(T), kAcross = BN / kRun;
        const size_t c = n0 + t % kAcross * kRun;
        for (int r = t / kAcross; r < height; r += kThreads / kAcross)
            if (c < a.n) store_columns<T>(a, m0 + r, c, (u32x4){0, 0, 0, 0});
        return;
    }
    // The matrix row behind each row of the tile, the output's rows first,
    // counted from the tile's first (from the matrix's where they are
    // gathered; row 0 is read for one that is not there); rows past the tile's
    // end stand in for the last one and are not stored.
    const size_t w_first = (size_t)rt.expert * a.n + n0, a_first = a.rows ? 0 : m0;
    const unsigned pieces = (unsigned)(a.kp / 16);
    float scale = 0.0f, other = 0.0f;  // the row's, and its weight or the column's bias
    bool real = true;
    if (t < kRows) {
        int row;
        if (t >= BM) {
            row = n0 + (t - BM) < a.n ? t - BM : (int)(a.n - 1 - n0);
            scale = a.w_scales[w_first + row];
            if (a.bias) other = a.bias[w_first + row];
        } else {
            const int in = t < height ? t : height - 1;
            row = a.rows ? a.rows[m0 + in] : in;
            real = !a.rows || (row >= 0 && (size_t)row < a.a_rows);
            row = real ? row : 0;
            scale = a.a_scales[a_first + row];
            other = a.row_scale ? a.row_scale[m0 + in] : 1.0f;
        }
        row_code[t] = (unsigned)row * pieces;
    }
    __syncthreads();

    i32x4 acc[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = (i32x4){0, 0, 0, 0};

    // A load's rows lie on one side.
    const int row0 = wave * kLoads * 8;
    unsigned from[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
        from[i] = row_code[row0 + i * 8 + (lane >> 3)] +
                  ((lane & 7) ^ (row0 + i * 8 >= BM ? spread_of<T>(row0 + i * 8 - BM + (lane >> 3))
                                                    : lane >> 3));
    const unsigned slices = (unsigned)(a.kp / kPad);
    const unsigned char *a_base = a.a_codes + a_first * a.kp, *w_base = a.w_codes + w_first * a.kp;
    const unsigned lds = (unsigned)(uintptr_t)(LdsPtr)codes;
    auto load_one = [&](unsigned slice, unsigned stage, int i) {
        const int first = row0 + i * 8;
        const unsigned char *base = (first >= BM ? w_base : a_base) + (size_t)slice * kPad;
        fetch(base + (size_t)from[i] * 16, lds + stage + first * kPad);
    };
    const int row_x = wm * MT * 16, row_w = BM + wn * NT * 16;
    const int lane_row = low * kPad, slot = (part ^ (low & 7)) * 16;
    // The same slot for every column tile: they differ in bits that spread_of leaves out.
    const int w_row = column_of<T>(0, low), w_slot = (part ^ spread_of<T>(w_row)) * 16;
    // Read `r` of a step's operands, the rows' first.
    auto read_one = [&](unsigned stage, int s, Operands<MT, NT> &o, int r) {
        if (r < MT) {
            const unsigned char *p = codes + stage + lane_row + (slot ^ (s * kStep));
            o.x[r] = *reinterpret_cast<const i32x4 *>(p + (row_x + r * 16) * kPad);
        } else {
            const int i = r - MT;
            const unsigned char *p = codes + stage + w_row * kPad + (w_slot ^ (s * kStep));
            o.w[i] =
                *reinterpret_cast<const i32x4 *>(p + (row_w + column_of<T>(i, 0)) * kPad);
        }
    };
    Operands<MT, NT> even, odd;
#pragma unroll
    for (int i = 0; i < STAGES; ++i)
        if (i < slices)
#pragma unroll
            for (int j = 0; j < kLoads; ++j) load_one(i, i * kStage, j);
    if (t >= BM && t < kRows) {
        scale_of[t - BM] = scale;
        bias_of[t - BM] = other;
    } else if (t < BM) {
        scale_of_row[t] = scale;
        weight_of_row[t] = other;
        real_row[t] = real;
    }
    // Slice `next` is there when all loads but those of later slices are.
    auto await = [&](unsigned next) {
        const unsigned later = slices - 1 - next;
        if (later >= STAGES - 1 && next == 0)
            arrive_but<(STAGES - 1) * kLoads>();
        else if (STAGES > 3 && later >= 2)
            arrive_but<2 * kLoads>();
        else if (STAGES > 2 && later >= 1)
            arrive_but<kLoads>();
        else
            arrive_but<0>();
    };
    await(0);
#pragma unroll
    for (int r = 0; r < kReads; ++r) read_one(0, 0, even, r);
#pragma unroll
    for (int r = 0; r < kReads; ++r) read_one(0, 1, odd, r);
    multiply<MT, NT>(even, acc);
    unsigned stage = 0;
    // Half a turn: a step's products in NT groups, the next step's reads and a
    // share of the loads among them.
    constexpr int kEach = (kReads + NT - 1) / NT;
    constexpr int kShare = STAGES > 2 ? (kLoads + 2 * NT - 1) / (2 * NT) : (kLoads + NT - 1) / NT;
    auto half = [&](auto loads, int h, unsigned slice, unsigned to, unsigned from_stage,
                    Operands<MT, NT> &now, Operands<MT, NT> &next) {
#pragma unroll
        for (int g = 0; g < NT; ++g) {
            if (decltype(loads)::value)
#pragma unroll
                for (int i = 0; i < kShare; ++i)
                    if ((h * NT + g) * kShare + i < kLoads)
                        load_one(slice, to, (h * NT + g) * kShare + i);
#pragma unroll
            for (int r = g * kEach; r < (g + 1) * kEach && r < kReads; ++r)
                read_one(from_stage, h, next, r);
#pragma unroll
            for (int j = 0; j < MT; ++j) acc[g][j] = step_of(now.w[g], now.x[j], acc[g][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto turn = [&](auto loads, unsigned slice) {
        await(slice + 1);
        const unsigned free = stage;
        stage = stage + kStage < STAGES * kStage ? stage + kStage : 0;
        half(loads, 0, slice + STAGES, free, stage, odd, even);
        half(loads, 1, slice + STAGES, free, stage, even, odd);
    };
    unsigned slice = 0;
    for (; slice + STAGES < slices; ++slice) turn(Int<1>(), slice);
    for (; slice + 1 < slices; ++slice) turn(Int<0>(), slice);
    multiply<MT, NT>(odd, acc);

    // Columns of row `in` of the tile that the lane holds in row tile j.
    const bool weighted = a.rows || a.row_scale;
    f32x4 bias[NT], column[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int c = wn * NT * 16 + column_of<T>(i, part * 4);
        bias[i] = *reinterpret_cast<const f32x4 *>(bias_of + c);
        column[i] = *reinterpret_cast<const f32x4 *>(scale_of + c);
    }
    auto results = [&](int j, int in, float (&v)[NT][4]) {
        const float row_scale = scale_of_row[in];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                v[i][q] = act_of<kFine<T>, ACT>(
                    fmaf((float)acc[i][j][q] * row_scale, column[i][q], bias[i][q]));
        if (weighted) {
            const float weight = weight_of_row[in];
            const bool there = real_row[in];
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) v[i][q] = there ? v[i][q] * weight : 0.0f;
        }
    };
    constexpr int kRun = 16 / sizeof(T);
    if (sizeof(T) == 2 && a.direct) {
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            const int in = (wm * MT + j) * 16 + low;
            float v[NT][4];
            results(j, in, v);
            if (in >= height) continue;
#pragma unroll
            for (int i = 0; i < NT; i += 2) {
                float run[kRun];
#pragma unroll
                for (int q = 0; q < kRun; ++q) run[q] = v[i + q / 4][q % 4];
                const size_t c = n0 + wn * NT * 16 + column_of<T>(i, part * 4);
                if (c < a.n) store_columns<T>(a, m0 + in, c, Vec<T, 16>::pack(run));
            }
        }
        return;
    }
    arrive_but<0>();
    // Through LDS, whose rows leave in runs: kPass rows of the tile at a time, two
    // buffers in turn, so that a pass is read before the next but one is written.
    // Four columns are one piece; piece c of a wave's row r lies at c ^ 4 r, so
    // that the rows of a write fall on different banks.
    typedef Vec<T, 4 * sizeof(T)> Four;
    constexpr int kPassTiles = pass_tiles(MT, WM * 16 * BN * sizeof(T), (int)kStage);
    constexpr int kPass = kPassTiles * WM * 16, kPieces = BN / 4;
    constexpr int kAcross = BN / kRun, kSweep = kThreads / kAcross;
    static_assert(MT % kPassTiles == 0);
    const int c = t % kAcross * kRun;
    const size_t n1 = n0 + c;
#pragma unroll
    for (int j0 = 0; j0 < MT; j0 += kPassTiles) {
        unsigned char *passed = codes + j0 / kPassTiles % 2 * kStage;
#pragma unroll
        for (int j = 0; j < kPassTiles; ++j) {
            const int at = (wm * kPassTiles + j) * 16 + low;
            float v[NT][4];
            results(j0 + j, (wm * MT + j0 + j) * 16 + low, v);
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const int piece = ((wn * NT * 16 + column_of<T>(i, part * 4)) / 4) ^
                                  (low * 4 & (kPieces - 1));
                reinterpret_cast<typename Four::raw *>(passed)[at * kPieces + piece] =
                    Four::pack(v[i]);
            }
        }
        __syncthreads();
        if (n1 >= a.n) continue;
#pragma unroll 4
        for (int row = t / kAcross; row < kPass; row += kSweep) {
            const int in = row / (kPassTiles * 16) * (MT * 16) + j0 * 16 + row % (kPassTiles * 16);
            const int piece = c / 4 ^ (row % 16 * 4 & (kPieces - 1));
            const u32x4 run = *reinterpret_cast<const u32x4 *>(
                passed + (row * kPieces + piece) * sizeof(typename Four::raw));
            if (in < height) store_columns<T>(a, m0 + in, n1, run);
        }
    }
}

// A workgroup's tile, how many workgroups run at once, and what a round of them
// is taken to cost in 0.01 us: start and end, and each slice of k; the same for
// the last round where it has one workgroup to a CU.
struct Shape {
    int rows, columns, slots, start, slice, lone_start, lone_slice;
};
constexpr Shape kShapes[] = {{16, 16, 256, 0, 13, 0, 13},
                             {64, 64, 512, 360, 42, 360, 21},
                             {64, 128, 512, 330, 61, 380, 30},
                             {128, 128, 512, 550, 100, 330, 72},
                             {192, 256, 256, 850, 130, 850, 130},
                             {256, 256, 256, 1000, 160, 1000, 160}};
constexpr int kFewStart = 300;  // once, not in each round
enum { kFew, kSmall, kLow, kMiddle, kHigh, kLarge, kCount };

size_t tiles_of(const ProductArgs &a, int shape) {
    const Shape t = kShapes[shape];
    // Every run of rows may end within a tile.
    const size_t high = (a.m + t.rows - 1) / t.rows + (a.offsets ? a.experts + 2 : 0);
    return high * ((a.n + t.columns - 1) / t.columns);
}

// The tiles with rows: of an expert with many about half a tile more than they
// fill, of one with few a single one.
size_t likely_tiles(const ProductArgs &a, int shape) {
    const Shape t = kShapes[shape];
    const size_t experts = (size_t)a.experts < a.m ? a.experts : a.m, each = a.m / experts;
    size_t high = (a.m + t.rows - 1) / t.rows;
    if (experts > 1) high = each < (size_t)t.rows / 2 ? experts : high + experts / 2;
    return high * ((a.n + t.columns - 1) / t.columns);
}

// A dimension of a grid holds less than 2^32 threads, 512 to a tile.  More than
// 2^22 tiles of few rows take rows of 2^22 workgroups, the last of which find
// no tile; staged tiles leave products of 2^23 tiles and more to them.
constexpr unsigned kGridRow = 1 << 22;
static_assert(64 * kFewWaves * (size_t)kGridRow < size_t(1) << 32);

// Measured (us, bf16 out; large / high / middle / low / small / few):
//   m 16,384 n 4,096 k 4,096: 241 / 266 / 292 / 366 / 435
//   m 16,384 n 4,096 k 1,024: 92 / 104 / 108 / 132 / 172
//   m 16,384 n 2,048 k 1,024, 8 experts: 69 / 63 / 68 / 83 / 105 / 585
//   m 10,000 n 3,000 k 2,000: 76 / 83 / 90 / 106 / 134
//   m  3,000 n 3,500 k 3,500: 51 / 46 / 57 / 67 / 81
//   m  8,192 n 2,048 k   512: 17.1 / 23.0 / 18.9 / 24.6 / 33.9 / 139
//   m  1,024 n 4,096 k 4,096: 43.4 / 38.0 / 26.9 / 25.5 / 34.5 / 228
//   m  2,000 n 1,000 k 4,000: 42.1 / 36.8 / 24.1 / 16.1 / 16.8
//   m  1,000 n 1,000 k 1,000: 16.4 / 14.1 / 8.3 / 6.9 / 6.1
//   m    300 n 4,096 k 4,096: 41.6 / 36.1 / 23.6 / 14.7 / 14.5
//   m     64 n 4,096 k 4,096: 39.8 / 34.4 / 22.3 / 13.5 / 10.3 / 18.1
//   m     64 n 4,096 k 1,024: 6.3 (low) / 5.3 / 7.1
//   m     32 n 4,096 k 4,096: 13.1 (low) / 10.0 / 10.7
//   m     16 n 4,096 k 4,096: 12.8 (low) / 10.0 / 7.6
// The cheapest by the costs above: the fastest in every line, or within 2% of it;
// elsewhere within 7% (12,000 x 1,500 x 700: 32 us in middle tiles, 30 in high).
int shape_for(const ProductArgs &a) {
    // The staged kernels count a matrix in 32 bits of 16 bytes, from a tile's
    // first row (from the first of all where rows are gathered).
    const size_t reach = 0xffffffffu / (a.kp / 16), slices = a.kp / kPad;
    const bool staged = !a.rows || a.a_rows <= reach;
    int best = kFew;
    size_t least = ~size_t(0);
    for (int shape = kFew; shape < kCount; ++shape) {
        if (shape > kFew && (!staged || tiles_of(a, shape) >= 2 * kGridRow)) continue;
        const Shape t = kShapes[shape];
        const size_t tiles = likely_tiles(a, shape), rest = tiles % t.slots;
        size_t cost = (tiles / t.slots) * (t.start + t.slice * slices);
        if (rest > 256)
            cost += t.start + t.slice * slices;
        else if (rest)
            cost += t.lone_start + t.lone_slice * slices;
        if (shape == kFew) cost += kFewStart;
        if (cost < least) {
            least = cost;
            best = shape;
        }
    }
    return best;
}

template <class T>
void launch_product(const ProductArgs &a, int act, int shape, unsigned tiles, hipStream_t q) {
    const dim3 few = tiles < kGridRow ? dim3(tiles)
                                      : dim3(kGridRow, (tiles + kGridRow - 1) / kGridRow);
    with_act(act, [&](auto which) {
        constexpr int ACT = decltype(which)::value;
        switch (shape) {
            case kFew: few_kernel<T, ACT><<<few, 64 * kFewWaves, 0, q>>>(a); break;
            case kSmall: tile_kernel<T, ACT, 2, 2, 2, 2, 4><<<tiles, 256, 0, q>>>(a); break;
            case kLow: tile_kernel<T, ACT, 2, 2, 2, 4, 3><<<tiles, 256, 0, q>>>(a); break;
            case kMiddle: tile_kernel<T, ACT, 2, 2, 4, 4, 2><<<tiles, 256, 0, q>>>(a); break;
            case kHigh: tile_kernel<T, ACT, 2, 4, 6, 4, 2><<<tiles, 512, 0, q>>>(a); break;
            default: tile_kernel<T, ACT, 2, 4, 8, 4, 2><<<tiles, 512, 0, q>>>(a); break;
        }
    });
}

unsigned grid_of(size_t items, size_t per) {
    const size_t want = (items + per - 1) / per;
    return (unsigned)(want < kMaxGrid ? want : kMaxGrid);
}

template <class T, bool STREAM>
void launch_rows(const QuantArgs &a, hipStream_t q) {
    const size_t per = a.pieces <= 64 * kHeld ? kQuantThreads / 64 : 1;
    const unsigned grid = grid_of(a.rows, per);
    if (per > 1)
        quantise_kernel<T, 64, STREAM><<<grid, kQuantThreads, 0, q>>>(a);
    else
        quantise_kernel<T, kQuantThreads, STREAM><<<grid, kQuantThreads, 0, q>>>(a);
}

template <class T>
void launch_quantise(const QuantArgs &a, hipStream_t q) {
    // Of longer rows than a workgroup holds the rest is read twice.
    const bool held = a.pieces <= kQuantThreads * kHeld;
    if (held && a.rows * a.k * sizeof(T) > kStreamBytes)
        launch_rows<T, true>(a, q);
    else
        launch_rows<T, false>(a, q);
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
        !words_ok(a_scales, w_scales, rows, offsets, bias, row_scale) ||
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
    a.direct = dtype != TB_HIP_F32 && multiple_of(out, 64) && n * type_size(dtype) % 64 == 0;
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
