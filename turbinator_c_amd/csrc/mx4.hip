// Microscaled 4-bit floating point (hip_layers.h): quantisation, the values it
// stands for, and products on the scaled matrix instructions.  Acting on a few
// tokens reads far more weights than it multiplies: a quarter of bf16's bytes
// is what this form is for.
//
//   scale  2^(s - 127), s = max(exponent bits of the largest magnitude - 2, 0)
//   code   value / scale (exact: a power of two) rounded to 0, 0.5, 1, 1.5, 2,
//          3, 4, 6, ties to even, by v_cvt_scalef32_pk_fp4_f32
//   out    = act(sum_k a_k w_k + bias) row_scale, summed in fp32 by
//          v_mfma_scale_f32_16x16x128_f8f6f4: lane l holds row l % 16, values
//          32 (l / 16) .. + 31 of a step of 128, one scale block, in 16 bytes
#include "product_tiles.h"
#include "xcd_order.h"

namespace {

using namespace layer;

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr size_t kMaxCount = 0x7fffffffu, kMaxOutputs = size_t(1) << 38;
constexpr size_t kMaxGrid = 1 << 20;
constexpr int kBlock = 32, kPad = 128;

__host__ __device__ inline size_t padded(size_t k) { return (k + kPad - 1) / kPad * kPad; }

// --------------------------------------------------------------------------
// Quantisation: four lanes to a block of 32, eight values each, one vector in
// and one word out.  Bound by memory where rows start on 16 bytes: 40,960 x
// 2,000 bf16 44 us, the values back 37 us (4.7 and 5.6 TB/s of what they read
// and write).  Other rows go by single elements: k 2,002 takes 2.3 and 2.7
// times as long (89 and 104 us for 38 and 39, in a row on the same rows).

constexpr int kQuantThreads = 256;

struct QuantArgs {
    const char *x;
    size_t stride;
    unsigned *codes;
    unsigned char *scales;
    size_t items;    // rows * kp / 8
    unsigned per;    // kp / 8
    unsigned k;
    int vector;      // rows start on 16 bytes
};

template <class T>
__device__ __forceinline__ void load8(const QuantArgs &a, const char *row, unsigned k0,
                                      float (&v)[8]) {
    if (a.vector && k0 + 8 <= a.k) {
        typedef Vec<T, 16> X;
#pragma unroll
        for (int i = 0; i < 8 / X::n; ++i) {
            float part[X::n];
            X::unpack(*reinterpret_cast<const typename X::raw *>(
                          row + (size_t)(k0 + i * X::n) * sizeof(T)),
                      part);
#pragma unroll
            for (int j = 0; j < X::n; ++j) v[i * X::n + j] = part[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = k0 + j < a.k ? (float)reinterpret_cast<const T *>(row)[k0 + j] : 0.0f;
    }
}

template <class T>
__global__ __launch_bounds__(kQuantThreads) void quantise_kernel(QuantArgs a) {
    // Whole blocks: kp / 8 and the grid's step are multiples of four.
    for (size_t i = (size_t)blockIdx.x * kQuantThreads + threadIdx.x; i < a.items;
         i += (size_t)gridDim.x * kQuantThreads) {
        const size_t row = i / a.per;
        const unsigned at = (unsigned)(i - row * a.per);
        float v[8];
        load8<T>(a, a.x + row * a.stride, at * 8, v);
        // Magnitudes order as integers; Inf and NaN have the exponent 255.
        unsigned most = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const unsigned m = __builtin_bit_cast(unsigned, v[j]) & 0x7fffffffu;
            most = m > most ? m : most;
        }
        for (int off = 1; off < 4; off *= 2) {
            const unsigned o = __shfl_xor(most, off);
            most = o > most ? o : most;
        }
        const unsigned e = most >> 23;
        const unsigned s = e == 255 ? 255 : e > 2 ? e - 2 : 0;
        const float inverse = __builtin_bit_cast(float, (254u - s) << 23);
        unsigned codes = 0;
        if (s != 255) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= inverse;
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[0], v[1], 1.0f, 0);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[2], v[3], 1.0f, 1);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[4], v[5], 1.0f, 2);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[6], v[7], 1.0f, 3);
        }
        a.codes[i] = codes;
        if ((i & 3) == 0) a.scales[i / 4] = (unsigned char)s;
    }
}

// 2^(s - 127), a subnormal for 0, NaN for 255.
__device__ __forceinline__ float scale_of(unsigned s) {
    return __builtin_bit_cast(float, s == 255 ? 0x7fc00000u : s ? s << 23 : 1u << 22);
}

// Code c's value from its doubled magnitudes, a nibble each.
__device__ __forceinline__ float value_of(unsigned c) {
    const float m = 0.5f * (float)((0xc8643210u >> (4 * (c & 7))) & 15);
    return c & 8 ? -m : m;
}

struct ValueArgs {
    const unsigned *codes;
    const unsigned char *scales;
    char *out;
    size_t items;
    unsigned per, k;
    int vector;
};

template <class T>
__global__ __launch_bounds__(kQuantThreads) void values_kernel(ValueArgs a) {
    typedef Vec<T, 16> X;
    for (size_t i = (size_t)blockIdx.x * kQuantThreads + threadIdx.x; i < a.items;
         i += (size_t)gridDim.x * kQuantThreads) {
        const size_t row = i / a.per;
        const unsigned k0 = (unsigned)(i - row * a.per) * 8;
        const float scale = scale_of(a.scales[i / 4]);
        const unsigned codes = a.codes[i];
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = value_of(codes >> (4 * j)) * scale;
        T *out = reinterpret_cast<T *>(a.out) + row * a.k;
        if (a.vector && k0 + 8 <= a.k) {
#pragma unroll
            for (int p = 0; p < 8 / X::n; ++p) {
                float part[X::n];
#pragma unroll
                for (int j = 0; j < X::n; ++j) part[j] = v[p * X::n + j];
                *reinterpret_cast<typename X::raw *>(out + k0 + p * X::n) = X::pack(part);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (k0 + j < a.k) out[k0 + j] = (T)v[j];
        }
    }
}

// --------------------------------------------------------------------------
// Products

struct ProductArgs {
    const unsigned char *a_codes, *a_scales, *w_codes, *w_scales;
    const int *rows, *offsets;
    const float *bias, *row_scale;
    char *out;
    size_t a_rows, m, n, kp;
    int experts, act, vector;
};

__device__ __forceinline__ f32x4 step16(i32x4 w, int ws, i32x4 x, int xs, f32x4 c) {
    const i32x8 A = {w[0], w[1], w[2], w[3], 0, 0, 0, 0}, B = {x[0], x[1], x[2], x[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, c, 4, 4, 0, ws, 0, xs);
}

// Four consecutive columns n0 .. of row r: bias, activation, row scale.
template <class T, int ACT>
__device__ __forceinline__ void store4(const ProductArgs &a, int expert, bool real, size_t r,
                                       size_t n0, f32x4 c) {
    T *out = reinterpret_cast<T *>(a.out) + r * a.n + n0;
    float v[4];
    const float scale = a.row_scale && real ? a.row_scale[r] : 1.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = 0.0f;
        if (real && n0 + i < a.n) {
            const float z = a.bias ? c[i] + a.bias[(size_t)expert * a.n + n0 + i] : c[i];
            v[i] = act_of<kFine<T>, ACT>(z) * scale;
        }
    }
    if (a.vector && n0 + 4 <= a.n) {
        typedef Vec<T, 4 * sizeof(T)> X;
        *reinterpret_cast<typename X::raw *>(out) = X::pack(v);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n0 + i < a.n) out[i] = (T)v[i];
    }
}

// Few rows: tiles of 16 columns and 16 MT rows, operands straight from memory
// in the instruction's layout, k split over the workgroup's waves in pairs of
// steps (128 bytes of a row) and joined in LDS.  The weights are the first
// operand, so a lane ends with four consecutive columns of one row.  10 rows,
// 2,048 columns, k 2,048: 4.4 us, of which the 2.2 MB of weights would take
// 0.5: a launch, two loads in turn (rows or offsets, then codes) and the join.
constexpr int kFewWaves = 8;

template <class T, int ACT, int MT>
__global__ __launch_bounds__(64 * kFewWaves) void few_kernel(ProductArgs a) {
    __shared__ f32x4 sums[kFewWaves][MT][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int low = lane & 15, part = lane >> 4;
    const unsigned block = blockIdx.y * gridDim.x + blockIdx.x;
    const unsigned columns = (unsigned)((a.n + 15) / 16), tile = block / columns;
    RowTile rt;
    if (!find_rows(a, tile, 16 * MT, rt)) return;
    const size_t n0 = (size_t)(block - tile * columns) * 16;
    const bool some = rt.expert < a.experts;
    const size_t code_row = a.kp / 2, scale_row = a.kp / kBlock;
    const size_t wr = (n0 + low < a.n ? n0 + low : a.n - 1) + (some ? rt.expert * a.n : 0);
    const unsigned char *wc = a.w_codes + wr * code_row + part * 16;
    const unsigned char *ws = a.w_scales + wr * scale_row + part;
    const unsigned char *xc[MT], *xs[MT];
    unsigned real = 0;  // a bit for each row tile
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        size_t m = rt.r0 + j * 16 + low;
        m = m < rt.r1 ? m : rt.r1 - 1;
        const long long row = a.rows ? a.rows[m] : (long long)m;
        const bool there = row >= 0 && (size_t)row < a.a_rows;
        real |= (some && there ? 1u : 0u) << j;
        xc[j] = a.a_codes + (there ? row : 0) * code_row + part * 16;
        xs[j] = a.a_scales + (there ? row : 0) * scale_row + part;
    }
    f32x4 acc[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[j] = (f32x4){0, 0, 0, 0};
    const size_t steps = some ? a.kp / kPad : 0;
    for (size_t s = 2 * wave; s < steps; s += 2 * kFewWaves) {
        // A step behind the last is the last again, times nothing.
        const size_t next = s + 1 < steps ? s + 1 : s;
        const i32x4 w0 = *reinterpret_cast<const i32x4 *>(wc + s * 64);
        const i32x4 w1 = *reinterpret_cast<const i32x4 *>(wc + next * 64);
        const int sw0 = ws[s * 4], sw1 = ws[next * 4];
        i32x4 x0[MT], x1[MT];
        int sx0[MT], sx1[MT];
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            x0[j] = *reinterpret_cast<const i32x4 *>(xc[j] + s * 64);
            x1[j] = *reinterpret_cast<const i32x4 *>(xc[j] + next * 64);
            sx0[j] = xs[j][s * 4];
            sx1[j] = xs[j][next * 4];
        }
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[j] = step16(w0, sw0, x0[j], sx0[j], acc[j]);
        if (next > s)
#pragma unroll
            for (int j = 0; j < MT; ++j) acc[j] = step16(w1, sw1, x1[j], sx1[j], acc[j]);
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) sums[wave][j][lane] = acc[j];
    __syncthreads();
    for (int j = wave; j < MT; j += kFewWaves) {
        f32x4 sum = sums[0][j][lane];
        for (int w = 1; w < kFewWaves; ++w) sum += sums[w][j][lane];
        const size_t r = rt.r0 + j * 16 + low, c = n0 + part * 4;
        if (r < rt.r1 && c < a.n) store4<T, ACT>(a, rt.expert, real >> j & 1, r, c, sum);
    }
}

// Large products: tiles of BM rows and BN columns, staged through LDS in
// slices of two steps (256 values, 128 bytes a row), two slices in turn.
//
// Codes come by loads that write LDS themselves: a wave's load fills 1 KB,
// eight rows, in lane order.  16-byte piece c of row r lies at slot c ^ (r & 7)
// of its row, so that the rows of an operand read, 128 bytes apart, fall on
// all banks.  Scales come through registers, the eight of a row at once (a
// request of the L2 costs the same for four bytes as for a line), and are
// turned while they are stored: lane l's word holds the scales of its part of
// four row tiles, which the instruction picks by number.
//
// Turn s: read step 1 of slice s while multiplying step 0; wait for the loads
// of slice s + 1; barrier: all waves have them, and have read slice s; load
// slice s + 2 over it, and read step 0 of slice s + 1 while multiplying step 1.
//
// m 16,384, n 4,096, k 4,096: 168 to 176 us, 3.1 to 3.3 PFLOP/s, half of what
// the instruction does from registers on such values (6.4): the waves of a CU
// meet at a barrier every 64 matrix instructions.  At short k the ends count: k
// 1,024 takes 18.1 us for 8,192 x 2,048, of which 8 are starting and storing.
// Outputs whose rows are off 16 bytes leave by single elements: n 4,095 takes
// 223 us, and with k 256 114 us where n 4,096 takes 48.
//
// With experts the grid holds tiles for the runs' ends that may not be there,
// the last ones of each band of columns, which the contiguous order gives to
// some of the XCDs: 8,200 rows of 8 experts leave 94 tiles to two of them and
// 150 to the others.
constexpr int kSlice = 2 * kPad, kSliceBytes = kSlice / 2;

typedef const __attribute__((address_space(1))) void *GlobalPtr;

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

__device__ __forceinline__ f32x4 step_of(int sel, i32x4 w, int ws, i32x4 x, int xs, f32x4 c) {
    const i32x8 A = {w[0], w[1], w[2], w[3], 0, 0, 0, 0}, B = {x[0], x[1], x[2], x[3], 0, 0, 0, 0};
#define TB_STEP(i, j)                                                                       \
    case 4 * i + j:                                                                         \
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, c, 4, 4, i, ws, j, xs);
    switch (sel) {
        TB_STEP(0, 0) TB_STEP(0, 1) TB_STEP(0, 2) TB_STEP(0, 3)
        TB_STEP(1, 0) TB_STEP(1, 1) TB_STEP(1, 2) TB_STEP(1, 3)
        TB_STEP(2, 0) TB_STEP(2, 1) TB_STEP(2, 2) TB_STEP(2, 3)
        TB_STEP(3, 0) TB_STEP(3, 1) TB_STEP(3, 2)
        default:
            return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, c, 4, 4, 3, ws, 3, xs);
    }
#undef TB_STEP
}

// The operands of one step of a wave: MT row tiles and NT column tiles.
template <int MT, int NT>
struct Operands {
    i32x4 x[MT], w[NT];
    int xs[MT / 4], ws[NT / 4];
};

// Lane 16 j + r holds the four scale bytes of row 16 j + r: out, lane 16 p + r
// holds byte p of the rows r, 16 + r, 32 + r and 48 + r.  Two exchanges between
// lanes 32 and 16 apart, each followed by a choice of bytes.
__device__ __forceinline__ int turned(unsigned v, int p) {
    const auto far = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = __builtin_amdgcn_perm(far[1], far[0], p & 2 ? 0x07060302 : 0x05040100);
    const auto near = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return (int)__builtin_amdgcn_perm(near[1], near[0], p & 1 ? 0x07030501 : 0x06020400);
}

// `codes` and `scales` at the lane's place of step 0 or 1.
template <int MT, int NT>
__device__ __forceinline__ void read_step(const unsigned char *__restrict codes,
                                          const int *__restrict scales, int row_x, int row_w,
                                          Operands<MT, NT> &__restrict o) {
#pragma unroll
    for (int j = 0; j < MT / 4; ++j) o.xs[j] = scales[row_x * 2 + j * 128];
#pragma unroll
    for (int i = 0; i < NT / 4; ++i) o.ws[i] = scales[row_w * 2 + i * 128];
#pragma unroll
    for (int j = 0; j < MT; ++j)
        o.x[j] = *reinterpret_cast<const i32x4 *>(codes + row_x * kSliceBytes +
                                                  j * 16 * kSliceBytes);
#pragma unroll
    for (int i = 0; i < NT; ++i)
        o.w[i] = *reinterpret_cast<const i32x4 *>(codes + row_w * kSliceBytes +
                                                  i * 16 * kSliceBytes);
}

template <int MT, int NT>
__device__ __forceinline__ void multiply(const Operands<MT, NT> &o, f32x4 (&acc)[NT][MT]) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j)
            acc[i][j] = step_of(4 * (i % 4) + j % 4, o.w[i], o.ws[i / 4], o.x[j], o.xs[j / 4],
                                acc[i][j]);
}

// 16 bytes of columns from n0 on of row r.  Nothing here reads them again:
// stores past the caches (8,192 x 2,048 results, k 1,024: 20.7 us, else 22.4).
template <class T>
__device__ __forceinline__ void store_run(const ProductArgs &a, size_t r, size_t n0, u32x4 run) {
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

template <class T, int ACT, int WM, int WN, int MT, int NT>
__global__ __launch_bounds__(64 * WM * WN) void tile_kernel(ProductArgs a) {
    constexpr int BM = 16 * MT * WM, BN = 16 * NT * WN, kWaves = WM * WN, kThreads = 64 * kWaves;
    constexpr int kRows = BM + BN, kLoads = kRows / 8 / kWaves;  // 1 KB a load of a wave
    constexpr int kReads = MT + NT + 2;  // of a step
    static_assert(kRows == kThreads && BM % (kLoads * 8) == 0);
    constexpr int kGroup = 8;  // column tiles that neighbours in time share
    // Two arrays each, chosen at compile time: the compiler knows that a read
    // of one need not wait for the loads into the other.
    __shared__ __attribute__((aligned(1024))) unsigned char codes0[kRows * kSliceBytes];
    __shared__ __attribute__((aligned(1024))) unsigned char codes1[kRows * kSliceBytes];
    // [group of 64 rows][step][lane]
    __shared__ __attribute__((aligned(4096))) int scales0[kRows * 2], scales1[kRows * 2];
    // Byte offset of each row's codes, by the loading wave, lane / 8 and load.
    __shared__ __attribute__((aligned(16))) unsigned row_code[kRows];
    __shared__ float scale_of_row[BM];
    __shared__ __attribute__((aligned(16))) float bias_of[BN];
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
    const bool none = rt.expert >= a.experts;
    const size_t code_row = a.kp / 2, scale_row = a.kp / kBlock;
    const size_t w_first = none ? 0 : (size_t)rt.expert * a.n;

    if (none) {
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
        bias_of[t - BM] = a.bias ? a.bias[w_first + n0 + row] : 0.0f;
    } else {
        const int in = t < height ? t : height - 1;
        row = a.rows ? a.rows[m0 + in] : in;
        const bool real = !a.rows || (row >= 0 && (size_t)row < a.a_rows);
        row = real ? row : 0;
        real_row[t] = real;
        scale_of_row[t] = a.row_scale ? a.row_scale[m0 + in] : 1.0f;
    }
    row_code[(t / (8 * kLoads) * 8 + t % 8) * kLoads + t / 8 % kLoads] = (unsigned)(row * code_row);
    __syncthreads();

    f32x4 acc[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = (f32x4){0, 0, 0, 0};

    // Codes: a base of the wave's side, 32 bits to the row, and a column that
    // stays within it (the second step of a last slice may lie past its end:
    // what is read for it is not used).
    const int row0 = wave * kLoads * 8;
    const bool w_side = row0 >= BM;
    const size_t first = w_side ? w_first + n0 : a.rows ? 0 : m0;
    const unsigned char *base = (w_side ? a.w_codes : a.a_codes) + first * code_row;
    unsigned from[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) from[i] = row_code[(t >> 3) * kLoads + i];
    const unsigned column = ((lane & 7) ^ (lane >> 3)) * 16, code_end = (unsigned)code_row - 16;
    auto load = [&](unsigned slice, unsigned char *codes) {
        unsigned at = slice * kSliceBytes + column;
        at = at < code_end ? at : code_end;
        unsigned char *to = codes + row0 * kSliceBytes;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) load_to_lds(base + (from[i] + at), to + i * 1024);
    };
    // Scales: thread t has row t, on the same side as its wave's chunks.
    const unsigned char *sbase = (w_side ? a.w_scales : a.a_scales) + first * scale_row;
    const unsigned scale_from = (unsigned)(row * scale_row);
    const unsigned scale_end = (unsigned)scale_row - 8;
    u32x2 held;
    auto load_scales = [&](unsigned slice) {
        const unsigned at = slice * 8 < scale_end ? slice * 8 : scale_end;
        held = *reinterpret_cast<const u32x2 *>(sbase + (scale_from + at));
    };
    // Steps behind the last get scales of 2^-127 on both sides, whose products
    // vanish: the loop runs over whole pairs of slices.
    auto store_scales = [&](unsigned slice, int *scales) {
        unsigned one = held[0], two = held[1];
        if (slice * 8 > scale_end) {  // uniform: a row's end, read four bytes early
            one = slice * 8 - scale_end == 4 ? two : 0;
            two = 0;
        }
        scales[(t >> 6) * 128 + lane] = turned(one, part);
        scales[(t >> 6) * 128 + 64 + lane] = turned(two, part);
    };
    const int row_x = wm * MT * 16, row_w = BM + wn * NT * 16;
    const int lane_row = low * kSliceBytes, slot = (part ^ (low & 7)) * 16;
    auto read = [&](const unsigned char *codes, const int *scales, int s, Operands<MT, NT> &o) {
        read_step<MT, NT>(codes + lane_row + (slot ^ (s * 64)), scales + s * 64 + lane, row_x,
                          row_w, o);
    };
    Operands<MT, NT> even, odd;
    auto turn = [&](unsigned slice, unsigned char *codes, int *scales, unsigned char *codes_next,
                    int *scales_next) {
        store_scales(slice + 1, scales_next);
        read(codes, scales, 1, odd);
        multiply<MT, NT>(even, acc);
#pragma unroll
        for (int i = 0; i < kReads; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
        }
        arrive();
        load_scales(slice + 2);
        load(slice + 2, codes);
        read(codes_next, scales_next, 0, even);
        multiply<MT, NT>(odd, acc);
#pragma unroll
        for (int i = 0; i < kLoads + 2; ++i) {
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
    load_scales(0);
    load(0, codes0);
    store_scales(0, scales0);
    load_scales(1);
    arrive();
    read(codes0, scales0, 0, even);
    load(1, codes1);
    const unsigned steps = (unsigned)(a.kp / kPad);
    for (unsigned slice = 0; 2 * slice < steps; slice += 2) {
        turn(slice, codes0, scales0, codes1, scales1);
        turn(slice + 1, codes1, scales1, codes0, scales0);
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
    f32x4 bias[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
        bias[i] = *reinterpret_cast<const f32x4 *>(bias_of + (wn * NT + i) * 16 + part * 4);
#pragma unroll
    for (int j0 = 0; j0 < MT; j0 += kPassTiles) {
        unsigned char *results = j0 / kPassTiles % 2 ? codes1 : codes0;
#pragma unroll
        for (int j = 0; j < kPassTiles; ++j) {
            const int in = (wm * MT + j0 + j) * 16 + low, at = (wm * kPassTiles + j) * 16 + low;
            const float scale = scale_of_row[in];
            const bool real = real_row[in];
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                float v[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    v[q] = act_of<kFine<T>, ACT>(acc[i][j0 + j][q] + bias[i][q]) * scale;
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

// Measured (us; large / middle / few rows with 4, 2 and 1 row tiles; bf16 out):
//   m 16,384 n 4,096 k 4,096: 168 / 210 / 2,210 / 2,650 / 3,537
//   m  8,192 n 2,048 k 2,048: 25.5 / 36.2 / 283 / 340 / 447     (256 large tiles)
//   m  8,192 n 2,048 k 1,024: 18.1 / 23.9 / 185 / 193 / 227
//   m  8,192 n 2,048 k   512: 14.7 / 17.1 / 99 / 99 / 131
//   m  8,192 n 2,048 k   256: 15.3 / 17.1 / 78 / 82 / 119
//   m  8,200 n 2,048 k 1,024: 28.5 / 25.5 / 186 / 193 / 228
//   m 16,384 n   512 k   512: 12.0 / 9.4 / 55 / 55 / 69         (128 large tiles)
//   m    320 n 2,048 k 2,048: 18.0 / 10.5 / 17.7 / 16.5 / 20.7
//   m    128 n 4,096 k 4,096: 27.8 / 16.9 / 21.5 / 24.5 / 30.9
//   m     64 n 4,096 k 4,096: 27.2 / 16.1 / 12.4 / 13.8 / 17.2
//   m     64 n 1,024 k 1,024: 12.0 / 7.3 / 5.6 / 4.5 / 3.9
//   m     10 n 2,048 k 2,048: 16.8 / 9.8 / 5.3 / 4.8 / 4.4
// So: staged tiles where the output has more than 2^18 values (a lone staged
// tile takes about 0.7 us for 256 values of k, the few-row kernel about 3 ns
// for a thousand outputs) and experts fill more than a quarter of a middle
// tile; large ones, one to a CU, or middle ones, two to a CU, by what a round
// of them is taken to cost, 8.2 + 2.4 and 3.9 + 1.8 us for each slice of k.
// That is within a tenth where a round or two of k 1,024 and 2,048 run, a
// third too little at k 256 and an eighth to a quarter too much at 16 slices
// and many rounds, on both sides alike: the faster one is chosen in every line
// above.  Else as many row tiles as leave a workgroup to every CU.
//
// What no staged tile takes goes to the few-row kernel at any size: k up to 128
// (16,384 x 4,096: 239 us, where k 256 takes 48; 4,096 x 1,024: 18.4 and 7.6)
// and gathered rows out of more than 4 GiB of codes (16,384 x 4,096 x 4,096:
// 2,233 us, 176 out of less).
int shape_for(const ProductArgs &a) {
    // The staged kernels address a matrix with 32 bits from a tile's first row
    // (from the first of all where rows are gathered) and read whole slices.
    const size_t code_row = a.kp / 2, reach = 0xffffffffu / code_row;
    const bool staged = a.kp >= kSlice && reach >= 256 && (!a.rows || a.a_rows <= reach) &&
                        tiles_of(a, kMiddle) < 2 * kGridRow;
    const size_t per = a.m / a.experts;
    if (staged && per > 32 && a.m * a.n > (1 << 18)) {
        // Half of the runs of rows end within a tile of their own, about.
        const size_t slices = (a.kp + kSlice - 1) / kSlice, ends = a.experts / 2;
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
void launch_product(const ProductArgs &a, int shape, unsigned tiles, hipStream_t q) {
    const dim3 few = tiles < kGridRow ? dim3(tiles)
                                      : dim3(kGridRow, (tiles + kGridRow - 1) / kGridRow);
    with_act(a.act, [&](auto act) {
        constexpr int ACT = decltype(act)::value;
        switch (shape) {
            case kFew1: few_kernel<T, ACT, 1><<<few, 64 * kFewWaves, 0, q>>>(a); break;
            case kFew2: few_kernel<T, ACT, 2><<<few, 64 * kFewWaves, 0, q>>>(a); break;
            case kFew4: few_kernel<T, ACT, 4><<<few, 64 * kFewWaves, 0, q>>>(a); break;
            case kMiddle: tile_kernel<T, ACT, 2, 2, 4, 4><<<tiles, 256, 0, q>>>(a); break;
            default: tile_kernel<T, ACT, 2, 4, 8, 4><<<tiles, 512, 0, q>>>(a); break;
        }
    });
}

unsigned grid_for(size_t items) {
    const size_t want = (items + kQuantThreads - 1) / kQuantThreads;
    return (unsigned)(want < kMaxGrid ? want : kMaxGrid);
}

}  // namespace

extern "C" size_t tb_hip_mx4_padded(size_t k) { return padded(k); }

extern "C" int tb_hip_mx4_quantise_device(const void *x, size_t row_stride, void *codes,
                                          void *scales, size_t rows, size_t k, int dtype,
                                          void *stream) {
    if (!x || !codes || !scales || !rows || rows > kMaxCount || !k || k > kMaxCount ||
        !known_type(dtype) || !multiple_of(codes, 16) || !multiple_of(scales, 4) ||
        !multiple_of(x, type_size(dtype)) || row_stride % type_size(dtype))
        return 0;
    QuantArgs a = {};
    a.x = static_cast<const char *>(x);
    a.stride = row_stride;
    a.codes = static_cast<unsigned *>(codes);
    a.scales = static_cast<unsigned char *>(scales);
    a.per = (unsigned)(padded(k) / 8);
    a.items = rows * a.per;
    a.k = (unsigned)k;
    a.vector = multiple_of(x, 16) && row_stride % 16 == 0;
    hipStream_t q = reinterpret_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    const unsigned grid = grid_for(a.items);
    if (dtype == TB_HIP_F32)
        quantise_kernel<float><<<grid, kQuantThreads, 0, q>>>(a);
    else if (dtype == TB_HIP_BF16)
        quantise_kernel<__bf16><<<grid, kQuantThreads, 0, q>>>(a);
    else
        quantise_kernel<_Float16><<<grid, kQuantThreads, 0, q>>>(a);
    return hipGetLastError() == hipSuccess;
}

extern "C" int tb_hip_mx4_values_device(const void *codes, const void *scales, void *values,
                                        size_t rows, size_t k, int dtype, void *stream) {
    if (!codes || !scales || !values || !rows || rows > kMaxCount || !k || k > kMaxCount ||
        !known_type(dtype) || !multiple_of(codes, 16) || !multiple_of(scales, 4) ||
        !multiple_of(values, type_size(dtype)))
        return 0;
    ValueArgs a = {};
    a.codes = static_cast<const unsigned *>(codes);
    a.scales = static_cast<const unsigned char *>(scales);
    a.out = static_cast<char *>(values);
    a.per = (unsigned)(padded(k) / 8);
    a.items = rows * a.per;
    a.k = (unsigned)k;
    a.vector = multiple_of(values, 16) && k * type_size(dtype) % 16 == 0;
    hipStream_t q = reinterpret_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    const unsigned grid = grid_for(a.items);
    if (dtype == TB_HIP_F32)
        values_kernel<float><<<grid, kQuantThreads, 0, q>>>(a);
    else if (dtype == TB_HIP_BF16)
        values_kernel<__bf16><<<grid, kQuantThreads, 0, q>>>(a);
    else
        values_kernel<_Float16><<<grid, kQuantThreads, 0, q>>>(a);
    return hipGetLastError() == hipSuccess;
}

extern "C" int tb_hip_mx4_product_device(const void *a_codes, const void *a_scales,
                                         size_t a_rows, const int *rows, const void *w_codes,
                                         const void *w_scales, const int *offsets,
                                         const float *bias, const float *row_scale, void *out,
                                         size_t m, size_t n, size_t k, int experts, int act,
                                         int dtype, void *stream) {
    if (!a_codes || !a_scales || !w_codes || !w_scales || !out || !a_rows ||
        a_rows > kMaxCount || !m || m > kMaxCount || !n || n > kMaxCount || !k ||
        k > kMaxCount || experts < 1 || experts > TB_HIP_ROUTE_MAX_EXPERTS ||
        (experts > 1 && !offsets) || n > kMaxCount / experts || m > kMaxOutputs / n ||
        (!rows && m != a_rows) ||
        !known_act(act) || !known_type(dtype) || !multiple_of(a_codes, 16) ||
        !multiple_of(w_codes, 16) || !multiple_of(a_scales, 4) || !multiple_of(w_scales, 4) ||
        !words_ok(rows, offsets, bias, row_scale) || !multiple_of(out, type_size(dtype)))
        return 0;
    ProductArgs a = {};
    a.a_codes = static_cast<const unsigned char *>(a_codes);
    a.a_scales = static_cast<const unsigned char *>(a_scales);
    a.w_codes = static_cast<const unsigned char *>(w_codes);
    a.w_scales = static_cast<const unsigned char *>(w_scales);
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
    a.act = act;
    a.vector = multiple_of(out, 16) && n * type_size(dtype) % 16 == 0;
    hipStream_t q = reinterpret_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    const int shape = shape_for(a);
    // Below 2^31: 2^30 for 2^38 values in tiles of 16 x 16, and the runs' ends.
    const size_t tiles = tiles_of(a, shape);
    if (dtype == TB_HIP_F32)
        launch_product<float>(a, shape, (unsigned)tiles, q);
    else if (dtype == TB_HIP_BF16)
        launch_product<__bf16>(a, shape, (unsigned)tiles, q);
    else
        launch_product<_Float16>(a, shape, (unsigned)tiles, q);
    return hipGetLastError() == hipSuccess;
}
