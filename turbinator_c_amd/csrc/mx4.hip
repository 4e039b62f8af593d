// Microscaled 4-bit floating point (hip_layers.h): quantisation, the values it
// stands for, and products on the scaled matrix instructions.  The reference's
// actor multiplies in fp32 through a library; acting reads far more weights
// than it multiplies, so a quarter of bf16's bytes is what this form is for.
//
//   scale  2^(s - 127), s = max(exponent bits of the largest magnitude - 2, 0)
//   code   value / scale (exact: a power of two) rounded to 0, 0.5, 1, 1.5, 2,
//          3, 4, 6, ties to even, by v_cvt_scalef32_pk_fp4_f32
//   out    = act(sum_k a_k w_k + bias) row_scale, summed in fp32 by
//          v_mfma_scale_f32_16x16x128_f8f6f4: lane l holds row l % 16, values
//          32 (l / 16) .. + 31 of a step of 128, one scale block, in 16 bytes
#include "layer_math.h"

namespace {

using namespace layer;

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr size_t kMaxCount = 0x7fffffffu;
constexpr size_t kMaxGrid = 1 << 20;
constexpr int kBlock = 32, kPad = 128;

__host__ __device__ inline size_t padded(size_t k) { return (k + kPad - 1) / kPad * kPad; }

// --------------------------------------------------------------------------
// Quantisation: four lanes to a block of 32, eight values each.

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

// Rows r0 .. r1-1 of the output, one tile of one expert's (expert = experts:
// of none's, which come out as 0).
struct RowTile {
    int expert;
    size_t r0, r1;
};

__device__ __forceinline__ size_t bound_of(const ProductArgs &a, int x) {
    if (!a.offsets) return x <= 0 ? 0 : a.m;
    const int v = a.offsets[x];
    return v < 0 ? 0 : (size_t)v < a.m ? (size_t)v : a.m;
}

// The rows fall into runs: before the first expert, each expert's, behind the
// last.  The wave counts the runs' tiles 64 runs at a time until it reaches
// `tile`; false if there are fewer.
__device__ __forceinline__ bool find_rows(const ProductArgs &a, size_t tile, int height,
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
        unsigned sum = tiles;
        for (int off = 1; off < 64; off *= 2) {
            const unsigned o = __shfl_up(sum, off);
            if (lane >= off) sum += o;
        }
        const unsigned long long reach = __ballot(tile < sum);
        if (reach) {
            const int at = __ffsll(reach) - 1;
            const unsigned before = __shfl(sum - tiles, at);
            const int expert = base + at - 1;
            lo = __shfl((unsigned long long)lo, at);
            hi = __shfl((unsigned long long)hi, at);
            t.expert = expert < 0 ? a.experts : expert;
            t.r0 = lo + (tile - before) * height;
            t.r1 = t.r0 + height < hi ? t.r0 + height : hi;
            return true;
        }
        tile -= __shfl(sum, 63);
    }
    return false;
}

__device__ __forceinline__ f32x4 step16(i32x4 w, int ws, i32x4 x, int xs, f32x4 c) {
    const i32x8 A = {w[0], w[1], w[2], w[3], 0, 0, 0, 0}, B = {x[0], x[1], x[2], x[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, c, 4, 4, 0, ws, 0, xs);
}

// Four consecutive columns n0 .. of row r: bias, activation, row scale.
template <class T>
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
            v[i] = act_of<kFine<T>>(z, a.act) * scale;
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

// Tiles of 64 columns and 64 rows, 32 by 32 a wave, operands straight from
// memory in the instruction's layout.  The weights are the first operand, so
// a lane ends with four consecutive columns of one row.
constexpr int kTile = 64;

template <class T>
__global__ __launch_bounds__(256) void product_kernel(ProductArgs a) {
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63, low = lane & 15, part = lane >> 4;
    const size_t columns = (a.n + kTile - 1) / kTile;
    const size_t tile = blockIdx.x / columns;
    RowTile rt;
    if (!find_rows(a, tile, kTile, rt)) return;
    const size_t n0 = (blockIdx.x - tile * columns) * kTile + (wave & 1) * 32;
    const size_t m0 = rt.r0 + (wave >> 1) * 32;
    const size_t codes = a.kp / 2, scales = a.kp / kBlock;
    f32x4 acc[2][2] = {};
    const unsigned char *wc[2], *ws[2], *xc[2], *xs[2];
    bool real[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        size_t r = n0 + i * 16 + low;
        r = (r < a.n ? r : a.n - 1) + (rt.expert < a.experts ? rt.expert * a.n : 0);
        wc[i] = a.w_codes + r * codes + part * 16;
        ws[i] = a.w_scales + r * scales + part;
        size_t m = m0 + i * 16 + low;
        m = m < rt.r1 ? m : rt.r1 - 1;
        const long long row = a.rows ? a.rows[m] : (long long)m;
        real[i] = rt.expert < a.experts && row >= 0 && (size_t)row < a.a_rows;
        xc[i] = a.a_codes + (real[i] ? row : 0) * codes + part * 16;
        xs[i] = a.a_scales + (real[i] ? row : 0) * scales + part;
    }
    if (rt.expert < a.experts)
        for (size_t k = 0; k < a.kp; k += kPad) {
            i32x4 w[2], x[2];
            int sw[2], sx[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                w[i] = *reinterpret_cast<const i32x4 *>(wc[i] + k / 2);
                x[i] = *reinterpret_cast<const i32x4 *>(xc[i] + k / 2);
                sw[i] = ws[i][k / kBlock];
                sx[i] = xs[i][k / kBlock];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    acc[i][j] = step16(w[i], sw[i], x[j], sx[j], acc[i][j]);
        }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const size_t r = m0 + j * 16 + low;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const size_t c = n0 + i * 16 + part * 4;
            if (r < rt.r1 && c < a.n) store4<T>(a, rt.expert, real[j], r, c, acc[i][j]);
        }
    }
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
        (experts > 1 && !offsets) || n > kMaxCount / experts || (!rows && m != a_rows) ||
        !known_act(act) || !known_type(dtype) || !multiple_of(a_codes, 16) ||
        !multiple_of(w_codes, 16) || !multiple_of(a_scales, 4) || !multiple_of(w_scales, 4) ||
        !multiple_of(out, type_size(dtype)))
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
    const size_t four = 4 * type_size(dtype);
    a.vector = multiple_of(out, four) && n * type_size(dtype) % four == 0;
    const size_t tiles = ((m + kTile - 1) / kTile + (offsets ? experts + 2 : 0)) *
                         ((n + kTile - 1) / kTile);
    if (tiles > 0x7fffffffu) return 0;
    hipStream_t q = reinterpret_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    if (dtype == TB_HIP_F32)
        product_kernel<float><<<(unsigned)tiles, 256, 0, q>>>(a);
    else if (dtype == TB_HIP_BF16)
        product_kernel<__bf16><<<(unsigned)tiles, 256, 0, q>>>(a);
    else
        product_kernel<_Float16><<<(unsigned)tiles, 256, 0, q>>>(a);
    return hipGetLastError() == hipSuccess;
}
