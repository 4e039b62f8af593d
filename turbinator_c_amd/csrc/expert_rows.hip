// Tokens to their experts' rows and back (hip_layers.h), with the gradients of
// both.  Choice (t, j) of token t has row p = positions[t, j] and weight w:
//
//   rows           rows[p] = w x[t]                 the rest of the rows 0
//   its gradient   dx[t] = sum_j w drows[p]         dw = <x[t], drows[p]>
//   sum            out[t] = residual[t] + sum_j w rows[p]
//   its gradient   drows[p] = w dout[t]             dw = <rows[p], dout[t]>
//
// All four go over the tokens: a token's vector is read once and its choices'
// rows are read or written once, whole runs of a row at a time, so that memory
// sees each byte once and nothing is added up by more than one thread.  Sums
// are held in 32 bits, in the order of the choices, and rounded once.
//
// Bound by memory: counters show at most 3% more traffic than the inputs and
// outputs (9% where rows are no whole lines).  bf16: 65,536 tokens x 2,048 to four experts 235 us (5.7 TB/s),
// summed back on a residual 300 (5.4); 40,960 x 1,024 to two, the sum's gradient
// 65 (6.5, the last cache helps); to eight, the rows' gradient 143 (5.9) and the
// sum's 260 (5.5).  fp32: 20,483 x 1,001 to three, the rows' gradient 67 (6.2).
// One token, eight rows of 4,096: 4.2 us, a launch and two loads in turn.
#include "layer_math.h"

namespace {

using namespace layer;

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr size_t kMaxCount = 0x7fffffffu, kMaxGrid = 1 << 20;

struct TokenArgs {
    const char *token_in;  // x, dout or the residual (may be NULL there)
    const char *rows_in;
    const int *positions, *end;  // end: one behind the last expert's rows
    const float *weights;
    char *token_out, *rows_out;
    float *dweights;
    size_t token_stride, row_stride, tokens, choices;
    unsigned k, width, vectors, pieces, lanes;
};

// kDot: the weights' gradient alone.
enum Kind { kRows, kRowsBack, kSum, kSumBack, kDot };
constexpr bool has_dots(int kind) { return kind >= kRowsBack && kind != kSum; }
// Choices taken at a time: as many as there are, up to a power of two.  What is
// left over costs instructions and registers: 65,536 tokens x 2,048 bf16, four
// each, summed in 300 us, and in 332 with room for eight.
constexpr int kFew = 2, kSome = 4, kMost = 8;

// A choice's row, -1 for none.  `end` is one behind the last expert's rows where
// the entry has offsets, else of all rows: positions from the former on are the
// caller's to set to -1, for the gradients' sake.
__device__ __forceinline__ long long row_of(const TokenArgs &a, size_t choice, size_t end) {
    const int p = a.positions[choice];
    return p >= 0 && (size_t)p < end ? p : -1;
}

// A token, or one of the pieces of a wide one, belongs to LANES lanes (0:
// a.lanes of them, a power of two below 64), each with a vector of B bytes at a
// time; the last vector of a row ends with the row and repeats some of the one
// before.  Without dot products a lane has one vector of an item.  Choices are
// taken K at a time, whose loads are all on their way at once.  STREAM: rows are
// read past the caches, what the token has is not.
template <class T, int B, int K, int KIND, int LANES, bool STREAM>
__global__ __launch_bounds__(kThreads) void token_kernel(TokenArgs a) {
    typedef Vec<T, B> X;
    typedef typename X::raw raw;
    constexpr bool kReadsToken = KIND != kSum, kReadsRows = KIND != kRows;
    constexpr bool kWritesRows = KIND == kRows || KIND == kSumBack;
    constexpr bool kAdds = KIND == kSum || KIND == kRowsBack, kDots = has_dots(KIND);
    const unsigned lanes = LANES ? LANES : a.lanes, lane = threadIdx.x & (lanes - 1);
    const unsigned k = a.k, groups = kThreads / lanes;
    size_t end = a.choices;
    if (kWritesRows) {
        const int e = *a.end;
        end = e < 0 ? 0 : (size_t)e < end ? (size_t)e : end;
    }
    const size_t items = a.tokens * a.pieces, row_bytes = (size_t)a.width * sizeof(T);
    unsigned group = threadIdx.x / lanes;
    if (LANES >= 64) group = __builtin_amdgcn_readfirstlane(group);
    for (size_t item = (size_t)blockIdx.x * groups + group; item < items;
         item += (size_t)gridDim.x * groups) {
        const size_t t = a.pieces > 1 ? item / a.pieces : item;
        const unsigned v0 = (unsigned)(item - t * a.pieces) * lanes + lane;
        // The vector's first element, and how many of its own the vector before has.
        auto start = [&](unsigned v) {
            return (v + 1) * X::n <= a.width ? v * X::n : a.width - X::n;
        };
        float sum[X::n] = {};
        for (unsigned j0 = 0; j0 < k; j0 += K) {
            const size_t c = t * k + j0;
            long long at[K];
            float w[K], dot[K];
#pragma unroll
            for (int j = 0; j < K; ++j) {
                dot[j] = 0.0f;
                w[j] = 1.0f;
                at[j] = -1;
                if (j0 + j < k) {
                    at[j] = row_of(a, c + j, end);
                    if (a.weights) w[j] = a.weights[c + j];
                }
            }
            for (unsigned v = v0; v < a.vectors; v += kDots ? lanes : a.vectors) {
                const unsigned e = start(v), again = v * X::n - e;
                raw token = {}, rows[K];
                float x[X::n];
                if (kReadsToken) token = load_loose<T, B>(a.token_in + t * a.token_stride, e);
                X::unpack(token, x);
                if (kReadsRows)
#pragma unroll
                    for (int j = 0; j < K; ++j) {
                        const char *row = a.rows_in + at[j] * a.row_stride;
                        if (at[j] >= 0)
                            rows[j] = STREAM ? stream_in<T, B>(row, e) : load_loose<T, B>(row, e);
                    }
                if (KIND == kRowsBack)
#pragma unroll
                    for (int i = 0; i < X::n; ++i) sum[i] = 0.0f;
#pragma unroll
                for (int j = 0; j < K; ++j) {
                    if (kWritesRows && j0 + j < k && c + j >= end)
                        store_loose<T, B>(a.rows_out + (c + j) * row_bytes, e, raw{});
                    if (at[j] < 0) continue;
                    if (kReadsRows) {
                        float y[X::n];
                        X::unpack(rows[j], y);
#pragma unroll
                        for (int i = 0; i < X::n; ++i) {
                            if (kAdds) sum[i] = fmaf(w[j], y[i], sum[i]);
                            if (kDots && i >= again) dot[j] = fmaf(x[i], y[i], dot[j]);
                        }
                    }
                    if (kWritesRows) {
                        raw out = token;
                        if (a.weights) {
                            float y[X::n];
#pragma unroll
                            for (int i = 0; i < X::n; ++i) y[i] = w[j] * x[i];
                            out = X::pack(y);
                        }
                        stream_out<T, B>(a.rows_out + at[j] * row_bytes, e, out);
                    }
                }
                if (KIND == kRowsBack)
                    stream_out<T, B>(a.token_out + t * row_bytes, e, X::pack(sum));
            }
            if (kDots) {
                __shared__ float part[kWaves][K];
#pragma unroll
                for (int j = 0; j < K; ++j) {
                    for (unsigned off = 1; off < lanes && off < 64; off *= 2)
                        dot[j] += __shfl_xor(dot[j], off);
                    if (LANES > 64) {
                        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6][j] = dot[j];
                    } else if (j0 + j < k && lane == (j & (lanes - 1))) {
                        a.dweights[c + j] = dot[j];
                    }
                }
                if (LANES > 64) {
                    __syncthreads();
                    if (threadIdx.x < K && j0 + threadIdx.x < k) {
                        float all = 0.0f;
                        for (int i = 0; i < kWaves; ++i) all += part[i][threadIdx.x];
                        a.dweights[c + threadIdx.x] = all;
                    }
                    __syncthreads();
                }
            }
        }
        if (KIND == kSum && v0 < a.vectors) {
            const unsigned e = start(v0);
            if (a.token_in) {
                float x[X::n];
                X::unpack(load_loose<T, B>(a.token_in + t * a.token_stride, e), x);
#pragma unroll
                for (int i = 0; i < X::n; ++i) sum[i] += x[i];
            }
            stream_out<T, B>(a.token_out + t * row_bytes, e, X::pack(sum));
        }
    }
}

// --------------------------------------------------------------------------

template <class T, int B, int K, int KIND>
void launch_lanes(TokenArgs &a, hipStream_t q) {
    a.vectors = (unsigned)(((size_t)a.width * sizeof(T) + B - 1) / B);
    a.pieces = has_dots(KIND) ? 1 : (a.vectors + 63) / 64;
    a.lanes = 1;
    while (a.lanes < a.vectors && a.lanes < 64) a.lanes *= 2;
    const bool block = has_dots(KIND) && a.vectors > 64 && a.tokens < 4096;
    if (block) a.lanes = kThreads;
    const size_t items = a.tokens * a.pieces, per = kThreads / a.lanes;
    const size_t want = (items + per - 1) / per;
    const unsigned grid = (unsigned)(want < kMaxGrid ? want : kMaxGrid);
    constexpr bool kWide = B == 16, kStreams = kWide && KIND != kRows;
    const bool stream = kStreams && a.choices * a.width * sizeof(T) > kStreamBytes;
    if constexpr (kWide && has_dots(KIND))
        if (block) {
            token_kernel<T, B, K, KIND, kThreads, false><<<grid, kThreads, 0, q>>>(a);
            return;
        }
    if constexpr (kWide)
        if (a.lanes == 64) {
            if (stream)
                token_kernel<T, B, K, KIND, 64, kStreams><<<grid, kThreads, 0, q>>>(a);
            else
                token_kernel<T, B, K, KIND, 64, false><<<grid, kThreads, 0, q>>>(a);
            return;
        }
    if (stream)
        token_kernel<T, B, K, KIND, 0, kStreams><<<grid, kThreads, 0, q>>>(a);
    else
        token_kernel<T, B, K, KIND, 0, false><<<grid, kThreads, 0, q>>>(a);
}

template <class T, int KIND>
void launch_type(TokenArgs &a, hipStream_t q) {
    // Rows shorter than a vector go by single elements.
    if (a.width * sizeof(T) < 16)
        launch_lanes<T, sizeof(T), kMost, KIND>(a, q);
    else if (a.k <= kFew)
        launch_lanes<T, 16, kFew, KIND>(a, q);
    else if (a.k <= kSome)
        launch_lanes<T, 16, kSome, KIND>(a, q);
    else
        launch_lanes<T, 16, kMost, KIND>(a, q);
}

template <int KIND>
int launch(TokenArgs a, int dtype, void *stream) {
    hipStream_t q = reinterpret_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    if (dtype == TB_HIP_F32)
        launch_type<float, KIND>(a, q);
    else if (dtype == TB_HIP_BF16)
        launch_type<__bf16, KIND>(a, q);
    else
        launch_type<_Float16, KIND>(a, q);
    return hipGetLastError() == hipSuccess;
}

bool sizes_ok(size_t tokens, int k, size_t width, int dtype) {
    return tokens && k >= 1 && k <= TB_HIP_ROUTE_MAX_K && tokens <= kMaxCount / k && width &&
           width <= kMaxCount && known_type(dtype);
}

// An input of strided rows, an output of dense ones.
bool rows_ok(const void *p, size_t stride, int dtype) {
    return p && multiple_of(p, type_size(dtype)) && stride % type_size(dtype) == 0;
}

TokenArgs args_of(const int *positions, const float *weights, size_t tokens, int k, size_t width) {
    TokenArgs a = {};
    a.positions = positions;
    a.weights = weights;
    a.tokens = tokens;
    a.choices = tokens * k;
    a.k = k;
    a.width = (unsigned)width;
    return a;
}

TokenArgs without_token(TokenArgs a) {
    a.token_in = nullptr;
    return a;
}

}  // namespace

extern "C" int tb_hip_expert_rows_device(const void *x, size_t row_stride, const int *offsets,
                                         const int *positions, const float *weights, void *rows,
                                         size_t tokens, int n_experts, int k, size_t width,
                                         int dtype, void *stream) {
    if (!sizes_ok(tokens, k, width, dtype) || n_experts < 1 ||
        n_experts > TB_HIP_ROUTE_MAX_EXPERTS || !offsets || !positions ||
        !words_ok(offsets, positions, weights) || !rows_ok(x, row_stride, dtype) ||
        !rows_ok(rows, 0, dtype))
        return 0;
    TokenArgs a = args_of(positions, weights, tokens, k, width);
    a.token_in = static_cast<const char *>(x);
    a.token_stride = row_stride;
    a.end = offsets + n_experts;
    a.rows_out = static_cast<char *>(rows);
    return launch<kRows>(a, dtype, stream);
}

extern "C" int tb_hip_expert_rows_backward_device(const void *drows, size_t drow_stride,
                                                  const void *x, size_t row_stride,
                                                  const int *positions, const float *weights,
                                                  void *dx, float *dweights, size_t tokens, int k,
                                                  size_t width, int dtype, void *stream) {
    if (!sizes_ok(tokens, k, width, dtype) || !positions ||
        !words_ok(positions, weights, dweights) || !rows_ok(drows, drow_stride, dtype) ||
        !rows_ok(dx, 0, dtype) || (dweights && !rows_ok(x, row_stride, dtype)))
        return 0;
    TokenArgs a = args_of(positions, weights, tokens, k, width);
    a.rows_in = static_cast<const char *>(drows);
    a.row_stride = drow_stride;
    a.token_out = static_cast<char *>(dx);
    if (!dweights) return launch<kSum>(a, dtype, stream);
    a.token_in = static_cast<const char *>(x);
    a.token_stride = row_stride;
    a.dweights = dweights;
    if (k <= kMost) return launch<kRowsBack>(a, dtype, stream);
    // The sums hold for all choices, the dot products for those of one turn.
    return launch<kDot>(a, dtype, stream) && launch<kSum>(without_token(a), dtype, stream);
}

extern "C" int tb_hip_expert_sum_device(const void *rows, size_t row_stride, const int *positions,
                                        const float *weights, const void *residual,
                                        size_t residual_stride, void *out, size_t tokens, int k,
                                        size_t width, int dtype, void *stream) {
    if (!sizes_ok(tokens, k, width, dtype) || !positions || !words_ok(positions, weights) ||
        !rows_ok(rows, row_stride, dtype) || !rows_ok(out, 0, dtype) ||
        (residual && !rows_ok(residual, residual_stride, dtype)))
        return 0;
    TokenArgs a = args_of(positions, weights, tokens, k, width);
    a.rows_in = static_cast<const char *>(rows);
    a.row_stride = row_stride;
    a.token_in = static_cast<const char *>(residual);
    a.token_stride = residual_stride;
    a.token_out = static_cast<char *>(out);
    return launch<kSum>(a, dtype, stream);
}

extern "C" int tb_hip_expert_sum_backward_device(const void *dout, size_t dout_stride,
                                                 const void *rows, size_t row_stride,
                                                 const int *offsets, const int *positions,
                                                 const float *weights, void *drows,
                                                 float *dweights, size_t tokens, int n_experts,
                                                 int k, size_t width, int dtype, void *stream) {
    if (!sizes_ok(tokens, k, width, dtype) || n_experts < 1 ||
        n_experts > TB_HIP_ROUTE_MAX_EXPERTS || !offsets || !positions ||
        !words_ok(offsets, positions, weights, dweights) || !rows_ok(dout, dout_stride, dtype) ||
        !rows_ok(drows, 0, dtype) || (dweights && !rows_ok(rows, row_stride, dtype)))
        return 0;
    TokenArgs a = args_of(positions, weights, tokens, k, width);
    a.token_in = static_cast<const char *>(dout);
    a.token_stride = dout_stride;
    a.end = offsets + n_experts;
    a.rows_out = static_cast<char *>(drows);
    if (!dweights) return launch<kRows>(a, dtype, stream);
    a.rows_in = static_cast<const char *>(rows);
    a.row_stride = row_stride;
    a.dweights = dweights;
    return launch<kSumBack>(a, dtype, stream);
}
