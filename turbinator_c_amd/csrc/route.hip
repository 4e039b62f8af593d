// Routing of tokens to experts, its gradient, and the order of the choices by
// expert (hip_layers.h).  The reference's actor mixes the two best experts of
// every token densely (moe_mix, src/network/network_gpu.cu:373-390); here the
// choice leaves as indices and weights, so each expert's product runs on its
// own tokens only.
//
//   s = softmax(l) or sigmoid(l);  key = l, or s + b with a bias
//   w_i = scale s_i, renormalised scale s_i / S, S the sum over the chosen
// Gradient at the chosen i, w' = s / S, g = scale dw:
//   renormalised      ds_i = (g_i - sum_j g_j w'_j) / S
//   softmax           dl = s (ds - sum_j ds_j s_j); renormalised the second
//                     sum is 0 and s / S = w', so dl_i = w'_i (g_i - sum g w')
//                     and 0 elsewhere, without S
//   sigmoid           dl = ds s (1 - s)
//
// A token belongs to W lanes of one wave, W a power of two; a lane holds Q
// consecutive experts in registers, so the first of equal keys is the lowest
// lane's first.  Rows of the best keys come from k rounds of a maximum over
// the lanes; all else is one pass over the logits.
#include "layer_math.h"

namespace {

using namespace layer;

constexpr int kThreads = 256;
constexpr size_t kMaxChoices = 0x7fffffffu;

struct RouteArgs {
    const char *logits;
    size_t stride;
    const float *bias;
    const unsigned char *valid;
    const int *chosen;
    const float *dweights;
    int *experts;
    float *weights;
    char *dlogits;
    size_t tokens;
    int n, k, groups, kept, lanes, score, renorm;
    float scale;
};

// Floats as unsigned integers of the same order: -0 as +0, NaN above all, and
// 0 for -inf, which is never chosen.
__device__ __forceinline__ unsigned key_of(float x) {
    if (x != x) return 0xffffffffu;
    const unsigned u = __builtin_bit_cast(unsigned, x + 0.0f);
    if (u == 0xff800000u) return 0u;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float lanes_max(float v, int lanes) {
    for (int off = 1; off < lanes; off *= 2) v = fmaxf(v, __shfl_xor(v, off));
    return v;
}

__device__ __forceinline__ float lanes_sum(float v, int lanes) {
    for (int off = 1; off < lanes; off *= 2) v += __shfl_xor(v, off);
    return v;
}

__device__ __forceinline__ unsigned lanes_max_key(unsigned v, int lanes) {
    for (int off = 1; off < lanes; off *= 2) {
        const unsigned o = __shfl_xor(v, off);
        v = o > v ? o : v;
    }
    return v;
}

// LDS that only the calling wave uses: its accesses are in order.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <class T>
__device__ __forceinline__ float element(const char *row, int i) {
    return (float)reinterpret_cast<const T *>(row)[i];
}

template <class T, int Q>
__device__ __forceinline__ void load_row(const char *row, int e0, int n, float (&x)[Q]) {
#pragma unroll
    for (int j = 0; j < Q; ++j) x[j] = e0 + j < n ? element<T>(row, e0 + j) : -__builtin_inff();
}

// Whether v is among the kept highest of all[count], ties to the lower index.
__device__ __forceinline__ bool in_best(const unsigned *all, int count, int i, int kept) {
    const unsigned v = all[i];
    int before = 0;
    for (int j = 0; j < count; ++j) before += all[j] > v || (all[j] == v && j < i);
    return before < kept;
}

template <class T, int Q>
__global__ __launch_bounds__(kThreads) void route_kernel(RouteArgs a) {
    // Per token: with groups the keys and the groups' standings, then the
    // picks (a token's span of 8 or more experts or its 32 picks at most).
    __shared__ unsigned keys[kThreads * Q], stands[kThreads * Q];
    __shared__ int pick_at[kThreads * 8];
    __shared__ float pick_s[kThreads * 8];
    const int W = a.lanes, per_block = kThreads / W, t = threadIdx.x;
    const int lane = t & (W - 1), slot = t / W;
    const int e0 = lane * Q, span = W * Q;
    unsigned *my_keys = keys + slot * span, *my_stands = stands + slot * span;
    const int picks = span < TB_HIP_ROUTE_MAX_K ? span : TB_HIP_ROUTE_MAX_K;
    int *at = pick_at + slot * picks;
    float *ps = pick_s + slot * picks;
    const unsigned long long mine = (W == 64 ? ~0ull : ((1ull << W) - 1)) << ((t & 63) - lane);
    for (size_t base = (size_t)blockIdx.x * per_block; base < a.tokens;
         base += (size_t)gridDim.x * per_block) {
        const size_t token = base + slot;
        const bool live = token < a.tokens && (!a.valid || a.valid[token]);
        float x[Q], s[Q];
        unsigned key[Q];
        if (live)
            load_row<T, Q>(a.logits + token * a.stride, e0, a.n, x);
        else
#pragma unroll
            for (int j = 0; j < Q; ++j) x[j] = -__builtin_inff();
        float top = -__builtin_inff(), sum = 0.0f;
        if (a.score == TB_HIP_SCORE_SOFTMAX) {
#pragma unroll
            for (int j = 0; j < Q; ++j) top = fmaxf(top, x[j]);
            top = lanes_max(top, W);
#pragma unroll
            for (int j = 0; j < Q; ++j) {
                s[j] = e0 + j < a.n ? exp_of<true>(x[j] - top) : 0.0f;
                sum += s[j];
            }
            const float inverse = 1.0f / lanes_sum(sum, W);
#pragma unroll
            for (int j = 0; j < Q; ++j) s[j] *= inverse;
        } else {
#pragma unroll
            for (int j = 0; j < Q; ++j) s[j] = sigmoid_of<true>(x[j]);
        }
#pragma unroll
        for (int j = 0; j < Q; ++j) {
            key[j] = key_of(x[j]);
            if (a.bias && key[j]) key[j] = key_of(s[j] + a.bias[e0 + j]);
        }
        if (a.kept < a.groups) {
            const int per = a.n / a.groups;
#pragma unroll
            for (int j = 0; j < Q; ++j) my_keys[e0 + j] = key[j];
            wave_fence();
            for (int g = lane; g < a.groups; g += W) {
                unsigned best = 0, next = 0;
                for (int i = 0; i < per; ++i) {
                    const unsigned v = my_keys[g * per + i];
                    next = v > best ? best : v > next ? v : next;
                    best = v > best ? v : best;
                }
                if (a.bias && next) {
                    // Back to floats; NaN keys stay above all.
                    const unsigned b = best & 0x80000000u ? best & 0x7fffffffu : ~best;
                    const unsigned c = next & 0x80000000u ? next & 0x7fffffffu : ~next;
                    const float both =
                        __builtin_bit_cast(float, b) + __builtin_bit_cast(float, c);
                    best = best == 0xffffffffu ? best : key_of(both);
                }
                my_stands[g] = best;
            }
            wave_fence();
            int g = e0 / per, left = per - (e0 - g * per);
            bool keep = g < a.groups && in_best(my_stands, a.groups, g, a.kept);
#pragma unroll
            for (int j = 0; j < Q; ++j) {
                if (left == 0) {
                    ++g;
                    left = per;
                    keep = g < a.groups && in_best(my_stands, a.groups, g, a.kept);
                }
                if (!keep) key[j] = 0;
                --left;
            }
        }
        for (int i = 0; i < a.k; ++i) {
            unsigned best = 0;
#pragma unroll
            for (int j = 0; j < Q; ++j) best = key[j] > best ? key[j] : best;
            const unsigned most = lanes_max_key(best, W);
            const unsigned long long has = __ballot(best == most) & mine;
            if (lane == 0 && most == 0) {
                at[i] = -1;
                ps[i] = 0.0f;
            }
            if (most && (t & 63) == __ffsll(has) - 1) {
                bool found = false;
#pragma unroll
                for (int j = 0; j < Q; ++j)
                    if (!found && key[j] == most) {
                        found = true;
                        key[j] = 0;
                        at[i] = e0 + j;
                        // Renormalised softmax weights need no row sum: they
                        // are formed from the chosen logits, below.
                        ps[i] = a.score == TB_HIP_SCORE_SOFTMAX && a.renorm ? x[j] : s[j];
                    }
            }
        }
        wave_fence();
        if (token < a.tokens) {
            const bool from_logits = a.score == TB_HIP_SCORE_SOFTMAX && a.renorm;
            float total = 0.0f, most = -__builtin_inff();
            if (a.renorm) {
                if (from_logits)
                    for (int i = 0; i < a.k; ++i)
                        if (at[i] >= 0) most = fmaxf(most, ps[i]);
                for (int i = 0; i < a.k; ++i)
                    if (at[i] >= 0) total += from_logits ? exp_of<true>(ps[i] - most) : ps[i];
            }
            for (int i = lane; i < a.k; i += W) {
                float w = 0.0f;
                if (at[i] >= 0) {
                    w = from_logits ? exp_of<true>(ps[i] - most) : ps[i];
                    if (a.renorm) w = total == 0.0f ? 0.0f : w / total;
                }
                a.experts[token * a.k + i] = at[i];
                a.weights[token * a.k + i] = w * a.scale;
            }
        }
        wave_fence();
    }
}

template <class T, int Q>
__global__ __launch_bounds__(kThreads) void route_backward_kernel(RouteArgs a) {
    const int W = a.lanes, per_block = kThreads / W, t = threadIdx.x;
    const int lane = t & (W - 1), slot = t / W;
    const int e0 = lane * Q;
    const bool soft = a.score == TB_HIP_SCORE_SOFTMAX;
    for (size_t base = (size_t)blockIdx.x * per_block; base < a.tokens;
         base += (size_t)gridDim.x * per_block) {
        const size_t token = base + slot;
        const bool live = token < a.tokens;
        const char *row = a.logits + token * a.stride;
        const int *at = a.chosen + token * a.k;
        const float *dw = a.dweights + token * a.k;
        float d[Q];
#pragma unroll
        for (int j = 0; j < Q; ++j) d[j] = 0.0f;
        int used = 0;
        if (live)
            for (int i = 0; i < a.k; ++i) used += (unsigned)at[i] < (unsigned)a.n;
        if (a.renorm) {
            // w' of the chosen from their logits alone, as quotients: a single
            // choice has w' = 1 and no gradient, exactly.
            float most = -__builtin_inff(), total = 0.0f, dot = 0.0f;
            if (used) {
                if (soft)
                    for (int i = 0; i < a.k; ++i)
                        if ((unsigned)at[i] < (unsigned)a.n)
                            most = fmaxf(most, element<T>(row, at[i]));
                for (int i = 0; i < a.k; ++i)
                    if ((unsigned)at[i] < (unsigned)a.n) {
                        const float x = element<T>(row, at[i]);
                        total += soft ? exp_of<true>(x - most) : sigmoid_of<true>(x);
                    }
                // A sum of 0 gave weights of 0.
                if (total == 0.0f) used = 0;
            }
            if (used) {
                for (int i = 0; i < a.k; ++i)
                    if ((unsigned)at[i] < (unsigned)a.n) {
                        const float x = element<T>(row, at[i]);
                        const float s = soft ? exp_of<true>(x - most) : sigmoid_of<true>(x);
                        dot += s / total * (a.scale * dw[i]);
                    }
                for (int i = 0; i < a.k; ++i)
                    if (at[i] >= e0 && at[i] < e0 + Q && at[i] < a.n) {
                        const float x = element<T>(row, at[i]);
                        const float s = soft ? exp_of<true>(x - most) : sigmoid_of<true>(x);
                        // 1 - s as the sigmoid of -x, without cancelling.
                        const float rest = soft ? 1.0f : sigmoid_of<true>(-x);
                        const float v = s / total * rest * (a.scale * dw[i] - dot);
#pragma unroll
                        for (int j = 0; j < Q; ++j) d[j] += at[i] == e0 + j ? v : 0.0f;
                    }
            }
        } else {
            if (used)
                for (int i = 0; i < a.k; ++i)
#pragma unroll
                    for (int j = 0; j < Q; ++j)
                        d[j] += at[i] == e0 + j ? a.scale * dw[i] : 0.0f;
            float x[Q];
            if (used)
                load_row<T, Q>(row, e0, a.n, x);
            else
#pragma unroll
                for (int j = 0; j < Q; ++j) x[j] = 0.0f;
            if (soft) {
                float top = -__builtin_inff(), sum = 0.0f, dot = 0.0f;
#pragma unroll
                for (int j = 0; j < Q; ++j) top = fmaxf(top, x[j]);
                top = lanes_max(top, W);
#pragma unroll
                for (int j = 0; j < Q; ++j) {
                    x[j] = e0 + j < a.n ? exp_of<true>(x[j] - top) : 0.0f;
                    sum += x[j];
                }
                const float inverse = 1.0f / lanes_sum(sum, W);
#pragma unroll
                for (int j = 0; j < Q; ++j) {
                    x[j] *= inverse;
                    dot += d[j] * x[j];
                }
                dot = lanes_sum(dot, W);
#pragma unroll
                for (int j = 0; j < Q; ++j) d[j] = used ? x[j] * (d[j] - dot) : 0.0f;
            } else {
#pragma unroll
                for (int j = 0; j < Q; ++j)
                    if (d[j] != 0.0f) d[j] *= sigmoid_of<true>(x[j]) * sigmoid_of<true>(-x[j]);
            }
        }
        if (live) {
            T *out = reinterpret_cast<T *>(a.dlogits) + token * a.n;
#pragma unroll
            for (int j = 0; j < Q; ++j)
                if (e0 + j < a.n) out[e0 + j] = (T)d[j];
        }
    }
}

// --------------------------------------------------------------------------
// The order of the choices by expert: a stable counting sort.  The choices are
// cut into segments, one to a wave: (1) every segment's count of each expert,
// (2) for each expert the running sum over the segments, (3) the segments
// again, each choice to its expert's start plus its running sum plus its rank
// in the segment.  Choices outside the experts count as expert n.

constexpr int kOrderWaves = 4;
constexpr size_t kSegment = 512, kMaxSegments = 4096;

struct OrderArgs {
    const int *experts;
    const float *weights;
    int *offsets, *tokens, *positions;
    float *row_weights;
    int *counts;  // [n + 1][segments], then their running sums
    int *totals;  // [n + 1]
    size_t choices, segment;
    unsigned segments;
    int n, k;
};

__device__ __forceinline__ int expert_of(const OrderArgs &a, size_t c) {
    const int e = a.experts[c];
    return (unsigned)e < (unsigned)a.n ? e : a.n;
}

__global__ __launch_bounds__(kOrderWaves * 64) void order_count_kernel(OrderArgs a) {
    extern __shared__ int lds[];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int *count = lds + wave * (a.n + 1);
    const unsigned seg = blockIdx.x * kOrderWaves + wave;
    if (seg >= a.segments) return;
    for (int e = lane; e <= a.n; e += 64) count[e] = 0;
    wave_fence();
    const size_t c0 = seg * a.segment;
    const size_t c1 = c0 + a.segment < a.choices ? c0 + a.segment : a.choices;
    for (size_t c = c0 + lane; c < c1; c += 64) atomicAdd(&count[expert_of(a, c)], 1);
    wave_fence();
    for (int e = lane; e <= a.n; e += 64) a.counts[(size_t)e * a.segments + seg] = count[e];
}

// One workgroup per expert: counts to exclusive running sums.
__global__ __launch_bounds__(256) void order_sum_kernel(OrderArgs a) {
    __shared__ int wave_total[4];
    const int t = threadIdx.x, lane = t & 63;
    int *row = a.counts + (size_t)blockIdx.x * a.segments;
    int before = 0;
    for (unsigned s0 = 0; s0 < a.segments; s0 += 256) {
        const unsigned s = s0 + t;
        const int v = s < a.segments ? row[s] : 0;
        int sum = v;
        for (int off = 1; off < 64; off *= 2) {
            const int o = __shfl_up(sum, off);
            if (lane >= off) sum += o;
        }
        if (lane == 63) wave_total[t >> 6] = sum;
        __syncthreads();
        int below = 0, all = 0;
        for (int w = 0; w < 4; ++w) {
            below += w < (t >> 6) ? wave_total[w] : 0;
            all += wave_total[w];
        }
        if (s < a.segments) row[s] = before + below + sum - v;
        before += all;
        __syncthreads();
    }
    if (t == 0) a.totals[blockIdx.x] = before;
}

__global__ __launch_bounds__(kOrderWaves * 64) void order_place_kernel(OrderArgs a) {
    extern __shared__ int lds[];
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    int *start = lds, *next = lds + (a.n + 1) * (1 + wave);
    // Every expert's start: wave 0 runs along the totals.
    if (wave == 0) {
        int before = 0;
        for (int e0 = 0; e0 <= a.n; e0 += 64) {
            const int e = e0 + lane, v = e <= a.n ? a.totals[e] : 0;
            int sum = v;
            for (int off = 1; off < 64; off *= 2) {
                const int o = __shfl_up(sum, off);
                if (lane >= off) sum += o;
            }
            if (e <= a.n) {
                start[e] = before + sum - v;
                if (blockIdx.x == 0) a.offsets[e] = before + sum - v;
            }
            before += __shfl(sum, 63);
        }
    }
    __syncthreads();
    const unsigned seg = blockIdx.x * kOrderWaves + wave;
    if (seg >= a.segments) return;
    for (int e = lane; e <= a.n; e += 64)
        next[e] = start[e] + a.counts[(size_t)e * a.segments + seg];
    wave_fence();
    int bits = 1;
    while ((1 << bits) <= a.n) ++bits;
    const size_t c0 = seg * a.segment;
    const size_t c1 = c0 + a.segment < a.choices ? c0 + a.segment : a.choices;
    for (size_t i = c0; i < c1; i += 64) {
        const size_t c = i + lane;
        const bool live = c < c1;
        const int e = live ? expert_of(a, c) : 0;
        // The lanes with the same expert.
        unsigned long long same = __ballot(live);
        for (int b = 0; b < bits; ++b) {
            const unsigned long long set = __ballot((e >> b) & 1);
            same &= (e >> b) & 1 ? set : ~set;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        const int row = live ? next[e] + rank : 0;
        wave_fence();
        if (live && rank == 0) next[e] = row + __popcll(same);
        wave_fence();
        if (live) {
            const bool known = e < a.n;
            a.tokens[row] = known ? (int)(c / (unsigned)a.k) : -1;
            a.positions[c] = known ? row : -1;
            if (a.weights) a.row_weights[row] = known ? a.weights[c] : 0.0f;
        }
    }
}

// --------------------------------------------------------------------------

bool route_ok(const void *logits, size_t stride, size_t tokens, int n, int k, int score,
              int dtype) {
    if (!logits || !tokens || n < 1 || n > TB_HIP_ROUTE_MAX_EXPERTS || k < 1 || k > n ||
        k > TB_HIP_ROUTE_MAX_K || tokens > kMaxChoices / k || !known_type(dtype) ||
        (score != TB_HIP_SCORE_SOFTMAX && score != TB_HIP_SCORE_SIGMOID))
        return false;
    const size_t size = type_size(dtype);
    return multiple_of(logits, size) && stride % size == 0;
}

constexpr size_t kMaxGrid = 1 << 20;

int lanes_for(int n, int q) {
    int lanes = 1;
    while (lanes * q < n) lanes *= 2;
    return lanes;
}

unsigned grid_for(const RouteArgs &a) {
    const size_t per = kThreads / a.lanes, want = (a.tokens + per - 1) / per;
    return (unsigned)(want < kMaxGrid ? want : kMaxGrid);
}

// 8 experts a lane up to 512 experts, 16 above, where 64 lanes need them.
template <class T>
void launch_route(RouteArgs &a, hipStream_t q) {
    if (a.n <= 512) {
        a.lanes = lanes_for(a.n, 8);
        route_kernel<T, 8><<<grid_for(a), kThreads, 0, q>>>(a);
    } else {
        a.lanes = 64;
        route_kernel<T, 16><<<grid_for(a), kThreads, 0, q>>>(a);
    }
}

template <class T>
void launch_backward(RouteArgs &a, hipStream_t q) {
    if (a.n <= 512) {
        a.lanes = lanes_for(a.n, 8);
        route_backward_kernel<T, 8><<<grid_for(a), kThreads, 0, q>>>(a);
    } else {
        a.lanes = 64;
        route_backward_kernel<T, 16><<<grid_for(a), kThreads, 0, q>>>(a);
    }
}

struct OrderShape {
    size_t segment;
    unsigned segments;
};

OrderShape order_shape(size_t choices) {
    OrderShape s;
    s.segment = kSegment;
    const size_t least = (choices + kMaxSegments - 1) / kMaxSegments;
    if (least > s.segment) s.segment = (least + 63) / 64 * 64;
    s.segments = (unsigned)((choices + s.segment - 1) / s.segment);
    return s;
}

bool order_ok(size_t tokens, int n, int k) {
    return tokens && n >= 1 && n <= TB_HIP_ROUTE_MAX_EXPERTS && k >= 1 &&
           k <= TB_HIP_ROUTE_MAX_K && tokens <= kMaxChoices / k;
}

}  // namespace

extern "C" int tb_hip_route_device(const void *logits, size_t row_stride, const float *bias,
                                   const unsigned char *valid, int *experts, float *weights,
                                   size_t tokens, int n_experts, int k, int groups,
                                   int groups_kept, int score, int renormalise, float scale,
                                   int dtype, void *stream) {
    if (!route_ok(logits, row_stride, tokens, n_experts, k, score, dtype) || !experts ||
        !weights || groups < 1 || n_experts % groups || groups_kept < 1 ||
        groups_kept > groups || groups_kept * (n_experts / groups) < k)
        return 0;
    RouteArgs a = {};
    a.logits = static_cast<const char *>(logits);
    a.stride = row_stride;
    a.bias = bias;
    a.valid = valid;
    a.experts = experts;
    a.weights = weights;
    a.tokens = tokens;
    a.n = n_experts;
    a.k = k;
    a.groups = groups;
    a.kept = groups_kept;
    a.score = score;
    a.renorm = renormalise != 0;
    a.scale = scale;
    hipStream_t q = reinterpret_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    if (dtype == TB_HIP_F32)
        launch_route<float>(a, q);
    else if (dtype == TB_HIP_BF16)
        launch_route<__bf16>(a, q);
    else
        launch_route<_Float16>(a, q);
    return hipGetLastError() == hipSuccess;
}

extern "C" int tb_hip_route_backward_device(const void *logits, size_t row_stride,
                                            const int *experts, const float *dweights,
                                            void *dlogits, size_t tokens, int n_experts, int k,
                                            int score, int renormalise, float scale, int dtype,
                                            void *stream) {
    if (!route_ok(logits, row_stride, tokens, n_experts, k, score, dtype) || !experts ||
        !dweights || !dlogits || !multiple_of(dlogits, type_size(dtype)))
        return 0;
    RouteArgs a = {};
    a.logits = static_cast<const char *>(logits);
    a.stride = row_stride;
    a.chosen = experts;
    a.dweights = dweights;
    a.dlogits = static_cast<char *>(dlogits);
    a.tokens = tokens;
    a.n = n_experts;
    a.k = k;
    a.score = score;
    a.renorm = renormalise != 0;
    a.scale = scale;
    hipStream_t q = reinterpret_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    if (dtype == TB_HIP_F32)
        launch_backward<float>(a, q);
    else if (dtype == TB_HIP_BF16)
        launch_backward<__bf16>(a, q);
    else
        launch_backward<_Float16>(a, q);
    return hipGetLastError() == hipSuccess;
}

extern "C" size_t tb_hip_expert_order_workspace_bytes(size_t tokens, int n_experts, int k) {
    if (!order_ok(tokens, n_experts, k)) return 0;
    const OrderShape s = order_shape(tokens * k);
    const size_t ints = (size_t)(n_experts + 1) * (s.segments + 1);
    return (ints * sizeof(int) + 15) & ~size_t(15);
}

extern "C" int tb_hip_expert_order_device(const int *experts, const float *weights, int *offsets,
                                          int *tokens_out, int *positions, float *row_weights,
                                          void *workspace, size_t tokens, int n_experts, int k,
                                          void *stream) {
    if (!experts || !offsets || !tokens_out || !positions || !weights != !row_weights ||
        !workspace || !multiple_of(workspace, 16) || !order_ok(tokens, n_experts, k))
        return 0;
    const OrderShape s = order_shape(tokens * k);
    OrderArgs a = {};
    a.experts = experts;
    a.weights = weights;
    a.offsets = offsets;
    a.tokens = tokens_out;
    a.positions = positions;
    a.row_weights = row_weights;
    a.counts = static_cast<int *>(workspace);
    a.totals = a.counts + (size_t)(n_experts + 1) * s.segments;
    a.choices = tokens * k;
    a.segment = s.segment;
    a.segments = s.segments;
    a.n = n_experts;
    a.k = k;
    hipStream_t q = reinterpret_cast<hipStream_t>(stream);
    const unsigned blocks = (s.segments + kOrderWaves - 1) / kOrderWaves;
    const size_t row = (n_experts + 1) * sizeof(int);
    (void)hipGetLastError();
    order_count_kernel<<<blocks, kOrderWaves * 64, kOrderWaves * row, q>>>(a);
    order_sum_kernel<<<n_experts + 1, 256, 0, q>>>(a);
    order_place_kernel<<<blocks, kOrderWaves * 64, (1 + kOrderWaves) * row, q>>>(a);
    return hipGetLastError() == hipSuccess;
}
