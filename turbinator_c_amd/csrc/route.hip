// Routing of tokens to experts, its gradient, and the order of the choices by
// expert (hip_layers.h).  The choice leaves as indices and weights, so each
// expert's product runs on its own tokens only.
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
    int n, k, groups, kept, lanes, score, renorm, vector, vector_bias;
    int log_per;  // of a group's experts, -1 if they are no power of two
    float scale;
};

// Floats as integers of the same order: -0 as +0, NaN above all.  kNone and
// below, -inf and kGone, are never chosen.
constexpr int kNone = (int)0x807fffff, kGone = (int)0x80000000;

__device__ __forceinline__ int key_of(float x) {
    const int u = __builtin_bit_cast(int, x + 0.0f);
    return x != x ? 0x7fffffff : u ^ ((u >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float float_of(int key) {
    return __builtin_bit_cast(float, key ^ ((key >> 31) & 0x7fffffff));
}

// f over the values of a token's lanes, the same in all of them where f does
// not depend on the order.
template <class F>
__device__ __forceinline__ int over_lanes(int v, int lanes, F f) {
    // Exchanges within 2, 4 and 8 lanes (mirrors of the groups below them).
    if (lanes > 1) v = f(v, __builtin_amdgcn_update_dpp(0, v, 0xb1, 15, 15, true));   // quad 1 0 3 2
    if (lanes > 2) v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x4e, 15, 15, true));   // quad 2 3 0 1
    if (lanes > 4) v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 15, 15, true));  // half mirror
    if (lanes > 8) v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x140, 15, 15, true));  // mirror
    if (lanes > 16) v = across(v, false, f);
    if (lanes > 32) v = across(v, true, f);
    return v;
}
__device__ __forceinline__ float lanes_max(float v, int lanes) {
    return __builtin_bit_cast(float, over_lanes(__builtin_bit_cast(int, v), lanes, [](int a, int b) {
        return __builtin_bit_cast(int, fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)));
    }));
}
// The lanes' orders differ, but a pair's sum does not, so neither does theirs.
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
    return __builtin_bit_cast(float, over_lanes(__builtin_bit_cast(int, v), lanes, [](int a, int b) {
        return __builtin_bit_cast(int, __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b));
    }));
}
__device__ __forceinline__ int lanes_max_int(int v, int lanes) {
    return over_lanes(v, lanes, [](int a, int b) { return a > b ? a : b; });
}
__device__ __forceinline__ int lanes_min_int(int v, int lanes) {
    return over_lanes(v, lanes, [](int a, int b) { return a < b ? a : b; });
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

// Q consecutive logits, -inf past the last; with `vector` rows start on 16
// bytes and hold whole vectors.
template <class T, int Q>
__device__ __forceinline__ void load_row(const char *row, int e0, int n, int vector,
                                         float (&x)[Q]) {
    typedef Vec<T, 16> X;
    if (vector) {
        if (e0 < n) {
#pragma unroll
            for (int p = 0; p < Q / X::n; ++p) {
                float part[X::n];
                X::unpack(reinterpret_cast<const typename X::raw *>(row + e0 * sizeof(T))[p],
                          part);
#pragma unroll
                for (int j = 0; j < X::n; ++j) x[p * X::n + j] = part[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < Q; ++j) x[j] = -__builtin_inff();
        }
    } else {
#pragma unroll
        for (int j = 0; j < Q; ++j)
            x[j] = e0 + j < n ? element<T>(row, e0 + j) : -__builtin_inff();
    }
}

// Whether all[i] is among the `kept` highest of all[count], ties to the lower
// index.  Keys above kGone, and kGone behind the last up to a whole eight.
__device__ __forceinline__ bool in_best(const int *all, int count, int i, int kept) {
    const int v = all[i];
    int before = 0;
    for (int j0 = 0; j0 < count; j0 += 8)
#pragma unroll
        for (int j = 0; j < 8; ++j) before += all[j0 + j] > (j0 + j < i ? v - 1 : v);
    return before < kept;
}
__device__ __forceinline__ void pad_standings(int *all, int count, int lane, int lanes) {
    for (int i = count + lane; i < (count + 7) / 8 * 8; i += lanes) all[i] = kGone;
}

// The two best keys of a set.
struct Two {
    int best, next;
};
__device__ __forceinline__ Two joined(Two a, Two b) {
    const int low = a.best < b.best ? a.best : b.best, next = a.next > b.next ? a.next : b.next;
    return {a.best > b.best ? a.best : b.best, low > next ? low : next};
}
// A group's: the best key, with a bias the sum of the two best that can be
// chosen.  A NaN's key stays above all.
__device__ __forceinline__ int standing(Two t, const float *bias) {
    int v = t.best;
    if (bias && t.next > kNone && v != 0x7fffffff) v = key_of(float_of(v) + float_of(t.next));
    return v > kGone ? v : kGone + 1;
}

// The keys of the kept groups, groups of 2^log_per experts: the two best of
// each in registers and between lanes, the standings through LDS.  LOG is
// log_per, Q's logarithm for groups of several lanes.
template <int Q, int LOG>
__device__ __forceinline__ void keep_groups(const RouteArgs &a, int e0, int lane, int *stands,
                                            int (&key)[Q]) {
    constexpr int kStep = 1 << LOG;
    Two two[Q];
#pragma unroll
    for (int j = 0; j < Q; ++j) two[j] = {key[j], kGone};
    // Leaders: the first of every group, or of the lane.
#pragma unroll
    for (int l = 0; l < LOG; ++l)
#pragma unroll
        for (int j = 0; j < Q; j += 2 << l) two[j] = joined(two[j], two[j + (1 << l)]);
    int share = 1;  // lanes of a group
    if constexpr (kStep == Q) {
        share = 1 << (a.log_per - LOG);
        for (int off = 1; off < share; off *= 2)
            two[0] =
                joined(two[0], Two{__shfl_xor(two[0].best, off), __shfl_xor(two[0].next, off)});
    }
#pragma unroll
    for (int j = 0; j < Q; j += kStep)
        if (e0 + j < a.n && (lane & (share - 1)) == 0)
            stands[(e0 + j) >> a.log_per] = standing(two[j], a.bias);
    pad_standings(stands, a.groups, lane, a.lanes);
    wave_fence();
#pragma unroll
    for (int j = 0; j < Q; j += kStep) {
        // Lanes past the last expert have no keys, and look at the first group.
        const int g = e0 + j < a.n ? (e0 + j) >> a.log_per : 0;
        const bool keep = in_best(stands, a.groups, g, a.kept);
#pragma unroll
        for (int i = j; i < j + kStep; ++i) key[i] = keep ? key[i] : kGone;
    }
}

// LDS of a token: its picks and their scores, with groups also the keys and
// the groups' standings, one word apart from the next token's so that tokens lie in
// different banks.
__host__ __device__ inline int route_words(int span, int k, int groups) {
    return (2 * k + (groups ? 2 * span : 0)) | 1;
}

// How groups are kept: not at all, of a power of two of experts, of others.
enum { kAll, kEven, kUneven };

// Bound by the vector units where a token has many experts: 4 of 64 in groups
// with a bias, 163,840 tokens, 22.7 us, of which 19 are 1,142 instructions a
// wave (the k maxima a third, the scores a quarter); its bytes would take 6.
// Without groups and bias 13.5 us; 2 of 8 experts 5.1 us.
template <class T, int Q, int GROUPS>
__global__ __launch_bounds__(kThreads) void route_kernel(RouteArgs given) {
    extern __shared__ int lds[];
    RouteArgs a = given;
    const int W = a.lanes, per_block = kThreads / W, t = threadIdx.x;
    const int lane = t & (W - 1), slot = t / W;
    const int e0 = lane * Q, span = W * Q;
    int *at = lds + slot * route_words(span, a.k, GROUPS), *keys = at + 2 * a.k,
        *stands = keys + span;
    float *scores = reinterpret_cast<float *>(at + a.k);
    const bool soft = a.score == TB_HIP_SCORE_SOFTMAX;
    for (size_t base = (size_t)blockIdx.x * per_block; base < a.tokens;
         base += (size_t)gridDim.x * per_block) {
        // Conditions on these stay inside the loop, which seldom turns twice:
        // kept over it they fill the scalar registers.
        asm volatile("" : "+s"(a.n), "+s"(a.log_per), "+s"(a.groups));
        const size_t token = base + slot;
        const bool live = token < a.tokens && (!a.valid || a.valid[token]);
        const char *row = a.logits + token * a.stride;
        float x[Q];
        int key[Q];
        if (live)
            load_row<T, Q>(row, e0, a.n, a.vector, x);
        else
#pragma unroll
            for (int j = 0; j < Q; ++j) x[j] = -__builtin_inff();
        // The row's largest logit and sum, where weights or keys need them.
        float top = -__builtin_inff(), inverse = 1.0f;
        if (soft && (a.bias || !a.renorm)) {
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < Q; ++j) top = fmaxf(top, x[j]);
            top = lanes_max(top, W);
#pragma unroll
            for (int j = 0; j < Q; ++j) sum += exp_of<true>(x[j] - top);  // -inf past the last
            inverse = 1.0f / lanes_sum(sum, W);
        }
        if (a.bias) {
            float b[Q];
            load_row<float, Q>(reinterpret_cast<const char *>(a.bias), e0, a.n, a.vector_bias, b);
            if (soft) {
#pragma unroll
                for (int j = 0; j < Q; ++j) b[j] += exp_of<true>(x[j] - top) * inverse;
            } else {
#pragma unroll
                for (int j = 0; j < Q; ++j) b[j] += sigmoid_of<true>(x[j]);
            }
#pragma unroll
            for (int j = 0; j < Q; ++j)
                key[j] = x[j] == -__builtin_inff() ? kGone : key_of(b[j]);
        } else {
#pragma unroll
            for (int j = 0; j < Q; ++j) key[j] = key_of(x[j]);
        }
        if constexpr (GROUPS == kEven) {
            switch (a.log_per) {
                case 0: keep_groups<Q, 0>(a, e0, lane, stands, key); break;
                case 1: keep_groups<Q, 1>(a, e0, lane, stands, key); break;
                case 2: keep_groups<Q, 2>(a, e0, lane, stands, key); break;
                case 3: keep_groups<Q, 3>(a, e0, lane, stands, key); break;
                // At eight a lane there are 16 experts at most, in groups of
                // no more than eight.
                default:
                    if constexpr (Q == 16) keep_groups<Q, 4>(a, e0, lane, stands, key);
            }
        }
        if constexpr (GROUPS == kUneven) {
            const int per = a.n / a.groups;
#pragma unroll
            for (int j = 0; j < Q; ++j) keys[e0 + j] = key[j];
            wave_fence();
            for (int g = lane; g < a.groups; g += W) {
                Two two = {kGone, kGone};
                for (int i = 0; i < per; ++i) two = joined(two, Two{keys[g * per + i], kGone});
                stands[g] = standing(two, a.bias);
            }
            pad_standings(stands, a.groups, lane, W);
            wave_fence();
            int g = e0 / per, left = per - (e0 - g * per);
            bool keep = g < a.groups && in_best(stands, a.groups, g, a.kept);
#pragma unroll
            for (int j = 0; j < Q; ++j) {
                if (left == 0) {
                    ++g;
                    left = per;
                    keep = g < a.groups && in_best(stands, a.groups, g, a.kept);
                }
                if (!keep) key[j] = kGone;
                --left;
            }
        }
        for (int i = 0; i < a.k; ++i) {
            int best = key[0];
#pragma unroll
            for (int j = 1; j < Q; ++j) best = key[j] > best ? key[j] : best;
            best = lanes_max_int(best, W);
            // The lowest index of that key; then it is gone.
            int expert = 0x7fffffff;
#pragma unroll
            for (int j = Q - 1; j >= 0; --j) expert = key[j] == best ? e0 + j : expert;
            expert = lanes_min_int(expert, W);
#pragma unroll
            for (int j = 0; j < Q; ++j) key[j] = expert == e0 + j ? kGone : key[j];
            if (lane == 0) at[i] = best > kNone ? expert : -1;
        }
        wave_fence();
        // The weights of the picks, from their logits again.  Renormalised
        // softmax weights need only the picks': relative to the largest of
        // them no sum is 0.
        const bool among = soft && a.renorm;
        float total = 0.0f;
        if (among) {
            top = -__builtin_inff();
            for (int i = lane; i < a.k; i += W)
                if (at[i] >= 0) top = fmaxf(top, element<T>(row, at[i]));
            top = lanes_max(top, W);
        }
        for (int i = lane; i < a.k; i += W) {
            float s = 0.0f;
            if (at[i] >= 0) {
                const float v = element<T>(row, at[i]);
                s = soft ? exp_of<true>(v - top) : sigmoid_of<true>(v);
            }
            scores[i] = s;
            total += s;
        }
        float factor = a.scale;
        if (a.renorm) {
            total = lanes_sum(total, W);
            // A NaN logit makes the row's scores NaN, picked or not.
            if (soft && a.bias) total += inverse - inverse;
        } else {
            factor *= inverse;
        }
        if (token < a.tokens)
            for (int i = lane; i < a.k; i += W) {
                float w = scores[i];
                if (a.renorm) w = total == 0.0f ? 0.0f : w / total;
                // No pick has weight 0 also where the row is NaN.
                a.experts[token * a.k + i] = at[i];
                a.weights[token * a.k + i] = at[i] >= 0 ? w * factor : 0.0f;
            }
        wave_fence();
    }
}

// A lane forms what belongs to its picks and puts it into the token's row in
// LDS, from which every lane takes its experts'.  Only softmax scores that are
// not renormalised need the whole row of logits.  163,840 tokens of 64 bf16
// logits, k 4: 16.4 us; 40,961 of 128, k 8, with the whole rows: 9.1 us, twice
// what its 24 MB take.
template <class T, int Q>
__global__ __launch_bounds__(kThreads) void route_backward_kernel(RouteArgs a) {
    __shared__ __attribute__((aligned(16))) float rows[kThreads * Q];
    typedef float floats __attribute__((ext_vector_type(4)));
    const int W = a.lanes, per_block = kThreads / W, t = threadIdx.x;
    const int lane = t & (W - 1), slot = t / W, e0 = lane * Q;
    const bool soft = a.score == TB_HIP_SCORE_SOFTMAX, whole = soft && !a.renorm;
    float *d = rows + slot * W * Q;
    floats *mine = reinterpret_cast<floats *>(d + e0);
    for (size_t base = (size_t)blockIdx.x * per_block; base < a.tokens;
         base += (size_t)gridDim.x * per_block) {
        const size_t token = base + slot;
        const bool live = token < a.tokens;
        const char *row = a.logits + token * a.stride;
        const int *at = a.chosen + token * a.k;
        const float *dw = a.dweights + token * a.k;
#pragma unroll
        for (int j = 0; j < Q / 4; ++j) mine[j] = (floats){0, 0, 0, 0};
        wave_fence();
        int used = 0;
        float top = -__builtin_inff();
        if (live)
            for (int i = lane; i < a.k; i += W)
                if ((unsigned)at[i] < (unsigned)a.n) {
                    used = 1;
                    if (soft && a.renorm) top = fmaxf(top, element<T>(row, at[i]));
                }
        used = lanes_max_int(used, W);
        if (a.renorm) {
            // w' of the picks, as quotients: a single one has w' = 1 and no
            // gradient, exactly.
            if (soft) top = lanes_max(top, W);
            float total = 0.0f, dot = 0.0f;
            if (live)
                for (int i = lane; i < a.k; i += W)
                    if ((unsigned)at[i] < (unsigned)a.n) {
                        const float x = element<T>(row, at[i]);
                        const float s = soft ? exp_of<true>(x - top) : sigmoid_of<true>(x);
                        d[at[i]] = s;
                        total += s;
                    }
            total = lanes_sum(total, W);
            wave_fence();
            if (live)
                for (int i = lane; i < a.k; i += W)
                    if ((unsigned)at[i] < (unsigned)a.n)
                        dot += d[at[i]] / total * (a.scale * dw[i]);
            dot = lanes_sum(dot, W);
            if (live)
                for (int i = lane; i < a.k; i += W)
                    if ((unsigned)at[i] < (unsigned)a.n) {
                        // 1 - s as the sigmoid of -x, without cancelling.  A sum
                        // of 0 gave weights of 0.
                        const float rest =
                            soft ? 1.0f : sigmoid_of<true>(-element<T>(row, at[i]));
                        const float w = d[at[i]] / total;
                        d[at[i]] = total == 0.0f ? 0.0f : w * rest * (a.scale * dw[i] - dot);
                    }
        } else if (live) {
            for (int i = lane; i < a.k; i += W)
                if ((unsigned)at[i] < (unsigned)a.n) {
                    float g = a.scale * dw[i];
                    if (!soft) {
                        const float x = element<T>(row, at[i]);
                        g *= sigmoid_of<true>(x) * sigmoid_of<true>(-x);
                    }
                    d[at[i]] = g;
                }
        }
        wave_fence();
        float v[Q];
#pragma unroll
        for (int j = 0; j < Q; ++j) v[j] = mine[j / 4][j % 4];
        if (whole) {
            float x[Q];
            if (used)
                load_row<T, Q>(row, e0, a.n, a.vector, x);
            else
#pragma unroll
                for (int j = 0; j < Q; ++j) x[j] = 0.0f;
            float sum = 0.0f, dot = 0.0f;
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
                dot += v[j] * x[j];
            }
            dot = lanes_sum(dot, W);
#pragma unroll
            for (int j = 0; j < Q; ++j) v[j] = used ? x[j] * (v[j] - dot) : 0.0f;
        }
        if (live) {
            T *out = reinterpret_cast<T *>(a.dlogits) + token * a.n + e0;
            if (a.vector) {
                typedef Vec<T, 16> X;
                if (e0 < a.n)
#pragma unroll
                    for (int p = 0; p < Q / X::n; ++p) {
                        float part[X::n];
#pragma unroll
                        for (int j = 0; j < X::n; ++j) part[j] = v[p * X::n + j];
                        reinterpret_cast<typename X::raw *>(out)[p] = X::pack(part);
                    }
            } else {
#pragma unroll
                for (int j = 0; j < Q; ++j)
                    if (e0 + j < a.n) out[j] = (T)v[j];
            }
        }
        wave_fence();
    }
}

// --------------------------------------------------------------------------
// The order of the choices by expert: a stable counting sort.  The choices are
// cut into segments, one to a wave: (1) every segment's count of each expert,
// (2) for each expert the running sum over the segments, (3) the segments
// again, each choice to its expert's start plus its running sum plus its rank
// in the segment.  Choices outside the experts count as expert n.  Up to
// kSmallChoices one workgroup does all three (us, that / three launches, 64
// experts: 640 choices 4.9 / 9.2, 4,000 7.9 / 9.8, 6,000 10.9 / 9.8).  655,360
// choices of 64 experts take 18.8 us in the three launches: a wave has 256
// choices, so that all are on their way at once, and what is left is each
// launch's chain of loads, about 5, 4 and 9 us.

constexpr int kOrderWaves = 4, kSmallWaves = 16, kSumThreads = 1024;
constexpr int kBatch = 4;  // choices of a lane on their way at once
constexpr size_t kSegment = 64 * kBatch, kMaxSegments = 4096, kSmallChoices = 5120;

struct OrderArgs {
    const int *experts;
    const float *weights;
    int *offsets, *tokens, *positions;
    float *row_weights;
    int *counts;  // [n + 1][padded], then their running sums
    int *totals;  // [n + 1]
    size_t choices, segment;
    unsigned segments, padded;  // padded: to whole workgroups
    int n, k, bits;
};

// The experts of choices c0 + lane, + 64, ...; n past c1.
__device__ __forceinline__ void load_choices(const OrderArgs &a, size_t c0, size_t c1,
                                             int (&e)[kBatch]) {
    const size_t c = c0 + (threadIdx.x & 63);
#pragma unroll
    for (int j = 0; j < kBatch; ++j) e[j] = c + 64 * j < c1 ? a.experts[c + 64 * j] : a.n;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) e[j] = (unsigned)e[j] < (unsigned)a.n ? e[j] : a.n;
}

// Adds a wave's segment to its counts in LDS.
__device__ __forceinline__ void count_segment(const OrderArgs &a, size_t c0, size_t c1,
                                              int *count) {
    const int lane = threadIdx.x & 63;
    for (size_t c = c0; c < c1; c += kSegment) {
        int e[kBatch];
        load_choices(a, c, c1, e);
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
            if (c + lane + 64 * j < c1) atomicAdd(&count[e[j]], 1);
    }
}

// A lane's choices of one turn, and their weights.
struct Choices {
    int e[kBatch];
    float w[kBatch];
    __device__ __forceinline__ void load(const OrderArgs &a, size_t cb, size_t c1) {
        const int lane = threadIdx.x & 63;
        load_choices(a, cb, c1, e);
        if (a.weights)
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
                w[j] = cb + lane + 64 * j < c1 ? a.weights[cb + lane + 64 * j] : 0.0f;
    }
};

// Writes a wave's segment; next[e] is the row of its next choice of expert e,
// `now` holds the first choices.
__device__ __forceinline__ void place_segment(const OrderArgs &a, size_t c0, size_t c1, int *next,
                                              Choices now) {
    const int lane = threadIdx.x & 63;
    for (size_t cb = c0; cb < c1; cb += kSegment) {
        int row[kBatch];
        if (cb > c0) now.load(a, cb, c1);
        const int(&e)[kBatch] = now.e;
        const float(&w)[kBatch] = now.w;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const bool live = cb + lane + 64 * j < c1;
            // The lanes with the same expert.
            unsigned long long same = __ballot(live);
            for (int b = 0; b < a.bits; ++b) {
                const bool set = (e[j] >> b) & 1;
                const unsigned long long all = __ballot(set);
                same &= set ? all : ~all;
            }
            const int rank = __popcll(same & ((1ull << lane) - 1));
            row[j] = live ? next[e[j]] + rank : 0;
            wave_fence();
            if (live && rank == 0) next[e[j]] = row[j] + __popcll(same);
            wave_fence();
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const size_t c = cb + lane + 64 * j;
            if (c < c1) {
                const bool known = e[j] < a.n;
                a.tokens[row[j]] = known ? (int)((unsigned)c / (unsigned)a.k) : -1;
                a.positions[c] = known ? row[j] : -1;
                if (a.weights) a.row_weights[row[j]] = known ? w[j] : 0.0f;
            }
        }
    }
}

// The counts of expert e in a workgroup's segments, those past the last too.
typedef int i32x4 __attribute__((ext_vector_type(4)));
static_assert(kOrderWaves == 4);
__device__ __forceinline__ i32x4 *counts_of(const OrderArgs &a, int e, unsigned block) {
    return reinterpret_cast<i32x4 *>(a.counts + (size_t)e * a.padded) + block;
}

__global__ __launch_bounds__(kOrderWaves * 64) void order_count_kernel(OrderArgs a) {
    extern __shared__ int lds[];
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63, columns = a.n + 1;
    int *count = lds + wave * columns;
    const unsigned seg = blockIdx.x * kOrderWaves + wave;
    for (int e = lane; e < columns; e += 64) count[e] = 0;
    wave_fence();
    const size_t c0 = seg * a.segment;
    if (seg < a.segments)
        count_segment(a, c0, c0 + a.segment < a.choices ? c0 + a.segment : a.choices, count);
    __syncthreads();
    for (int e = t; e < columns; e += kOrderWaves * 64)
        *counts_of(a, e, blockIdx.x) = (i32x4){lds[e], lds[columns + e], lds[2 * columns + e],
                                               lds[3 * columns + e]};
}

// One workgroup per expert: counts to exclusive running sums.
__global__ __launch_bounds__(kSumThreads) void order_sum_kernel(OrderArgs a) {
    __shared__ int wave_total[kSumThreads / 64];
    const int t = threadIdx.x, lane = t & 63;
    int *row = a.counts + (size_t)blockIdx.x * a.padded;
    int before = 0;
    for (unsigned s0 = 0; s0 < a.segments; s0 += kSumThreads) {
        const unsigned s = s0 + t;
        const int v = s < a.segments ? row[s] : 0, sum = running_sum(v);
        if (lane == 63) wave_total[t >> 6] = sum;
        __syncthreads();
        int below = 0, all = 0;
        for (int w = 0; w < kSumThreads / 64; ++w) {
            below += w < (t >> 6) ? wave_total[w] : 0;
            all += wave_total[w];
        }
        if (s < a.segments) row[s] = before + below + sum - v;
        before += all;
        __syncthreads();
    }
    if (t == 0) a.totals[blockIdx.x] = before;
}

// Every expert's start from the totals, by one wave.
__device__ __forceinline__ void find_starts(const OrderArgs &a, const int *totals, int *start,
                                            bool write) {
    const int lane = threadIdx.x & 63;
    int before = 0, ahead = lane <= a.n ? totals[lane] : 0;
    for (int e0 = 0; e0 <= a.n; e0 += 64) {
        const int e = e0 + lane, v = ahead, sum = running_sum(v);
        ahead = e + 64 <= a.n ? totals[e + 64] : 0;
        if (e <= a.n) {
            start[e] = before + sum - v;
            if (write) a.offsets[e] = before + sum - v;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
}

__global__ __launch_bounds__(kOrderWaves * 64) void order_place_kernel(OrderArgs a) {
    extern __shared__ int lds[];
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const int columns = a.n + 1;
    int *start = lds, *next = lds + columns * (1 + wave);
    const unsigned seg = blockIdx.x * kOrderWaves + wave;
    const size_t c0 = seg * a.segment;
    const size_t c1 = c0 + a.segment < a.choices ? c0 + a.segment : a.choices;
    Choices first;
    first.load(a, c0, c1);  // on their way meanwhile
    if (wave == 0) find_starts(a, a.totals, start, blockIdx.x == 0);
    for (int e = t; e < columns; e += kOrderWaves * 64) {
        const i32x4 before = *counts_of(a, e, blockIdx.x);
#pragma unroll
        for (int w = 0; w < kOrderWaves; ++w) lds[columns * (1 + w) + e] = before[w];
    }
    __syncthreads();
    if (seg >= a.segments) return;
    for (int e = lane; e < columns; e += 64) next[e] += start[e];
    wave_fence();
    place_segment(a, c0, c1, next, first);
}

// All of it in one workgroup: LDS holds the totals and each wave's counts.
__global__ __launch_bounds__(kSmallWaves * 64) void order_small_kernel(OrderArgs a) {
    extern __shared__ int lds[];
    const int t = threadIdx.x, wave = t >> 6, columns = a.n + 1;
    int *start = lds, *next = lds + columns * (1 + wave);
    for (int i = t; i < columns * (1 + kSmallWaves); i += kSmallWaves * 64) lds[i] = 0;
    __syncthreads();
    const size_t c0 = wave * a.segment < a.choices ? wave * a.segment : a.choices;
    const size_t c1 = c0 + a.segment < a.choices ? c0 + a.segment : a.choices;
    Choices first;
    first.load(a, c0, c1);
    count_segment(a, c0, c1, next);
    __syncthreads();
    // Counts to running sums over the waves; the totals behind.
    for (int e = t; e < columns; e += kSmallWaves * 64) {
        int before = 0;
        for (int w = 0; w < kSmallWaves; ++w) {
            const int v = lds[columns * (1 + w) + e];
            lds[columns * (1 + w) + e] = before;
            before += v;
        }
        start[e] = before;
    }
    __syncthreads();
    if (wave == 0) find_starts(a, start, start, true);
    __syncthreads();
    for (int i = t; i < columns * kSmallWaves; i += kSmallWaves * 64) {
        const int e = i % columns;
        lds[columns + i] += start[e];
    }
    __syncthreads();
    place_segment(a, c0, c1, next, first);
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

// Experts a lane.  Forward 16 above 16 experts, which halves what lanes do for
// their token (163,840 tokens, us, 8 / 16 a lane: 4 of 64 20.5 / 13.3, 2 of 16
// 5.6 / 7.0, 8 of 128 of 81,920 tokens 30.0 / 22.5); backward 8, which
// keeps more loads under way, as long as 64 lanes hold a token's.
constexpr int kForwardEight = 16, kBackwardEight = 512;

template <class T, int Q, int GROUPS>
void launch_route(RouteArgs &a, hipStream_t q) {
    a.lanes = lanes_for(a.n, Q);
    const size_t words = route_words(a.lanes * Q, a.k, GROUPS);
    route_kernel<T, Q, GROUPS>
        <<<grid_for(a), kThreads, kThreads / a.lanes * words * sizeof(int), q>>>(a);
}

template <class T, int Q>
void launch_backward(RouteArgs &a, hipStream_t q) {
    a.lanes = lanes_for(a.n, Q);
    route_backward_kernel<T, Q><<<grid_for(a), kThreads, 0, q>>>(a);
}

// Rows that start on 16 bytes and hold whole lanes' experts.
int vector_rows(const void *p, size_t stride, int n, int q) {
    return multiple_of(p, 16) && stride % 16 == 0 && n % q == 0;
}

// Calls f with a zero of the type.
template <class F>
void with_type(int dtype, F f) {
    if (dtype == TB_HIP_F32)
        f(0.0f);
    else if (dtype == TB_HIP_BF16)
        f((__bf16)0.0f);
    else
        f((_Float16)0.0f);
}

struct OrderShape {
    size_t segment;
    unsigned segments, blocks;
};

OrderShape order_shape(size_t choices) {
    OrderShape s;
    s.segment = kSegment;
    const size_t least = (choices + kMaxSegments - 1) / kMaxSegments;
    if (least > s.segment) s.segment = (least + 63) / 64 * 64;
    s.segments = (unsigned)((choices + s.segment - 1) / s.segment);
    s.blocks = (s.segments + kOrderWaves - 1) / kOrderWaves;
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
    const int per = n_experts / groups;
    a.log_per = per & (per - 1) ? -1 : __builtin_ctz(per);
    a.score = score;
    a.renorm = renormalise != 0;
    a.scale = scale;
    hipStream_t q = reinterpret_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    const bool eight = n_experts <= kForwardEight;
    a.vector = vector_rows(logits, row_stride, n_experts, eight ? 8 : 16);
    a.vector_bias = vector_rows(bias, 0, n_experts, eight ? 8 : 16);
    with_type(dtype, [&](auto zero) {
        typedef decltype(zero) T;
        if (groups_kept == groups)
            eight ? launch_route<T, 8, kAll>(a, q) : launch_route<T, 16, kAll>(a, q);
        else if (a.log_per >= 0)
            eight ? launch_route<T, 8, kEven>(a, q) : launch_route<T, 16, kEven>(a, q);
        else
            eight ? launch_route<T, 8, kUneven>(a, q) : launch_route<T, 16, kUneven>(a, q);
    });
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
    const bool eight = n_experts <= kBackwardEight;
    a.vector = vector_rows(logits, row_stride, n_experts, eight ? 8 : 16) &&
               multiple_of(dlogits, 16);
    with_type(dtype, [&](auto zero) {
        if (eight)
            launch_backward<decltype(zero), 8>(a, q);
        else
            launch_backward<decltype(zero), 16>(a, q);
    });
    return hipGetLastError() == hipSuccess;
}

extern "C" size_t tb_hip_expert_order_workspace_bytes(size_t tokens, int n_experts, int k) {
    if (!order_ok(tokens, n_experts, k)) return 0;
    const OrderShape s = order_shape(tokens * k);
    const size_t ints = (size_t)(n_experts + 1) * (s.blocks * kOrderWaves + 1);
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
    a.padded = s.blocks * kOrderWaves;
    a.totals = a.counts + (size_t)(n_experts + 1) * a.padded;
    a.choices = tokens * k;
    a.segment = s.segment;
    a.segments = s.segments;
    a.n = n_experts;
    a.k = k;
    while ((1 << a.bits) <= n_experts) ++a.bits;
    hipStream_t q = reinterpret_cast<hipStream_t>(stream);
    const size_t row = (n_experts + 1) * sizeof(int);
    (void)hipGetLastError();
    if (a.choices <= kSmallChoices && row * (1 + kSmallWaves) <= 64 * 1024) {
        a.segment = (a.choices + kSmallWaves * 64 - 1) / (kSmallWaves * 64) * 64;
        order_small_kernel<<<1, kSmallWaves * 64, row * (1 + kSmallWaves), q>>>(a);
        return hipGetLastError() == hipSuccess;
    }
    order_count_kernel<<<s.blocks, kOrderWaves * 64, kOrderWaves * row, q>>>(a);
    order_sum_kernel<<<n_experts + 1, kSumThreads, 0, q>>>(a);
    order_place_kernel<<<s.blocks, kOrderWaves * 64, (1 + kOrderWaves) * row, q>>>(a);
    return hipGetLastError() == hipSuccess;
}
