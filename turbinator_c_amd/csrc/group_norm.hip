// Group norm with an activation over channels-last planes, forward and
// backward (hip_layers.h).  The activation is in the same pass, and the planes
// are channels last, as a matrix-core convolution leaves them.
//
//   h = (x - mean) rstd,  z = h gamma + beta,  y = act(z)
//   u = dy act'(z):  dbeta = sum u,  dgamma = sum u h  (images, pixels)
//   dx = rstd (u gamma - m1 - h m2),  m1 = mean(u gamma), m2 = mean(u gamma h)
//   over the group; both follow from the per-channel sums of u and u h.
//
// A workgroup takes a slab of whole groups of one image: thread t owns lane
// t % lanes (a vector of channels) of the pixels t / lanes, + rows, ..., so
// every load is a run of the slab's bytes and every thread's channels stay
// the same.  Sums go lane by lane, then through LDS per wave (or per row
// where the lanes of a pixel do not divide a wave), always in the same order.
//
// A slab whose pixels fit the registers of a workgroup is read once.  Larger
// ones take two launches: partial statistics of chunks of pixels, then the
// elements, each workgroup joining its image's partials first.
#include <initializer_list>

#include "layer_math.h"
#include "xcd_order.h"

namespace {

using namespace layer;

constexpr int kMaxSlab = 1024;     // channels of a workgroup
constexpr int kMaxChunks = 1024;   // chunks of an image
constexpr size_t kMaxCount = 0x7fffffffu;
constexpr int kThreads = 512;      // of a workgroup; kMaxThreads where a pixel has more lanes
constexpr int kMaxThreads = 1024;
constexpr int kVectors = 8;        // a chunk holds this many vectors a thread
constexpr int kAhead = 4;          // of them a thread loads before it uses the first
constexpr size_t kMaxGrid = 1 << 20;

// How a launch divides the planes.
struct Shape {
    int bytes;        // of a vector
    int lanes;        // vectors of one pixel of the slab
    int slab;         // channels of the slab
    int slabs;
    int threads;
    int rows;         // pixels per sweep of the workgroup
    int fold;         // lanes divide a wave: sums fold within it
    unsigned chunk;   // pixels of a chunk, whole sweeps
    unsigned chunks;
    int whole;        // the slab's pixels fit whole: vectors a thread holds
    unsigned spans;   // workgroups that share a slab's images, backward
};

struct NormArgs {
    const char *x, *dy;
    size_t x_image, x_pixel, dy_image, dy_pixel;
    const float *gamma, *beta, *mean_in, *rstd_in;
    char *out;
    float *mean, *rstd;
    float *parts;
    size_t images;
    unsigned pixels;
    int channels, groups, per;  // per: channels of a group
    float eps;
    int act;
    Shape s;
};

template <int N>
__device__ __forceinline__ float plus_rotated(float v) {
    return v + __builtin_bit_cast(float, rotated<N>(__builtin_bit_cast(int, v)));
}
__device__ __forceinline__ float plus_far(float v, bool far) {
    return __builtin_bit_cast(float, across(__builtin_bit_cast(int, v), far, [](int a, int b) {
        return __builtin_bit_cast(int, __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b));
    }));
}

// Sums over the lanes of a wave that are a multiple of `lanes` apart, lanes a
// power of two: rotations within sixteen lanes, exchanges between them.
template <int V>
__device__ __forceinline__ void fold(float (&v)[V], int lanes) {
#define TB_FOLD(limit, step)                          \
    if (lanes <= limit)                               \
        _Pragma("unroll") for (int i = 0; i < V; ++i) v[i] = step;
    TB_FOLD(1, plus_rotated<1>(v[i]))
    TB_FOLD(2, plus_rotated<2>(v[i]))
    TB_FOLD(4, plus_rotated<4>(v[i]))
    TB_FOLD(8, plus_rotated<8>(v[i]))
    TB_FOLD(16, plus_far(v[i], false))
    TB_FOLD(32, plus_far(v[i], true))
#undef TB_FOLD
}

// Writes the workgroup's sums of v over the rows that fold within a wave to
// part[row][channel]; the caller synchronises.
template <int V>
__device__ __forceinline__ void row_sums(float (&v)[V], const Shape &s, float *part) {
    const int t = threadIdx.x;
    if (s.fold) {
        fold(v, s.lanes);
        const int lane = t & 63;
        if (lane < s.lanes)
#pragma unroll
            for (int i = 0; i < V; ++i) part[(t >> 6) * s.slab + lane * V + i] = v[i];
    } else if (t < s.rows * s.lanes) {
#pragma unroll
        for (int i = 0; i < V; ++i) part[t * V + i] = v[i];
    }
}

__device__ __forceinline__ int part_rows(const Shape &s) {
    return s.fold ? (int)(blockDim.x >> 6) : s.rows;
}

__device__ __forceinline__ float wave_sum(float v) {
    float one[1] = {v};
    fold(one, 1);
    // The lanes add in orders of their own: all take the first one's sum.
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(
                                         __builtin_bit_cast(int, one[0])));
}

// The sum of part[rows][slab] over all rows and the `per` channels from c0,
// in every lane of the calling wave.
__device__ __forceinline__ float group_sum(const float *part, int rows, int slab, int c0,
                                           int per) {
    const int lane = threadIdx.x & 63;
    float sum = 0.0f;
    if (per >= 64) {
        for (int r = 0; r < rows; ++r)
            for (int c = lane; c < per; c += 64) sum += part[r * slab + c0 + c];
    } else {
        const int step = 64 / per, r0 = lane / per, c = lane - r0 * per;
        if (r0 < step)
            for (int r = r0; r < rows; r += step) sum += part[r * slab + c0 + c];
    }
    return wave_sum(sum);
}

struct Place {
    size_t image;
    int c0;             // first channel of the slab
    unsigned p0, p1;    // pixels of the chunk
    size_t chunk;       // index of (image, chunk)
};

__device__ __forceinline__ Place place_of(const NormArgs &a, size_t item) {
    Place w;
    const size_t per_image = (size_t)a.s.slabs * a.s.chunks;
    w.image = item / per_image;
    const unsigned rest = (unsigned)(item - w.image * per_image);
    const unsigned chunk = rest / a.s.slabs;
    w.c0 = (int)(rest - chunk * a.s.slabs) * a.s.slab;
    w.p0 = chunk * a.s.chunk;
    w.p1 = w.p0 + a.s.chunk < a.pixels ? w.p0 + a.s.chunk : a.pixels;
    w.chunk = w.image * a.s.chunks + chunk;
    return w;
}

// Mean and sum of squared deviations of each group over one chunk.  A sweep
// of kVectors vectors a thread stays in registers for both; sweeps of a longer
// chunk are joined with Chan's formula.  Bound by memory, which the second
// launch reads again, from the last cache where the planes fit it: both take
// 77 us for 16 x 65,536 x 64 bf16 (3.5 TB/s of x and y), 334 us for 128 x
// 16,384 x 128 (3.2).
template <class T, int B>
__global__ __launch_bounds__(kMaxThreads) void norm_parts_kernel(NormArgs a) {
    typedef Vec<T, B> X;
    constexpr int V = X::n;
    extern __shared__ float lds[];
    const Shape s = a.s;
    const int t = threadIdx.x, rows = part_rows(s), wave = t >> 6, waves = blockDim.x >> 6;
    float *part = lds, *means = part + rows * s.slab, *sofar = means + s.slab;
    const int lane = t % s.lanes, row = t / s.lanes;
    const size_t items = a.images * s.slabs * s.chunks;
    for (size_t item = blockIdx.x; item < items; item += gridDim.x) {
        const Place w = place_of(a, xcd_contiguous(item, items));
        const char *x = a.x + w.image * a.x_image + (size_t)(w.c0 + lane * V) * sizeof(T);
        float count = 0.0f;
        for (unsigned p0 = w.p0; p0 < w.p1; p0 += s.rows * kVectors) {
            typename X::raw raw[kVectors];
            float sum[V];
#pragma unroll
            for (int i = 0; i < V; ++i) sum[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < kVectors; ++j) {
                const unsigned p = p0 + j * s.rows + row;
                if (row < s.rows && p < w.p1)
                    raw[j] = *reinterpret_cast<const typename X::raw *>(x + p * a.x_pixel);
            }
#pragma unroll
            for (int j = 0; j < kVectors; ++j) {
                const unsigned p = p0 + j * s.rows + row;
                if (row < s.rows && p < w.p1) {
                    float v[V];
                    X::unpack(raw[j], v);
#pragma unroll
                    for (int i = 0; i < V; ++i) sum[i] += v[i];
                }
            }
            const unsigned end = p0 + s.rows * kVectors < w.p1 ? p0 + s.rows * kVectors : w.p1;
            const float n = (float)(end - p0) * a.per;
            row_sums<V>(sum, s, part);
            __syncthreads();
            for (int g = wave; g < s.slab / a.per; g += waves) {
                const float m = group_sum(part, rows, s.slab, g * a.per, a.per) / n;
                for (int c = t & 63; c < a.per; c += 64) means[g * a.per + c] = m;
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < V; ++i) sum[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < kVectors; ++j) {
                const unsigned p = p0 + j * s.rows + row;
                if (row < s.rows && p < w.p1) {
                    float v[V];
                    X::unpack(raw[j], v);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float d = v[i] - means[lane * V + i];
                        sum[i] = fmaf(d, d, sum[i]);
                    }
                }
            }
            row_sums<V>(sum, s, part);
            __syncthreads();
            for (int g = wave; g < s.slab / a.per; g += waves) {
                const float m2 = group_sum(part, rows, s.slab, g * a.per, a.per);
                if ((t & 63) == 0) {
                    const float m = means[g * a.per];
                    if (count == 0.0f) {
                        sofar[2 * g] = m;
                        sofar[2 * g + 1] = m2;
                    } else {
                        const float d = m - sofar[2 * g], all = count + n;
                        sofar[2 * g] += d * (n / all);
                        sofar[2 * g + 1] += m2 + d * d * (count * (n / all));
                    }
                }
            }
            count += n;
            __syncthreads();
        }
        for (int g = t; g < s.slab / a.per; g += blockDim.x) {
            const size_t at = (w.chunk * a.groups + w.c0 / a.per + g) * 2;
            a.parts[at] = sofar[2 * g];
            a.parts[at + 1] = sofar[2 * g + 1];
        }
        __syncthreads();
    }
}

// Joins an image's chunks and writes the chunk's elements.
template <class T, int B, int ACT>
__global__ __launch_bounds__(kMaxThreads) void norm_apply_kernel(NormArgs a) {
    typedef Vec<T, B> X;
    constexpr int V = X::n;
    extern __shared__ float lds[];
    const Shape s = a.s;
    const int t = threadIdx.x, wave = t >> 6, waves = blockDim.x >> 6;
    float *means = lds, *rstds = lds + s.slab;
    const int lane = t % s.lanes, row = t / s.lanes;
    const size_t items = a.images * s.slabs * s.chunks;
    for (size_t item = blockIdx.x; item < items; item += gridDim.x) {
        const Place w = place_of(a, xcd_contiguous(item, items));
        for (int g = wave; g < s.slab / a.per; g += waves) {
            const int group = w.c0 / a.per + g;
            const float *parts = a.parts + (w.image * s.chunks * a.groups + group) * 2;
            const float full = (float)s.chunk * a.per, all = (float)a.pixels * a.per;
            const float last = (float)(a.pixels - (s.chunks - 1) * s.chunk) * a.per;
            float sum = 0.0f, m2 = 0.0f;
            for (unsigned i = t & 63; i < s.chunks; i += 64)
                sum += parts[(size_t)i * a.groups * 2] * (i + 1 < s.chunks ? full : last);
            const float mean = wave_sum(sum) / all;
            for (unsigned i = t & 63; i < s.chunks; i += 64) {
                const float d = parts[(size_t)i * a.groups * 2] - mean;
                m2 += parts[(size_t)i * a.groups * 2 + 1] +
                      d * d * (i + 1 < s.chunks ? full : last);
            }
            const float rstd = 1.0f / sqrtf(wave_sum(m2) / all + a.eps);
            for (int c = t & 63; c < a.per; c += 64) {
                means[g * a.per + c] = mean;
                rstds[g * a.per + c] = rstd;
            }
            if ((t & 63) == 0 && w.p0 == 0) {
                if (a.mean) a.mean[w.image * a.groups + group] = mean;
                if (a.rstd) a.rstd[w.image * a.groups + group] = rstd;
            }
        }
        __syncthreads();
        if (row < s.rows) {
            const int c0 = w.c0 + lane * V;
            float mean[V], scale[V], shift[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                mean[i] = means[lane * V + i];
                scale[i] = rstds[lane * V + i] * (a.gamma ? a.gamma[c0 + i] : 1.0f);
                shift[i] = a.beta ? a.beta[c0 + i] : 0.0f;
            }
            const char *x = a.x + w.image * a.x_image + (size_t)c0 * sizeof(T);
            char *y = a.out + (w.image * a.pixels * a.channels + c0) * sizeof(T);
            for (unsigned p0 = w.p0 + row; p0 < w.p1; p0 += s.rows * kAhead) {
                typename X::raw raw[kAhead];
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
                    const unsigned p = p0 + j * s.rows;
                    if (p < w.p1)
                        raw[j] = *reinterpret_cast<const typename X::raw *>(x + p * a.x_pixel);
                }
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
                    const unsigned p = p0 + j * s.rows;
                    if (p >= w.p1) break;
                    float v[V];
                    X::unpack(raw[j], v);
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        v[i] = act_of<kFine<T>, ACT>(fmaf(v[i] - mean[i], scale[i], shift[i]));
                    *reinterpret_cast<typename X::raw *>(y + (size_t)p * a.channels * sizeof(T)) =
                        X::pack(v);
                }
            }
        }
        __syncthreads();
    }
}

// u = dy act'(z) and d = x - mean of one vector.
template <class T, int B, int ACT>
__device__ __forceinline__ void grad_terms(typename Vec<T, B>::raw xr,
                                           typename Vec<T, B>::raw gr,
                                           const float (&mean)[Vec<T, B>::n],
                                           const float (&scale)[Vec<T, B>::n],
                                           const float (&beta)[Vec<T, B>::n],
                                           float (&u)[Vec<T, B>::n], float (&d)[Vec<T, B>::n]) {
    Vec<T, B>::unpack(xr, d);
    Vec<T, B>::unpack(gr, u);
#pragma unroll
    for (int i = 0; i < Vec<T, B>::n; ++i) {
        d[i] -= mean[i];
        if constexpr (ACT != TB_HIP_ACT_NONE)
            u[i] *= act_slope<kFine<T>, ACT>(fmaf(d[i], scale[i], beta[i]));
    }
}

// A thread's channels: z = (x - mean) scale + beta, scale = rstd gamma.
template <int V>
struct Channels {
    float mean[V], rstd[V], scale[V], beta[V];
    __device__ __forceinline__ void load(const NormArgs &a, size_t image, int c0) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const size_t g = image * a.groups + (c0 + i) / a.per;
            mean[i] = a.mean_in[g];
            rstd[i] = a.rstd_in[g];
            scale[i] = rstd[i] * (a.gamma ? a.gamma[c0 + i] : 1.0f);
            beta[i] = a.beta ? a.beta[c0 + i] : 0.0f;
        }
    }
};

// f(pixel, u, d) of a thread's vectors of a chunk, kAhead of them loaded at once.
template <class T, int B, int ACT, class F>
__device__ __forceinline__ void grad_sweep(const NormArgs &a, const Place &w, int row,
                                           const char *x, const char *dy,
                                           const Channels<Vec<T, B>::n> &ch, F f) {
    typedef Vec<T, B> X;
    const int rows = a.s.rows;
    for (unsigned p0 = w.p0 + row; p0 < w.p1; p0 += rows * kAhead) {
        typename X::raw xr[kAhead], gr[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const unsigned p = p0 + j * rows;
            if (p < w.p1) {
                xr[j] = *reinterpret_cast<const typename X::raw *>(x + p * a.x_pixel);
                gr[j] = *reinterpret_cast<const typename X::raw *>(dy + p * a.dy_pixel);
            }
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const unsigned p = p0 + j * rows;
            if (p >= w.p1) break;
            float u[X::n], d[X::n];
            grad_terms<T, B, ACT>(xr[j], gr[j], ch.mean, ch.scale, ch.beta, u, d);
            f(p, u, d);
        }
    }
}

// The sums of u and u h of every channel over one chunk:
// parts[(image, chunk)][channel][2].  With grad_apply_kernel 176 us for 16 x
// 65,536 x 64 bf16 (2.3 TB/s of x, dy and dx, five passes for three), 550 us
// for 128 x 16,384 x 128 (2.9).
template <class T, int B, int ACT>
__global__ __launch_bounds__(kMaxThreads) void grad_parts_kernel(NormArgs a) {
    typedef Vec<T, B> X;
    constexpr int V = X::n;
    extern __shared__ float lds[];
    const Shape s = a.s;
    const int t = threadIdx.x, rows = part_rows(s);
    float *part = lds, *part2 = part + rows * s.slab;
    const int lane = t % s.lanes, row = t / s.lanes;
    const size_t items = a.images * s.slabs * s.chunks;
    for (size_t item = blockIdx.x; item < items; item += gridDim.x) {
        const Place w = place_of(a, xcd_contiguous(item, items));
        const int c0 = w.c0 + lane * V;
        float su[V], sh[V];
#pragma unroll
        for (int i = 0; i < V; ++i) su[i] = sh[i] = 0.0f;
        if (row < s.rows) {
            Channels<V> ch;
            ch.load(a, w.image, c0);
            const char *x = a.x + w.image * a.x_image + (size_t)c0 * sizeof(T);
            const char *dy = a.dy + w.image * a.dy_image + (size_t)c0 * sizeof(T);
            grad_sweep<T, B, ACT>(a, w, row, x, dy, ch,
                                  [&](unsigned, const float(&u)[V], const float(&d)[V]) {
#pragma unroll
                                      for (int i = 0; i < V; ++i) {
                                          su[i] += u[i];
                                          sh[i] = fmaf(u[i], d[i], sh[i]);
                                      }
                                  });
#pragma unroll
            for (int i = 0; i < V; ++i) sh[i] *= ch.rstd[i];
        }
        row_sums<V>(su, s, part);
        row_sums<V>(sh, s, part2);
        __syncthreads();
        for (int c = t; c < s.slab; c += blockDim.x) {
            float one = 0.0f, two = 0.0f;
            for (int r = 0; r < rows; ++r) {
                one += part[r * s.slab + c];
                two += part2[r * s.slab + c];
            }
            float *at = a.parts + (w.chunk * a.channels + w.c0 + c) * 2;
            at[0] = one;
            at[1] = two;
        }
        __syncthreads();
    }
}

typedef float Pair __attribute__((ext_vector_type(2)));
__host__ __device__ __forceinline__ int shares_of(const Shape &s) {
    return s.threads > s.slab ? s.threads / s.slab : 1;
}

template <class T, int B, int ACT>
__global__ __launch_bounds__(kMaxThreads) void grad_apply_kernel(NormArgs a) {
    typedef Vec<T, B> X;
    constexpr int V = X::n;
    extern __shared__ float lds[];
    const Shape s = a.s;
    const int t = threadIdx.x, wave = t >> 6, waves = blockDim.x >> 6;
    const int shares = shares_of(s);
    float *m1 = lds, *m2 = m1 + s.slab, *sum1 = m2 + s.slab, *sum2 = sum1 + s.slab * shares;
    const int lane = t % s.lanes, row = t / s.lanes;
    const size_t items = a.images * s.slabs * s.chunks;
    const float inverse = 1.0f / ((float)a.pixels * a.per);
    for (size_t item = blockIdx.x; item < items; item += gridDim.x) {
        const Place w = place_of(a, xcd_contiguous(item, items));
        // A channel's chunks are summed by `shares` threads, then those sums.
        for (int i = t; i < s.slab * shares; i += blockDim.x) {
            const int share = i / s.slab, c = i - share * s.slab;
            const Pair *at = reinterpret_cast<const Pair *>(a.parts) +
                             w.image * s.chunks * a.channels + w.c0 + c;
            float one = 0.0f, two = 0.0f;
#pragma unroll 4
            for (unsigned j = share; j < s.chunks; j += shares) {
                const Pair v = at[(size_t)j * a.channels];
                one += v[0];
                two += v[1];
            }
            sum1[i] = one;
            sum2[i] = two;
        }
        __syncthreads();
        for (int c = t; c < s.slab; c += blockDim.x) {
            float one = 0.0f, two = 0.0f;
            for (int i = 0; i < shares; ++i) {
                one += sum1[i * s.slab + c];
                two += sum2[i * s.slab + c];
            }
            const float gamma = a.gamma ? a.gamma[w.c0 + c] : 1.0f;
            m1[c] = one * gamma;
            m2[c] = two * gamma;
        }
        __syncthreads();
        for (int g = wave; g < s.slab / a.per; g += waves) {
            const float one = group_sum(m1, 1, s.slab, g * a.per, a.per) * inverse;
            const float two = group_sum(m2, 1, s.slab, g * a.per, a.per) * inverse;
            for (int c = t & 63; c < a.per; c += 64) {
                m1[g * a.per + c] = one;
                m2[g * a.per + c] = two;
            }
        }
        __syncthreads();
        if (row < s.rows) {
            const int c0 = w.c0 + lane * V;
            Channels<V> ch;
            ch.load(a, w.image, c0);
            const char *x = a.x + w.image * a.x_image + (size_t)c0 * sizeof(T);
            const char *dy = a.dy + w.image * a.dy_image + (size_t)c0 * sizeof(T);
            char *dx = a.out + (w.image * a.pixels * a.channels + c0) * sizeof(T);
            // dx = u rstd gamma - rstd m1 - d rstd^2 m2
            float less[V], slope[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                less[i] = ch.rstd[i] * m1[lane * V + i];
                slope[i] = ch.rstd[i] * ch.rstd[i] * m2[lane * V + i];
            }
            grad_sweep<T, B, ACT>(
                a, w, row, x, dy, ch, [&](unsigned p, const float(&u)[V], const float(&d)[V]) {
                    float v[V];
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        v[i] = fmaf(-d[i], slope[i], fmaf(u[i], ch.scale[i], -less[i]));
                    *reinterpret_cast<typename X::raw *>(
                        dx + (size_t)p * a.channels * sizeof(T)) = X::pack(v);
                });
        }
        __syncthreads();
    }
}

// Planes whose slab fits the registers of one workgroup: one pass over memory.
// Every thread holds NV vectors; the means, then the squared deviations, then
// the elements come from them.  4,096 x 1,024 x 64 bf16 with SiLU: 250 us, 4.3
// TB/s of x and y, where a copy of 4 GiB moves 4.8; 257 x 1,023 x 48 fp32 with
// GELU: 26.5 us, 3.8 TB/s, 771 workgroups on 256 CUs.
template <class T, int B, int NV, int ACT>
__global__ __launch_bounds__(kMaxThreads) void norm_whole_kernel(NormArgs a) {
    typedef Vec<T, B> X;
    constexpr int V = X::n;
    extern __shared__ float lds[];
    const Shape s = a.s;
    const int t = threadIdx.x, rows = part_rows(s), wave = t >> 6, waves = blockDim.x >> 6;
    float *part = lds, *part2 = part + rows * s.slab, *means = part2 + rows * s.slab,
          *rstds = means + s.slab;
    const int lane = t % s.lanes, row = t / s.lanes;
    const size_t items = a.images * s.slabs;
    const float inverse = 1.0f / ((float)a.pixels * a.per);
    // Pixels of a thread: row, row + rows, ... below `count` vectors.
    const int count = row < s.rows && (unsigned)row < a.pixels
                          ? (int)((a.pixels - row + s.rows - 1) / s.rows) : 0;
    for (size_t item = blockIdx.x; item < items; item += gridDim.x) {
        const size_t at = xcd_contiguous(item, items), image = at / s.slabs;
        const int first = (int)(at - image * s.slabs) * s.slab, c0 = first + lane * V;
        const char *x = a.x + image * a.x_image + (size_t)c0 * sizeof(T) + row * a.x_pixel;
        const size_t step = s.rows * a.x_pixel;
        typename X::raw raw[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j < count) raw[j] = *reinterpret_cast<const typename X::raw *>(x + j * step);
        float sum[V];
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j < count) {
                float v[V];
                X::unpack(raw[j], v);
#pragma unroll
                for (int i = 0; i < V; ++i) sum[i] += v[i];
            }
        row_sums<V>(sum, s, part);
        __syncthreads();
        for (int g = wave; g < s.slab / a.per; g += waves) {
            const float m = group_sum(part, rows, s.slab, g * a.per, a.per) * inverse;
            for (int c = t & 63; c < a.per; c += 64) means[g * a.per + c] = m;
        }
        __syncthreads();
        float mean[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            mean[i] = means[lane * V + i];
            sum[i] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j < count) {
                float v[V];
                X::unpack(raw[j], v);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float d = v[i] - mean[i];
                    sum[i] = fmaf(d, d, sum[i]);
                }
            }
        row_sums<V>(sum, s, part2);
        __syncthreads();
        for (int g = wave; g < s.slab / a.per; g += waves) {
            const float var = group_sum(part2, rows, s.slab, g * a.per, a.per) * inverse;
            const float rstd = 1.0f / sqrtf(var + a.eps);
            for (int c = t & 63; c < a.per; c += 64) rstds[g * a.per + c] = rstd;
            if ((t & 63) == 0) {
                const size_t to = image * a.groups + first / a.per + g;
                if (a.mean) a.mean[to] = means[g * a.per];
                if (a.rstd) a.rstd[to] = rstd;
            }
        }
        __syncthreads();
        float scale[V], shift[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            scale[i] = rstds[lane * V + i] * (count && a.gamma ? a.gamma[c0 + i] : 1.0f);
            shift[i] = count && a.beta ? a.beta[c0 + i] : 0.0f;
        }
        char *y = a.out + ((image * a.pixels + row) * a.channels + c0) * sizeof(T);
        const size_t out_step = (size_t)s.rows * a.channels * sizeof(T);
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j < count) {
                float v[V];
                X::unpack(raw[j], v);
#pragma unroll
                for (int i = 0; i < V; ++i)
                    v[i] = act_of<kFine<T>, ACT>(fmaf(v[i] - mean[i], scale[i], shift[i]));
                *reinterpret_cast<typename X::raw *>(y + j * out_step) = X::pack(v);
            }
    }
}

// The backward pass of such planes: x and dy stay in registers between the
// sums and the elements.  A workgroup takes every so manieth image of its slab
// and keeps its channels' sums: parts[workgroup of the slab][channel][2].
// What belongs to a channel is formed by one thread and read from LDS.
// 1,024 x 2,048 x 64 bf16 with SiLU: 244 us, 3.3 TB/s of x, dy and dx.  A
// plane's x and dy take half of a CU's registers, so one workgroup has the CU
// and its loads, sums and stores take turns; reading both twice, with two to
// four workgroups to a CU, took 240 to 298 us.
template <class T, int B, int NV, int ACT>
__global__ __launch_bounds__(kMaxThreads) void grad_whole_kernel(NormArgs a) {
    typedef Vec<T, B> X;
    constexpr int V = X::n;
    extern __shared__ float lds[];
    const Shape s = a.s;
    const int t = threadIdx.x, rows = part_rows(s), wave = t >> 6, waves = blockDim.x >> 6;
    float *part = lds, *part2 = part + rows * s.slab, *m1 = part2 + rows * s.slab,
          *m2 = m1 + s.slab, *all1 = m2 + s.slab, *all2 = all1 + s.slab, *means = all2 + s.slab,
          *rstds = means + s.slab, *scales = rstds + s.slab;
    const int lane = t % s.lanes, row = t / s.lanes;
    const float inverse = 1.0f / ((float)a.pixels * a.per);
    const int count = row < s.rows && (unsigned)row < a.pixels
                          ? (int)((a.pixels - row + s.rows - 1) / s.rows) : 0;
    const unsigned at = (unsigned)xcd_contiguous(blockIdx.x, gridDim.x), spans = gridDim.x / s.slabs;
    const int first = (int)(at % s.slabs) * s.slab, c0 = first + lane * V;
    float beta[V];
#pragma unroll
    for (int i = 0; i < V; ++i) beta[i] = count && a.beta ? a.beta[c0 + i] : 0.0f;
    for (int c = t; c < s.slab; c += blockDim.x) all1[c] = all2[c] = 0.0f;
    for (size_t image = at / s.slabs; image < a.images; image += spans) {
        const char *x = a.x + image * a.x_image + (size_t)c0 * sizeof(T) + row * a.x_pixel;
        const char *dy = a.dy + image * a.dy_image + (size_t)c0 * sizeof(T) + row * a.dy_pixel;
        const size_t x_step = s.rows * a.x_pixel, dy_step = s.rows * a.dy_pixel;
        typename X::raw xr[NV], gr[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j < count) {
                xr[j] = *reinterpret_cast<const typename X::raw *>(x + j * x_step);
                gr[j] = *reinterpret_cast<const typename X::raw *>(dy + j * dy_step);
            }
        for (int c = t; c < s.slab; c += blockDim.x) {
            const size_t g = image * a.groups + (first + c) / a.per;
            const float rstd = a.rstd_in[g];
            means[c] = a.mean_in[g];
            rstds[c] = rstd;
            scales[c] = a.gamma ? rstd * a.gamma[first + c] : rstd;
        }
        __syncthreads();
        float mean[V], scale[V], su[V], sh[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            mean[i] = means[lane * V + i];
            scale[i] = scales[lane * V + i];
            su[i] = sh[i] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j < count) {
                float u[V], d[V];
                grad_terms<T, B, ACT>(xr[j], gr[j], mean, scale, beta, u, d);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    su[i] += u[i];
                    sh[i] = fmaf(u[i], d[i], sh[i]);
                }
            }
        row_sums<V>(su, s, part);
        row_sums<V>(sh, s, part2);
        __syncthreads();
        for (int c = t; c < s.slab; c += blockDim.x) {
            float one = 0.0f, two = 0.0f;
            for (int r = 0; r < rows; ++r) {
                one += part[r * s.slab + c];
                two += part2[r * s.slab + c];
            }
            two *= rstds[c];
            all1[c] += one;
            all2[c] += two;
            const float gamma = a.gamma ? a.gamma[first + c] : 1.0f;
            m1[c] = one * gamma;
            m2[c] = two * gamma;
        }
        __syncthreads();
        // dx = u rstd gamma - rstd m1 - d rstd^2 m2
        for (int g = wave; g < s.slab / a.per; g += waves) {
            const float rstd = rstds[g * a.per] * inverse;
            const float one = group_sum(m1, 1, s.slab, g * a.per, a.per) * rstd;
            const float two = group_sum(m2, 1, s.slab, g * a.per, a.per) * rstd * rstds[g * a.per];
            for (int c = t & 63; c < a.per; c += 64) {
                m1[g * a.per + c] = one;
                m2[g * a.per + c] = two;
            }
        }
        __syncthreads();
        float less[V], slope[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            less[i] = m1[lane * V + i];
            slope[i] = m2[lane * V + i];
        }
        char *dx = a.out + ((image * a.pixels + row) * a.channels + c0) * sizeof(T);
        const size_t out_step = (size_t)s.rows * a.channels * sizeof(T);
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j < count) {
                float u[V], d[V];
                grad_terms<T, B, ACT>(xr[j], gr[j], mean, scale, beta, u, d);
#pragma unroll
                for (int i = 0; i < V; ++i)
                    u[i] = fmaf(-d[i], slope[i], fmaf(u[i], scale[i], -less[i]));
                *reinterpret_cast<typename X::raw *>(dx + j * out_step) = X::pack(u);
            }
        // The next image's tables, sums and means are each written at least
        // one barrier after their last reads here.
    }
    for (int c = t; c < s.slab; c += blockDim.x) {
        float *to = a.parts + ((size_t)(at / s.slabs) * a.channels + first + c) * 2;
        to[0] = all1[c];
        to[1] = all2[c];
    }
}

// parts[rows][channels][2] summed over the rows of each of gridDim.y spans:
// to `parts` of the next level, or to dbeta and dgamma.  32 channels and 32
// rows at a time a workgroup: 4.6 us for 128 rows of 64 channels, a launch's
// time.
constexpr int kSumChannels = 32, kSumRows = 32;

__global__ __launch_bounds__(kSumChannels *kSumRows) void grad_sum_kernel(
    const float *parts, size_t rows, int channels, float *out, float *dgamma, float *dbeta) {
    __shared__ float one[kSumRows][kSumChannels], two[kSumRows][kSumChannels];
    const int lane = threadIdx.x % kSumChannels, row = threadIdx.x / kSumChannels;
    const int c = blockIdx.x * kSumChannels + lane;
    const size_t span = (rows + gridDim.y - 1) / gridDim.y, r0 = blockIdx.y * span;
    const size_t r1 = r0 + span < rows ? r0 + span : rows;
    float su = 0.0f, sh = 0.0f;
    if (c < channels)
        for (size_t r = r0 + row; r < r1; r += kSumRows) {
            su += parts[(r * channels + c) * 2];
            sh += parts[(r * channels + c) * 2 + 1];
        }
    one[row][lane] = su;
    two[row][lane] = sh;
    __syncthreads();
    for (int half = kSumRows / 2; half; half /= 2) {
        if (row < half) {
            one[row][lane] += one[row + half][lane];
            two[row][lane] += two[row + half][lane];
        }
        __syncthreads();
    }
    if (row == 0 && c < channels) {
        if (out) {
            out[((size_t)blockIdx.y * channels + c) * 2] = one[0][lane];
            out[((size_t)blockIdx.y * channels + c) * 2 + 1] = two[0][lane];
        } else {
            dbeta[c] = one[0][lane];
            dgamma[c] = two[0][lane];
        }
    }
}

// --------------------------------------------------------------------------

// A slab is whole groups; its vectors are `widest` bytes, 4 or one element, by
// what the strides, the channels and the addresses allow.  f(bytes, slab,
// lanes) sees the slabs of the widest vectors that give any.
template <class F>
void slabs_of(size_t align, int widest, int channels, int groups, int size, F f) {
    const int per = channels / groups, widths[3] = {widest, 4, size};
    for (int bytes : widths) {
        if (bytes < size || align % bytes || (size_t)channels * size % bytes) continue;
        const int v = bytes / size;
        bool any = false;
        for (int n = 1; n <= groups && n * per <= kMaxSlab; ++n)
            if (groups % n == 0 && n * per % v == 0 && n * per / v <= kMaxThreads) {
                any = true;
                f(bytes, n * per, n * per / v);
            }
        if (any) return;
    }
}

// The most vectors a thread holds: 128 bytes of x, and of dy.
constexpr int held_most(int bytes) { return bytes == 16 ? 8 : 16; }

int log2_up(size_t n) {
    int bits = 0;
    while (((size_t)1 << bits) < n) ++bits;
    return bits;
}

bool divides_wave(int lanes) { return lanes <= 64 && 64 % lanes == 0; }

// Slabs that fit the registers of a workgroup: of them the one whose runs are
// nearest to 64 bytes and that fills the CUs (4,096 x 1,024 x 64 bf16, us:
// runs of 32 bytes 317, 64 251, 128 289; gradients of 1,024 x 2,048 x 64: 283,
// 256 and more than the registers).  A workgroup too few costs more than a run of half
// a line, lanes that do not divide a wave more than both.  Vectors are four
// values: eight of 16 bits would take as many registers for a channel's
// statistics and parameters as for the data.
bool whole_shape(Shape &s, size_t align, size_t images, size_t pixels, int channels, int groups,
                 int size) {
    int best = 1 << 30;
    slabs_of(align, 4 * size, channels, groups, size, [&](int bytes, int slab, int lanes) {
        if (bytes < 4 || (size_t)(kMaxThreads / lanes) * held_most(bytes) < pixels) return;
        const size_t work = images * (channels / slab);
        const int run = slab * size;
        int cost = divides_wave(lanes) ? 0 : 16;
        if (work < 256) cost += 4 * log2_up((256 + work - 1) / work);
        cost += 3 * (run < 64 ? log2_up((64 + run - 1) / run) : log2_up((run + 63) / 64));
        if (cost >= best) return;
        best = cost;
        s.bytes = bytes;
        s.slab = slab;
        s.lanes = lanes;
    });
    if (best == 1 << 30) return false;
    s.slabs = channels / s.slab;
    // Few workgroups: more threads with fewer vectors each.
    const int most = held_most(s.bytes);
    s.whole = images * s.slabs < 512 && (size_t)(kMaxThreads / s.lanes) * 4 >= pixels ? 4 : most;
    const size_t need = ((pixels + s.whole - 1) / s.whole * s.lanes + 63) / 64 * 64;
    s.threads = (int)(need < (size_t)kMaxThreads ? need : kMaxThreads);
    s.rows = s.threads / s.lanes;
    s.fold = divides_wave(s.lanes);
    s.chunk = (unsigned)pixels;
    s.chunks = 1;
    // Backward: one workgroup of 1,024 threads to a CU, or as many threads.
    const size_t at_once = 256 * (size_t)(kMaxThreads / s.threads);
    const size_t spans = (at_once + s.slabs - 1) / s.slabs;
    s.spans = (unsigned)(spans < images ? spans : images);
    return true;
}

// Else slabs of at least 64-byte runs, in chunks of pixels.
Shape shape_of(size_t align, size_t images, size_t pixels, int channels, int groups, int size) {
    Shape s = {};
    if (whole_shape(s, align, images, pixels, channels, groups, size)) return s;
    int best = 1 << 30;
    slabs_of(align, 16, channels, groups, size, [&](int bytes, int slab, int lanes) {
        const int run = slab * size;
        const int cost = (run < 64 ? 64 / run : run / 64) + (divides_wave(lanes) ? 0 : 16);
        if (cost >= best) return;
        best = cost;
        s.bytes = bytes;
        s.slab = slab;
        s.lanes = lanes;
    });
    s.slabs = channels / s.slab;
    s.threads = s.lanes > kThreads ? kMaxThreads : kThreads;
    s.rows = s.threads / s.lanes;
    s.fold = divides_wave(s.lanes);
    const size_t sweep = (size_t)s.rows * kVectors;
    size_t sweeps = (pixels + sweep - 1) / sweep;
    sweeps = (sweeps + kMaxChunks - 1) / kMaxChunks;
    s.chunk = (unsigned)(sweeps * sweep);
    s.chunks = (unsigned)((pixels + s.chunk - 1) / s.chunk);
    return s;
}

bool sizes_ok(size_t images, size_t pixels, int channels, int groups, int dtype) {
    return images && images <= kMaxCount && pixels && pixels <= kMaxCount && channels > 0 &&
           channels <= TB_HIP_NORM_MAX_CHANNELS && groups > 0 && channels % groups == 0 &&
           channels / groups <= TB_HIP_NORM_MAX_GROUP && known_type(dtype);
}

// Rows of the second level of the parameters' sums.
constexpr size_t kSumSpans = 128, kSumDirect = 1024;

// Rows of the channels' partial sums, backward.
size_t sum_rows(size_t images, const Shape &s) { return s.whole ? s.spans : images * s.chunks; }

size_t grid_of(const NormArgs &a) {
    const size_t items = a.images * a.s.slabs * a.s.chunks;
    return items < kMaxGrid ? items : kMaxGrid;
}

size_t part_floats(const Shape &s) { return (size_t)(s.fold ? s.threads / 64 : s.rows) * s.slab; }

template <class T, int B, int ACT>
void launch_forward(const NormArgs &a, hipStream_t q) {
    const Shape &s = a.s;
    const size_t part = part_floats(s) * sizeof(float), slab = s.slab * sizeof(float);
    const unsigned grid = (unsigned)grid_of(a);
    if constexpr (B == 4 * sizeof(T) || B == 4) {
        constexpr int most = held_most(B);
        if (s.whole == 4)
            norm_whole_kernel<T, B, 4, ACT><<<grid, s.threads, 2 * part + 2 * slab, q>>>(a);
        if (s.whole == most)
            norm_whole_kernel<T, B, most, ACT><<<grid, s.threads, 2 * part + 2 * slab, q>>>(a);
        if (s.whole) return;
    }
    if constexpr (B != 8) {
        norm_parts_kernel<T, B><<<grid, s.threads, part + 3 * slab, q>>>(a);
        norm_apply_kernel<T, B, ACT><<<grid, s.threads, 2 * slab, q>>>(a);
    }
}

template <class T, int B, int ACT>
void launch_backward(const NormArgs &a, hipStream_t q) {
    const Shape &s = a.s;
    const size_t part = part_floats(s) * sizeof(float), slab = s.slab * sizeof(float);
    if constexpr (B == 4 * sizeof(T) || B == 4) {
        constexpr int most = held_most(B);
        const unsigned grid = s.spans * s.slabs;
        if (s.whole == 4)
            grad_whole_kernel<T, B, 4, ACT><<<grid, s.threads, 2 * part + 7 * slab, q>>>(a);
        if (s.whole == most)
            grad_whole_kernel<T, B, most, ACT><<<grid, s.threads, 2 * part + 7 * slab, q>>>(a);
        if (s.whole) return;
    }
    if constexpr (B != 8) {
        const unsigned grid = (unsigned)grid_of(a);
        grad_parts_kernel<T, B, ACT><<<grid, s.threads, 2 * part, q>>>(a);
        grad_apply_kernel<T, B, ACT>
            <<<grid, s.threads, 2 * slab * (1 + shares_of(s)), q>>>(a);
    }
}

struct Forward {
    template <class T, int B, int ACT>
    static void run(const NormArgs &a, hipStream_t q) { launch_forward<T, B, ACT>(a, q); }
};
struct Backward {
    template <class T, int B, int ACT>
    static void run(const NormArgs &a, hipStream_t q) { launch_backward<T, B, ACT>(a, q); }
};

template <class F, class T>
void by_width(const NormArgs &a, hipStream_t q) {
    with_act(a.act, [&](auto act) {
        constexpr int ACT = decltype(act)::value;
        switch (a.s.bytes) {
            case 16: F::template run<T, 16, ACT>(a, q); break;
            case 4: F::template run<T, 4, ACT>(a, q); break;
            default:
                if constexpr (sizeof(T) == 2) {
                    if (a.s.bytes == 8)
                        F::template run<T, 8, ACT>(a, q);
                    else
                        F::template run<T, 2, ACT>(a, q);
                }
        }
    });
}

template <class F>
void dispatch(const NormArgs &a, int dtype, hipStream_t q) {
    if (dtype == TB_HIP_F32)
        by_width<F, float>(a, q);
    else if (dtype == TB_HIP_BF16)
        by_width<F, __bf16>(a, q);
    else
        by_width<F, _Float16>(a, q);
}

// The common alignment of the addresses and strides.
size_t alignment(std::initializer_list<size_t> all) {
    size_t bits = 16;
    for (size_t v : all) bits |= v;
    return bits & (~bits + 1);
}

size_t address(const void *p) { return reinterpret_cast<uintptr_t>(p); }

}  // namespace

extern "C" size_t tb_hip_group_norm_workspace_bytes(size_t images, size_t pixels, int channels,
                                                    int groups, int dtype, int backward) {
    if (!sizes_ok(images, pixels, channels, groups, dtype)) return 0;
    const int size = type_size(dtype);
    size_t most = 0;
    for (size_t align : {size_t(16), size_t(8), size_t(4), size_t(size)}) {
        const Shape s = shape_of(align, images, pixels, channels, groups, size);
        const size_t need =
            backward ? (sum_rows(images, s) + kSumSpans) * channels : images * s.chunks * groups;
        most = need > most ? need : most;
    }
    most *= 2 * sizeof(float);
    return (most + 15) & ~size_t(15);
}

extern "C" int tb_hip_group_norm_device(const void *x, size_t image_stride, size_t pixel_stride,
                                        const float *gamma, const float *beta, void *y,
                                        float *mean, float *rstd, void *workspace,
                                        size_t images, size_t pixels, int channels, int groups,
                                        float eps, int act, int dtype, void *stream) {
    if (!x || !y || !sizes_ok(images, pixels, channels, groups, dtype) || !known_act(act) ||
        !(eps > 0.0f) || !(eps < __builtin_inff()) || !workspace || !multiple_of(workspace, 16))
        return 0;
    const int size = type_size(dtype);
    const size_t align = alignment({address(x), address(y), image_stride, pixel_stride});
    if (align % size) return 0;
    NormArgs a = {};
    a.x = static_cast<const char *>(x);
    a.x_image = image_stride;
    a.x_pixel = pixel_stride;
    a.gamma = gamma;
    a.beta = beta;
    a.out = static_cast<char *>(y);
    a.mean = mean;
    a.rstd = rstd;
    a.parts = static_cast<float *>(workspace);
    a.images = images;
    a.pixels = (unsigned)pixels;
    a.channels = channels;
    a.groups = groups;
    a.per = channels / groups;
    a.eps = eps;
    a.act = act;
    a.s = shape_of(align, images, pixels, channels, groups, size);
    (void)hipGetLastError();
    dispatch<Forward>(a, dtype, reinterpret_cast<hipStream_t>(stream));
    return hipGetLastError() == hipSuccess;
}

extern "C" int tb_hip_group_norm_backward_device(
    const void *x, size_t x_image_stride, size_t x_pixel_stride, const void *dy,
    size_t dy_image_stride, size_t dy_pixel_stride, const float *gamma, const float *beta,
    const float *mean, const float *rstd, void *dx, float *dgamma, float *dbeta,
    void *workspace, size_t images, size_t pixels, int channels, int groups, int act, int dtype,
    void *stream) {
    if (!x || !dy || !mean || !rstd || !dx || !dgamma != !dbeta ||
        !sizes_ok(images, pixels, channels, groups, dtype) || !known_act(act) || !workspace ||
        !multiple_of(workspace, 16))
        return 0;
    const int size = type_size(dtype);
    const size_t align = alignment({address(x), address(dy), address(dx), x_image_stride,
                                    x_pixel_stride, dy_image_stride, dy_pixel_stride});
    if (align % size) return 0;
    NormArgs a = {};
    a.x = static_cast<const char *>(x);
    a.x_image = x_image_stride;
    a.x_pixel = x_pixel_stride;
    a.dy = static_cast<const char *>(dy);
    a.dy_image = dy_image_stride;
    a.dy_pixel = dy_pixel_stride;
    a.gamma = gamma;
    a.beta = beta;
    a.mean_in = mean;
    a.rstd_in = rstd;
    a.out = static_cast<char *>(dx);
    a.parts = static_cast<float *>(workspace);
    a.images = images;
    a.pixels = (unsigned)pixels;
    a.channels = channels;
    a.groups = groups;
    a.per = channels / groups;
    a.act = act;
    a.s = shape_of(align, images, pixels, channels, groups, size);
    hipStream_t q = reinterpret_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    dispatch<Backward>(a, dtype, q);
    if (dgamma) {
        const unsigned tiles = (unsigned)((channels + kSumChannels - 1) / kSumChannels);
        const float *parts = a.parts;
        size_t rows = sum_rows(images, a.s);
        if (rows > kSumDirect) {
            float *next = a.parts + rows * channels * 2;
            grad_sum_kernel<<<dim3(tiles, kSumSpans), kSumChannels * kSumRows, 0, q>>>(
                parts, rows, channels, next, nullptr, nullptr);
            parts = next;
            rows = kSumSpans;
        }
        grad_sum_kernel<<<dim3(tiles, 1), kSumChannels * kSumRows, 0, q>>>(
            parts, rows, channels, nullptr, dgamma, dbeta);
    }
    return hipGetLastError() == hipSuccess;
}
