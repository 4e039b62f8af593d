// Group norm with an activation over channels-last planes, forward and
// backward (hip_layers.h).  The reference's stems normalise its planes with
// kernels of their own (groupnorm_stats, _apply and _backward of
// src/network/network_gpu.cu, channels first); here the activation is in the
// same pass and the planes are channels last, as a matrix-core convolution
// leaves them.
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
// Two launches: partial statistics of chunks of pixels, then the elements,
// each workgroup joining its image's partials first.
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

// Writes the workgroup's sums of v over the rows that fold within a wave to
// part[row][channel]; the caller synchronises.
template <int V>
__device__ __forceinline__ void row_sums(float (&v)[V], const Shape &s, float *part) {
    const int t = threadIdx.x;
    if (s.fold) {
        for (int off = s.lanes; off < 64; off *= 2)
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] += __shfl_xor(v[i], off);
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
    for (int off = 32; off; off >>= 1) v += __shfl_xor(v, off);
    return v;
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
// chunk are joined with Chan's formula.
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
template <class T, int B>
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
            for (unsigned p = w.p0 + row; p < w.p1; p += s.rows) {
                float v[V];
                X::unpack(*reinterpret_cast<const typename X::raw *>(x + p * a.x_pixel), v);
#pragma unroll
                for (int i = 0; i < V; ++i)
                    v[i] = act_of<kFine<T>>(fmaf(v[i] - mean[i], scale[i], shift[i]), a.act);
                *reinterpret_cast<typename X::raw *>(y + (size_t)p * a.channels * sizeof(T)) =
                    X::pack(v);
            }
        }
        __syncthreads();
    }
}

// u = dy act'(z) and h of one vector.
template <class T, int B>
__device__ __forceinline__ void grad_terms(typename Vec<T, B>::raw xr,
                                           typename Vec<T, B>::raw gr,
                                           const float (&mean)[Vec<T, B>::n],
                                           const float (&rstd)[Vec<T, B>::n],
                                           const float (&gamma)[Vec<T, B>::n],
                                           const float (&beta)[Vec<T, B>::n], int act,
                                           float (&u)[Vec<T, B>::n], float (&h)[Vec<T, B>::n]) {
    Vec<T, B>::unpack(xr, h);
    Vec<T, B>::unpack(gr, u);
#pragma unroll
    for (int i = 0; i < Vec<T, B>::n; ++i) {
        h[i] = (h[i] - mean[i]) * rstd[i];
        u[i] *= act_slope<kFine<T>>(fmaf(h[i], gamma[i], beta[i]), act);
    }
}

// A thread's channels: statistics and parameters.
template <int V>
struct Channels {
    float mean[V], rstd[V], gamma[V], beta[V];
    __device__ __forceinline__ void load(const NormArgs &a, size_t image, int c0) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const size_t g = image * a.groups + (c0 + i) / a.per;
            mean[i] = a.mean_in[g];
            rstd[i] = a.rstd_in[g];
            gamma[i] = a.gamma ? a.gamma[c0 + i] : 1.0f;
            beta[i] = a.beta ? a.beta[c0 + i] : 0.0f;
        }
    }
};

// The sums of u and u h of every channel over one chunk:
// parts[(image, chunk)][channel][2].
template <class T, int B>
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
            for (unsigned p = w.p0 + row; p < w.p1; p += s.rows) {
                float u[V], h[V];
                grad_terms<T, B>(*reinterpret_cast<const typename X::raw *>(x + p * a.x_pixel),
                                 *reinterpret_cast<const typename X::raw *>(dy + p * a.dy_pixel),
                                 ch.mean, ch.rstd, ch.gamma, ch.beta, a.act, u, h);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    su[i] += u[i];
                    sh[i] = fmaf(u[i], h[i], sh[i]);
                }
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
            float *at = a.parts + (w.chunk * a.channels + w.c0 + c) * 2;
            at[0] = one;
            at[1] = two;
        }
        __syncthreads();
    }
}

template <class T, int B>
__global__ __launch_bounds__(kMaxThreads) void grad_apply_kernel(NormArgs a) {
    typedef Vec<T, B> X;
    constexpr int V = X::n;
    extern __shared__ float lds[];
    const Shape s = a.s;
    const int t = threadIdx.x, wave = t >> 6, waves = blockDim.x >> 6;
    float *m1 = lds, *m2 = lds + s.slab;
    const int lane = t % s.lanes, row = t / s.lanes;
    const size_t items = a.images * s.slabs * s.chunks;
    const float inverse = 1.0f / ((float)a.pixels * a.per);
    for (size_t item = blockIdx.x; item < items; item += gridDim.x) {
        const Place w = place_of(a, xcd_contiguous(item, items));
        for (int c = t; c < s.slab; c += blockDim.x) {
            const float *at = a.parts + (w.image * s.chunks * a.channels + w.c0 + c) * 2;
            float one = 0.0f, two = 0.0f;
            for (unsigned i = 0; i < s.chunks; ++i) {
                one += at[(size_t)i * a.channels * 2];
                two += at[(size_t)i * a.channels * 2 + 1];
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
            for (unsigned p = w.p0 + row; p < w.p1; p += s.rows) {
                float u[V], h[V];
                grad_terms<T, B>(*reinterpret_cast<const typename X::raw *>(x + p * a.x_pixel),
                                 *reinterpret_cast<const typename X::raw *>(dy + p * a.dy_pixel),
                                 ch.mean, ch.rstd, ch.gamma, ch.beta, a.act, u, h);
#pragma unroll
                for (int i = 0; i < V; ++i)
                    u[i] = ch.rstd[i] * (fmaf(u[i], ch.gamma[i], -m1[lane * V + i]) -
                                         h[i] * m2[lane * V + i]);
                *reinterpret_cast<typename X::raw *>(dx + (size_t)p * a.channels * sizeof(T)) =
                    X::pack(u);
            }
        }
        __syncthreads();
    }
}

// parts[rows][channels][2] summed over the rows of each of gridDim.y spans:
// to `parts` of the next level, or to dbeta and dgamma.  32 channels and 32
// rows at a time a workgroup.
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

// The slab is the fewest whole groups whose vectors fill 64-byte runs, with
// lanes that divide a wave where there are such.  Vectors are 16 bytes, 4 or
// one element, by what the strides, the channels and the addresses allow.
Shape shape_of(size_t align, size_t pixels, int channels, int groups, int size) {
    Shape s = {};
    const int per = channels / groups;
    const int widths[3] = {16, 4, size};
    for (int bytes : widths) {
        if (bytes < size || align % bytes || (size_t)channels * size % bytes) continue;
        const int v = bytes / size;
        int best = 1 << 30;
        for (int n = 1; n <= groups; ++n) {
            const int slab = n * per;
            if (slab > kMaxSlab) break;
            if (groups % n || slab % v || slab / v > kMaxThreads) continue;
            const int lanes = slab / v, run = slab * size;
            int cost = run < 64 ? 64 / run : run / 64;
            if (lanes > 64 || 64 % lanes) cost += 16;
            if (cost < best) {
                best = cost;
                s.bytes = bytes;
                s.slab = slab;
                s.lanes = lanes;
            }
        }
        if (s.slab) break;
    }
    s.slabs = channels / s.slab;
    s.threads = s.lanes > kThreads ? kMaxThreads : kThreads;
    s.rows = s.threads / s.lanes;
    s.fold = s.lanes <= 64 && 64 % s.lanes == 0;
    const size_t sweep = (size_t)s.rows * kVectors;
    size_t sweeps = (pixels + sweep - 1) / sweep;
    sweeps = (sweeps + kMaxChunks - 1) / kMaxChunks;
    s.chunk = (unsigned)(sweeps * sweep);
    s.chunks = (unsigned)((pixels + s.chunk - 1) / s.chunk);
    return s;
}

bool sizes_ok(size_t images, size_t pixels, int channels, int groups, int dtype) {
    return images && images <= kMaxCount && pixels && pixels <= kMaxCount && channels > 0 &&
           channels <= TB_HIP_NORM_MAX_CHANNELS && groups > 0 && channels % groups == 0 && channels / groups <= TB_HIP_NORM_MAX_GROUP &&
           known_type(dtype);
}

// Rows of the second level of the parameters' sums.
constexpr size_t kSumSpans = 128, kSumDirect = 1024;

size_t part_bytes(size_t images, const Shape &s, int columns) {
    return images * s.chunks * columns * 2 * sizeof(float);
}

size_t grid_of(const NormArgs &a) {
    const size_t items = a.images * a.s.slabs * a.s.chunks;
    return items < kMaxGrid ? items : kMaxGrid;
}

template <class T, int B>
void forward(const NormArgs &a, hipStream_t q) {
    const Shape &s = a.s;
    const int rows = s.fold ? s.threads / 64 : s.rows;
    const size_t lds = ((size_t)rows * s.slab + 3 * s.slab) * sizeof(float);
    norm_parts_kernel<T, B><<<(unsigned)grid_of(a), s.threads, lds, q>>>(a);
    norm_apply_kernel<T, B>
        <<<(unsigned)grid_of(a), s.threads, 2 * s.slab * sizeof(float), q>>>(a);
}

template <class T, int B>
void backward(const NormArgs &a, hipStream_t q) {
    const Shape &s = a.s;
    const int rows = s.fold ? s.threads / 64 : s.rows;
    grad_parts_kernel<T, B>
        <<<(unsigned)grid_of(a), s.threads, (size_t)2 * rows * s.slab * sizeof(float), q>>>(a);
    grad_apply_kernel<T, B>
        <<<(unsigned)grid_of(a), s.threads, 2 * s.slab * sizeof(float), q>>>(a);
}

struct Forward {
    template <class T, int B>
    static void run(const NormArgs &a, hipStream_t q) { forward<T, B>(a, q); }
};
struct Backward {
    template <class T, int B>
    static void run(const NormArgs &a, hipStream_t q) { backward<T, B>(a, q); }
};

template <class F>
void dispatch(const NormArgs &a, int dtype, hipStream_t q) {
    const int b = a.s.bytes;
    if (dtype == TB_HIP_F32)
        b == 16 ? F::template run<float, 16>(a, q) : F::template run<float, 4>(a, q);
    else if (dtype == TB_HIP_BF16)
        b == 16  ? F::template run<__bf16, 16>(a, q)
        : b == 4 ? F::template run<__bf16, 4>(a, q)
                 : F::template run<__bf16, 2>(a, q);
    else
        b == 16  ? F::template run<_Float16, 16>(a, q)
        : b == 4 ? F::template run<_Float16, 4>(a, q)
                 : F::template run<_Float16, 2>(a, q);
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
    for (size_t align : {size_t(16), size_t(4), size_t(size)}) {
        const Shape s = shape_of(align, pixels, channels, groups, size);
        const size_t need = backward ? part_bytes(images, s, channels) +
                                           kSumSpans * channels * 2 * sizeof(float)
                                     : part_bytes(images, s, groups);
        most = need > most ? need : most;
    }
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
    a.s = shape_of(align, pixels, channels, groups, size);
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
    a.s = shape_of(align, pixels, channels, groups, size);
    hipStream_t q = reinterpret_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    dispatch<Backward>(a, dtype, q);
    if (dgamma) {
        const unsigned tiles = (unsigned)((channels + kSumChannels - 1) / kSumChannels);
        const float *parts = a.parts;
        size_t rows = images * a.s.chunks;
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
