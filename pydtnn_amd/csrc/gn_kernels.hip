// Group normalisation with an activation, forward and backward.
//
// x is (images, pixels, channels) channels last, or (images, channels, pixels).  A group is cg consecutive channels
// over all pixels of an image; with M = cg * pixels and sums over a group
//   mean = sum(x) / M     var = sum((x - mean)^2) / M     inv_std = 1 / sqrt(var + eps)
//   xn = (x - mean) inv_std     z = gamma xn + beta     y = act(z)
//   dz = dy act'(z)     dgamma = sum over images and pixels of dz xn     dbeta = the same of dz
//   dx = inv_std (gamma dz - A - xn B),   A = sum(gamma dz) / M,   B = sum(gamma dz xn) / M
// The backward pass keeps nothing of the forward pass but x and the two statistics of each group: xn and z are
// computed again.  Both passes are bound by memory: forward reads x and writes y, backward reads x and dy and writes dx.
//
// Every pass is two steps: sums of pieces of each group, then the map with the joined sums.  Sums are held in 32 bits
// (64 for double), as (mean, sum of squared differences from it) of a piece, and pieces are joined in double through
// their common mean, so that a mean far from zero costs no digits of the variance.
#include <cmath>
#include "../../include/pydtnn_hip.h"
#include "conv_internal.h"
#include "dtypes.h"

namespace {

constexpr int kT = 256;
constexpr int kWave = 64;
constexpr int kWaves = kT / kWave;

enum { kIdentity = 0, kRelu = 1, kSilu = 2 };

__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }

template <int ACT, typename A>
__device__ __forceinline__ A act(A z)
{
    if (ACT == kRelu) return z > (A)0 ? z : (A)0;
    if (ACT == kSilu) return z / ((A)1 + exp_of(-z));
    return z;
}

template <typename A>
__device__ __forceinline__ A wave_sum(A v)
{
#pragma unroll
    for (int o = kWave / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    return v;
}

// A group's sums as pieces of them are stored: the mean of a piece and the sum of (x - mean)^2 over it.
template <typename A>
struct Moments {
    A mean, m2;
};

// ---------------------------------------------------------------------------------------------- channels last
// A workgroup takes a slab of whole groups (slab_groups of them, `width` channels) of one image and a run of its pixels.
// Its threads stand as `rows` pixels by `tx` packs of V channels; a slab wider than that (a single very wide group, or
// groups that no pack divides) is walked in steps of tx * V channels.
struct GnLast {
    long images;
    int pixels, channels, groups, cg;
    int slab_groups, width, slabs;     // groups and channels of a slab, slabs of an image
    int tx, rows;
    int splits, run;                   // runs of pixels of an image, pixels of a run
};

struct Place {
    long image;
    int slab, split, p0, p1, tx, ty;
};

__device__ __forceinline__ Place place_of(const GnLast& g)
{
    Place at;
    const unsigned b = blockIdx.x, per = (unsigned)(g.slabs * g.splits);
    at.image = b / per;
    const unsigned r = b % per;
    at.slab = r / g.splits;
    at.split = r % g.splits;
    at.p0 = at.split * g.run;
    at.p1 = min(at.p0 + g.run, g.pixels);
    at.tx = threadIdx.x % g.tx;
    at.ty = threadIdx.x / g.tx;
    return at;
}

// The moments of each group's piece: partial[(image * groups + group) * splits + split].
template <typename T, int V>
__global__ void __launch_bounds__(kT) gn_last_moments(const T* __restrict__ x, Moments<wide_t<T>>* __restrict__ partial,
                                                      GnLast g)
{
    using A = wide_t<T>;
    __shared__ A part_mean[kT * V], part_m2[kT * V];
    __shared__ int part_n[kT];
    const Place at = place_of(g);
    const T* base = x + (at.image * g.pixels) * g.channels + at.slab * g.width;
    // differences from the thread's own first value keep the sums small
    A first[V], s1[V] = {}, s2[V] = {};
    int n = 0;
    if (at.ty < g.rows) {
        for (int c = at.tx * V; c < g.width; c += g.tx * V) {
            for (int p = at.p0 + at.ty; p < at.p1; p += g.rows) {
                const Pack<T, V> v = *reinterpret_cast<const Pack<T, V>*>(base + (long)p * g.channels + c);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    if (n == 0) first[j] = (A)v.v[j];
                    const A d = (A)v.v[j] - first[j];
                    s1[j] += d;
                    s2[j] += d * d;
                }
                ++n;
            }
        }
    }
    part_n[threadIdx.x] = n;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const A m = n ? s1[j] / (A)n : (A)0;
        part_mean[threadIdx.x * V + j] = n ? first[j] + m : (A)0;
        part_m2[threadIdx.x * V + j] = n ? s2[j] - s1[j] * m : (A)0;
    }
    __syncthreads();
    // a group's channels are every column of a slab that is one group, else columns k cg .. of each row
    const int columns = g.tx * V, mine = g.slab_groups == 1 ? columns : g.cg;
    for (int k = threadIdx.x / kWave; k < g.slab_groups; k += kWaves) {
        const int entries = mine * g.rows;
        double count = 0, sum = 0, m2 = 0;
        for (int e = threadIdx.x % kWave; e < entries; e += kWave) {
            const int i = (e / mine) * columns + k * mine + e % mine;
            count += part_n[i / V];
            sum += part_n[i / V] * (double)part_mean[i];
        }
        count = wave_sum(count);
        const double mean = wave_sum(sum) / count;
        for (int e = threadIdx.x % kWave; e < entries; e += kWave) {
            const int i = (e / mine) * columns + k * mine + e % mine;
            const double d = (double)part_mean[i] - mean;
            m2 += part_n[i / V] * d * d + (double)part_m2[i];
        }
        m2 = wave_sum(m2);
        if (threadIdx.x % kWave == 0) {
            const long group = at.image * g.groups + at.slab * g.slab_groups + k;
            partial[group * g.splits + at.split] = Moments<A>{(A)mean, (A)m2};
        }
    }
}

// Mean and 1/std of one group from the moments of its pieces, `run_of(i)` elements each.
template <typename A, typename F>
__device__ __forceinline__ void join_moments(const Moments<A>* part, int pieces, F run_of, double m, double eps, A* mean_out,
                                             A* inv_std_out)
{
    double sum = 0, m2 = 0;
    for (int i = 0; i < pieces; ++i) sum += run_of(i) * (double)part[i].mean;
    const double mean = sum / m;
    for (int i = 0; i < pieces; ++i) {
        const double d = (double)part[i].mean - mean;
        m2 += run_of(i) * d * d + (double)part[i].m2;
    }
    *mean_out = (A)mean;
    *inv_std_out = (A)(1.0 / sqrt(m2 / m + eps));
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kT) gn_last_apply(const T* __restrict__ x, const wide_t<T>* __restrict__ gamma,
                                                    const wide_t<T>* __restrict__ beta,
                                                    const Moments<wide_t<T>>* __restrict__ partial, T* __restrict__ y,
                                                    wide_t<T>* __restrict__ mean_out, wide_t<T>* __restrict__ inv_std_out,
                                                    double eps, GnLast g)
{
    using A = wide_t<T>;
    __shared__ A mean[kT * V], inv_std[kT * V];      // of the slab's groups: at most a group to a column
    const Place at = place_of(g);
    for (int k = threadIdx.x; k < g.slab_groups; k += kT) {
        const long group = at.image * g.groups + at.slab * g.slab_groups + k;
        join_moments<A>(partial + group * g.splits, g.splits,
                        [&](int i) { return (double)(min(g.run, g.pixels - i * g.run)) * g.cg; },
                        (double)g.pixels * g.cg, eps, &mean[k], &inv_std[k]);
        if (at.split == 0) {
            mean_out[group] = mean[k];
            inv_std_out[group] = inv_std[k];
        }
    }
    __syncthreads();
    if (at.ty >= g.rows) return;
    const long base = (at.image * g.pixels) * g.channels + at.slab * g.width;
    for (int c = at.tx * V; c < g.width; c += g.tx * V) {
        A mu[V], scale[V], shift[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int k = (c + j) / g.cg, ch = at.slab * g.width + c + j;
            mu[j] = mean[k];
            scale[j] = inv_std[k] * gamma[ch];
            shift[j] = beta[ch];
        }
        for (int p = at.p0 + at.ty; p < at.p1; p += g.rows) {
            const long i = base + (long)p * g.channels + c;
            Pack<T, V> v = *reinterpret_cast<const Pack<T, V>*>(x + i);
#pragma unroll
            for (int j = 0; j < V; ++j) v.v[j] = (T)act<ACT>(((A)v.v[j] - mu[j]) * scale[j] + shift[j]);
            *reinterpret_cast<Pack<T, V>*>(y + i) = v;
        }
    }
}

// What the backward pass needs of a channel of an image to compute dz from x and dy.
//
// The rectifier's border is decided exactly: z > 0 is x beyond mean - beta / (gamma inv_std), a number that is computed in
// double and rounded down, since for the x of its type "greater than the number" and "greater than the number rounded down"
// are the same.  A sign of gamma other than plus turns the comparison round through `sign`.
template <typename A>
struct ChanBwd {
    A mean, inv_std, gamma, beta, border, sign;
};

// The largest float that is not above v.
__device__ __forceinline__ float round_down(double v, float)
{
    const float f = (float)v;
    if (!((double)f > v)) return f;
    const int bits = __float_as_int(f);
    return __int_as_float(f > 0.0f ? bits - 1 : f < 0.0f ? bits + 1 : (int)0x80000001);
}
__device__ __forceinline__ double round_down(double v, double) { return v; }

template <int ACT, typename A>
__device__ __forceinline__ ChanBwd<A> chan_bwd(A mean, A inv_std, A gamma, A beta)
{
    ChanBwd<A> c = {mean, inv_std, gamma, beta, (A)0, (A)1};
    if (ACT == kRelu) {
        const double slope = (double)gamma * (double)inv_std;
        c.sign = gamma < (A)0 ? (A)-1 : (A)1;
        if (slope != 0.0) c.border = round_down((double)c.sign * ((double)mean - (double)beta / slope), (A)0);
        else c.border = beta > (A)0 ? -(A)INFINITY : (A)INFINITY;
    }
    return c;
}

template <int ACT, typename A>
__device__ __forceinline__ A dz_of(const ChanBwd<A>& c, A x, A xn, A dy)
{
    if (ACT == kRelu) return x * c.sign > c.border ? dy : (A)0;
    if (ACT == kSilu) {
        const A z = xn * c.gamma + c.beta, p = (A)1 / ((A)1 + exp_of(-z));
        return dy * (p * ((A)1 + z * ((A)1 - p)));
    }
    return dy;
}

// inv_std (gamma dz - A - xn B).  Without contraction: where a group is one element, gamma dz - A is exactly zero.
template <typename A>
__device__ __forceinline__ A dx_of(const ChanBwd<A>& c, A xn, A dz, A a, A b)
{
#pragma clang fp contract(off)
    const A g = c.gamma * dz;
    return c.inv_std * ((g - a) - xn * b);
}

// Sums of dz and dz xn over a run's pixels: sums[(image * splits + split) * channels + channel], then the same of dz xn.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kT) gn_last_bwd_sums(const T* __restrict__ dy, const T* __restrict__ x,
                                                       const wide_t<T>* __restrict__ gamma,
                                                       const wide_t<T>* __restrict__ beta,
                                                       const wide_t<T>* __restrict__ mean,
                                                       const wide_t<T>* __restrict__ inv_std,
                                                       wide_t<T>* __restrict__ sums, GnLast g)
{
    using A = wide_t<T>;
    __shared__ A part1[kT * V], part2[kT * V];
    const Place at = place_of(g);
    const long base = (at.image * g.pixels) * g.channels + at.slab * g.width;
    A* out1 = sums + (at.image * g.splits + at.split) * g.channels + at.slab * g.width;
    A* out2 = out1 + g.images * g.splits * g.channels;
    const int columns = g.tx * V;
    for (int c0 = 0; c0 < g.width; c0 += columns) {
        const int c = c0 + at.tx * V;
        A s1[V] = {}, s2[V] = {};
        if (at.ty < g.rows && c < g.width) {
            ChanBwd<A> ch[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int i = at.slab * g.width + c + j;
                const long group = at.image * g.groups + i / g.cg;
                ch[j] = chan_bwd<ACT>(mean[group], inv_std[group], gamma[i], beta[i]);
            }
            for (int p = at.p0 + at.ty; p < at.p1; p += g.rows) {
                const long i = base + (long)p * g.channels + c;
                const Pack<T, V> xv = *reinterpret_cast<const Pack<T, V>*>(x + i);
                const Pack<T, V> dv = *reinterpret_cast<const Pack<T, V>*>(dy + i);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const A xn = ((A)xv.v[j] - ch[j].mean) * ch[j].inv_std;
                    const A dz = dz_of<ACT>(ch[j], (A)xv.v[j], xn, (A)dv.v[j]);
                    s1[j] += dz;
                    s2[j] += dz * xn;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            part1[threadIdx.x * V + j] = s1[j];
            part2[threadIdx.x * V + j] = s2[j];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < min(columns, g.width - c0); i += kT) {
            A t1 = (A)0, t2 = (A)0;
            for (int r = 0; r < g.rows; ++r) {
                t1 += part1[r * columns + i];
                t2 += part2[r * columns + i];
            }
            out1[c0 + i] = t1;
            out2[c0 + i] = t2;
        }
        __syncthreads();
    }
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kT) gn_last_bwd_apply(const T* __restrict__ dy, const T* __restrict__ x,
                                                        const wide_t<T>* __restrict__ gamma,
                                                        const wide_t<T>* __restrict__ beta,
                                                        const wide_t<T>* __restrict__ mean,
                                                        const wide_t<T>* __restrict__ inv_std,
                                                        const wide_t<T>* __restrict__ ab, T* __restrict__ dx, GnLast g)
{
    using A = wide_t<T>;
    const Place at = place_of(g);
    if (at.ty >= g.rows) return;
    const long base = (at.image * g.pixels) * g.channels + at.slab * g.width;
    for (int c = at.tx * V; c < g.width; c += g.tx * V) {
        ChanBwd<A> ch[V];
        A a[V], b[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int i = at.slab * g.width + c + j;
            const long group = at.image * g.groups + i / g.cg;
            ch[j] = chan_bwd<ACT>(mean[group], inv_std[group], gamma[i], beta[i]);
            a[j] = ab[2 * group];
            b[j] = ab[2 * group + 1];
        }
        for (int p = at.p0 + at.ty; p < at.p1; p += g.rows) {
            const long i = base + (long)p * g.channels + c;
            const Pack<T, V> xv = *reinterpret_cast<const Pack<T, V>*>(x + i);
            Pack<T, V> dv = *reinterpret_cast<const Pack<T, V>*>(dy + i);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const A xn = ((A)xv.v[j] - ch[j].mean) * ch[j].inv_std;
                const A dz = dz_of<ACT>(ch[j], (A)xv.v[j], xn, (A)dv.v[j]);
                dv.v[j] = (T)dx_of(ch[j], xn, dz, a[j], b[j]);
            }
            *reinterpret_cast<Pack<T, V>*>(dx + i) = dv;
        }
    }
}

// ---------------------------------------------------------------------------------------------- channels first
// A wave, or a workgroup where planes are large, takes a plane: one channel of one image.
template <typename T, int THREADS>
__device__ __forceinline__ wide_t<T> plane_sum(wide_t<T> v, wide_t<T>* part)
{
    v = wave_sum(v);
    if (THREADS == kWave) return v;
    __syncthreads();
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += part[w];
    return v;
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(kT) gn_first_moments(const T* __restrict__ x, Moments<wide_t<T>>* __restrict__ partial,
                                                       long planes, int pixels)
{
    using A = wide_t<T>;
    __shared__ A part[kWaves];
    const long plane = (long)blockIdx.x * (kT / THREADS) + threadIdx.x / THREADS;
    if (plane >= planes) return;
    const T* base = x + plane * pixels;
    const A first = (A)base[0];
    A s1 = (A)0;
    for (int p = threadIdx.x % THREADS; p < pixels; p += THREADS) s1 += (A)base[p] - first;
    const A mean = first + plane_sum<T, THREADS>(s1, part) / (A)pixels;
    A s2 = (A)0;
    for (int p = threadIdx.x % THREADS; p < pixels; p += THREADS) {
        const A d = (A)base[p] - mean;
        s2 += d * d;
    }
    s2 = plane_sum<T, THREADS>(s2, part);
    if (threadIdx.x % THREADS == 0) partial[plane] = Moments<A>{mean, s2};
}

template <typename T, int THREADS, int ACT>
__global__ void __launch_bounds__(kT) gn_first_apply(const T* __restrict__ x, const wide_t<T>* __restrict__ gamma,
                                                     const wide_t<T>* __restrict__ beta,
                                                     const Moments<wide_t<T>>* __restrict__ partial, T* __restrict__ y,
                                                     wide_t<T>* __restrict__ mean_out, wide_t<T>* __restrict__ inv_std_out,
                                                     double eps, long planes, int pixels, int channels, int cg)
{
    using A = wide_t<T>;
    const long plane = (long)blockIdx.x * (kT / THREADS) + threadIdx.x / THREADS;
    if (plane >= planes) return;
    const long group = plane / cg;
    const int c = (int)(plane % channels);
    A mean, inv_std;
    join_moments<A>(partial + group * cg, cg, [&](int) { return (double)pixels; }, (double)pixels * cg, eps, &mean, &inv_std);
    if (plane % cg == 0 && threadIdx.x % THREADS == 0) {
        mean_out[group] = mean;
        inv_std_out[group] = inv_std;
    }
    const A scale = inv_std * gamma[c], shift = beta[c];
    for (int p = threadIdx.x % THREADS; p < pixels; p += THREADS) {
        const long i = plane * pixels + p;
        y[i] = (T)act<ACT>(((A)x[i] - mean) * scale + shift);
    }
}

template <typename T, int THREADS, int ACT>
__global__ void __launch_bounds__(kT) gn_first_bwd_sums(const T* __restrict__ dy, const T* __restrict__ x,
                                                        const wide_t<T>* __restrict__ gamma,
                                                        const wide_t<T>* __restrict__ beta,
                                                        const wide_t<T>* __restrict__ mean,
                                                        const wide_t<T>* __restrict__ inv_std,
                                                        wide_t<T>* __restrict__ sums, long planes, int pixels, int channels,
                                                        int cg)
{
    using A = wide_t<T>;
    __shared__ A part[kWaves];
    const long plane = (long)blockIdx.x * (kT / THREADS) + threadIdx.x / THREADS;
    if (plane >= planes) return;
    const int c = (int)(plane % channels);
    const ChanBwd<A> ch = chan_bwd<ACT>(mean[plane / cg], inv_std[plane / cg], gamma[c], beta[c]);
    A s1 = (A)0, s2 = (A)0;
    for (int p = threadIdx.x % THREADS; p < pixels; p += THREADS) {
        const long i = plane * pixels + p;
        const A xn = ((A)x[i] - ch.mean) * ch.inv_std;
        const A dz = dz_of<ACT>(ch, (A)x[i], xn, (A)dy[i]);
        s1 += dz;
        s2 += dz * xn;
    }
    s1 = plane_sum<T, THREADS>(s1, part);
    s2 = plane_sum<T, THREADS>(s2, part);
    if (threadIdx.x % THREADS == 0) {
        sums[plane] = s1;
        sums[planes + plane] = s2;
    }
}

template <typename T, int THREADS, int ACT>
__global__ void __launch_bounds__(kT) gn_first_bwd_apply(const T* __restrict__ dy, const T* __restrict__ x,
                                                         const wide_t<T>* __restrict__ gamma,
                                                         const wide_t<T>* __restrict__ beta,
                                                         const wide_t<T>* __restrict__ mean,
                                                         const wide_t<T>* __restrict__ inv_std,
                                                         const wide_t<T>* __restrict__ ab, T* __restrict__ dx, long planes,
                                                         int pixels, int channels, int cg)
{
    using A = wide_t<T>;
    const long plane = (long)blockIdx.x * (kT / THREADS) + threadIdx.x / THREADS;
    if (plane >= planes) return;
    const int c = (int)(plane % channels);
    const long group = plane / cg;
    const ChanBwd<A> ch = chan_bwd<ACT>(mean[group], inv_std[group], gamma[c], beta[c]);
    const A a = ab[2 * group], b = ab[2 * group + 1];
    for (int p = threadIdx.x % THREADS; p < pixels; p += THREADS) {
        const long i = plane * pixels + p;
        const A xn = ((A)x[i] - ch.mean) * ch.inv_std;
        dx[i] = (T)dx_of(ch, xn, dz_of<ACT>(ch, (A)x[i], xn, (A)dy[i]), a, b);
    }
}

// ---------------------------------------------------------------------------------------------- joining the sums
// A and B of each group from the channel sums of its runs: one wave a group.
template <typename A>
__global__ void __launch_bounds__(kT) gn_bwd_groups(const A* __restrict__ sums, const A* __restrict__ gamma,
                                                    A* __restrict__ ab, long images, int splits, int channels, int groups,
                                                    double m)
{
    const long group = (long)blockIdx.x * kWaves + threadIdx.x / kWave;
    if (group >= images * groups) return;
    const int cg = channels / groups, c0 = (int)(group % groups) * cg;
    const A* s1 = sums + (group / groups) * splits * channels;
    const A* s2 = s1 + images * splits * channels;
    double a = 0, b = 0;
    for (int c = c0 + threadIdx.x % kWave; c < c0 + cg; c += kWave) {
        double t1 = 0, t2 = 0;
        for (int s = 0; s < splits; ++s) {
            t1 += (double)s1[(long)s * channels + c];
            t2 += (double)s2[(long)s * channels + c];
        }
        a += t1 * (double)gamma[c];
        b += t2 * (double)gamma[c];
    }
    a = wave_sum(a);
    b = wave_sum(b);
    if (threadIdx.x % kWave == 0) {
        ab[2 * group] = (A)(a / m);
        ab[2 * group + 1] = (A)(b / m);
    }
}

// dgamma and dbeta: the channel sums over images and runs.  A workgroup takes 16 channels, 16 threads each.
template <typename A>
__global__ void __launch_bounds__(kT) gn_bwd_params(const A* __restrict__ sums, A* __restrict__ dgamma,
                                                    A* __restrict__ dbeta, long pieces, int channels)
{
    __shared__ double part1[kT], part2[kT];
    const int c = blockIdx.x * 16 + threadIdx.x % 16, r = threadIdx.x / 16;
    double t1 = 0, t2 = 0;
    if (c < channels) {
        for (long i = r; i < pieces; i += 16) {
            t1 += (double)sums[i * channels + c];
            t2 += (double)sums[(pieces + i) * channels + c];
        }
    }
    part1[threadIdx.x] = t1;
    part2[threadIdx.x] = t2;
    __syncthreads();
    if (r == 0 && c < channels) {
        for (int k = 1; k < 16; ++k) {
            t1 += part1[k * 16 + threadIdx.x];
            t2 += part2[k * 16 + threadIdx.x];
        }
        dbeta[c] = (A)t1;
        dgamma[c] = (A)t2;
    }
}

// ---------------------------------------------------------------------------------------------- host
// The largest pack of consecutive channels that 16 bytes hold and that divides the channels (and, where a slab is not
// all of the channels, the channels of a group, so that slabs start on packs).
int pack_of(int size, int channels, int cg)
{
    int v = 16 / size;
    while (v > 1 && (channels % v || (channels / v > kT && cg % v))) v /= 2;
    return v;
}

GnLast last_shape(long images, int channels, int pixels, int groups, int v)
{
    GnLast g;
    g.images = images;
    g.pixels = pixels;
    g.channels = channels;
    g.groups = groups;
    g.cg = channels / groups;
    // as many whole groups as the threads have columns for, or one
    g.slab_groups = groups;
    if (channels > kT * v) {
        g.slab_groups = kT * v / g.cg > 0 ? kT * v / g.cg : 1;
        while (groups % g.slab_groups) --g.slab_groups;
    }
    g.width = g.slab_groups * g.cg;
    g.slabs = groups / g.slab_groups;
    const int packs = g.width / v;
    g.tx = packs < kT ? packs : kT;
    g.rows = kT / g.tx;
    // about eight workgroups to each of 256 compute units, and at least eight pixels to a thread
    long want = (2048 + images * g.slabs - 1) / (images * g.slabs);
    const long most = (pixels + 8l * g.rows - 1) / (8l * g.rows);
    if (want > most) want = most;
    g.run = (int)((pixels + want - 1) / want);
    g.splits = (pixels + g.run - 1) / g.run;
    return g;
}

int check(long images, long channels, long pixels, long groups)
{
    if (images <= 0 || channels <= 0 || pixels <= 0 || groups <= 0 || channels % groups) return PYDTNN_HIP_ERR_INVALID;
    // runs and planes are counted in 32 bits
    if (pixels > (1l << 30) || channels > (1l << 30) || images > (1l << 40) / channels) return PYDTNN_HIP_ERR_UNSUPPORTED;
    return PYDTNN_HIP_OK;
}

int size_of(int dtype) { return dtype == kDtypeF64 ? 8 : dtype == kDtypeF32 ? 4 : 2; }

struct Pieces {
    long moments, sums;      // moments of the forward pass, channel sums (of each kind) of the backward pass
    size_t wide;
};

// `v` is a pack that the tensors' addresses allow or a larger one: pieces depend on it, so the query asks for both.
Pieces pieces_of(int dtype, int nhwc, long images, int channels, int pixels, int groups, int v)
{
    Pieces p;
    p.wide = dtype == kDtypeF64 ? 8 : 4;
    if (nhwc) {
        const GnLast g = last_shape(images, channels, pixels, groups, v);
        p.moments = images * groups * g.splits;
        p.sums = images * g.splits * channels;
    } else {
        p.moments = p.sums = images * channels;
    }
    return p;
}

size_t workspace_of(const Pieces& p, long images, int groups, bool backward)
{
    return (backward ? 2 * p.sums + 2 * images * groups : 2 * p.moments) * p.wide;
}

template <typename F>
int with_act(int activation, F f)
{
    switch (activation) {
        case kIdentity: return f(std::integral_constant<int, kIdentity>());
        case kRelu: return f(std::integral_constant<int, kRelu>());
        case kSilu: return f(std::integral_constant<int, kSilu>());
        default: return PYDTNN_HIP_ERR_INVALID;
    }
}

template <typename F>
int with_pack(int v, F f)
{
    switch (v) {
        case 8: return f(std::integral_constant<int, 8>());
        case 4: return f(std::integral_constant<int, 4>());
        case 2: return f(std::integral_constant<int, 2>());
        default: return f(std::integral_constant<int, 1>());
    }
}

bool too_many(long blocks) { return blocks * kT >= (1l << 32); }      // a launch counts its threads in 32 bits

// Planes of fewer pixels than this go to a wave each.
constexpr int kPlaneOfGroup = 1024;

template <typename T, int ACT>
int forward(int nhwc, const T* x, const wide_t<T>* gamma, const wide_t<T>* beta, T* y, wide_t<T>* mean, wide_t<T>* inv_std,
            long images, int channels, int pixels, int groups, double eps, void* workspace, hipStream_t st)
{
    using A = wide_t<T>;
    Moments<A>* part = static_cast<Moments<A>*>(workspace);
    if (nhwc) {
        const int v = aligned16(x) && aligned16(y) ? pack_of(sizeof(T), channels, channels / groups) : 1;
        const GnLast g = last_shape(images, channels, pixels, groups, v);
        const long blocks = images * g.slabs * g.splits;
        if (too_many(blocks)) return PYDTNN_HIP_ERR_UNSUPPORTED;
        return with_pack(v, [&](auto pack) {
            constexpr int V = decltype(pack)::value * sizeof(T) <= 16 ? decltype(pack)::value : 1;
            hipLaunchKernelGGL((gn_last_moments<T, V>), dim3((unsigned)blocks), dim3(kT), 0, st, x, part, g);
            hipLaunchKernelGGL((gn_last_apply<T, V, ACT>), dim3((unsigned)blocks), dim3(kT), 0, st, x, gamma, beta, part, y,
                               mean, inv_std, eps, g);
            HIP_RETURN_IF_LAUNCH_FAILED();
            return PYDTNN_HIP_OK;
        });
    }
    const long planes = images * channels;
    const bool small = pixels < kPlaneOfGroup;
    const long blocks = small ? (planes + kWaves - 1) / kWaves : planes;
    if (too_many(blocks)) return PYDTNN_HIP_ERR_UNSUPPORTED;
    auto launch = [&](auto threads) {
        constexpr int N = decltype(threads)::value;
        hipLaunchKernelGGL((gn_first_moments<T, N>), dim3((unsigned)blocks), dim3(kT), 0, st, x, part, planes, pixels);
        hipLaunchKernelGGL((gn_first_apply<T, N, ACT>), dim3((unsigned)blocks), dim3(kT), 0, st, x, gamma, beta, part, y,
                           mean, inv_std, eps, planes, pixels, channels, channels / groups);
    };
    if (small) launch(std::integral_constant<int, kWave>());
    else launch(std::integral_constant<int, kT>());
    HIP_RETURN_IF_LAUNCH_FAILED();
    return PYDTNN_HIP_OK;
}

template <typename T, int ACT>
int backward(int nhwc, const T* dy, const T* x, const wide_t<T>* gamma, const wide_t<T>* beta, const wide_t<T>* mean,
             const wide_t<T>* inv_std, wide_t<T>* dgamma, wide_t<T>* dbeta, T* dx, long images, int channels, int pixels,
             int groups, void* workspace, hipStream_t st)
{
    using A = wide_t<T>;
    A* sums = static_cast<A*>(workspace);
    const int cg = channels / groups;
    const double m = (double)cg * pixels;
    const unsigned group_blocks = (unsigned)((images * groups + kWaves - 1) / kWaves);
    auto join = [&](long pieces, int splits) {
        if (dx) hipLaunchKernelGGL((gn_bwd_groups<A>), dim3(group_blocks), dim3(kT), 0, st, sums, gamma, sums + 2 * pieces * channels,
                                   images, splits, channels, groups, m);
        hipLaunchKernelGGL((gn_bwd_params<A>), dim3((unsigned)((channels + 15) / 16)), dim3(kT), 0, st, sums, dgamma, dbeta,
                           pieces, channels);
    };
    if (nhwc) {
        const int v = aligned16(x) && aligned16(dy) && aligned16(dx) ? pack_of(sizeof(T), channels, cg) : 1;
        const GnLast g = last_shape(images, channels, pixels, groups, v);
        const long blocks = images * g.slabs * g.splits;
        if (too_many(blocks)) return PYDTNN_HIP_ERR_UNSUPPORTED;
        return with_pack(v, [&](auto pack) {
            constexpr int V = decltype(pack)::value * sizeof(T) <= 16 ? decltype(pack)::value : 1;
            hipLaunchKernelGGL((gn_last_bwd_sums<T, V, ACT>), dim3((unsigned)blocks), dim3(kT), 0, st, dy, x, gamma, beta,
                               mean, inv_std, sums, g);
            join(images * g.splits, g.splits);
            if (dx) hipLaunchKernelGGL((gn_last_bwd_apply<T, V, ACT>), dim3((unsigned)blocks), dim3(kT), 0, st, dy, x, gamma,
                                       beta, mean, inv_std, sums + 2 * images * g.splits * channels, dx, g);
            HIP_RETURN_IF_LAUNCH_FAILED();
            return PYDTNN_HIP_OK;
        });
    }
    const long planes = images * channels;
    const bool small = pixels < kPlaneOfGroup;
    const long blocks = small ? (planes + kWaves - 1) / kWaves : planes;
    if (too_many(blocks)) return PYDTNN_HIP_ERR_UNSUPPORTED;
    auto launch = [&](auto threads) {
        constexpr int N = decltype(threads)::value;
        hipLaunchKernelGGL((gn_first_bwd_sums<T, N, ACT>), dim3((unsigned)blocks), dim3(kT), 0, st, dy, x, gamma, beta, mean,
                           inv_std, sums, planes, pixels, channels, cg);
        join(images, 1);
        if (dx) hipLaunchKernelGGL((gn_first_bwd_apply<T, N, ACT>), dim3((unsigned)blocks), dim3(kT), 0, st, dy, x, gamma, beta,
                                   mean, inv_std, sums + 2 * planes, dx, planes, pixels, channels, cg);
    };
    if (small) launch(std::integral_constant<int, kWave>());
    else launch(std::integral_constant<int, kT>());
    HIP_RETURN_IF_LAUNCH_FAILED();
    return PYDTNN_HIP_OK;
}

}  // namespace

extern "C" {

size_t pydtnn_hip_gn_workspace_bytes(int dtype, int nhwc, int backward, long images, long channels, long pixels, long groups)
{
    if (check(images, channels, pixels, groups) != PYDTNN_HIP_OK || dtype < kDtypeF32 || dtype > kDtypeBF16) return 0;
    const int c = (int)channels, p = (int)pixels, g = (int)groups;
    const size_t a = workspace_of(pieces_of(dtype, nhwc, images, c, p, g, 1), images, g, backward != 0);
    const size_t b = workspace_of(pieces_of(dtype, nhwc, images, c, p, g, pack_of(size_of(dtype), c, c / g)), images, g,
                                  backward != 0);
    return a > b ? a : b;
}

int pydtnn_hip_gn_forward(int dtype, int nhwc, const void* x, const void* gamma, const void* beta, void* y, void* mean,
                          void* inv_std, long images, long channels, long pixels, long groups, double eps, int activation,
                          void* workspace, size_t workspace_bytes, void* stream)
{
    if (!x || !gamma || !beta || !y || !mean || !inv_std || !(eps >= 0.0)) return PYDTNN_HIP_ERR_INVALID;
    const int rc = check(images, channels, pixels, groups);
    if (rc != PYDTNN_HIP_OK) return rc;
    if (!workspace || workspace_bytes < pydtnn_hip_gn_workspace_bytes(dtype, nhwc, 0, images, channels, pixels, groups))
        return PYDTNN_HIP_ERR_WORKSPACE;
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        using A = wide_t<T>;
        return with_act(activation, [&](auto a) {
            return forward<T, decltype(a)::value>(nhwc, (const T*)x, (const A*)gamma, (const A*)beta, (T*)y, (A*)mean,
                                                  (A*)inv_std, images, (int)channels, (int)pixels, (int)groups, eps,
                                                  workspace, convint::as_stream(stream));
        });
    });
}

int pydtnn_hip_gn_backward(int dtype, int nhwc, const void* dy, const void* x, const void* gamma, const void* beta,
                           const void* mean, const void* inv_std, void* dgamma, void* dbeta, void* dx, long images,
                           long channels, long pixels, long groups, int activation, void* workspace, size_t workspace_bytes,
                           void* stream)
{
    if (!dy || !x || !gamma || !beta || !mean || !inv_std || !dgamma || !dbeta) return PYDTNN_HIP_ERR_INVALID;
    const int rc = check(images, channels, pixels, groups);
    if (rc != PYDTNN_HIP_OK) return rc;
    if (!workspace || workspace_bytes < pydtnn_hip_gn_workspace_bytes(dtype, nhwc, 1, images, channels, pixels, groups))
        return PYDTNN_HIP_ERR_WORKSPACE;
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        using A = wide_t<T>;
        return with_act(activation, [&](auto a) {
            return backward<T, decltype(a)::value>(nhwc, (const T*)dy, (const T*)x, (const A*)gamma, (const A*)beta,
                                                   (const A*)mean, (const A*)inv_std, (A*)dgamma, (A*)dbeta, (T*)dx, images,
                                                   (int)channels, (int)pixels, (int)groups, workspace,
                                                   convint::as_stream(stream));
        });
    });
}

}  // extern "C"
