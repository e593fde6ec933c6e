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
// Each is sums of a group, then the map.  Where the registers of a workgroup hold whole groups, one kernel does both and
// x is read once (..._whole): 16 x 56 x 56 x 256 forward in float32 takes 21 us, 5.0 TB/s.  Elsewhere there are two passes:
// sums of pieces of each group (moments, bwd_sums), then the map with the joined sums (apply): 64 x 56 x 56 x 256 in float32
// takes 100 us forward, where a copy takes 76, and 179 backward (114), with 6.1 and 5.8 TB/s moved.  Each workgroup of the map
// joins the pieces of its groups, or where there are many kernels between the two do.  The smallest calls take 5 us, a launch.
//
// Sums are held in 32 bits (64 for double), as (mean, sum of squared differences from it) of a piece, and pieces are joined
// in double through their common mean, so that a mean far from zero costs no digits of the variance.
#include <algorithm>
#include <cmath>
#include "../../include/pydtnn_hip.h"
#include "conv_internal.h"
#include "dtypes.h"

namespace {

constexpr int kT = 256;
constexpr int kWave = 64;
constexpr int kWaves = kT / kWave;
constexpr int kWholeWidth = 512;      // channels of a slab that one kernel holds at most

enum { kIdentity = 0, kRelu = 1, kSilu = 2 };

// 1 / (1 + e^-z).  In 32 bits through the hardware's 2^v and 1/v, each within a step: their errors and that of the product
// -z log2(e) move the result by at most 3 + |z| steps.  Under z = -126 log 2 = -87.34 the reciprocal is below the smallest normal
// number and counts as 0.
__device__ __forceinline__ float sigmoid(float z)
{
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504f));
}
__device__ __forceinline__ double sigmoid(double z) { return 1.0 / (1.0 + exp(-z)); }

template <int ACT, typename A>
__device__ __forceinline__ A act(A z)
{
    if (ACT == kRelu) return z > (A)0 ? z : (A)0;
    if (ACT == kSilu) return z * sigmoid(z);
    return z;
}

// The sum over `lanes` consecutive lanes, a power of two, in each of them.
template <typename A>
__device__ __forceinline__ A lanes_sum(A v, int lanes)
{
    for (int o = lanes / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
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
    long pieces;                       // images * slabs * splits
    int group_lanes, column_lanes;     // threads that join the sums of one group, of one channel: powers of two, a wave at most
    FastDiv by_columns;                // by the columns that a group has in a row of threads (join_threads)
};

struct Place {
    long image;
    int slab, split, p0, p1, tx, ty;
};

__device__ __forceinline__ Place place_of(const GnLast& g, unsigned piece)
{
    Place at;
    const unsigned per = (unsigned)(g.slabs * g.splits);
    at.image = piece / per;
    const unsigned r = piece % per;
    at.slab = r / g.splits;
    at.split = r % g.splits;
    at.p0 = at.split * g.run;
    at.p1 = min(at.p0 + g.run, g.pixels);
    at.tx = threadIdx.x % g.tx;
    at.ty = threadIdx.x / g.tx;
    return at;
}

// The second pass walks the pieces from the last to the first, so that what the first pass read last is read again while
// the caches hold it; in eights, since eight consecutive workgroups go to the eight dies and a piece should find its die's
// second-level cache again.  The grid is a multiple of eight; places behind the last piece do nothing.
__device__ __forceinline__ unsigned piece_from_the_end(unsigned block, unsigned blocks)
{
    return (blocks / 8 - 1 - block / 8) * 8 + block % 8;
}

// Neighbouring slabs of an image share lines of memory where their rows are shorter than a line: they go to one die, whose
// second-level cache joins them.  Consecutive workgroups go to the eight dies in turn, so a die's pieces are every eighth.
__device__ __forceinline__ long piece_of_die(long pieces)
{
    return (long)(blockIdx.x % 8) * ((pieces + 7) / 8) + blockIdx.x / 8;
}

// What the second pass writes goes past the caches, and what the first pass reads does not wait for lines of it to be
// written back: forward 64 x 56 x 56 x 256 in float32 126 -> 102 us, backward 215 -> 182.  (Where one kernel does it all there
// is no first pass to spare: 103 us with plain stores, 112 with these.)
template <typename T, int V>
__device__ __forceinline__ void stream_out(Pack<T, V>* to, const Pack<T, V>& v)
{
    if constexpr (sizeof(T) * V == 16) {
        typedef uint32_t quad __attribute__((ext_vector_type(4)));
        __builtin_nontemporal_store(*reinterpret_cast<const quad*>(&v), reinterpret_cast<quad*>(to));
    } else {
        *to = v;
    }
}

// Loads of this many pixels are in flight before the first is used.
constexpr int kAhead = 4;

// Calls f(value of x at pixel p, p) for every pixel p of the thread's run, with kAhead loads under way at once.
template <typename P, typename F>
__device__ __forceinline__ void each_pixel(const Place& at, int rows, const P* x, long step, F f)
{
    int p = at.p0 + at.ty;
    for (; p + (kAhead - 1) * rows < at.p1; p += kAhead * rows) {
        P v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) v[u] = x[(p + u * rows) * step];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) f(v[u], p + u * rows);
    }
    for (; p < at.p1; p += rows) f(x[p * step], p);
}

template <typename P, typename F>
__device__ __forceinline__ void each_pixel_of_two(const Place& at, int rows, const P* x, const P* y, long step, F f)
{
    int p = at.p0 + at.ty;
    for (; p + (kAhead - 1) * rows < at.p1; p += kAhead * rows) {
        P v[kAhead], w[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            v[u] = x[(p + u * rows) * step];
            w[u] = y[(p + u * rows) * step];
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) f(v[u], w[u], p + u * rows);
    }
    for (; p < at.p1; p += rows) {
        P v = x[p * step], w = y[p * step];
        f(v, w, p);
    }
}

// Moments of one thread's elements of each of V channels, from differences from its own first element.
template <typename A, int V>
struct ThreadMoments {
    A first[V], s1[V], s2[V];
    int n;

    template <typename T>
    __device__ __forceinline__ void add(const Pack<T, V>& v)
    {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (n == 0) first[j] = (A)v.v[j];
            const A d = (A)v.v[j] - first[j];
            s1[j] += d;
            s2[j] += d * d;
        }
        ++n;
    }
};

// Joins the threads' moments to those of the slab's groups: calls f(group of the slab, count, mean, sum of squared
// differences) in one lane for each.  Where no pack straddles groups, a thread first joins its own V channels.
template <int THREADS, int V, typename A, typename F>
__device__ __forceinline__ void join_threads(const GnLast& g, const ThreadMoments<A, V>& t, F f)
{
    __shared__ A part_mean[THREADS * V], part_m2[THREADS * V];
    __shared__ int part_n[THREADS];
    const int unit = g.cg % V == 0 ? V : 1;      // channels of an entry
    A mean[V], m2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const A m = t.n ? t.s1[j] / (A)t.n : (A)0;
        mean[j] = t.n ? t.first[j] + m : (A)0;
        m2[j] = t.n ? t.s2[j] - t.s1[j] * m : (A)0;
    }
    part_n[threadIdx.x] = t.n * unit;
    if (unit == V) {
        // around the first channel's mean, as above around the first element
        A sum = (A)0, squares = (A)0, all = (A)0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const A d = mean[j] - mean[0];
            sum += d;
            squares += d * d;
            all += m2[j];
        }
        part_mean[threadIdx.x] = mean[0] + sum / (A)V;
        part_m2[threadIdx.x] = all + (A)t.n * (squares - sum * sum / (A)V);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            part_mean[threadIdx.x * V + j] = mean[j];
            part_m2[threadIdx.x * V + j] = m2[j];
        }
    }
    __syncthreads();
    // a group's entries are every column of a slab that is one group, else columns k mine .. of each row
    const int each = V / unit, columns = g.tx * each, mine = g.slab_groups == 1 ? columns : g.cg / unit;
    const int lane = threadIdx.x & (g.group_lanes - 1);
    for (int k = threadIdx.x / g.group_lanes; k < g.slab_groups; k += THREADS / g.group_lanes) {
        const int entries = mine * g.rows;
        double count = 0, sum = 0, squares = 0;
        for (int e = lane; e < entries; e += g.group_lanes) {
            const int row = (int)fd_div((uint32_t)e, g.by_columns), i = row * columns + k * mine + e - row * mine;
            const double n = part_n[unit == V ? i : i / V];
            count += n;
            sum += n * (double)part_mean[i];
        }
        count = lanes_sum(count, g.group_lanes);
        const double centre = lanes_sum(sum, g.group_lanes) / count;
        for (int e = lane; e < entries; e += g.group_lanes) {
            const int row = (int)fd_div((uint32_t)e, g.by_columns), i = row * columns + k * mine + e - row * mine;
            const double d = (double)part_mean[i] - centre;
            squares += part_n[unit == V ? i : i / V] * d * d + (double)part_m2[i];
        }
        squares = lanes_sum(squares, g.group_lanes);
        if (lane == 0) f(k, count, centre, squares);
    }
}

// The moments of each group's piece: partial[(image * groups + group) * splits + split].
template <typename T, int V>
__global__ void __launch_bounds__(kT) gn_last_moments(const T* __restrict__ x, Moments<wide_t<T>>* __restrict__ partial,
                                                      GnLast g)
{
    using A = wide_t<T>;
    const Place at = place_of(g, blockIdx.x);
    const T* base = x + (at.image * g.pixels) * g.channels + at.slab * g.width;
    ThreadMoments<A, V> t = {};
    if (at.ty < g.rows) {
        for (int c = at.tx * V; c < g.width; c += g.tx * V)
            each_pixel(at, g.rows, reinterpret_cast<const Pack<T, V>*>(base + c), g.channels / V,
                       [&](const Pack<T, V>& v, int) { t.add(v); });
    }
    join_threads<kT>(g, t, [&](int k, double, double mean, double m2) {
        const long group = at.image * g.groups + at.slab * g.slab_groups + k;
        partial[group * g.splits + at.split] = Moments<A>{(A)mean, (A)m2};
    });
}

// Mean and 1/std of one group from the moments of its pieces, `run_of(i)` elements each, by `lanes` consecutive threads;
// all of them get the results.
template <typename A, typename F>
__device__ __forceinline__ void join_moments(const Moments<A>* part, int pieces, F run_of, double m, double eps, int lanes,
                                             A* mean_out, A* inv_std_out)
{
    const int lane = threadIdx.x & (lanes - 1);
    double sum = 0, m2 = 0;
#pragma unroll 4
    for (int i = lane; i < pieces; i += lanes) sum += run_of(i) * (double)part[i].mean;
    const double mean = lanes_sum(sum, lanes) / m;
#pragma unroll 4
    for (int i = lane; i < pieces; i += lanes) {
        const double d = (double)part[i].mean - mean;
        m2 += run_of(i) * d * d + (double)part[i].m2;
    }
    m2 = lanes_sum(m2, lanes);
    *mean_out = (A)mean;
    *inv_std_out = (A)(1.0 / sqrt(m2 / m + eps));
}

// y = act((x - mean) scale + shift) of V channels.
template <typename A, int V>
struct ChanFwd {
    A mean[V], scale[V], shift[V];

    // channels c .. of the slab, whose groups' statistics are given
    __device__ __forceinline__ void set(const GnLast& g, int slab, int c, const A* group_mean, const A* group_inv_std,
                                        const A* gamma, const A* beta)
    {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int k = (c + j) / g.cg, ch = slab * g.width + c + j;
            mean[j] = group_mean[k];
            scale[j] = group_inv_std[k] * gamma[ch];
            shift[j] = beta[ch];
        }
    }

    template <int ACT, typename T>
    __device__ __forceinline__ Pack<T, V> apply(Pack<T, V> v) const
    {
#pragma unroll
        for (int j = 0; j < V; ++j) v.v[j] = (T)act<ACT>(((A)v.v[j] - mean[j]) * scale[j] + shift[j]);
        return v;
    }
};

// The same for every group by a kernel of its own, a wave a group, for passes whose workgroups would each join too much again.
// A group is `units` of `unit` elements, in pieces of `run` units.
template <typename A>
__global__ void __launch_bounds__(kT) gn_join_groups(const Moments<A>* __restrict__ partial, A* __restrict__ mean_out,
                                                     A* __restrict__ inv_std_out, long groups, int pieces, long units, long run,
                                                     int unit, double eps)
{
    const long group = (long)blockIdx.x * kWaves + threadIdx.x / kWave;
    if (group >= groups) return;
    A mean, inv_std;
    join_moments<A>(partial + group * pieces, pieces, [&](int i) { return (double)min(run, units - i * run) * unit; },
                    (double)units * unit, eps, kWave, &mean, &inv_std);
    if (threadIdx.x % kWave == 0) {
        mean_out[group] = mean;
        inv_std_out[group] = inv_std;
    }
}

// Without `partial`, mean and inv_std hold the groups' statistics already.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kT) gn_last_apply(const T* __restrict__ x, const wide_t<T>* __restrict__ gamma,
                                                    const wide_t<T>* __restrict__ beta,
                                                    const Moments<wide_t<T>>* __restrict__ partial, T* __restrict__ y,
                                                    wide_t<T>* __restrict__ mean_out, wide_t<T>* __restrict__ inv_std_out,
                                                    double eps, GnLast g)
{
    using A = wide_t<T>;
    __shared__ A mean[kT * V], inv_std[kT * V];      // of the slab's groups: at most a group to a column
    const unsigned piece = piece_from_the_end(blockIdx.x, gridDim.x);
    if (piece >= g.pieces) return;
    const Place at = place_of(g, piece);
    const long first_group = at.image * g.groups + at.slab * g.slab_groups;
    if (!partial) {
        for (int k = threadIdx.x; k < g.slab_groups; k += kT) {
            mean[k] = mean_out[first_group + k];
            inv_std[k] = inv_std_out[first_group + k];
        }
    }
    for (int k = threadIdx.x / g.group_lanes; partial && k < g.slab_groups; k += kT / g.group_lanes) {
        const long group = first_group + k;
        A m, r;
        join_moments<A>(partial + group * g.splits, g.splits,
                        [&](int i) { return (double)(min(g.run, g.pixels - i * g.run)) * g.cg; },
                        (double)g.pixels * g.cg, eps, g.group_lanes, &m, &r);
        if (threadIdx.x % g.group_lanes == 0) {
            mean[k] = m;
            inv_std[k] = r;
            if (at.split == 0) {
                mean_out[group] = m;
                inv_std_out[group] = r;
            }
        }
    }
    __syncthreads();
    if (at.ty >= g.rows) return;
    const long base = (at.image * g.pixels) * g.channels + at.slab * g.width;
    for (int c = at.tx * V; c < g.width; c += g.tx * V) {
        ChanFwd<A, V> ch;
        ch.set(g, at.slab, c, mean, inv_std, gamma, beta);
        const long step = -(g.channels / V), from = base + c + (long)(at.p0 + at.p1 - 1) * g.channels;
        Pack<T, V>* out = reinterpret_cast<Pack<T, V>*>(y + from);
        each_pixel(at, g.rows, reinterpret_cast<const Pack<T, V>*>(x + from), step,
                   [&](const Pack<T, V>& v, int p) { stream_out(out + p * step, ch.template apply<ACT>(v)); });
    }
}

// Both steps in one kernel where the registers of a workgroup hold a slab of an image: x is read once.
template <typename T, int V, int ACT, int THREADS, int PACKS>
__global__ void __launch_bounds__(THREADS) gn_last_whole(const T* __restrict__ x, const wide_t<T>* __restrict__ gamma,
                                                         const wide_t<T>* __restrict__ beta, T* __restrict__ y,
                                                         wide_t<T>* __restrict__ mean_out,
                                                         wide_t<T>* __restrict__ inv_std_out, double eps, GnLast g)
{
    using A = wide_t<T>;
    __shared__ A mean[kWholeWidth], inv_std[kWholeWidth];
    const long piece = piece_of_die(g.pieces);
    if (piece >= g.pieces) return;
    const Place at = place_of(g, (unsigned)piece);
    const long step = g.channels / V, base = (at.image * g.pixels) * g.channels + at.slab * g.width + at.tx * V;
    const Pack<T, V>* in = reinterpret_cast<const Pack<T, V>*>(x + base);
    Pack<T, V>* out = reinterpret_cast<Pack<T, V>*>(y + base);
    const int mine = at.ty < g.rows ? (g.pixels - at.ty + g.rows - 1) / g.rows : 0;      // pixels of this thread
    Pack<T, V> v[PACKS];
#pragma unroll
    for (int i = 0; i < PACKS; ++i)
        if (i < mine) v[i] = in[(at.ty + i * g.rows) * step];
    ThreadMoments<A, V> t = {};
#pragma unroll
    for (int i = 0; i < PACKS; ++i)
        if (i < mine) t.add(v[i]);
    join_threads<THREADS>(g, t, [&](int k, double count, double m, double m2) {
        const long group = at.image * g.groups + at.slab * g.slab_groups + k;
        mean_out[group] = mean[k] = (A)m;
        inv_std_out[group] = inv_std[k] = (A)(1.0 / sqrt(m2 / count + eps));
    });
    __syncthreads();
    if (!mine) return;
    ChanFwd<A, V> ch;
    ch.set(g, at.slab, at.tx * V, mean, inv_std, gamma, beta);
#pragma unroll
    for (int i = 0; i < PACKS; ++i)
        if (i < mine) out[(at.ty + i * g.rows) * step] = ch.template apply<ACT>(v[i]);
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
        const A z = xn * c.gamma + c.beta, p = sigmoid(z);
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

// V channels of an image: their constants, sums of dz and dz xn, and dx.
template <typename A, int V>
struct ChansBwd {
    ChanBwd<A> ch[V];

    template <int ACT>
    __device__ __forceinline__ void set(const GnLast& g, long image, int channel, const A* mean, const A* inv_std,
                                        const A* gamma, const A* beta)
    {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const long group = image * g.groups + (channel + j) / g.cg;
            ch[j] = chan_bwd<ACT>(mean[group], inv_std[group], gamma[channel + j], beta[channel + j]);
        }
    }

    // With KEEP, dz takes the place of dy: for apply<kIdentity> later.
    template <int ACT, bool KEEP, typename T>
    __device__ __forceinline__ void add(const Pack<T, V>& x, Pack<T, V>& dy, A* s1, A* s2) const
    {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const A xn = ((A)x.v[j] - ch[j].mean) * ch[j].inv_std;
            const A dz = dz_of<ACT>(ch[j], (A)x.v[j], xn, (A)dy.v[j]);
            s1[j] += dz;
            s2[j] += dz * xn;
            if (KEEP) dy.v[j] = (T)dz;
        }
    }

    template <int ACT, typename T>
    __device__ __forceinline__ Pack<T, V> apply(const Pack<T, V>& x, Pack<T, V> dy, const A* a, const A* b) const
    {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const A xn = ((A)x.v[j] - ch[j].mean) * ch[j].inv_std;
            const A dz = dz_of<ACT>(ch[j], (A)x.v[j], xn, (A)dy.v[j]);
            dy.v[j] = (T)dx_of(ch[j], xn, dz, a[j], b[j]);
        }
        return dy;
    }
};

// Sums of a run's dz and dz xn in each of the slab's channels c0 .. c0 + columns: f(channel of the slab, the two sums).
template <int THREADS, int V, typename A, typename F>
__device__ __forceinline__ void join_rows(const GnLast& g, int c0, const A* s1, const A* s2, F f)
{
    __shared__ A part1[THREADS * V], part2[THREADS * V];
    const int columns = g.tx * V;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < V; ++j) {
        part1[threadIdx.x * V + j] = s1[j];
        part2[threadIdx.x * V + j] = s2[j];
    }
    __syncthreads();
    const int lane = threadIdx.x & (g.column_lanes - 1);
    for (int i = threadIdx.x / g.column_lanes; i < min(columns, g.width - c0); i += THREADS / g.column_lanes) {
        A t1 = (A)0, t2 = (A)0;
        for (int r = lane; r < g.rows; r += g.column_lanes) {
            t1 += part1[r * columns + i];
            t2 += part2[r * columns + i];
        }
        t1 = lanes_sum(t1, g.column_lanes);
        t2 = lanes_sum(t2, g.column_lanes);
        if (lane == 0) f(c0 + i, t1, t2);
    }
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
    const Place at = place_of(g, blockIdx.x);
    const long base = (at.image * g.pixels) * g.channels + at.slab * g.width;
    A* out1 = sums + (at.image * g.splits + at.split) * g.channels + at.slab * g.width;
    A* out2 = out1 + g.images * g.splits * g.channels;
    for (int c0 = 0; c0 < g.width; c0 += g.tx * V) {
        const int c = c0 + at.tx * V;
        A s1[V] = {}, s2[V] = {};
        if (at.ty < g.rows && c < g.width) {
            ChansBwd<A, V> ch;
            ch.template set<ACT>(g, at.image, at.slab * g.width + c, mean, inv_std, gamma, beta);
            each_pixel_of_two(at, g.rows, reinterpret_cast<const Pack<T, V>*>(x + base + c),
                              reinterpret_cast<const Pack<T, V>*>(dy + base + c), g.channels / V,
                              [&](const Pack<T, V>& xv, Pack<T, V>& dv, int) { ch.template add<ACT, false>(xv, dv, s1, s2); });
        }
        join_rows<kT, V>(g, c0, s1, s2, [&](int i, A t1, A t2) {
            out1[i] = t1;
            out2[i] = t2;
        });
    }
}

// dgamma and dbeta of kParamChannels channels: the channel sums over images and runs, kParamRows threads a channel.
constexpr int kParamChannels = 4, kParamRows = kT / kParamChannels;

template <typename A>
__device__ __forceinline__ void bwd_params(const A* __restrict__ s1, const A* __restrict__ s2, A* __restrict__ dgamma,
                                           A* __restrict__ dbeta, long pieces, int channels, int block)
{
    __shared__ double part1[kT], part2[kT];
    const int c = block * kParamChannels + threadIdx.x % kParamChannels, r = threadIdx.x / kParamChannels;
    double t1 = 0, t2 = 0;
    if (c < channels) {
#pragma unroll 4
        for (long i = r; i < pieces; i += kParamRows) {
            t1 += (double)s1[i * channels + c];
            t2 += (double)s2[i * channels + c];
        }
    }
    part1[threadIdx.x] = t1;
    part2[threadIdx.x] = t2;
    __syncthreads();
    for (int half = kParamRows / 2; half > 0; half /= 2) {
        if (r < half) {
            part1[threadIdx.x] += part1[threadIdx.x + half * kParamChannels];
            part2[threadIdx.x] += part2[threadIdx.x + half * kParamChannels];
        }
        __syncthreads();
    }
    if (r == 0 && c < channels) {
        dbeta[c] = (A)part1[threadIdx.x];
        dgamma[c] = (A)part2[threadIdx.x];
    }
}

template <typename A>
__global__ void __launch_bounds__(kT) gn_bwd_params(const A* __restrict__ sums, A* __restrict__ dgamma,
                                                    A* __restrict__ dbeta, long pieces, int channels)
{
    bwd_params(sums, sums + pieces * channels, dgamma, dbeta, pieces, channels, blockIdx.x);
}

// The channel sums of each image from those of its runs, `blocks` workgroups an image: image_sums[image * channels + channel],
// then the same of dz xn.
template <typename A>
__global__ void __launch_bounds__(kT) gn_bwd_images(const A* __restrict__ sums, A* __restrict__ image_sums, long images,
                                                    int splits, int channels, int blocks)
{
    const long image = blockIdx.x / blocks;
    const A* s1 = sums + image * splits * channels;
    A* out = image_sums + image * channels;
    bwd_params(s1, s1 + images * splits * channels, out + images * channels, out, splits, channels, blockIdx.x % blocks);
}

// A and B of one group from the channel sums of its runs, by `lanes` consecutive threads.
template <typename A>
__device__ __forceinline__ void group_ab(const A* s1, const A* s2, const A* gamma, int c0, int cg, int splits, int channels,
                                         double m, int lanes, A* a_out, A* b_out)
{
    double a = 0, b = 0;
    const int lane = threadIdx.x & (lanes - 1);
    for (int c = c0 + lane; c < c0 + cg; c += lanes) {
#pragma unroll 4
        for (int s = 0; s < splits; ++s) {
            const long at = (long)s * channels + c;
            a += (double)s1[at] * (double)gamma[c];
            b += (double)s2[at] * (double)gamma[c];
        }
    }
    a = lanes_sum(a, lanes);
    b = lanes_sum(b, lanes);
    if (lane == 0) {
        *a_out = (A)(a / m);
        *b_out = (A)(b / m);
    }
}

// dx, and in the first workgroups dgamma and dbeta.  `ab`, unless it is null, holds A and B of each group.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kT) gn_last_bwd_apply(const T* __restrict__ dy, const T* __restrict__ x,
                                                        const wide_t<T>* __restrict__ gamma,
                                                        const wide_t<T>* __restrict__ beta,
                                                        const wide_t<T>* __restrict__ mean,
                                                        const wide_t<T>* __restrict__ inv_std,
                                                        const wide_t<T>* __restrict__ sums,
                                                        const wide_t<T>* __restrict__ ab, wide_t<T>* __restrict__ dgamma,
                                                        wide_t<T>* __restrict__ dbeta, T* __restrict__ dx, int param_blocks,
                                                        GnLast g)
{
    using A = wide_t<T>;
    __shared__ A group_a[kT * V], group_b[kT * V];
    const A* sums2 = sums + g.images * g.splits * g.channels;
    if ((int)blockIdx.x < param_blocks) {
        if ((int)blockIdx.x * kParamChannels < g.channels)
            bwd_params(sums, sums2, dgamma, dbeta, g.images * g.splits, g.channels, blockIdx.x);
        return;
    }
    const unsigned piece = piece_from_the_end(blockIdx.x - param_blocks, gridDim.x - param_blocks);
    if (piece >= g.pieces) return;
    const Place at = place_of(g, piece);
    if (ab) {
        const A* of_slab = ab + 2 * (at.image * g.groups + at.slab * g.slab_groups);
        for (int k = threadIdx.x; k < g.slab_groups; k += kT) {
            group_a[k] = of_slab[2 * k];
            group_b[k] = of_slab[2 * k + 1];
        }
    }
    const long from_run = at.image * g.splits * g.channels;
    for (int k = threadIdx.x / g.group_lanes; !ab && k < g.slab_groups; k += kT / g.group_lanes)
        group_ab(sums + from_run, sums2 + from_run, gamma, at.slab * g.width + k * g.cg, g.cg, g.splits, g.channels,
                 (double)g.cg * g.pixels, g.group_lanes, &group_a[k], &group_b[k]);
    __syncthreads();
    if (at.ty >= g.rows) return;
    const long base = (at.image * g.pixels) * g.channels + at.slab * g.width;
    for (int c = at.tx * V; c < g.width; c += g.tx * V) {
        ChansBwd<A, V> ch;
        ch.template set<ACT>(g, at.image, at.slab * g.width + c, mean, inv_std, gamma, beta);
        A a[V], b[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            a[j] = group_a[(c + j) / g.cg];
            b[j] = group_b[(c + j) / g.cg];
        }
        const long step = -(g.channels / V), from = base + c + (long)(at.p0 + at.p1 - 1) * g.channels;
        Pack<T, V>* out = reinterpret_cast<Pack<T, V>*>(dx + from);
        each_pixel_of_two(at, g.rows, reinterpret_cast<const Pack<T, V>*>(x + from),
                          reinterpret_cast<const Pack<T, V>*>(dy + from), step,
                          [&](const Pack<T, V>& xv, const Pack<T, V>& dv, int p) {
                              stream_out(out + p * step, ch.template apply<ACT>(xv, dv, a, b));
                          });
    }
}

// Sums and dx in one kernel where the registers of a workgroup hold a slab of an image of x and of dy: both are read once.
template <typename T, int V, int ACT, int THREADS, int PACKS>
__global__ void __launch_bounds__(THREADS) gn_last_bwd_whole(const T* __restrict__ dy, const T* __restrict__ x,
                                                             const wide_t<T>* __restrict__ gamma,
                                                             const wide_t<T>* __restrict__ beta,
                                                             const wide_t<T>* __restrict__ mean,
                                                             const wide_t<T>* __restrict__ inv_std,
                                                             wide_t<T>* __restrict__ sums, T* __restrict__ dx, GnLast g)
{
    using A = wide_t<T>;
    __shared__ A group_a[kWholeWidth], group_b[kWholeWidth], chan1[kWholeWidth], chan2[kWholeWidth];
    const long piece = piece_of_die(g.pieces);
    if (piece >= g.pieces) return;
    const Place at = place_of(g, (unsigned)piece);
    const long step = g.channels / V, base = (at.image * g.pixels) * g.channels + at.slab * g.width + at.tx * V;
    const Pack<T, V>* xin = reinterpret_cast<const Pack<T, V>*>(x + base);
    const Pack<T, V>* din = reinterpret_cast<const Pack<T, V>*>(dy + base);
    Pack<T, V>* out = reinterpret_cast<Pack<T, V>*>(dx + base);
    const int mine = at.ty < g.rows ? (g.pixels - at.ty + g.rows - 1) / g.rows : 0;      // pixels of this thread
    Pack<T, V> xv[PACKS], dv[PACKS];
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
        if (i < mine) {
            xv[i] = xin[(at.ty + i * g.rows) * step];
            dv[i] = din[(at.ty + i * g.rows) * step];
        }
    }
    // dz is computed once where its type holds it: of the rectifier it is dy or 0
    constexpr bool kKeep = ACT != kSilu || sizeof(T) >= 4;
    ChansBwd<A, V> ch;
    A s1[V] = {}, s2[V] = {};
    if (mine) ch.template set<ACT>(g, at.image, at.slab * g.width + at.tx * V, mean, inv_std, gamma, beta);
#pragma unroll
    for (int i = 0; i < PACKS; ++i)
        if (i < mine) ch.template add<ACT, kKeep>(xv[i], dv[i], s1, s2);
    A* out1 = sums + at.image * g.channels + at.slab * g.width;
    A* out2 = out1 + g.images * g.channels;
    join_rows<THREADS, V>(g, 0, s1, s2, [&](int i, A t1, A t2) {
        out1[i] = chan1[i] = t1;
        out2[i] = chan2[i] = t2;
    });
    if (!dx) return;
    __syncthreads();
    for (int k = threadIdx.x / g.group_lanes; k < g.slab_groups; k += THREADS / g.group_lanes)
        group_ab(chan1 + k * g.cg, chan2 + k * g.cg, gamma + at.slab * g.width + k * g.cg, 0, g.cg, 1, 0,
                 (double)g.cg * g.pixels, g.group_lanes, &group_a[k], &group_b[k]);
    __syncthreads();
    if (!mine) return;
    A a[V], b[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        a[j] = group_a[(at.tx * V + j) / g.cg];
        b[j] = group_b[(at.tx * V + j) / g.cg];
    }
#pragma unroll
    for (int i = 0; i < PACKS; ++i)
        if (i < mine) out[(at.ty + i * g.rows) * step] = ch.template apply<kKeep ? kIdentity : ACT>(xv[i], dv[i], a, b);
}

// ---------------------------------------------------------------------------------------------- channels first
// A group is one run of memory here.  Where a workgroup's registers hold it, one kernel does the forward pass; otherwise, and
// in the backward pass, whose sums are of channels, THREADS threads take a plane: one channel of one image.
// 64 x 256 x 56 x 56: forward 88 us in float32 and 55 in bfloat16 (196 and 148 in planes), backward 183 and 92.
struct GnFirst {
    long planes;                     // images * channels
    int pixels, channels, cg;
    FastDiv by_pixels;               // exact for the elements of a group that one kernel holds, at most 2^16
};

// V elements that start anywhere: planes of odd extents start off the boundaries of 16 bytes, where loads and stores of 16
// bytes still beat those of an element.
template <typename T, int V>
struct Loose {
    T v[V];
};

// Calls f(V elements of x, their first's number) for a plane, kAhead loads under way at once, and then f(one element, its
// number) for what is left.
template <int THREADS, int V, typename T, typename F>
__device__ __forceinline__ void each_pack(const T* x, int pixels, F f)
{
    using P = Loose<T, V>;
    int p = threadIdx.x % THREADS * V;
    for (; p + (kAhead - 1) * THREADS * V + V <= pixels; p += kAhead * THREADS * V) {
        P v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) __builtin_memcpy(&v[u], x + p + u * THREADS * V, sizeof(P));
#pragma unroll
        for (int u = 0; u < kAhead; ++u) f(v[u], p + u * THREADS * V);
    }
    for (; p + V <= pixels; p += THREADS * V) {
        P v;
        __builtin_memcpy(&v, x + p, sizeof(P));
        f(v, p);
    }
    for (p = pixels / V * V + threadIdx.x % THREADS; p < pixels; p += THREADS) f(Loose<T, 1>{{x[p]}}, p);
}

template <int THREADS, int V, typename T, typename F>
__device__ __forceinline__ void each_pack_of_two(const T* x, const T* y, int pixels, F f)
{
    using P = Loose<T, V>;
    int p = threadIdx.x % THREADS * V;
    for (; p + (kAhead - 1) * THREADS * V + V <= pixels; p += kAhead * THREADS * V) {
        P v[kAhead], w[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            __builtin_memcpy(&v[u], x + p + u * THREADS * V, sizeof(P));
            __builtin_memcpy(&w[u], y + p + u * THREADS * V, sizeof(P));
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) f(v[u], w[u], p + u * THREADS * V);
    }
    for (; p + V <= pixels; p += THREADS * V) {
        P v, w;
        __builtin_memcpy(&v, x + p, sizeof(P));
        __builtin_memcpy(&w, y + p, sizeof(P));
        f(v, w, p);
    }
    for (p = pixels / V * V + threadIdx.x % THREADS; p < pixels; p += THREADS)
        f(Loose<T, 1>{{x[p]}}, Loose<T, 1>{{y[p]}}, p);
}

// stream_out to anywhere.
template <typename T, int V>
__device__ __forceinline__ void stream_loose(T* to, const Loose<T, V>& v)
{
    if constexpr (sizeof(T) * V == 16) {
        typedef uint32_t quad __attribute__((ext_vector_type(4)));
        typedef quad loose_quad __attribute__((aligned(2)));
        __builtin_nontemporal_store(__builtin_bit_cast(quad, v), reinterpret_cast<loose_quad*>(to));
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) to[j] = v.v[j];
    }
}

template <int THREADS, typename A>
__device__ __forceinline__ A plane_sum(A v, A* part)
{
    v = lanes_sum(v, THREADS < kWave ? THREADS : kWave);
    if (THREADS <= kWave) return v;
    __syncthreads();
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += part[w];
    return v;
}

template <int THREADS>
__device__ __forceinline__ long plane_of()
{
    return (long)blockIdx.x * (kT / THREADS) + threadIdx.x / THREADS;
}

template <typename T, int V, int THREADS>
__global__ void __launch_bounds__(kT) gn_first_moments(const T* __restrict__ x, Moments<wide_t<T>>* __restrict__ partial,
                                                       GnFirst g)
{
    using A = wide_t<T>;
    __shared__ A part[kWaves];
    const long plane = plane_of<THREADS>();
    if (plane >= g.planes) return;
    const T* base = x + plane * g.pixels;
    const A first = (A)base[0];
    A s1 = (A)0;
    each_pack<THREADS, V>(base, g.pixels, [&](const auto& v, int) {
        for (const T& e : v.v) s1 += (A)e - first;
    });
    const A mean = first + plane_sum<THREADS>(s1, part) / (A)g.pixels;
    A s2 = (A)0;
    each_pack<THREADS, V>(base, g.pixels, [&](const auto& v, int) {
        for (const T& e : v.v) s2 += ((A)e - mean) * ((A)e - mean);
    });
    s2 = plane_sum<THREADS>(s2, part);
    if (threadIdx.x % THREADS == 0) partial[plane] = Moments<A>{mean, s2};
}

// Without `partial`, mean and inv_std hold the groups' statistics already.
template <typename T, int V, int THREADS, int ACT>
__global__ void __launch_bounds__(kT) gn_first_apply(const T* __restrict__ x, const wide_t<T>* __restrict__ gamma,
                                                     const wide_t<T>* __restrict__ beta,
                                                     const Moments<wide_t<T>>* __restrict__ partial, T* __restrict__ y,
                                                     wide_t<T>* __restrict__ mean_out, wide_t<T>* __restrict__ inv_std_out,
                                                     double eps, GnFirst g)
{
    using A = wide_t<T>;
    const long plane = plane_of<THREADS>();
    if (plane >= g.planes) return;
    const long group = plane / g.cg;
    const int c = (int)(plane % g.channels);
    A mean, inv_std;
    if (!partial) {
        mean = mean_out[group];
        inv_std = inv_std_out[group];
    } else {
        join_moments<A>(partial + group * g.cg, g.cg, [&](int) { return (double)g.pixels; }, (double)g.pixels * g.cg, eps,
                        THREADS < kWave ? THREADS : kWave, &mean, &inv_std);
        if (plane % g.cg == 0 && threadIdx.x % THREADS == 0) {
            mean_out[group] = mean;
            inv_std_out[group] = inv_std;
        }
    }
    const A scale = inv_std * gamma[c], shift = beta[c];
    T* out = y + plane * g.pixels;
    each_pack<THREADS, V>(x + plane * g.pixels, g.pixels, [&](auto v, int p) {
        for (T& e : v.v) e = (T)act<ACT>(((A)e - mean) * scale + shift);
        stream_loose(out + p, v);
    });
}

// A workgroup holds a group: x is read once.  `join` makes one group of all threads for join_threads.
template <typename T, int V, int ACT, int THREADS, int PACKS>
__global__ void __launch_bounds__(THREADS) gn_first_whole(const T* __restrict__ x, const wide_t<T>* __restrict__ gamma,
                                                          const wide_t<T>* __restrict__ beta, T* __restrict__ y,
                                                          wide_t<T>* __restrict__ mean_out,
                                                          wide_t<T>* __restrict__ inv_std_out, double eps, GnFirst g,
                                                          GnLast join)
{
    using A = wide_t<T>;
    __shared__ A mean, inv_std;
    const long group = blockIdx.x, elements = (long)g.cg * g.pixels;
    const int c0 = (int)(group % (g.channels / g.cg)) * g.cg, packs = (int)(elements / V);
    const Pack<T, V>* in = reinterpret_cast<const Pack<T, V>*>(x + group * elements);
    Pack<T, V>* out = reinterpret_cast<Pack<T, V>*>(y + group * elements);
    Pack<T, V> v[PACKS];
#pragma unroll
    for (int i = 0; i < PACKS; ++i)
        if ((int)threadIdx.x + i * THREADS < packs) v[i] = in[threadIdx.x + i * THREADS];
    ThreadMoments<A, 1> t = {};      // all of one group
    if ((int)threadIdx.x < packs) t.first[0] = (A)v[0].v[0];
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
        if ((int)threadIdx.x + i * THREADS >= packs) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const A d = (A)v[i].v[j] - t.first[0];
            t.s1[0] += d;
            t.s2[0] += d * d;
        }
        t.n += V;
    }
    join_threads<THREADS>(join, t, [&](int, double count, double m, double m2) {
        mean_out[group] = mean = (A)m;
        inv_std_out[group] = inv_std = (A)(1.0 / sqrt(m2 / count + eps));
    });
    __syncthreads();
    const A mu = mean, r = inv_std;
    const bool one = g.pixels % V == 0;      // whether each pack is of one channel
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
        const int p = threadIdx.x + i * THREADS;
        if (p >= packs) continue;
        const uint32_t k = fd_div((uint32_t)(p * V), g.by_pixels);
        if (one || k == fd_div((uint32_t)(p * V + V - 1), g.by_pixels)) {
            const A scale = r * gamma[c0 + k], shift = beta[c0 + k];
#pragma unroll
            for (int j = 0; j < V; ++j) v[i].v[j] = (T)act<ACT>(((A)v[i].v[j] - mu) * scale + shift);
        } else {      // a pack that straddles channels
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int c = c0 + (int)fd_div((uint32_t)(p * V + j), g.by_pixels);
                v[i].v[j] = (T)act<ACT>(((A)v[i].v[j] - mu) * (r * gamma[c]) + beta[c]);
            }
        }
        out[p] = v[i];
    }
}

template <typename T, int V, int THREADS, int ACT>
__global__ void __launch_bounds__(kT) gn_first_bwd_sums(const T* __restrict__ dy, const T* __restrict__ x,
                                                        const wide_t<T>* __restrict__ gamma,
                                                        const wide_t<T>* __restrict__ beta,
                                                        const wide_t<T>* __restrict__ mean,
                                                        const wide_t<T>* __restrict__ inv_std,
                                                        wide_t<T>* __restrict__ sums, GnFirst g)
{
    using A = wide_t<T>;
    __shared__ A part[kWaves];
    const long plane = plane_of<THREADS>();
    if (plane >= g.planes) return;
    const int c = (int)(plane % g.channels);
    const ChanBwd<A> ch = chan_bwd<ACT>(mean[plane / g.cg], inv_std[plane / g.cg], gamma[c], beta[c]);
    A s1 = (A)0, s2 = (A)0;
    auto add = [&](const auto& xv, const auto& dv, int) {
#pragma unroll
        for (unsigned j = 0; j < sizeof(xv) / sizeof(T); ++j) {
            const A xn = ((A)xv.v[j] - ch.mean) * ch.inv_std;
            const A dz = dz_of<ACT>(ch, (A)xv.v[j], xn, (A)dv.v[j]);
            s1 += dz;
            s2 += dz * xn;
        }
    };
    each_pack_of_two<THREADS, V>(x + plane * g.pixels, dy + plane * g.pixels, g.pixels, add);
    s1 = plane_sum<THREADS>(s1, part);
    s2 = plane_sum<THREADS>(s2, part);
    if (threadIdx.x % THREADS == 0) {
        sums[plane] = s1;
        sums[g.planes + plane] = s2;
    }
}

template <typename T, int V, int THREADS, int ACT>
__global__ void __launch_bounds__(kT) gn_first_bwd_apply(const T* __restrict__ dy, const T* __restrict__ x,
                                                         const wide_t<T>* __restrict__ gamma,
                                                         const wide_t<T>* __restrict__ beta,
                                                         const wide_t<T>* __restrict__ mean,
                                                         const wide_t<T>* __restrict__ inv_std,
                                                         const wide_t<T>* __restrict__ ab, T* __restrict__ dx, GnFirst g)
{
    using A = wide_t<T>;
    const long plane = plane_of<THREADS>();
    if (plane >= g.planes) return;
    const int c = (int)(plane % g.channels);
    const long group = plane / g.cg;
    const ChanBwd<A> ch = chan_bwd<ACT>(mean[group], inv_std[group], gamma[c], beta[c]);
    const A a = ab[2 * group], b = ab[2 * group + 1];
    T* out = dx + plane * g.pixels;
    each_pack_of_two<THREADS, V>(x + plane * g.pixels, dy + plane * g.pixels, g.pixels, [&](const auto& xv, auto dv, int p) {
#pragma unroll
        for (unsigned j = 0; j < sizeof(xv) / sizeof(T); ++j) {
            const A xn = ((A)xv.v[j] - ch.mean) * ch.inv_std;
            const A dz = dz_of<ACT>(ch, (A)xv.v[j], xn, (A)dv.v[j]);
            dv.v[j] = (T)dx_of(ch, xn, dz, a, b);
        }
        stream_loose(out + p, dv);
    });
}

// A and B of each group: one wave a group.
template <typename A>
__global__ void __launch_bounds__(kT) gn_bwd_groups(const A* __restrict__ sums, const A* __restrict__ gamma,
                                                    A* __restrict__ ab, long images, int channels, int groups, double m)
{
    const long group = (long)blockIdx.x * kWaves + threadIdx.x / kWave;
    if (group >= images * groups) return;
    const int cg = channels / groups;
    const A* s1 = sums + (group / groups) * channels;
    group_ab(s1, s1 + images * channels, gamma, (int)(group % groups) * cg, cg, 1, channels, m, kWave,
             &ab[2 * group], &ab[2 * group + 1]);
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

// A power of two of the threads that `items` can have each, a wave at most.
int lanes_of(int threads, int items)
{
    int lanes = kWave;
    while (lanes > 1 && (long)lanes * items > threads) lanes /= 2;
    return lanes;
}

void set_joins(GnLast* g, int threads, int v)
{
    const int unit = g->cg % v == 0 ? v : 1;
    g->group_lanes = lanes_of(threads, g->slab_groups);
    g->column_lanes = lanes_of(threads, g->tx * v);
    g->by_columns = make_fastdiv((uint32_t)(g->slab_groups == 1 ? g->tx * (v / unit) : g->cg / unit));
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
    g.rows = std::min(kT / g.tx, pixels);
    // three workgroups to each of 256 compute units, which hold them all at once (backward 64 x 56 x 56 x 256 in float32: 178
    // us against 188 with four and 199 with eight), and at least eight pixels to a thread
    long want = (768 + images * g.slabs - 1) / (images * g.slabs);
    const long most = (pixels + 8l * g.rows - 1) / (8l * g.rows);
    if (want > most) want = most;
    g.run = (int)((pixels + want - 1) / want);
    g.splits = (pixels + g.run - 1) / g.run;
    g.pieces = images * g.slabs * g.splits;
    set_joins(&g, kT, v);
    return g;
}

// Each workgroup of a second pass joins what the runs of its slab's groups left, which grows with the square of the runs: where
// a lane would take more than kJoinForward moments, or kJoinBackward channel sums, a kernel (backward two) of a wave a
// group joins them once.  1 x 112 x 112 x 1024 in float32 (738 runs): forward in groups of one 2600 us and 41 joined once, backward in
// groups of 16 600 and 58.  About the limits, forward in groups of 8: 4 x 112 x 112 x 256 (24 a lane) 31 and 27, 8 x 112 x 112 x 256
// (12) 48.8 and 48.5, 16 x 112 x 112 x 256 (6) 92.7 and 93.1.  Backward: 4 x 112 x 112 x 256 in groups of 8 (191 a lane) 54 and 47;
// 32 x 28 x 28 x 1024 in bfloat16 in groups of 16 (192) 82 and 70; 24 x 20 x 20 x 1024 in groups of 128 (128) 53 and 50, in
// bfloat16 45 and 44; 48 x 20 x 20 x 512 in one group (128) 46 and 47, in bfloat16 39 and 42; 64 x 20 x 20 x 2048 in bfloat16 in
// groups of 256 (96) 116 and 132.
constexpr long kJoinForward = 16, kJoinBackward = 128;

// What a lane of a workgroup joins where each group has that many entries.
long entries_of_lane(const GnLast& g, long entries)
{
    return ((long)g.slab_groups * g.group_lanes + kT - 1) / kT * ((entries + g.group_lanes - 1) / g.group_lanes);
}

bool joined_forward(const GnLast& g) { return entries_of_lane(g, g.splits) > kJoinForward; }

// (a slab that is one run joins nothing twice)
bool joined_backward(const GnLast& g) { return g.splits > 1 && entries_of_lane(g, g.cg) * g.splits > kJoinBackward; }

// Whether to take a slab of so many packs that leaves threads idle, where no other way holds one.  17 groups, two passes second.
// Forward: where there are few workgroups (float32, 64 x 7 x 7 x 544: 8.6 us and 10.9; but 18.2 and 15.3 for 256 images) or more
// packs than the smallest way holds (1024 x 14 x 14 x 544 160 and 223, 256 images 42 and 50).  Backward: 64 x 7 x 7 x 544 14 and 20,
// x 3 x 3 x 544 for 120 images 15.7 and 13.1; 1024 x 14 x 14 x 544 331 and 417, in float64 with 272 channels 324 and 383, 256 of those
// 96 and 85.
enum class Idle { kNever, kForward, kBackward };

bool takes_idle(Idle idle, long packs, long pieces)
{
    if (idle == Idle::kForward) return packs >= kWave && (pieces <= 2048 || packs > 1024);
    return idle == Idle::kBackward && (packs > 1024 ? pieces > 8192 : pieces <= 2048 && packs >= 256);
}

// Where one kernel can hold a slab of an image in the registers of `threads` threads, `packs` packs of 16 bytes each (of x,
// and in the backward pass as many of dy): the smallest slab of whole groups whose rows have at least `line` bytes, or all
// channels; at most `most` of them.  A slab of few packs leaves threads idle: it grows while there are workgroups enough.  Where no
// wider one fits (group counts with few divisors) the way is passed over, unless `idle` says that the idle slab is better than
// two passes.
bool whole_shape(GnLast* g, long images, int channels, int pixels, int groups, int v, int size, int line, long most, Idle idle,
                 int threads, int packs)
{
    if (v * size != 16) return false;
    const int cg = channels / groups;
    long slab = 0;      // packs of the slab
    bool is_idle = false;
    for (int sg = 1; sg <= groups && (long)sg * cg <= kWholeWidth; ++sg) {
        const int width = sg * cg;
        if (groups % sg || width % v || (width * size < line && sg != groups)) continue;
        const int tx = width / v;
        if (tx > threads || (pixels + threads / tx - 1) / (threads / tx) > packs) break;
        *g = GnLast{images, pixels, channels, groups, cg, sg, width, groups / sg, tx, std::min(threads / tx, pixels), 1, pixels,
                    images * (groups / sg), 1, 1, {}};
        slab = (long)pixels * tx;
        is_idle = 2 * slab < threads * packs && sg != groups && g->pieces > 1024;
        if (!is_idle) break;
    }
    if (!slab || (is_idle && !takes_idle(idle, slab, g->pieces))) return false;
    set_joins(g, threads, v);
    return g->pieces <= most && (g->pieces + 8) * threads < (1l << 32);      // (a launch counts its threads in 32 bits)
}

int check(long images, long channels, long pixels, long groups)
{
    if (images <= 0 || channels <= 0 || pixels <= 0 || groups <= 0 || channels % groups) return PYDTNN_HIP_ERR_INVALID;
    // runs and planes are counted in 32 bits
    if (pixels > (1l << 30) || channels > (1l << 30) || images > (1l << 40) / channels) return PYDTNN_HIP_ERR_UNSUPPORTED;
    return PYDTNN_HIP_OK;
}

int size_of(int dtype) { return dtype == kDtypeF64 ? 8 : dtype == kDtypeF32 ? 4 : 2; }

// A way to hold a slab: a workgroup's threads, and the packs that each holds.
template <int THREADS, int PACKS>
struct Hold {};

// Calls launch(line, most, idle, threads, packs) for these ways in turn, with whole lines of `first` bytes, then with half lines
// of 64 (forward 64 x 14 x 14 x 1024 in float32: 19 us with lines of 128, 22 with half lines), until one fits.
template <typename F, int... THREADS, int... PACKS>
bool hold_lines(int first, long most, Idle idle, F launch, Hold<THREADS, PACKS>...)
{
    for (int line = first; line >= std::min(first, 64); line /= 2)
        if ((launch(line, most, idle, std::integral_constant<int, THREADS>(), std::integral_constant<int, PACKS>()) || ...))
            return true;
    return false;
}

// The lines that slabs are made of.  Where the images' rows, of `rows_bytes` in all, make fewer than 256 whole lines, slabs are
// narrower, so that more compute units have one: caches hold tensors this small (4 x 28 x 28 x 128 in bfloat16: forward 10 -> 9
// us, backward 16 -> 12).
int first_line(long rows_bytes)
{
    int first = 128;
    while (first > 16 && rows_bytes / first < 256) first /= 2;
    return first;
}

// The ways to hold slabs, the better first: few threads before many (several workgroups to a compute unit, whose loads and
// stores overlap) and few packs to a thread before many (forward 16 x 28 x 28 x 512 in bfloat16: 12 us with eight packs to 512
// threads, 15 with sixteen to 256).  Sixteen packs to 512 threads still beat two passes (forward 64 x 28 x 28 x 512 in float64:
// 86 us against 104; 64 x 40 x 40 x 256 in float32: 48 against 52), and so do two tensors of eight packs to 1024 (backward:
// 156 against 187; 92 against 95).  A workgroup that has a compute unit to itself is taken where one round of them does it all:
// forward 56 x 56 x 256 in float32 takes 22 us against 30 in two passes for 16 images (256 slabs), 103 against 102 for 64.
// SHORT: packs of eight 16-bit values, whose sums leave registers for fewer of them (backward 64 x 28 x 28 x 512 in bfloat16:
// 61 us in two passes, 81 with twelve packs to 512 threads); idle slabs of them lose (1024 x 10 x 10 x 544: 72 us forward, 52 in
// two passes).
constexpr long kAny = 1l << 40, kOneRound = 256;

template <bool SHORT, typename F>
bool hold_forward(long rows_bytes, F launch)
{
    const int line = first_line(rows_bytes);
    if (hold_lines(line, kAny, Idle::kNever, launch, Hold<256, 4>(), Hold<512, 8>())) return true;
    if constexpr (SHORT)
        return hold_lines(128, kOneRound, Idle::kNever, launch, Hold<512, 24>());
    else
        return hold_lines(line, kAny, Idle::kNever, launch, Hold<512, 16>()) ||
               hold_lines(128, kOneRound, Idle::kNever, launch, Hold<1024, 16>()) ||
               hold_lines(line, kAny, Idle::kForward, launch, Hold<256, 4>(), Hold<512, 8>(), Hold<512, 16>());
}

template <bool SHORT, typename F>
bool hold_backward(long rows_bytes, F launch)
{
    const int line = first_line(rows_bytes);
    if constexpr (SHORT)
        return hold_lines(line, kAny, Idle::kNever, launch, Hold<256, 4>(), Hold<256, 8>()) ||
               hold_lines(128, kOneRound, Idle::kNever, launch, Hold<512, 12>());
    else
        return hold_lines(line, kAny, Idle::kNever, launch, Hold<256, 4>(), Hold<512, 8>()) ||
               hold_lines(line, kAny, Idle::kNever, launch, Hold<1024, 8>()) ||
               hold_lines(line, kAny, Idle::kBackward, launch, Hold<256, 4>(), Hold<512, 8>(), Hold<1024, 8>());
}

// Calls launch(threads, packs) for the smallest workgroup whose registers hold `packs` packs of a group that is one run of
// memory; whether there is one.  SHORT: packs of eight 16-bit values, of which a thread holds fewer (64 x 256 x 56 x 56 in
// bfloat16: 55 us with eight each to 512 threads, 72 with sixteen to 256; in float32 89 with sixteen to 512, 106 with eight to
// 1024).
template <bool SHORT, typename F>
bool hold_group(long packs, F launch)
{
    using std::integral_constant;
    if (packs <= 256 * 4) launch(integral_constant<int, 256>(), integral_constant<int, 4>());
    else if (packs <= 512 * 8) launch(integral_constant<int, 512>(), integral_constant<int, 8>());
    else if (packs <= 1024 * 8) launch(integral_constant<int, SHORT ? 1024 : 512>(), integral_constant<int, SHORT ? 8 : 16>());
    else if (packs <= 1024 * 16 && !SHORT) launch(integral_constant<int, 1024>(), integral_constant<int, SHORT ? 8 : 16>());
    else return false;
    return true;
}

bool first_whole(int size, int pixels, int cg, bool aligned, long groups)
{
    const long elements = (long)cg * pixels;
    auto any = [](auto, auto) {};
    return aligned && elements % (16 / size) == 0 && groups * 1024 < (1l << 32) &&
           (size == 2 ? hold_group<true>(elements * size / 16, any) : hold_group<false>(elements * size / 16, any));
}

size_t workspace_bytes_of(int dtype, bool nhwc, bool backward, long images, int channels, int pixels, int groups, bool aligned)
{
    const int size = size_of(dtype), wide = dtype == kDtypeF64 ? 8 : 4;
    const int v = aligned ? pack_of(size, channels, channels / groups) : 1;
    long moments = images * channels, sums = images * channels, joined = 0;      // pieces of groups, of channels, channels of images
    if (nhwc) {
        auto fits = [&](int line, long most, Idle idle, auto threads, auto packs) {
            GnLast g;
            return whole_shape(&g, images, channels, pixels, groups, v, size, line, most, idle, threads, packs);
        };
        const long rows_bytes = images * channels * size;
        if (!backward && (size == 2 ? hold_forward<true>(rows_bytes, fits) : hold_forward<false>(rows_bytes, fits))) return 0;
        const GnLast g = last_shape(images, channels, pixels, groups, v);
        moments = images * groups * g.splits;
        sums = images * channels * g.splits;
        if (joined_backward(g)) joined = images * channels;
    } else if (!backward && first_whole(size, pixels, channels / groups, aligned, images * groups)) {
        return 0;
    }
    return (size_t)(backward ? 2 * (sums + joined + images * groups) : 2 * moments) * wide;
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

// Calls launch(threads of a plane) for channels first: eight packs or more to a thread, where a plane has them, so that small
// planes share workgroups; four threads for the smallest, whose time goes into a plane's constants and sums (backward
// 64 x 1024 x 4 x 4 in float32: 13 us with four, 19 with sixteen; 64 x 2048 x 7 x 7, of twelve packs: 47 and 37, and of six in
// bfloat16: 29 and 36).
template <typename T, typename F>
int with_plane(int pixels, F launch)
{
    using std::integral_constant;
    const int packs = pixels / (16 / (int)sizeof(T));
    if (packs <= 4 * 2) return launch(integral_constant<int, 4>());
    if (packs < 16 * 8) return launch(integral_constant<int, 16>());
    if (packs < kWave * 8) return launch(integral_constant<int, kWave>());
    return launch(integral_constant<int, kT>());
}

long wave_blocks(long waves) { return (waves + kWaves - 1) / kWaves; }

long plane_blocks(long planes, int threads) { return (planes + kT / threads - 1) / (kT / threads); }

// The same choice as kJoinForward for channels first, where every plane would join the moments of its group's planes, by the
// plane's threads, a wave at most.  In bfloat16: 64 x 2048 x 7 x 7 in one group (512 moments a lane) 236 us and 24 joined once,
// 64 x 1024 x 14 x 14 (64) 74 and 25; in groups of 73, 64 x 1022 x 7 x 7 (19) 14.0 and 12.1; in groups of 51, x 1020 x 3 x 3 (13) 10.7
// and 9.7 for 64 images, 7.7 and 8.5 for eight; in groups of 37, 64 x 148 x 7 x 7 (10) 8.1 and 9.1; in groups of 131, 128 x 1048 x 13 x
// 13 in float32 (9) 63 and 69; in one group in float32, 64 x 256 x 56 x 56 (4) 101 and 104.
constexpr long kJoinPlanes = 12;

bool joined_planes(int cg, int threads)
{
    const int lanes = threads < kWave ? threads : kWave;
    return (cg + lanes - 1) / lanes > kJoinPlanes;
}

unsigned eights(long blocks) { return (unsigned)((blocks + 7) / 8 * 8); }

template <typename T, int ACT>
int forward(int nhwc, const T* x, const wide_t<T>* gamma, const wide_t<T>* beta, T* y, wide_t<T>* mean, wide_t<T>* inv_std,
            long images, int channels, int pixels, int groups, double eps, void* workspace, hipStream_t st)
{
    using A = wide_t<T>;
    Moments<A>* part = static_cast<Moments<A>*>(workspace);
    if (nhwc) {
        const int v = aligned16(x) && aligned16(y) ? pack_of(sizeof(T), channels, channels / groups) : 1;
        GnLast g;
        auto whole = [&](int line, long most, Idle idle, auto threads, auto packs) {
            constexpr int N = decltype(threads)::value, M = decltype(packs)::value;
            if (!whole_shape(&g, images, channels, pixels, groups, v, sizeof(T), line, most, idle, N, M)) return false;
            hipLaunchKernelGGL((gn_last_whole<T, 16 / (int)sizeof(T), ACT, N, M>), dim3(eights(g.pieces)), dim3(N), 0, st, x,
                               gamma, beta, y, mean, inv_std, eps, g);
            return true;
        };
        if (hold_forward<sizeof(T) == 2>(images * channels * (long)sizeof(T), whole)) {
            HIP_RETURN_IF_LAUNCH_FAILED();
            return PYDTNN_HIP_OK;
        }
        g = last_shape(images, channels, pixels, groups, v);
        if (too_many(g.pieces + 8) || (joined_forward(g) && too_many(wave_blocks(images * groups))))
            return PYDTNN_HIP_ERR_UNSUPPORTED;
        return with_pack(v, [&](auto pack) {
            constexpr int V = decltype(pack)::value * sizeof(T) <= 16 ? decltype(pack)::value : 1;
            hipLaunchKernelGGL((gn_last_moments<T, V>), dim3((unsigned)g.pieces), dim3(kT), 0, st, x, part, g);
            if (joined_forward(g))
                hipLaunchKernelGGL((gn_join_groups<A>), dim3((unsigned)wave_blocks(images * groups)), dim3(kT), 0, st, part, mean,
                                   inv_std, images * groups, g.splits, (long)pixels, (long)g.run, g.cg, eps);
            hipLaunchKernelGGL((gn_last_apply<T, V, ACT>), dim3(eights(g.pieces)), dim3(kT), 0, st, x, gamma, beta,
                               joined_forward(g) ? nullptr : part, y, mean, inv_std, eps, g);
            HIP_RETURN_IF_LAUNCH_FAILED();
            return PYDTNN_HIP_OK;
        });
    }
    const int cg = channels / groups;
    const GnFirst g = {images * channels, pixels, channels, cg, make_fastdiv((uint32_t)pixels)};
    const bool aligned = aligned16(x) && aligned16(y);
    if (first_whole(sizeof(T), pixels, cg, aligned, images * groups)) {
        constexpr int V = 16 / sizeof(T);
        hold_group<sizeof(T) == 2>((long)cg * pixels / V, [&](auto threads, auto packs) {
            constexpr int N = decltype(threads)::value, M = decltype(packs)::value;
            GnLast join = {images, pixels, 1, 1, 1, 1, 1, 1, N, 1, 1, 1, 1, 1, 1, {}};
            set_joins(&join, N, 1);
            hipLaunchKernelGGL((gn_first_whole<T, V, ACT, N, M>), dim3((unsigned)(images * groups)), dim3(N), 0, st, x, gamma,
                               beta, y, mean, inv_std, eps, g, join);
        });
        HIP_RETURN_IF_LAUNCH_FAILED();
        return PYDTNN_HIP_OK;
    }
    return with_plane<T>(pixels, [&](auto threads) {
        constexpr int V = 16 / sizeof(T), N = decltype(threads)::value;
        const long blocks = plane_blocks(g.planes, N);
        const bool joined = joined_planes(cg, N);
        if (too_many(blocks) || (joined && too_many(wave_blocks(images * groups)))) return PYDTNN_HIP_ERR_UNSUPPORTED;
        hipLaunchKernelGGL((gn_first_moments<T, V, N>), dim3((unsigned)blocks), dim3(kT), 0, st, x, part, g);
        if (joined)
            hipLaunchKernelGGL((gn_join_groups<A>), dim3((unsigned)wave_blocks(images * groups)), dim3(kT), 0, st, part, mean,
                               inv_std, images * groups, cg, (long)cg * pixels, (long)pixels, 1, eps);
        hipLaunchKernelGGL((gn_first_apply<T, V, N, ACT>), dim3((unsigned)blocks), dim3(kT), 0, st, x, gamma, beta,
                           joined ? nullptr : part, y, mean, inv_std, eps, g);
        HIP_RETURN_IF_LAUNCH_FAILED();
        return PYDTNN_HIP_OK;
    });
}

template <typename T, int ACT>
int backward(int nhwc, const T* dy, const T* x, const wide_t<T>* gamma, const wide_t<T>* beta, const wide_t<T>* mean,
             const wide_t<T>* inv_std, wide_t<T>* dgamma, wide_t<T>* dbeta, T* dx, long images, int channels, int pixels,
             int groups, void* workspace, hipStream_t st)
{
    using A = wide_t<T>;
    A* sums = static_cast<A*>(workspace);
    const int cg = channels / groups;
    const int param_blocks = (channels + kParamChannels - 1) / kParamChannels;
    auto params = [&](long pieces) {
        hipLaunchKernelGGL((gn_bwd_params<A>), dim3((unsigned)param_blocks), dim3(kT), 0, st, sums, dgamma, dbeta, pieces,
                           channels);
    };
    if (nhwc) {
        const int v = aligned16(x) && aligned16(dy) && aligned16(dx) ? pack_of(sizeof(T), channels, cg) : 1;
        GnLast g;
        auto whole = [&](int line, long most, Idle idle, auto threads, auto packs) {
            constexpr int N = decltype(threads)::value, M = decltype(packs)::value;
            if (!whole_shape(&g, images, channels, pixels, groups, v, sizeof(T), line, most, idle, N, M)) return false;
            hipLaunchKernelGGL((gn_last_bwd_whole<T, 16 / (int)sizeof(T), ACT, N, M>), dim3(eights(g.pieces)), dim3(N), 0, st,
                               dy, x, gamma, beta, mean, inv_std, sums, dx, g);
            params(images);
            return true;
        };
        if (hold_backward<sizeof(T) == 2>(images * channels * (long)sizeof(T), whole)) {
            HIP_RETURN_IF_LAUNCH_FAILED();
            return PYDTNN_HIP_OK;
        }
        g = last_shape(images, channels, pixels, groups, v);
        // the first workgroups of the second pass, in eights so that its pieces keep their dies, are those of the parameters
        const long ahead = eights(param_blocks);
        const bool joined = dx && joined_backward(g);
        if (too_many(g.pieces + 8 + ahead) || (joined && too_many(images * std::max((long)param_blocks, wave_blocks(groups)))))
            return PYDTNN_HIP_ERR_UNSUPPORTED;
        A* image_sums = sums + 2 * images * g.splits * channels;
        A* ab = joined ? image_sums + 2 * images * channels : nullptr;
        return with_pack(v, [&](auto pack) {
            constexpr int V = decltype(pack)::value * sizeof(T) <= 16 ? decltype(pack)::value : 1;
            hipLaunchKernelGGL((gn_last_bwd_sums<T, V, ACT>), dim3((unsigned)g.pieces), dim3(kT), 0, st, dy, x, gamma, beta,
                               mean, inv_std, sums, g);
            if (joined) {
                hipLaunchKernelGGL((gn_bwd_images<A>), dim3((unsigned)(images * param_blocks)), dim3(kT), 0, st, sums, image_sums,
                                   images, g.splits, channels, param_blocks);
                hipLaunchKernelGGL((gn_bwd_groups<A>), dim3((unsigned)wave_blocks(images * groups)), dim3(kT), 0, st, image_sums,
                                   gamma, ab, images, channels, groups, (double)cg * pixels);
            }
            if (dx) hipLaunchKernelGGL((gn_last_bwd_apply<T, V, ACT>), dim3((unsigned)(ahead + eights(g.pieces))), dim3(kT), 0,
                                       st, dy, x, gamma, beta, mean, inv_std, sums, ab, dgamma, dbeta, dx, (int)ahead, g);
            else params(images * g.splits);
            HIP_RETURN_IF_LAUNCH_FAILED();
            return PYDTNN_HIP_OK;
        });
    }
    const GnFirst g = {images * channels, pixels, channels, cg, make_fastdiv((uint32_t)pixels)};
    return with_plane<T>(pixels, [&](auto threads) {
        constexpr int V = 16 / sizeof(T), N = decltype(threads)::value;
        const long blocks = plane_blocks(g.planes, N);
        if (too_many(blocks)) return PYDTNN_HIP_ERR_UNSUPPORTED;
        A* ab = sums + 2 * g.planes;
        hipLaunchKernelGGL((gn_first_bwd_sums<T, V, N, ACT>), dim3((unsigned)blocks), dim3(kT), 0, st, dy, x, gamma, beta, mean,
                           inv_std, sums, g);
        params(images);
        if (dx) {
            hipLaunchKernelGGL((gn_bwd_groups<A>), dim3((unsigned)wave_blocks(images * groups)), dim3(kT), 0, st,
                               sums, gamma, ab, images, channels, groups, (double)cg * pixels);
            hipLaunchKernelGGL((gn_first_bwd_apply<T, V, N, ACT>), dim3((unsigned)blocks), dim3(kT), 0, st, dy, x, gamma, beta,
                               mean, inv_std, ab, dx, g);
        }
        HIP_RETURN_IF_LAUNCH_FAILED();
        return PYDTNN_HIP_OK;
    });
}

}  // namespace

extern "C" {

size_t pydtnn_hip_gn_workspace_bytes(int dtype, int nhwc, int backward, long images, long channels, long pixels, long groups,
                                     int aligned)
{
    if (check(images, channels, pixels, groups) != PYDTNN_HIP_OK || dtype < kDtypeF32 || dtype > kDtypeBF16) return 0;
    return workspace_bytes_of(dtype, nhwc != 0, backward != 0, images, (int)channels, (int)pixels, (int)groups, aligned != 0);
}

int pydtnn_hip_gn_forward(int dtype, int nhwc, const void* x, const void* gamma, const void* beta, void* y, void* mean,
                          void* inv_std, long images, long channels, long pixels, long groups, double eps, int activation,
                          void* workspace, size_t workspace_bytes, void* stream)
{
    if (!x || !gamma || !beta || !y || !mean || !inv_std || !(eps >= 0.0)) return PYDTNN_HIP_ERR_INVALID;
    const int rc = check(images, channels, pixels, groups);
    if (rc != PYDTNN_HIP_OK) return rc;
    const size_t need = pydtnn_hip_gn_workspace_bytes(dtype, nhwc, 0, images, channels, pixels, groups,
                                                      aligned16(x) && aligned16(y));
    if (need && (!workspace || !aligned16(workspace) || workspace_bytes < need)) return PYDTNN_HIP_ERR_WORKSPACE;
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
    const size_t need = pydtnn_hip_gn_workspace_bytes(dtype, nhwc, 1, images, channels, pixels, groups,
                                                      aligned16(x) && aligned16(dy) && aligned16(dx));
    if (!workspace || !aligned16(workspace) || workspace_bytes < need) return PYDTNN_HIP_ERR_WORKSPACE;
    // (the kernels of channels and of groups; those of x count their own)
    if (too_many((channels + kParamChannels - 1) / kParamChannels) ||
        (!nhwc && too_many(wave_blocks(images * groups))))
        return PYDTNN_HIP_ERR_UNSUPPORTED;
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
