// Group norm with an activation, channels last, and its gradient.
//
// Memory-bound: x (and dy) once for the sums and once for the result, which is three passes over an activation forward and five
// backward.  64 x 3999 x 512 bf16 forward 136 us (5.8 TB/s of what it moves; a copy of 1 GiB reaches 5.1 here), 16 x 3999 x 512 fp32
// forward 75 us and backward 110 us (5.3 and 6.0 TB/s); small calls are two launches of 5 us.
//
// A workgroup takes `width` neighbouring channels, the whole frame where it can, of some frames of one utterance.  Its sums go to the
// workspace per (chunk of frames, slice, group), a group's sums lie in every slice that it touches, and the workgroups that use a
// group's sums join them themselves: no atomics, the same order every time.
//
// The second read comes from the 256 MB cache behind the L2s as far as the first has left it there: what was read last is still
// there, so the second launch walks the work backwards, and results are stored past the caches (64 x 3999 x 512 bf16: the sums of the
// next call then find no results to write back, 48 us instead of 72).  A read from that cache is not much faster than one from memory
// (5.9 and 5.2 TB/s), so walking a batch in parts that fit it was no gain.
//
// Statistics: each thread sums u - K and (u - K)^2 over its frames, 64 at most, in 32 bits, K the first of its own values.  So a mean far
// from zero costs no digits of the variance, and an untypical K is that of one thread: as K is among the n values, the
// squares sum to no more than n times their squared deviations from the mean.  From there on everything is joined in 64 bits as (count,
// mean, sum of squared deviations); a K for the whole chunk and 32-bit joins lost 2.5 % of a variance to one frame.
#pragma once
#include <algorithm>
#include "msf2_rows.h"

namespace msf2 {

constexpr int GN_T = 512;                    // most threads of a workgroup
constexpr int GN_LANES = 128;                // most lanes over the channels of a frame
constexpr int GN_ROWS = 64;                  // frames a thread sums in 32 bits at most

// Division of the work: `slices` of `width` channels (`lanes` x V) by `chunks` of `rows` frames by utterances.  Within a slice a
// group counts from the first that touches it; at most `local` groups do.
struct GnPlan {
    int lanes, step, threads, width, slices, chunks, rows, local, D;     // step: frames that a workgroup takes side by side
    Divider by_D, by_width, by_step;
    __device__ int group(int c) const { return by_D.div(c); }
    __device__ int first(int slice) const { return group(slice * width); }
    __device__ int last(int slice, int C) const { return group(min((slice + 1) * width, C) - 1); }
};

// A thread's place.  The lane of the last channels is moved left to end with the row, so that every access is a whole vector: what
// it shares with its neighbour (below `own`) counts for nothing in sums and is stored twice with the same value -- but for the lane that
// is moved into the slice before (`astray`), whose groups this workgroup does not know: it stores its own channels only.
template <int V> struct GnPlace {
    int b, slice, chunk, c, r0, step, have, own;
    bool astray;
    __device__ GnPlace(const GnPlan& pl, unsigned block, int C) {
        slice = block % pl.slices;
        const unsigned rest = block / pl.slices;
        chunk = rest % pl.chunks;
        b = rest / pl.chunks;
        r0 = threadIdx.x / pl.lanes;
        c = slice * pl.width + (threadIdx.x - r0 * pl.lanes) * V;
        step = pl.step;
        have = r0 < step ? min(C - c, V) : 0;        // channels of this lane, none or less past the row's end
        own = C >= V && have > 0 ? V - have : 0;
        c -= own;
        astray = own && c < slice * pl.width;
    }
};

// z from a deviation from the mean, ga = gamma rstd: the same expression in every pass, so that the gradient of a ReLU is that of the
// side of zero on which its result was.
__device__ __forceinline__ float gn_affine(float dev, float ga, float be) { return fmaf(dev, ga, be); }

struct Moments {
    float n, mean, m2;
};

// V channels' values of a vector over channels (null: `none`), and of a pair of values per group.
template <int V> __device__ __forceinline__ void gn_channels(const float* p, int c, int C, float none, float (&f)[V]) {
    if (p && c + V <= C) {
        const auto u = load_vec<V>(p + c);
#pragma unroll
        for (int v = 0; v < V; ++v) f[v] = u[v];
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) f[v] = p && c + v < C ? p[c + v] : none;
    }
}
// g0: the first group that `pairs` holds.
template <int V>
__device__ __forceinline__ void gn_of_groups(const float* pairs, int g0, const GnPlan& pl, int c, int C, float (&a)[V], float (&b)[V]) {
    if (pl.D % V == 0) {                     // one group holds them all, and no lane is moved
        const int g = pl.group(min(c, C - 1)) - g0;
        const float p = pairs[2 * g], q = pairs[2 * g + 1];
#pragma unroll
        for (int v = 0; v < V; ++v) a[v] = p, b[v] = q;
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int k = max(pl.group(min(c + v, C - 1)) - g0, 0);
            a[v] = pairs[2 * k], b[v] = pairs[2 * k + 1];
        }
    }
}

// One vector of a frame.  C < V, the same for the whole launch: frames narrower than a vector.
template <int V, class T> __device__ __forceinline__ typename VecOf<T, V>::type gn_load(const T* p, int C) {
    return C >= V ? load_vec<V>(p) : load_some<V>(p, C);
}
template <int V, class T> __device__ __forceinline__ void gn_store(T* p, int C, const GnPlace<V>& at, const float (&f)[V]) {
    if (C < V) {
        store_some<V>(p, C, f);
    } else if (!at.astray) {
        store_vec<V, true>(p, f);
    } else {
#pragma unroll
        for (int v = 1; v < V; ++v)
            if (v >= at.own) p[v] = (T)f[v];
    }
}
// this thread's own channels into its row of a table [step][width]
template <int V> __device__ __forceinline__ void gn_note(float* table, const GnPlan& pl, const GnPlace<V>& at, const float (&f)[V]) {
    if (at.have <= 0) return;
    float* p = table + at.r0 * pl.width + at.c - at.slice * pl.width;
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (v >= at.own) p[v] = f[v];
}

template <int J> __device__ __forceinline__ double sum_lanes(double v) {
#pragma unroll
    for (int o = 1; o < J; o *= 2) v += __shfl_xor(v, o, 64);
    return v;
}
// f(J) with J threads a group: a wave where there are few
template <class F> __device__ __forceinline__ void gn_spread(int groups, F f) {
    if (groups <= (int)blockDim.x / 64) f(std::integral_constant<int, 64>());
    else if (groups <= (int)blockDim.x / 32) f(std::integral_constant<int, 32>());
    else f(std::integral_constant<int, 16>());
}

// f(J) with J neighbouring lanes a channel of a slice w wide: narrow frames are many side by side, and so a channel's sums are 32 at most
// for a lane.
template <class F> __device__ __forceinline__ void gn_columns(int w, F f) {
    if (w > (int)blockDim.x / 4) f(std::integral_constant<int, 1>());
    else if (w > (int)blockDim.x / 16) f(std::integral_constant<int, 4>());
    else if (w > (int)blockDim.x / 64) f(std::integral_constant<int, 16>());
    else f(std::integral_constant<int, 64>());
}

// Every group that touches a slice, J threads each: f(g, j, each), where each(h) calls h on the group's sums over all
// chunks and slices, a J-th of them a thread.
template <int J, class P, class F> __device__ __forceinline__ void gn_groups(const P* part, const GnPlan& pl, int b, int slice, int C, F f) {
    const int g0 = pl.first(slice), groups = pl.last(slice, C) - g0 + 1, j = threadIdx.x % J;
    for (int g = threadIdx.x / J; g < groups; g += blockDim.x / J) {
        const int a = pl.by_width.div((g0 + g) * pl.D), z = pl.by_width.div((g0 + g + 1) * pl.D - 1);
        f(g, j, [&](auto h) {
            for (int sl = a; sl <= z; ++sl) {
                const P* p = part + ((long)b * pl.chunks * pl.slices + sl) * pl.local + g0 + g - pl.first(sl);
                const long next = (long)pl.slices * pl.local;
#pragma unroll 4
                for (int k = j; k < pl.chunks; k += J) h(p[k * next]);
            }
        });
    }
}

// ---- statistics --------------------------------------------------------------------------------
// part [B][chunks][slices][local] of Moments
template <class T, int V, int PRE>
__global__ __launch_bounds__(GN_T) void gn_moments_kernel(Rows<const T> x, const int* lengths, Moments* part, GnPlan pl, int S, int C) {
    constexpr int U = 2;
    __shared__ float s_s[GN_T * V], q_s[GN_T * V];
    const GnPlace<V> at(pl, blockIdx.x, C);
    const int n = frames_of(lengths, at.b, S), s0 = at.chunk * pl.rows, s1 = min(s0 + pl.rows, n), c0 = at.slice * pl.width;
    const unsigned count = max(s1 - s0, 0), rounds = pl.by_step.div(count), more = count - rounds * at.step;
    auto frames = [&](int r0) { return rounds + ((unsigned)r0 < more); };       // of the threads r0 of the workgroup
    typename VecOf<T, V>::type u[U];
    const bool some = at.have > 0 && s0 + at.r0 < s1;
    auto fetch = [&](int r) {
#pragma unroll
        for (int j = 0; j < U; ++j) u[j] = gn_load<V>(x.at(at.b, min(r + j * at.step, s1 - 1)) + at.c, C);
    };
    float K[V], s[V], q[V];
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = q[v] = 0.f;
    if (some) {
        fetch(s0 + at.r0);
#pragma unroll
        for (int v = 0; v < V; ++v) K[v] = act_f<PRE, fine<T>()>((float)u[0][v]);
        for (int r = s0 + at.r0; r < s1; r += U * at.step) {
            typename VecOf<T, V>::type w[U];
#pragma unroll
            for (int j = 0; j < U; ++j) w[j] = u[j];
            if (r + U * at.step < s1) fetch(r + U * at.step);
#pragma unroll
            for (int j = 0; j < U; ++j) {
                if (r + j * at.step >= s1) break;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float d = act_f<PRE, fine<T>()>((float)w[j][v]) - K[v];
                    s[v] += d;
                    q[v] = fmaf(d, d, q[v]);
                }
            }
        }
    }
    if (some) {                              // s becomes the mean, q the squared deviations from it; not a number stays one
        const float inv = 1.f / (float)frames(at.r0);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float m = fmaf(-s[v] * inv, s[v], q[v]);
            q[v] = m < 0.f ? 0.f : m;
            s[v] = fmaf(s[v], inv, K[v]);
        }
    }
    gn_note<V>(s_s, pl, at, s);
    gn_note<V>(q_s, pl, at, q);
    __syncthreads();
    // a channel's frames together: (mean, squared deviations) over the chunk; the J lanes of column i alone read and write it
    const int w = min(pl.width, C - c0);
    gn_columns(count ? w : 0, [&](auto jj) {
        constexpr int J = decltype(jj)::value;
        const int j = threadIdx.x % J;
        const double inv = 1. / count;
        for (int i = threadIdx.x / J; i < (count ? w : 0); i += blockDim.x / J) {
            const double first = s_s[i];
            double p = 0, m = 0;
            for (int k = j; k < at.step; k += J) {
                const double d = s_s[k * pl.width + i] - first, n = frames(k);
                p += n * d;
                m += q_s[k * pl.width + i] + n * d * d;
            }
            p = sum_lanes<J>(p);
            m = sum_lanes<J>(m);
            m -= p * inv * p;
            if (j == 0) {
                s_s[i] = (float)(first + p * inv);
                q_s[i] = m < 0 ? 0.f : (float)m;
            }
        }
    });
    __syncthreads();
    const int g0 = pl.first(at.slice), groups = pl.last(at.slice, C) - g0 + 1;
    Moments* out = part + (((long)at.b * pl.chunks + at.chunk) * pl.slices + at.slice) * pl.local;
    gn_spread(groups, [&](auto jj) {
        constexpr int J = decltype(jj)::value;
        const int j = threadIdx.x % J;
        for (int g = threadIdx.x / J; g < groups; g += blockDim.x / J) {
            const int w0 = max((g0 + g) * pl.D - c0, 0), w1 = min((g0 + g + 1) * pl.D - c0, w);
            double mean = 0, m2 = 0;
            for (int i = w0 + j; i < w1; i += J) mean += s_s[i];
            mean = sum_lanes<J>(mean) / (w1 - w0);
            for (int i = w0 + j; i < w1; i += J) m2 += (double)count * (s_s[i] - mean) * (s_s[i] - mean) + q_s[i];
            m2 = sum_lanes<J>(m2);
            if (j == 0) out[g] = {(float)count * (float)(w1 - w0), (float)mean, (float)m2};
        }
    });
}

// (mean, rstd) of the groups that touch a slice: st[2 g], st[2 g + 1]; joined in 64 bits
__device__ __forceinline__ void gn_join_moments(const Moments* part, const GnPlan& pl, int b, int slice, int C, float eps, float* st) {
    gn_spread(pl.last(slice, C) - pl.first(slice) + 1, [&](auto jj) {
        constexpr int J = decltype(jj)::value;
        gn_groups<J>(part, pl, b, slice, C, [&](int g, int j, auto each) {
            double n = 0, sum = 0, sq = 0;
            each([&](const Moments& m) {
                const double u = m.mean, k = m.n * u;
                n += m.n;
                sum += k;
                sq += m.m2 + k * u;
            });
            n = sum_lanes<J>(n);
            sum = sum_lanes<J>(sum);
            sq = sum_lanes<J>(sq);
            if (j == 0) {
                const double mean = n > 0 ? sum / n : 0, var = n > 0 ? sq / n - mean * mean : 0;
                st[2 * g] = (float)mean;
                st[2 * g + 1] = n > 0 ? (float)(1 / sqrt((var < 0 ? 0 : var) + eps)) : 0.f;
            }
        });
    });
}

template <class T, int V, int PRE, int POST>
__global__ __launch_bounds__(GN_T) void gn_apply_kernel(Rows<const T> x, const float* gamma, const float* beta, const int* lengths,
                                                        const Moments* part, Rows<T> y, float* stats, float eps, GnPlan pl, int S, int C, int G) {
    constexpr int U = 2;
    extern __shared__ float st[];            // 2 local floats
    const GnPlace<V> at(pl, gridDim.x - 1 - blockIdx.x, C);
    const int n = frames_of(lengths, at.b, S), cap = max(n - 1, 0);        // frames past the end are not fetched
    const int s0 = at.chunk * pl.rows, s1 = min(s0 + pl.rows, S);
    typename VecOf<T, V>::type u[U];
    auto fetch = [&](int r) {
        if (at.have > 0) {
#pragma unroll
            for (int j = 0; j < U; ++j) u[j] = gn_load<V>(x.at(at.b, min(r + j * at.step, min(s1 - 1, cap))) + at.c, C);
        }
    };
    fetch(s0 + at.r0);                       // on its way while the sums are joined
    const int g0 = pl.first(at.slice), groups = pl.last(at.slice, C) - g0 + 1;
    gn_join_moments(part, pl, at.b, at.slice, C, eps, st);
    __syncthreads();
    if (at.chunk == 0)                       // slices that share a group write the same values
        for (int i = threadIdx.x; i < 2 * groups; i += blockDim.x) stats[2 * ((long)at.b * G + g0) + i] = st[i];
    if (at.have <= 0) return;
    float mean[V], ga[V], be[V], rstd[V];
    gn_of_groups<V>(st, g0, pl, at.c, C, mean, rstd);
    gn_channels<V>(gamma, at.c, C, 1.f, ga);
    gn_channels<V>(beta, at.c, C, 0.f, be);
#pragma unroll
    for (int v = 0; v < V; ++v) ga[v] *= rstd[v];
    for (int r = s0 + at.r0; r < s1; r += U * at.step) {
        typename VecOf<T, V>::type w[U];
#pragma unroll
        for (int j = 0; j < U; ++j) w[j] = u[j];
        if (r + U * at.step < s1) fetch(r + U * at.step);
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int s = r + j * at.step;
            if (s >= s1) break;
            float f[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                f[v] = act_f<POST, fine<T>()>(gn_affine(act_f<PRE, fine<T>()>((float)w[j][v]) - mean[v], ga[v], be[v]));
                if (s >= n) f[v] = 0.f;
            }
            gn_store<V>(y.at(at.b, s) + at.c, C, at, f);
        }
    }
}

// ---- gradient ------------------------------------------------------------------------------------
// Sums of dz and dz xh: per channel, chan [B][chunks][2][C], and of their products with gamma per group, part
// [B][chunks][slices][local] pairs.
template <class T, int V, int PRE, int POST>
__global__ __launch_bounds__(GN_T) void gn_grad_sums_kernel(Rows<const T> dy, Rows<const T> x, const float* gamma, const float* beta,
                                                            const float* stats, const int* lengths, float* chan, float2* part, GnPlan pl, int S,
                                                            int C, int G) {
    constexpr int U = 2;
    __shared__ float s1_s[GN_T * V], s2_s[GN_T * V];
    const GnPlace<V> at(pl, blockIdx.x, C);
    const int n = frames_of(lengths, at.b, S), s0 = at.chunk * pl.rows, s1 = min(s0 + pl.rows, n), c0 = at.slice * pl.width;
    typename VecOf<T, V>::type u[U], d[U];
    auto fetch = [&](int r) {
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int s = min(r + j * at.step, s1 - 1);
            u[j] = gn_load<V>(x.at(at.b, s) + at.c, C);
            d[j] = gn_load<V>(dy.at(at.b, s) + at.c, C);
        }
    };
    const bool some = at.have > 0 && s0 + at.r0 < s1;
    if (some) fetch(s0 + at.r0);
    float mean[V], rstd[V], ga[V], be[V], a1[V], a2[V];
    gn_of_groups<V>(stats + 2 * (long)at.b * G, 0, pl, at.c, C, mean, rstd);
    gn_channels<V>(gamma, at.c, C, 1.f, ga);
    gn_channels<V>(beta, at.c, C, 0.f, be);
#pragma unroll
    for (int v = 0; v < V; ++v) a1[v] = a2[v] = 0.f, ga[v] *= rstd[v];
    if (some)
        for (int r = s0 + at.r0; r < s1; r += U * at.step) {
            typename VecOf<T, V>::type w[U], e[U];
#pragma unroll
            for (int j = 0; j < U; ++j) w[j] = u[j], e[j] = d[j];
            if (r + U * at.step < s1) fetch(r + U * at.step);
#pragma unroll
            for (int j = 0; j < U; ++j) {
                if (r + j * at.step >= s1) break;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float dev = act_f<PRE, fine<T>()>((float)w[j][v]) - mean[v];
                    const float dz = (float)e[j][v] * act_grad_f<POST, fine<T>()>(gn_affine(dev, ga[v], be[v]));
                    a1[v] += dz;
                    a2[v] = fmaf(dz, dev * rstd[v], a2[v]);
                }
            }
        }
    gn_note<V>(s1_s, pl, at, a1);
    gn_note<V>(s2_s, pl, at, a2);
    __syncthreads();
    const int w = min(pl.width, C - c0);
    float* out = chan + ((long)at.b * pl.chunks + at.chunk) * 2 * C + c0;
    gn_columns(w, [&](auto jj) {
        constexpr int J = decltype(jj)::value;
        const int j = threadIdx.x % J;
        for (int i = threadIdx.x / J; i < w; i += blockDim.x / J) {
            double p = 0, q = 0;
            for (int k = j; k < at.step; k += J) p += s1_s[k * pl.width + i], q += s2_s[k * pl.width + i];
            p = sum_lanes<J>(p);
            q = sum_lanes<J>(q);
            if (j == 0) {
                out[i] = (float)p;
                out[C + i] = (float)q;
                const float k = gamma ? gamma[c0 + i] : 1.f;
                s1_s[i] = (float)p * k;      // the J lanes of column i alone read it
                s2_s[i] = (float)q * k;
            }
        }
    });
    __syncthreads();
    const int g0 = pl.first(at.slice), groups = pl.last(at.slice, C) - g0 + 1;
    gn_spread(groups, [&](auto jj) {
        constexpr int J = decltype(jj)::value;
        const int j = threadIdx.x % J;
        for (int g = threadIdx.x / J; g < groups; g += blockDim.x / J) {
            const int w0 = max((g0 + g) * pl.D - c0, 0), w1 = min((g0 + g + 1) * pl.D - c0, w);
            double p = 0, q = 0;
            for (int i = w0 + j; i < w1; i += J) p += s1_s[i], q += s2_s[i];
            p = sum_lanes<J>(p);
            q = sum_lanes<J>(q);
            if (j == 0) part[(((long)at.b * pl.chunks + at.chunk) * pl.slices + at.slice) * pl.local + g] = make_float2((float)p, (float)q);
        }
    });
}

constexpr int GN_SUM_C = 16;                 // channels of a workgroup that adds up dgamma and dbeta
// dgamma and dbeta of 16 channels over utterances and chunks, in 64 bits
__device__ __forceinline__ void gn_gain_sums(const float* chan, float* dgamma, float* dbeta, long parts, int C, unsigned block) {
    __shared__ double red[2][GN_T / GN_SUM_C][GN_SUM_C];
    const int K = blockDim.x / GN_SUM_C, i = threadIdx.x % GN_SUM_C, k = threadIdx.x / GN_SUM_C, c = block * GN_SUM_C + i;
    double p = 0, q = 0;
    if (c < C) {
#pragma unroll 8
        for (long m = k; m < parts; m += K) p += chan[m * 2 * C + c], q += chan[m * 2 * C + C + c];
    }
    red[0][k][i] = p;
    red[1][k][i] = q;
    __syncthreads();
    if (k == 0 && c < C) {
        p = q = 0;
        for (int m = 0; m < K; ++m) p += red[0][m][i], q += red[1][m][i];
        if (dbeta) dbeta[c] = (float)p;
        if (dgamma) dgamma[c] = (float)q;
    }
}

// The first `gains` workgroups add up dgamma and dbeta, the others give dx.
template <class T, int V, int PRE, int POST>
__global__ __launch_bounds__(GN_T) void gn_dx_kernel(Rows<const T> dy, Rows<const T> x, const float* gamma, const float* beta, const float* stats,
                                                     const int* lengths, const float* chan, const float2* part, Rows<T> dx, float* dgamma,
                                                     float* dbeta, GnPlan pl, unsigned gains, int B, int S, int C, int G) {
    constexpr int U = 2;
    extern __shared__ float st[];            // 2 local floats
    if (blockIdx.x < gains) {
        gn_gain_sums(chan, dgamma, dbeta, (long)B * pl.chunks, C, blockIdx.x);
        return;
    }
    const GnPlace<V> at(pl, gridDim.x - 1 - blockIdx.x, C);
    const int n = frames_of(lengths, at.b, S), cap = max(n - 1, 0), g0 = pl.first(at.slice);
    const int s0 = at.chunk * pl.rows, s1 = min(s0 + pl.rows, S);
    typename VecOf<T, V>::type u[U], d[U];
    auto fetch = [&](int r) {
        if (at.have > 0) {
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int s = min(r + j * at.step, min(s1 - 1, cap));
                u[j] = gn_load<V>(x.at(at.b, s) + at.c, C);
                d[j] = gn_load<V>(dy.at(at.b, s) + at.c, C);
            }
        }
    };
    fetch(s0 + at.r0);
    gn_spread(pl.last(at.slice, C) - g0 + 1, [&](auto jj) {
        constexpr int J = decltype(jj)::value;
        gn_groups<J>(part, pl, at.b, at.slice, C, [&](int g, int j, auto each) {
            double p = 0, q = 0;
            each([&](const float2& m) { p += m.x, q += m.y; });
            p = sum_lanes<J>(p);
            q = sum_lanes<J>(q);
            const double count = (double)n * pl.D;
            if (j == 0) st[2 * g] = n ? (float)(p / count) : 0.f, st[2 * g + 1] = n ? (float)(q / count) : 0.f;
        });
    });
    __syncthreads();
    if (at.have <= 0) return;
    float mean[V], rstd[V], ga[V], be[V], c1[V], c2[V];
    gn_of_groups<V>(stats + 2 * (long)at.b * G, 0, pl, at.c, C, mean, rstd);
    gn_of_groups<V>(st, g0, pl, at.c, C, c1, c2);
    gn_channels<V>(gamma, at.c, C, 1.f, ga);
    gn_channels<V>(beta, at.c, C, 0.f, be);
#pragma unroll
    for (int v = 0; v < V; ++v) ga[v] *= rstd[v], c1[v] *= rstd[v], c2[v] *= rstd[v];
    for (int r = s0 + at.r0; r < s1; r += U * at.step) {
        typename VecOf<T, V>::type w[U], e[U];
#pragma unroll
        for (int j = 0; j < U; ++j) w[j] = u[j], e[j] = d[j];
        if (r + U * at.step < s1) fetch(r + U * at.step);
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int s = r + j * at.step;
            if (s >= s1) break;
            float f[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float xv = (float)w[j][v], dev = act_f<PRE, fine<T>()>(xv) - mean[v];
                const float dz = (float)e[j][v] * act_grad_f<POST, fine<T>()>(gn_affine(dev, ga[v], be[v]));
                f[v] = (fmaf(dz, ga[v], -c1[v]) - dev * rstd[v] * c2[v]) * act_grad_f<PRE, fine<T>()>(xv);
                if (s >= n) f[v] = 0.f;
            }
            gn_store<V>(dx.at(at.b, s) + at.c, C, at, f);
        }
    }
}

constexpr int gn_vec(int bytes) { return 16 / bytes; }         // channels a lane: 16 bytes of a frame

static inline GnPlan gn_plan(int B, int S, int C, int G, int bytes) {
    GnPlan pl;
    const int V = gn_vec(bytes), vecs = (C + V - 1) / V;
    pl.D = C / G;
    pl.by_D = Divider(pl.D);
    // Whole frames up to 128 lanes, so that a workgroup's frames are one piece of memory whatever their width; wider ones in equal slices.
    // As many frames side by side as leave the fewest lanes of the waves idle, in 256 threads or 512.
    const int cuts = (vecs + GN_LANES - 1) / GN_LANES;
    pl.lanes = (vecs + cuts - 1) / cuts;
    pl.step = 256 / pl.lanes;
    auto idle = [&](int step) { const int t = step * pl.lanes; return 1. - (double)t / ((t + 63) / 64 * 64); };
    if (idle(512 / pl.lanes) + 0.05 < idle(pl.step)) pl.step = 512 / pl.lanes;
    pl.threads = (pl.step * pl.lanes + 63) / 64 * 64;
    pl.by_step = Divider(pl.step);
    pl.width = pl.lanes * V;
    pl.by_width = Divider(pl.width);
    pl.slices = (vecs + pl.lanes - 1) / pl.lanes;
    pl.local = std::min(G, (pl.width + pl.D - 2) / pl.D + 1);
    // Chunks for 1024 threads a CU, but no more than let a thread join 12 sums of its groups, while 512 a CU are left (1 x 61499 x 512 bf16
    // in 32 groups: 1009 chunks 91 us, 509 chunks 54); 4 frames a thread at least.
    const long cu256 = 256l * 256 / pl.threads / ((long)B * pl.slices), here = std::min(pl.local, G);
    const long joined = 12 * std::min<long>(pl.threads, 64 * here) / here;
    const long want = std::max(1l, std::min(4 * cu256, std::max(joined, 2 * cu256)));
    pl.rows = (int)std::min<long>(std::max<long>(4 * pl.step, (S + want - 1) / want), (long)GN_ROWS * pl.step);
    pl.chunks = (S + pl.rows - 1) / pl.rows;
    return pl;
}
static inline size_t gn_part_bytes(const GnPlan& pl, int B, size_t each) { return align_up((size_t)B * pl.chunks * pl.slices * pl.local * each); }
static inline size_t gn_ws_bytes(int B, int S, int C, int G, int bytes, bool backward) {
    const GnPlan pl = gn_plan(B, S, C, G, bytes);
    if (!backward) return gn_part_bytes(pl, B, sizeof(Moments));
    return gn_part_bytes(pl, B, sizeof(float2)) + align_up((size_t)B * pl.chunks * 2 * C * sizeof(float));
}

template <class T, int PRE, int POST>
static int run_group_norm(Rows<const T> x, const float* gamma, const float* beta, const int* lengths, Rows<T> y, float* stats, int B, int S, int C,
                          int G, float eps, void* ws, hipStream_t st) {
    constexpr int V = gn_vec(sizeof(T));
    const GnPlan pl = gn_plan(B, S, C, G, sizeof(T));
    const long grid = (long)B * pl.chunks * pl.slices;
    if (!launch_ok(grid, pl.threads)) return MSF2_ERR_ARG;
    gn_moments_kernel<T, V, PRE><<<grid, pl.threads, 0, st>>>(x, lengths, (Moments*)ws, pl, S, C);
    gn_apply_kernel<T, V, PRE, POST>
        <<<grid, pl.threads, pl.local * 2 * sizeof(float), st>>>(x, gamma, beta, lengths, (const Moments*)ws, y, stats, eps, pl, S, C, G);
    return check_launch();
}

template <class T, int PRE, int POST>
static int run_group_norm_backward(Rows<const T> dy, Rows<const T> x, const float* gamma, const float* beta, const float* stats, const int* lengths,
                                   Rows<T> dx, float* dgamma, float* dbeta, int B, int S, int C, int G, void* ws, hipStream_t st) {
    constexpr int V = gn_vec(sizeof(T));
    const GnPlan pl = gn_plan(B, S, C, G, sizeof(T));
    const long grid = (long)B * pl.chunks * pl.slices;
    const long gains = dgamma || dbeta ? (C + GN_SUM_C - 1) / GN_SUM_C : 0;
    if (!launch_ok(grid + gains, pl.threads)) return MSF2_ERR_ARG;
    float2* part = (float2*)ws;
    float* chan = (float*)((char*)ws + gn_part_bytes(pl, B, sizeof(float2)));
    gn_grad_sums_kernel<T, V, PRE, POST><<<grid, pl.threads, 0, st>>>(dy, x, gamma, beta, stats, lengths, chan, part, pl, S, C, G);
    gn_dx_kernel<T, V, PRE, POST><<<grid + gains, pl.threads, pl.local * 2 * sizeof(float), st>>>(
        dy, x, gamma, beta, stats, lengths, chan, part, dx, dgamma, dbeta, pl, (unsigned)gains, B, S, C, G);
    return check_launch();
}

}  // namespace msf2
