// Group norm with an activation, channels last, and its gradient.
//
// Memory-bound: x (and dy) once for the sums and once for the result, the second time from the memory-side cache as far as they
// fit it.  A workgroup takes `slice` neighbouring channels of some frames of one utterance; lanes run over channels first, so a
// frame's part of a slice is whole lines.  Its sums go to the workspace per (chunk of frames, slice, group), a group's sums lie in
// every slice that it touches, and the workgroups of the second launch join those of their groups themselves: two launches a
// pass, no atomics, the same order every time.
//
// Statistics: each thread sums (u - K) and (u - K)^2 over its frames in 32 bits, K the first value that its channel has in the
// chunk, and everything above a thread joins (count, mean, sum of squared deviations) by the pairwise rule
//   n = n1 + n2, mean = mean1 + (mean2 - mean1) n2 / n, M2 = M2_1 + M2_2 + (mean2 - mean1)^2 n1 n2 / n,
// so a mean far from zero costs no digits of the variance.
#pragma once
#include <algorithm>
#include "msf2_rows.h"

namespace msf2 {

constexpr int GN_T = 256;                    // threads of a workgroup
constexpr int GN_JOIN = 16;                  // threads that join the sums of one group where there are many
constexpr int GN_ROWS = 64;                  // frames a thread sums in 32 bits at most

// Division of the work: `slices` of 64 lanes x V channels, or fewer lanes where C is narrow; `chunks` of `rows` frames.
// Within a slice a group counts from the first that touches it; at most `local` groups do.
struct GnPlan {
    int lanes, width, slices, chunks, rows, local, D;
    __host__ __device__ int first(int slice) const { return slice * width / D; }
    __host__ __device__ int last(int slice, int C) const { return (min((slice + 1) * width, C) - 1) / D; }
};

template <int V> struct GnPlace {
    int b, slice, chunk, c, lane, r0, step, have;
    __device__ GnPlace(const GnPlan& pl, int C) {
        slice = blockIdx.x % pl.slices;
        const unsigned rest = blockIdx.x / pl.slices;
        chunk = rest % pl.chunks;
        b = rest / pl.chunks;
        lane = threadIdx.x % pl.lanes;
        c = slice * pl.width + lane * V;
        have = min(C - c, V);                // channels of this lane, none or less past the row's end
        r0 = threadIdx.x / pl.lanes;
        step = GN_T / pl.lanes;
    }
};

struct Moments {
    float n, mean, m2;
    __device__ __forceinline__ void join(const Moments& o) {
        const float t = n + o.n, d = o.mean - mean, k = t > 0.f ? o.n / t : 0.f;
        mean = fmaf(d, k, mean);
        m2 += o.m2 + d * d * n * k;
        n = t;
    }
};

// One vector of a frame: whole, or the last channels of the row.
template <int V, class T> __device__ __forceinline__ typename VecOf<T, V>::type gn_load(const T* p, int have) {
    return have >= V ? load_vec<V>(p) : load_some<V>(p, have);
}
template <int V, class T> __device__ __forceinline__ void gn_store(T* p, int have, const float (&f)[V]) {
    if (have >= V) store_vec<V, true>(p, f);
    else store_some<V>(p, have, f);
}

// ---- sums for the statistics -------------------------------------------------------------------
// part [B][chunks][slices][local] of Moments
template <class T, int V, int PRE>
__global__ __launch_bounds__(GN_T) void gn_moments_kernel(Rows<const T> x, const int* lengths, Moments* part, GnPlan pl, int S, int C) {
    constexpr int U = 4;
    __shared__ float mean_s[GN_T * V], m2_s[GN_T * V];
    __shared__ float rows_s[GN_T];
    const GnPlace<V> at(pl, C);
    const int n = frames_of(lengths, at.b, S);
    const int s0 = at.chunk * pl.rows, s1 = min(s0 + pl.rows, n);
    float K[V], s[V], q[V];
    int count = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) K[v] = s[v] = q[v] = 0.f;
    if (at.have > 0 && s0 + at.r0 < s1) {
        const auto k = gn_load<V>(x.at(at.b, s0 + at.r0) + at.c, at.have);
#pragma unroll
        for (int v = 0; v < V; ++v) K[v] = act_f<PRE, fine<T>()>((float)k[v]);
        for (int r = s0 + at.r0; r < s1; r += U * at.step) {
            typename VecOf<T, V>::type u[U];
#pragma unroll
            for (int j = 0; j < U; ++j) u[j] = gn_load<V>(x.at(at.b, min(r + j * at.step, s1 - 1)) + at.c, at.have);
#pragma unroll
            for (int j = 0; j < U; ++j) {
                if (r + j * at.step >= s1) break;
                ++count;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float d = act_f<PRE, fine<T>()>((float)u[j][v]) - K[v];
                    s[v] += d;
                    q[v] = fmaf(d, d, q[v]);
                }
            }
        }
    }
    const float cnt = (float)count, inv = count ? 1.f / cnt : 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        mean_s[threadIdx.x * V + v] = fmaf(s[v], inv, K[v]);
        m2_s[threadIdx.x * V + v] = fmaxf(fmaf(-s[v] * inv, s[v], q[v]), 0.f);
    }
    rows_s[threadIdx.x] = cnt;
    __syncthreads();
    // a group's channels, and for each the threads that took its frames
    const int g0 = pl.first(at.slice), groups = pl.last(at.slice, C) - g0 + 1, j = threadIdx.x % GN_JOIN;
    Moments* out = part + (((long)at.b * pl.chunks + at.chunk) * pl.slices + at.slice) * pl.local;
    for (int g = threadIdx.x / GN_JOIN; g < groups; g += GN_T / GN_JOIN) {
        const int w0 = max((g0 + g) * pl.D, at.slice * pl.width) - at.slice * pl.width;
        const int w1 = min(min((g0 + g + 1) * pl.D, (at.slice + 1) * pl.width), C) - at.slice * pl.width;
        Moments m = {0.f, 0.f, 0.f};
        for (int w = w0 + j; w < w1; w += GN_JOIN)
            for (int k = 0; k < at.step; ++k) m.join({rows_s[k * pl.lanes], mean_s[k * pl.width + w], m2_s[k * pl.width + w]});
#pragma unroll
        for (int o = 1; o < GN_JOIN; o *= 2) m.join({__shfl_xor(m.n, o, 64), __shfl_xor(m.mean, o, 64), __shfl_xor(m.m2, o, 64)});
        if (j == 0) out[g] = m;
    }
}

// Every group that touches a slice, by J threads each: f(g, each, j), where each(h) calls h on the group's sums over all
// chunks and slices, a J-th of them a thread.
template <int J, class P, class F> __device__ __forceinline__ void gn_groups(const P* part, const GnPlan& pl, int b, int slice, int C, F f) {
    const int g0 = pl.first(slice), groups = pl.last(slice, C) - g0 + 1, j = threadIdx.x % J;
    for (int g = threadIdx.x / J; g < groups; g += GN_T / J) {
        const int a = (g0 + g) * pl.D / pl.width, z = ((g0 + g + 1) * pl.D - 1) / pl.width, over = z - a + 1;
        f(g, j, [&](auto h) {
            for (int i = j; i < pl.chunks * over; i += J) {
                const int k = i / over, sl = a + i % over;
                h(part[(((long)b * pl.chunks + k) * pl.slices + sl) * pl.local + g0 + g - pl.first(sl)]);
            }
        });
    }
}
template <int J> __device__ __forceinline__ double sum_lanes(double v) {
#pragma unroll
    for (int o = 1; o < J; o *= 2) v += __shfl_xor(v, o, 64);
    return v;
}

// (mean, rstd) of the groups that touch this workgroup's slice, in LDS: st[2 g], st[2 g + 1]; joined in 64 bits
template <int J> __device__ __forceinline__ void gn_join_moments(const Moments* part, const GnPlan& pl, int b, int slice, int C, float eps, float* st) {
    gn_groups<J>(part, pl, b, slice, C, [&](int g, int j, auto each) {
        double n = 0, sum = 0, m2 = 0;
        each([&](const Moments& m) { n += m.n; sum += (double)m.n * m.mean; });
        n = sum_lanes<J>(n);
        sum = sum_lanes<J>(sum);
        const double mean = n > 0 ? sum / n : 0;
        each([&](const Moments& m) { m2 += m.m2 + m.n * (m.mean - mean) * (m.mean - mean); });
        m2 = sum_lanes<J>(m2);
        if (j == 0) {
            st[2 * g] = (float)mean;
            st[2 * g + 1] = n > 0 ? (float)(1 / sqrt(m2 / n + eps)) : 0.f;
        }
    });
}
// (c1, c2) likewise, n the group's count of values
template <int J> __device__ __forceinline__ void gn_join_sums(const float2* part, const GnPlan& pl, int b, int slice, int C, double n, float* st) {
    gn_groups<J>(part, pl, b, slice, C, [&](int g, int j, auto each) {
        double p = 0, q = 0;
        each([&](const float2& m) { p += m.x; q += m.y; });
        p = sum_lanes<J>(p);
        q = sum_lanes<J>(q);
        if (j == 0) st[2 * g] = n > 0 ? (float)(p / n) : 0.f, st[2 * g + 1] = n > 0 ? (float)(q / n) : 0.f;
    });
}

template <class T, int V, int PRE, int POST>
__global__ __launch_bounds__(GN_T) void gn_apply_kernel(Rows<const T> x, const float* gamma, const float* beta, const int* lengths,
                                                        const Moments* part, Rows<T> y, float* stats, float eps, GnPlan pl, int S, int C, int G) {
    constexpr int U = 4;
    extern __shared__ float st[];
    const GnPlace<V> at(pl, C);
    const int g0 = pl.first(at.slice), groups = pl.last(at.slice, C) - g0 + 1;
    if (groups <= GN_T / 64) gn_join_moments<64>(part, pl, at.b, at.slice, C, eps, st);
    else gn_join_moments<GN_JOIN>(part, pl, at.b, at.slice, C, eps, st);
    __syncthreads();
    if (at.chunk == 0)                       // slices that share a group write the same values
        for (int i = threadIdx.x; i < 2 * groups; i += GN_T) stats[2 * ((long)at.b * G + g0) + i] = st[i];
    if (at.have <= 0) return;
    float mean[V], ga[V], be[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = min(at.c + v, C - 1), g = c / pl.D - g0;
        mean[v] = st[2 * g];
        ga[v] = st[2 * g + 1] * (gamma ? gamma[c] : 1.f);
        be[v] = beta ? beta[c] : 0.f;
    }
    const int n = frames_of(lengths, at.b, S), cap = max(n - 1, 0);        // frames past the end are not fetched
    const int s0 = at.chunk * pl.rows, s1 = min(s0 + pl.rows, S);
    for (int r = s0 + at.r0; r < s1; r += U * at.step) {
        typename VecOf<T, V>::type u[U];
#pragma unroll
        for (int j = 0; j < U; ++j) u[j] = gn_load<V>(x.at(at.b, min(r + j * at.step, min(s1 - 1, cap))) + at.c, at.have);
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int s = r + j * at.step;
            if (s >= s1) break;
            float f[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                f[v] = act_f<POST, fine<T>()>(fmaf(act_f<PRE, fine<T>()>((float)u[j][v]) - mean[v], ga[v], be[v]));
                if (s >= n) f[v] = 0.f;
            }
            gn_store<V>(y.at(at.b, s) + at.c, at.have, f);
        }
    }
}

// ---- gradient ------------------------------------------------------------------------------------
// Sums of dz and dz xh: per channel, chan [B][chunks][2][C], and of their products with gamma per group, part
// [B][chunks][slices][local] pairs.
template <class T, int V, int PRE, int POST>
__global__ __launch_bounds__(GN_T) void gn_grad_sums_kernel(Rows<const T> dy, Rows<const T> x, const float* gamma, const float* beta,
                                                            const float* stats, const int* lengths, float* chan, float2* part, GnPlan pl,
                                                            int S, int C, int G) {
    constexpr int U = 4;
    __shared__ float s1_s[GN_T * V], s2_s[GN_T * V];
    const GnPlace<V> at(pl, C);
    const int n = frames_of(lengths, at.b, S);
    const int s0 = at.chunk * pl.rows, s1 = min(s0 + pl.rows, n);
    float mean[V], rstd[V], ga[V], be[V], a1[V], a2[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = min(at.c + v, C - 1);
        const float* st = stats + 2 * ((long)at.b * G + c / pl.D);
        mean[v] = st[0];
        rstd[v] = st[1];
        ga[v] = gamma ? gamma[c] : 1.f;
        be[v] = beta ? beta[c] : 0.f;
        a1[v] = a2[v] = 0.f;
    }
    if (at.have > 0)
        for (int r = s0 + at.r0; r < s1; r += U * at.step) {
            typename VecOf<T, V>::type u[U], d[U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int s = min(r + j * at.step, s1 - 1);
                u[j] = gn_load<V>(x.at(at.b, s) + at.c, at.have);
                d[j] = gn_load<V>(dy.at(at.b, s) + at.c, at.have);
            }
#pragma unroll
            for (int j = 0; j < U; ++j) {
                if (r + j * at.step >= s1) break;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float xh = (act_f<PRE, fine<T>()>((float)u[j][v]) - mean[v]) * rstd[v];
                    const float dz = (float)d[j][v] * act_grad_f<POST, fine<T>()>(fmaf(xh, ga[v], be[v]));
                    a1[v] += dz;
                    a2[v] = fmaf(dz, xh, a2[v]);
                }
            }
        }
#pragma unroll
    for (int v = 0; v < V; ++v) {
        s1_s[threadIdx.x * V + v] = a1[v];
        s2_s[threadIdx.x * V + v] = a2[v];
    }
    __syncthreads();
    const int w = min(pl.width, C - at.slice * pl.width);
    float* out = chan + ((long)at.b * pl.chunks + at.chunk) * 2 * C + at.slice * pl.width;
    for (int i = threadIdx.x; i < w; i += GN_T) {
        float p = 0.f, q = 0.f;
        for (int k = 0; k < at.step; ++k) p += s1_s[k * pl.width + i], q += s2_s[k * pl.width + i];
        out[i] = s1_s[i] = p;                // this thread alone reads column i
        out[C + i] = s2_s[i] = q;
    }
    __syncthreads();
    const int g0 = pl.first(at.slice), groups = pl.last(at.slice, C) - g0 + 1, j = threadIdx.x % GN_JOIN, c0 = at.slice * pl.width;
    for (int g = threadIdx.x / GN_JOIN; g < groups; g += GN_T / GN_JOIN) {
        const int w0 = max((g0 + g) * pl.D, c0) - c0, w1 = min((g0 + g + 1) * pl.D - c0, w);
        float p = 0.f, q = 0.f;
        for (int i = w0 + j; i < w1; i += GN_JOIN) {
            const float k = gamma ? gamma[c0 + i] : 1.f;
            p = fmaf(k, s1_s[i], p);
            q = fmaf(k, s2_s[i], q);
        }
        for (int o = 1; o < GN_JOIN; o *= 2) p += __shfl_xor(p, o, 64), q += __shfl_xor(q, o, 64);
        if (j == 0) part[(((long)at.b * pl.chunks + at.chunk) * pl.slices + at.slice) * pl.local + g] = make_float2(p, q);
    }
}

constexpr int GN_DGAMMA_C = 16;              // channels of a workgroup that sums dgamma and dbeta

// The first `sum_blocks` workgroups add up dgamma and dbeta over utterances and chunks; the others give dx.
template <class T, int V, int PRE, int POST>
__global__ __launch_bounds__(GN_T) void gn_dx_kernel(Rows<const T> dy, Rows<const T> x, const float* gamma, const float* beta,
                                                     const float* stats, const int* lengths, const float* chan, const float2* part,
                                                     Rows<T> dx, float* dgamma, float* dbeta, GnPlan pl, int B, int S, int C, int G,
                                                     int sum_blocks) {
    constexpr int U = 4;
    extern __shared__ float st[];
    if ((int)blockIdx.x < sum_blocks) {
        const int c = blockIdx.x * GN_DGAMMA_C + threadIdx.x % GN_DGAMMA_C, k = threadIdx.x / GN_DGAMMA_C;
        constexpr int K = GN_T / GN_DGAMMA_C;
        __shared__ double red[2][K][GN_DGAMMA_C];
        double p = 0, q = 0;
        if (c < C)
#pragma unroll 8
            for (long i = k; i < (long)B * pl.chunks; i += K) p += chan[i * 2 * C + c], q += chan[i * 2 * C + C + c];
        red[0][k][threadIdx.x % GN_DGAMMA_C] = p;
        red[1][k][threadIdx.x % GN_DGAMMA_C] = q;
        __syncthreads();
        if (k == 0 && c < C) {
            p = q = 0;
            for (int i = 0; i < K; ++i) p += red[0][i][threadIdx.x], q += red[1][i][threadIdx.x];
            if (dbeta) dbeta[c] = (float)p;
            if (dgamma) dgamma[c] = (float)q;
        }
        return;
    }
    GnPlace<V> at(pl, C);
    {
        const unsigned id = blockIdx.x - sum_blocks;
        at.slice = id % pl.slices;
        at.chunk = id / pl.slices % pl.chunks;
        at.b = id / pl.slices / pl.chunks;
        at.c = at.slice * pl.width + at.lane * V;
        at.have = min(C - at.c, V);
    }
    const int n = frames_of(lengths, at.b, S);
    const int g0 = pl.first(at.slice);
    if (pl.last(at.slice, C) - g0 < GN_T / 64) gn_join_sums<64>(part, pl, at.b, at.slice, C, (double)n * pl.D, st);
    else gn_join_sums<GN_JOIN>(part, pl, at.b, at.slice, C, (double)n * pl.D, st);
    __syncthreads();
    if (at.have <= 0) return;
    float mean[V], rstd[V], ga[V], be[V], c1[V], c2[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = min(at.c + v, C - 1), g = c / pl.D;
        mean[v] = stats[2 * ((long)at.b * G + g)];
        rstd[v] = stats[2 * ((long)at.b * G + g) + 1];
        ga[v] = gamma ? gamma[c] : 1.f;
        be[v] = beta ? beta[c] : 0.f;
        c1[v] = st[2 * (g - g0)];
        c2[v] = st[2 * (g - g0) + 1];
    }
    const int s0 = at.chunk * pl.rows, s1 = min(s0 + pl.rows, S), cap = max(n - 1, 0);
    for (int r = s0 + at.r0; r < s1; r += U * at.step) {
        typename VecOf<T, V>::type u[U], d[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int s = min(r + j * at.step, min(s1 - 1, cap));
            u[j] = gn_load<V>(x.at(at.b, s) + at.c, at.have);
            d[j] = gn_load<V>(dy.at(at.b, s) + at.c, at.have);
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int s = r + j * at.step;
            if (s >= s1) break;
            float f[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float xv = (float)u[j][v], xh = (act_f<PRE, fine<T>()>(xv) - mean[v]) * rstd[v];
                const float dz = (float)d[j][v] * act_grad_f<POST, fine<T>()>(fmaf(xh, ga[v], be[v]));
                f[v] = rstd[v] * (fmaf(dz, ga[v], -c1[v]) - xh * c2[v]) * act_grad_f<PRE, fine<T>()>(xv);
                if (s >= n) f[v] = 0.f;
            }
            gn_store<V>(dx.at(at.b, s) + at.c, at.have, f);
        }
    }
}

constexpr int gn_vec(int bytes) { return 16 / bytes; }         // channels a lane: 16 bytes of a frame

static inline GnPlan gn_plan(int B, int S, int C, int G, int bytes) {
    GnPlan pl;
    const int V = gn_vec(bytes), vecs = (C + V - 1) / V;
    pl.D = C / G;
    pl.lanes = 1;
    while (pl.lanes < 64 && pl.lanes < vecs) pl.lanes *= 2;
    pl.width = pl.lanes * V;
    pl.slices = (vecs + pl.lanes - 1) / pl.lanes;
    pl.local = std::min(G, (pl.width + pl.D - 2) / pl.D + 1);
    // 8 workgroups a CU, each with 4 frames a thread at least
    const int least = 4 * GN_T / pl.lanes;
    const long want = std::max(1l, 2048 / ((long)B * pl.slices));
    pl.rows = (int)std::min<long>(std::max<long>(least, (S + want - 1) / want), GN_ROWS * GN_T / pl.lanes);
    pl.chunks = (S + pl.rows - 1) / pl.rows;
    return pl;
}
static inline size_t gn_part_bytes(const GnPlan& pl, int B) { return align_up((size_t)B * pl.chunks * pl.slices * pl.local * sizeof(Moments)); }
static inline size_t gn_ws_bytes(int B, int S, int C, int G, int bytes, bool backward) {
    const GnPlan pl = gn_plan(B, S, C, G, bytes);
    return gn_part_bytes(pl, B) + (backward ? align_up((size_t)B * pl.chunks * 2 * C * sizeof(float)) : 0);
}

template <class T, int PRE, int POST>
static int run_group_norm(Rows<const T> x, const float* gamma, const float* beta, const int* lengths, Rows<T> y, float* stats, int B, int S, int C,
                          int G, float eps, void* ws, hipStream_t st) {
    constexpr int V = gn_vec(sizeof(T));
    const GnPlan pl = gn_plan(B, S, C, G, sizeof(T));
    const long grid = (long)B * pl.chunks * pl.slices;
    if (grid > 0x7fffffff) return MSF2_ERR_ARG;
    gn_moments_kernel<T, V, PRE><<<grid, GN_T, 0, st>>>(x, lengths, (Moments*)ws, pl, S, C);
    gn_apply_kernel<T, V, PRE, POST><<<grid, GN_T, pl.local * 2 * sizeof(float), st>>>(x, gamma, beta, lengths, (const Moments*)ws, y, stats, eps, pl, S, C, G);
    return check_launch();
}

template <class T, int PRE, int POST>
static int run_group_norm_backward(Rows<const T> dy, Rows<const T> x, const float* gamma, const float* beta, const float* stats, const int* lengths,
                                   Rows<T> dx, float* dgamma, float* dbeta, int B, int S, int C, int G, void* ws, hipStream_t st) {
    constexpr int V = gn_vec(sizeof(T));
    const GnPlan pl = gn_plan(B, S, C, G, sizeof(T));
    const long grid = (long)B * pl.chunks * pl.slices;
    const int sums = dgamma || dbeta ? (C + GN_DGAMMA_C - 1) / GN_DGAMMA_C : 0;
    if (grid + sums > 0x7fffffff) return MSF2_ERR_ARG;
    float2* part = (float2*)ws;
    float* chan = (float*)((char*)ws + gn_part_bytes(pl, B));
    gn_grad_sums_kernel<T, V, PRE, POST><<<grid, GN_T, 0, st>>>(dy, x, gamma, beta, stats, lengths, chan, part, pl, S, C, G);
    gn_dx_kernel<T, V, PRE, POST><<<grid + sums, GN_T, pl.local * 2 * sizeof(float), st>>>(dy, x, gamma, beta, stats, lengths, chan, part, dx, dgamma,
                                                                                        dbeta, pl, B, S, C, G, sums);
    return check_launch();
}

}  // namespace msf2
