// Group norm with an activation, channels last, and its gradient.
#pragma once
#include "msf2_rows.h"

namespace msf2 {

// grid B * groups, block 256: (mean, rstd) of one group
template <class T, int PRE>
__global__ __launch_bounds__(256) void gn_stats_kernel(Rows<const T> x, const int* lengths, float* stats, int S, int G, int D, float eps) {
    __shared__ double red[4];
    const int b = blockIdx.x / G, g = blockIdx.x % G;
    const long n = (long)frames_of(lengths, b, S) * D;
    auto sum = [&](double mean, int power) {
        double v = 0;
        for (long i = threadIdx.x; i < n; i += 256) {
            const double u = (double)act_f<PRE>((float)x.at(b, i / D)[g * D + i % D]) - mean;
            v += power == 2 ? u * u : u;
        }
        for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        return red[0] + red[1] + red[2] + red[3];
    };
    const double mean = n ? sum(0, 1) / n : 0, var = n ? sum(mean, 2) / n : 0;
    if (threadIdx.x == 0) {
        stats[2 * blockIdx.x] = (float)mean;
        stats[2 * blockIdx.x + 1] = n ? (float)(1 / sqrt(var + eps)) : 0.f;
    }
}

template <class T, int PRE, int POST>
__global__ __launch_bounds__(256) void gn_apply_kernel(Rows<const T> x, const float* gamma, const float* beta, const int* lengths,
                                                       const float* stats, Rows<T> y, int B, int S, int C, int G) {
    const int D = C / G;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < (long)B * S * C; i += (long)gridDim.x * 256) {
        const int c = i % C, s = i / C % S, b = i / C / S;
        const float* st = stats + 2 * (b * G + c / D);
        float v = 0.f;
        if (s < frames_of(lengths, b, S))
            v = act_f<POST>(fmaf((act_f<PRE>((float)x.at(b, s)[c]) - st[0]) * st[1], gamma ? gamma[c] : 1.f, beta ? beta[c] : 0.f));
        y.at(b, s)[c] = (T)v;
    }
}

// dz and xh of one element
template <class T, int PRE, int POST>
__device__ __forceinline__ void gn_grad_at(float xv, float dy, float mean, float rstd, float ga, float be, float& dz, float& xh) {
    xh = (act_f<PRE>(xv) - mean) * rstd;
    dz = dy * act_grad_f<POST>(fmaf(xh, ga, be));
}

// grid B * groups: coef[b][g] = (c1, c2);  grid.y = 1: one block a channel, dgamma and dbeta
template <class T, int PRE, int POST>
__global__ __launch_bounds__(256) void gn_sums_kernel(Rows<const T> dy, Rows<const T> x, const float* gamma, const float* beta,
                                                      const float* stats, const int* lengths, float* coef, float* dgamma,
                                                      float* dbeta, int B, int S, int C, int G, int per_channel) {
    __shared__ double red[8];
    const int D = C / G;
    double s1 = 0, s2 = 0;
    long n = 0;
    const int b0 = per_channel ? 0 : blockIdx.x / G, b1 = per_channel ? B : b0 + 1;
    const int c0 = per_channel ? blockIdx.x : blockIdx.x % G * D, w = per_channel ? 1 : D;
    for (int b = b0; b < b1; ++b) {
        n = (long)frames_of(lengths, b, S) * w;
        for (long i = threadIdx.x; i < n; i += 256) {
            const int s = i / w, c = c0 + i % w;
            const float* st = stats + 2 * (b * G + c / D);
            const float ga = gamma ? gamma[c] : 1.f;
            float dz, xh;
            gn_grad_at<T, PRE, POST>((float)x.at(b, s)[c], (float)dy.at(b, s)[c], st[0], st[1], ga, beta ? beta[c] : 0.f, dz, xh);
            const double k = per_channel ? dz : (double)dz * ga;
            s1 += k;
            s2 += k * xh;
        }
    }
    for (int o = 32; o > 0; o >>= 1) { s1 += __shfl_xor(s1, o, 64); s2 += __shfl_xor(s2, o, 64); }
    if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6] = s1; red[4 + (threadIdx.x >> 6)] = s2; }
    __syncthreads();
    if (threadIdx.x == 0) {
        s1 = red[0] + red[1] + red[2] + red[3];
        s2 = red[4] + red[5] + red[6] + red[7];
        if (per_channel) {
            if (dbeta) dbeta[blockIdx.x] = (float)s1;
            if (dgamma) dgamma[blockIdx.x] = (float)s2;
        } else {
            coef[2 * blockIdx.x] = n ? (float)(s1 / n) : 0.f;
            coef[2 * blockIdx.x + 1] = n ? (float)(s2 / n) : 0.f;
        }
    }
}

template <class T, int PRE, int POST>
__global__ __launch_bounds__(256) void gn_dx_kernel(Rows<const T> dy, Rows<const T> x, const float* gamma, const float* beta,
                                                    const float* stats, const int* lengths, const float* coef, Rows<T> dx,
                                                    int B, int S, int C, int G) {
    const int D = C / G;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < (long)B * S * C; i += (long)gridDim.x * 256) {
        const int c = i % C, s = i / C % S, b = i / C / S, at = 2 * (b * G + c / D);
        float v = 0.f;
        if (s < frames_of(lengths, b, S)) {
            const float ga = gamma ? gamma[c] : 1.f, xv = (float)x.at(b, s)[c];
            float dz, xh;
            gn_grad_at<T, PRE, POST>(xv, (float)dy.at(b, s)[c], stats[at], stats[at + 1], ga, beta ? beta[c] : 0.f, dz, xh);
            v = stats[at + 1] * (dz * ga - coef[at] - xh * coef[at + 1]) * act_grad_f<PRE>(xv);
        }
        dx.at(b, s)[c] = (T)v;
    }
}

}  // namespace msf2
