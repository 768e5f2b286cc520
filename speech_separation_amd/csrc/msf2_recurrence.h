// Gated linear recurrence and its gradient.
#pragma once
#include "msf2_rows.h"

namespace msf2 {

constexpr int REC_SAVE = MSF2_RECURRENCE_SAVE;

// one thread a channel of an utterance; t counts the frames walked, the frame itself is t or S - 1 - t
template <class T>
__global__ __launch_bounds__(256) void rec_forward_kernel(Rows<const T> x, Rows<const T> gate, const float* h0, const int* lengths,
                                                          Rows<T> h, float* last, float* saved, int B, int S, int C, int reverse) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long)B * C) return;
    const int b = i / C, c = i % C, n = frames_of(lengths, b, S);
    float v = h0 ? h0[i] : 0.f;
    for (int t = 0; t < S; ++t) {
        const int s = reverse ? S - 1 - t : t;
        if (saved && t % REC_SAVE == 0) saved[((long)b * ((S + REC_SAVE - 1) / REC_SAVE) + t / REC_SAVE) * C + c] = v;
        if (s < n) {
            float a, na;
            sigmoid_pair((float)gate.at(b, s)[c], a, na);
            v = fmaf(a, v, na * (float)x.at(b, s)[c]);
        }
        h.at(b, s)[c] = s < n ? (T)v : (T)0.f;
    }
    if (last) last[i] = v;
}

template <class T>
__global__ __launch_bounds__(256) void rec_backward_kernel(Rows<const T> dh, Rows<const T> x, Rows<const T> gate, const float* saved,
                                                           const float* dlast, const int* lengths, Rows<T> dx, Rows<T> dgate,
                                                           float* dh0, int B, int S, int C, int reverse) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long)B * C) return;
    const int b = i / C, c = i % C, n = frames_of(lengths, b, S), blocks = (S + REC_SAVE - 1) / REC_SAVE;
    float e = dlast ? dlast[i] : 0.f;
    for (int k = blocks - 1; k >= 0; --k) {
        float before[REC_SAVE], v = saved[((long)b * blocks + k) * C + c];
        for (int j = 0; j < REC_SAVE; ++j) {
            const int t = k * REC_SAVE + j, s = reverse ? S - 1 - t : t;
            before[j] = v;
            if (t < S && s < n) {
                float a, na;
                sigmoid_pair((float)gate.at(b, s)[c], a, na);
                v = fmaf(a, v, na * (float)x.at(b, s)[c]);
            }
        }
        for (int j = REC_SAVE - 1; j >= 0; --j) {
            const int t = k * REC_SAVE + j, s = reverse ? S - 1 - t : t;
            if (t >= S) continue;
            float gx = 0.f, gg = 0.f;
            if (s < n) {
                float a, na;
                sigmoid_pair((float)gate.at(b, s)[c], a, na);
                const float d = (float)dh.at(b, s)[c] + e;
                gx = na * d;
                gg = a * gx * (before[j] - (float)x.at(b, s)[c]);
                e = a * d;
            }
            dx.at(b, s)[c] = (T)gx;
            dgate.at(b, s)[c] = (T)gg;
        }
    }
    if (dh0) dh0[i] = e;
}

}  // namespace msf2
