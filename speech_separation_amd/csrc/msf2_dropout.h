// Dropout from a counter-based generator, with the residual addition.
#pragma once
#include "msf2_rows.h"

namespace msf2 {

// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011).
__device__ __forceinline__ uint4 philox10(uint4 c, uint2 k) {
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t p = (uint64_t)0xD2511F53u * c.x, q = (uint64_t)0xCD9E8D57u * c.z;
        c = make_uint4((unsigned)(q >> 32) ^ c.y ^ k.x, (unsigned)q, (unsigned)(p >> 32) ^ c.w ^ k.y, (unsigned)p);
        k.x += 0x9E3779B9u;
        k.y += 0xBB67AE85u;
    }
    return c;
}

// one thread 8 neighbouring channels of a frame: the 128 bits of one generator call
template <class TX, class TY>
__global__ __launch_bounds__(256) void dropout_kernel(Rows<const TX> x, Rows<const TY> res, Rows<TY> y, const int64_t* rng,
                                                      unsigned site, unsigned thr, float scale, int B, int S, int C) {
    const int per = (C + 7) / 8;
    const uint64_t seed = rng[0], step = rng[1];
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < (long)B * S * per; i += (long)gridDim.x * 256) {
        const int c0 = i % per * 8, s = i / per % S, b = i / per / S;
        const uint4 r = philox10(make_uint4((unsigned)i, (unsigned)((uint64_t)i >> 32), (unsigned)step, site),
                                 make_uint2((unsigned)seed, (unsigned)(seed >> 32)));
        const unsigned w[4] = {r.x, r.y, r.z, r.w};
        for (int j = 0; j < 8 && c0 + j < C; ++j) {
            const unsigned bits = j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xFFFF;
            float v = bits >= thr ? (float)x.at(b, s)[c0 + j] * scale : 0.f;
            if (res.p) v += (float)res.at(b, s)[c0 + j];
            y.at(b, s)[c0 + j] = (TY)v;
        }
    }
}

}  // namespace msf2
