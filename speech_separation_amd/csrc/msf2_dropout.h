// Dropout from a counter-based generator, with the residual addition.  One pass, no mask in memory.  Memory-bound: 64 x 3999 x 512, bf16
// onto an fp32 residual, 227 us and its gradient 135 us (5.8 TB/s); 55 x 3398 x 701 fp16 100 us (5.2 TB/s).
#pragma once
#include <algorithm>
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

// y = residual + x keep scale of `rows` frames (of utterance blockIdx.y where the operands' utterances do not follow one
// another).  A thread takes U times 8 neighbouring channels of a frame, the 128 bits of one generator call: 16 bits an element, because the
// generator's 20 wide multiplications (a quarter of the vector rate each) would otherwise bind the kernel before memory does.
// All loads go out before the first of them.  The last, narrower block of a frame is loaded as the frame's last 8 channels, its
// bits are moved up to them, and only its own channels are stored: loads without a branch (one here cost 5 % at widths that are
// multiples of 8, and element by element it was 10 to 40 % at others).  TAIL: there is such a block.
template <class TX, class TY, bool RES, bool TAIL, int U>
__global__ __launch_bounds__(256) void dropout_kernel(Rows<const TX> x, Rows<const TY> res, Rows<TY> y, const int64_t* rng,
                                                      unsigned site, unsigned thr, float scale, Divider per, unsigned blocks,
                                                      long block0, long block_batch, int C) {
    const uint64_t seed = rng[0], step = rng[1];
    const long b = blockIdx.y;
    const unsigned i0 = blockIdx.x * (256u * U) + threadIdx.x;
    typename VecOf<TX, 8>::type xv[U];
    typename VecOf<TY, 8>::type rv[U];
    unsigned row[U];
    int c[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned i = min(i0 + u * 256u, blocks - 1);
        row[u] = per.div(i);
        c[u] = (int)(i - row[u] * per.d) * 8;
        if (!TAIL || C >= 8) {
            const int at = TAIL ? min(c[u], C - 8) : c[u];
            xv[u] = load_vec<8>(x.at(b, row[u]) + at);
            if constexpr (RES) rv[u] = load_vec<8>(res.at(b, row[u]) + at);
        } else {
            xv[u] = load_some<8>(x.at(b, row[u]), C);
            if constexpr (RES) rv[u] = load_some<8>(res.at(b, row[u]), C);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint64_t block = (uint64_t)(block0 + b * block_batch) + i0 + u * 256u;
        const uint4 r = philox10(make_uint4((unsigned)block, (unsigned)(block >> 32), (unsigned)step, site),
                                 make_uint2((unsigned)seed, (unsigned)(seed >> 32)));
        unsigned w[4] = {r.x, r.y, r.z, r.w};
        const bool last = TAIL && C >= 8 && c[u] > C - 8;
        if (last)
            for (int k = C % 8; k < 8; ++k) {        // 8 - C % 8 half-words up
#pragma unroll
                for (int j = 3; j > 0; --j) w[j] = w[j] << 16 | w[j - 1] >> 16;
                w[0] <<= 16;
            }
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const unsigned bits = j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xFFFF;
            v[j] = bits >= thr ? (float)xv[u][j] * scale : 0.f;
            if constexpr (RES) v[j] += (float)rv[u][j];
        }
        if (i0 + u * 256u >= blocks) continue;
        TY* out = y.at(b, row[u]);
        if (TAIL && C < 8) store_some<8>(out, C, v);
        else if (last) store_last<8>(out + C - 8, 8 - C % 8, v);
        else store_vec<8>(out + c[u], v);
    }
}

// Utterances that follow one another without a gap are walked as one; a launch takes less than 2^31 generator calls.
template <class TX, class TY>
static int run_dropout(Rows<const TX> x, Rows<const TY> res, Rows<TY> y, const int64_t* rng, unsigned site, unsigned thr, float scale,
                       int B, int S, int C, hipStream_t st) {
    constexpr int U = 2;
    long rows = S, batches = B;
    auto whole = [&](long batch, long row) { return batch == (long)S * row; };
    if (S == 1) {
        x.row = x.batch; res.row = res.batch; y.row = y.batch;
        rows = B; batches = 1;
    } else if (B > 1 && whole(x.batch, x.row) && whole(y.batch, y.row) && (!res.p || whole(res.batch, res.row))) {
        rows = (long)B * S; batches = 1;
    }
    const long per = (C + 7) / 8, most = ((1l << 31) - 1) / per;
    const Divider by((unsigned)per);
    for (long b = 0; b < batches; b += 65535)
        for (long r = 0; r < rows; r += most) {
            const unsigned blocks = (unsigned)(std::min(most, rows - r) * per);
            const dim3 grid((blocks + 256u * U - 1) / (256u * U), (unsigned)std::min(65535l, batches - b));
            const Rows<const TX> xr = {x.at(b, r), x.batch, x.row};
            const Rows<const TY> rr = {res.p ? res.at(b, r) : nullptr, res.batch, res.row};
            const Rows<TY> yr = {y.at(b, r), y.batch, y.row};
            const long block0 = (b * rows + r) * per;
            auto go = [&](auto has_res, auto tail) {
                dropout_kernel<TX, TY, decltype(has_res)::value, decltype(tail)::value, U>
                    <<<grid, 256, 0, st>>>(xr, rr, yr, rng, site, thr, scale, by, blocks, block0, rows * per, C);
            };
            const std::true_type yes;
            const std::false_type no;
            if (res.p) C % 8 ? go(yes, yes) : go(yes, no);
            else C % 8 ? go(no, yes) : go(no, no);
        }
    return check_launch();
}

}  // namespace msf2
