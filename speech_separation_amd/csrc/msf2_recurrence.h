// Gated linear recurrence and its gradient: h_t = a_t h_{t-1} + (1 - a_t) x_t per channel, a = sigmoid(gate).
//
// A run of frames acts on the state as h -> A h + B, with A the product of its gates and B what it adds; runs join as
// (A, B) then (A', B') = (A A', A' B + B').  So a workgroup takes a tile of frames by channels into registers in one go: every
// thread joins its R frames, a scan over the time lanes gives each thread the state before its first frame, and a second walk
// over the registers gives every h_t.  x and gate are read once and h is written once.  The gradient is the same recurrence
// from the last frame back, E_t = a_t (dh_t + E_{t+1}); the h_{t-1} that dgate needs are scanned again within 32 frames from
// a state that the forward pass saved, which costs 1/32 of a row per frame instead of reading h, and keeps them in 32 bits.
// t counts frames in walking order; frame s is t, or S - 1 - t in reverse.  Frames past an utterance's end count as a = 1, B = 0.
#pragma once
#include <algorithm>
#include "msf2_rows.h"

namespace msf2 {

constexpr int REC_SAVE = MSF2_RECURRENCE_SAVE;
constexpr int REC_LC = 16;                   // lanes side by side over channels; the four rows of lanes of a wave follow in time
constexpr int REC_LT = 64 / REC_LC;
constexpr int REC_WIDE = 8;                  // waves of a workgroup, where a sequence is longer than one wave's frames

// How the work is dealt out: `slices` of channels by `pieces` of `piece` frames by utterances.
struct RecPlan {
    int slices, pieces, waves;
    long piece;
};

// What a workgroup works on, and a thread's place in it.  The lane of the last channels is moved left to end with the
// row, so that every load is a whole vector; what it shares with its neighbour is computed twice and written once (`own` on).
// Slices of the same frames share lines where rows are not aligned to them, and go to the same XCD one after the other: blocks are dealt
// to the 8 XCDs in turn, so block i of XCD k takes the i-th of the k-th eighth of the work.
template <int V> struct RecPlace {
    int b, p, n, tl, wave, c, own;
    bool whole;                              // no lane of the workgroup is past the row's end
    __device__ RecPlace(const RecPlan& pl, const int* lengths, int S, int C) {
        const unsigned each = gridDim.x / 8, more = gridDim.x % 8, xcd = blockIdx.x % 8;
        const unsigned id = xcd * each + min(xcd, more) + blockIdx.x / 8;
        const int slice = id % pl.slices;
        const unsigned rest = id / pl.slices;
        p = rest % pl.pieces;
        b = rest / pl.pieces;
        n = frames_of(lengths, b, S);
        const int lane = threadIdx.x & 63;
        wave = threadIdx.x >> 6;
        tl = lane / REC_LC;
        const int c0 = (slice * REC_LC + lane % REC_LC) * V;
        c = min(c0, C - V);
        own = c0 - c;                        // V and more: nothing is this lane's own
        whole = (slice + 1) * REC_LC * V <= C;
    }
};

// Runs of V neighbouring channels.
template <int V> struct Run {
    float a[V], b[V];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int v = 0; v < V; ++v) a[v] = 1.f, b[v] = 0.f;
    }
    // what `first` and then this run do
    __device__ __forceinline__ void after(const Run& first) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            b[v] = fmaf(a[v], first.b[v], b[v]);
            a[v] *= first.a[v];
        }
    }
    __device__ __forceinline__ void apply(float (&h)[V]) const {
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = fmaf(a[v], h[v], b[v]);
    }
};

// One level of a scan over the rows of 16 lanes: every lane gets the run of the earlier (lo) and of the later (hi) half of its
// pair, rows 2k and 2k + 1 with D = 16, the two halves of the wave with D = 32.  v_permlane*_swap exchanges the odd half of its
// first register with the even half of its second, so with the same value in both it leaves lo in the first, hi in the second.
template <int D, int V> __device__ __forceinline__ void halves(const Run<V>& r, Run<V>& lo, Run<V>& hi) {
    auto swap = [](float f, float& l, float& h) {
        const unsigned u = __builtin_bit_cast(unsigned, f);
        const auto p = D == 16 ? __builtin_amdgcn_permlane16_swap(u, u, false, false) : __builtin_amdgcn_permlane32_swap(u, u, false, false);
        l = __builtin_bit_cast(float, (unsigned)p[0]);
        h = __builtin_bit_cast(float, (unsigned)p[1]);
    };
#pragma unroll
    for (int v = 0; v < V; ++v) {
        swap(r.a[v], lo.a[v], hi.a[v]);
        swap(r.b[v], lo.b[v], hi.b[v]);
    }
}
// From each time lane's run: `before`, the run of all earlier lanes of the wave, and `all`, the run of the whole wave, in
// every lane.  BACK: later lanes come first.
template <bool BACK, int V> __device__ __forceinline__ void wave_scan(const Run<V>& r, int tl, Run<V>& before, Run<V>& all) {
    Run<V> lo, hi, pair;
    halves<16, V>(r, lo, hi);
    const bool second = BACK ? !(tl & 1) : tl & 1, late = BACK ? tl < 2 : tl >= 2;
    const Run<V>&first = BACK ? hi : lo, &then = BACK ? lo : hi;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        before.a[v] = second ? first.a[v] : 1.f;
        before.b[v] = second ? first.b[v] : 0.f;
    }
    pair = then;
    pair.after(first);
    halves<32, V>(pair, lo, hi);
    Run<V> skip;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        skip.a[v] = late ? first.a[v] : 1.f;
        skip.b[v] = late ? first.b[v] : 0.f;
    }
    before.after(skip);
    all = then;
    all.after(first);
}

// The waves of a workgroup in turn: h, the state before the tile, becomes the state after it, and `mine` the one before this
// wave's frames.  `runs` is one of two buffers that tiles take in turn, so one barrier a tile is enough: who fills a buffer
// again has passed the barrier of the tile between, which nobody passes before having read it.
template <bool BACK, int V, int W>
__device__ __forceinline__ void join_waves(const Run<V>& all, int wave, int tl, Run<V> (*runs)[REC_LC], float (&h)[V], float (&mine)[V]) {
    const int cl = threadIdx.x & (REC_LC - 1);
    if constexpr (W == 1) {
#pragma unroll
        for (int v = 0; v < V; ++v) mine[v] = h[v];
        all.apply(h);
        return;
    }
    if (tl == 0) runs[wave][cl] = all;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < W; ++k) {
        const int w = BACK ? W - 1 - k : k;
        if (w == wave) {
#pragma unroll
            for (int v = 0; v < V; ++v) mine[v] = h[v];
        }
        runs[w][cl].apply(h);
    }
}

// The gate: a = 1 / (1 + t) and na = 1 - a = t a, t = e^-g.  1 - a has to come from t, and h from a h + (1 - a) x: the shorter
// x + a (h - x) rounds at the size of x, which a gate near 1 lets through to a state that is far smaller.  A rounding d of g log2 e is a
// relative error d ln 2 of t, all of which 1 - a takes: FINE (fp32) adds the part that the product's rounding left out.  Gates beyond 87
// are held there (e^87 and its inverse are normal numbers; max and min keep NaN).
template <bool FINE> __device__ __forceinline__ void rec_gate(float g, float& a, float& na) {
    constexpr float LOG2E = 1.44269504088896f, LN2 = 0.693147180559945f;
    g = __builtin_elementwise_maximum(g, -87.f);
    if constexpr (FINE) g = __builtin_elementwise_minimum(g, 87.f);
    const float u = -g * LOG2E;
    float t = __builtin_amdgcn_exp2f(u);
    if constexpr (FINE) t = fmaf(t * LN2, fmaf(-g, LOG2E, -u), t);
    a = __builtin_amdgcn_rcpf(1.f + t);
    na = t * a;
}
template <class T> constexpr bool rec_fine() { return sizeof(T) == 4; }

// Frames outside the utterance: a gate of 87 is a = 1 exactly, and nothing is added.
template <int V, class T> __device__ __forceinline__ void rec_shut(typename VecOf<T, V>::type& g) {
#pragma unroll
    for (int v = 0; v < V; ++v) g[v] = (T)87.f;
}

template <int V, class T> __device__ __forceinline__ void rec_store(T* row, int own, const float (&f)[V]) {
    if (own <= 0) {
        store_vec<V>(row, f);
    } else {
#pragma unroll
        for (int v = 1; v < V; ++v)
            if (v >= own) row[v] = (T)f[v];
    }
}
template <int V> __device__ __forceinline__ void rec_read(const float* p, float (&f)[V]) {
    const auto u = load_vec<V>(p);
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = u[v];
}

// The state before piece p: `start` and the runs of the pieces before it (BACK: behind it), agg [b][pieces][2][C].
template <bool BACK, int V>
__device__ __forceinline__ void rec_carry(const RecPlan& pl, const float* agg, const float* start, int b, int p, int c, int C, float (&h)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = 0.f;
    if (start) rec_read<V>(start + (long)b * C + c, h);
    const int k0 = BACK ? pl.pieces - 1 : 0, n = BACK ? pl.pieces - 1 - p : p;
    for (int k = 0; k < n; ++k) {
        const float* q = agg + ((long)b * pl.pieces + (BACK ? k0 - k : k)) * 2 * C + c;
        Run<V> r;
        rec_read<V>(q, r.a);
        rec_read<V>(q + C, r.b);
        r.apply(h);
    }
}

// A thread's R frames of a tile; which of them are in the utterance, and whether all of the tile's are.
template <int R> struct RecFrames {
    long t, s0;
    int n, step;
    bool all;
    // first: this thread's first frame walked; tile, rows: the workgroup's
    __device__ __forceinline__ RecFrames(long first, long tile, int rows, long end, int n_, int S, int reverse) : t(first), n(n_) {
        s0 = reverse ? S - 1 - t : t;
        step = reverse ? -1 : 1;
        all = tile + rows <= end && (reverse ? tile >= S - n : tile + rows <= n);
    }
    __device__ __forceinline__ long s(int j) const { return s0 + step * j; }
    __device__ __forceinline__ bool live(int j) const { return s(j) >= 0 && s(j) < n; }
    __device__ __forceinline__ long held(int j) const { return min(max(s(j), 0l), (long)max(n - 1, 0)); }   // in memory at least
};

// The run of one piece, for sequences too few to fill the chip: agg, and `start` copied to `kept`, because the pieces of the
// next launch read it while one of them may write the last state into the same memory.  u is x, or dh with BACK; a thread
// walks piece / (W REC_LT) frames on end.
template <bool BACK, class T, int V, int W>
__global__ __launch_bounds__(64 * W) void rec_piece_kernel(Rows<const T> u, Rows<const T> gate, const float* start, const int* lengths,
                                                           float* agg, float* kept, RecPlan pl, int S, int C, int reverse) {
    constexpr int R = 8;
    __shared__ Run<V> runs[W][REC_LC];
    const RecPlace<V> at(pl, lengths, S, C);
    const bool writes = at.wave == 0 && at.tl == 0;
    if (at.p == (BACK ? pl.pieces - 1 : 0) && writes) {
        float h[V];
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = 0.f;
        if (start) rec_read<V>(start + (long)at.b * C + at.c, h);
        rec_store<V>(kept + (long)at.b * C + at.c, at.own, h);
    }
    if (at.p == (BACK ? 0 : pl.pieces - 1)) return;         // nothing follows it
    const int steps = (int)(pl.piece / (W * REC_LT));       // a multiple of R
    const long t0 = at.p * pl.piece + (long)(at.wave * REC_LT + at.tl) * steps;
    Run<V> r;
    r.clear();
    for (int k = 0; k < steps; k += R) {
        const RecFrames<R> fr(BACK ? t0 + steps - R - k : t0 + k, 0, 0, 0, at.n, S, reverse);
        typename VecOf<T, V>::type uv[R], gv[R];
#pragma unroll
        for (int j = 0; j < R; ++j) {
            uv[j] = load_vec<V>(u.at(at.b, fr.held(j)) + at.c);
            gv[j] = load_vec<V>(gate.at(at.b, fr.held(j)) + at.c);
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int j = BACK ? R - 1 - i : i;
            if (!fr.live(j) || fr.t + j >= S) rec_shut<V, T>(gv[j]), uv[j] = 0;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float a, na;
                rec_gate<rec_fine<T>()>((float)gv[j][v], a, na);
                const float f = (float)uv[j][v];
                r.b[v] = BACK ? a * (r.b[v] + f) : fmaf(a, r.b[v], na * f);
                r.a[v] *= a;
            }
        }
    }
    Run<V> before, all;
    wave_scan<BACK, V>(r, at.tl, before, all);
    if (at.tl == 0) runs[at.wave][threadIdx.x & (REC_LC - 1)] = all;
    __syncthreads();
    if (writes) {
        r.clear();
        for (int k = 0; k < W; ++k) {
            Run<V> next = runs[BACK ? W - 1 - k : k][threadIdx.x];
            next.after(r);
            r = next;
        }
        float* q = agg + ((long)at.b * pl.pieces + at.p) * 2 * C + at.c;
        rec_store<V>(q, at.own, r.a);
        rec_store<V>(q + C, at.own, r.b);
    }
}

template <class T, int V, int R, int W>
__global__ __launch_bounds__(64 * W) void rec_forward_kernel(Rows<const T> x, Rows<const T> gate, const float* start, const int* lengths,
                                                             Rows<T> h, float* last, float* saved, const float* agg, RecPlan pl,
                                                             int S, int C, int reverse) {
    constexpr int TILE = W * REC_LT * R;
    __shared__ Run<V> runs[2][W][REC_LC];
    const RecPlace<V> at(pl, lengths, S, C);
    const long t0 = at.p * pl.piece, t1 = min(t0 + pl.piece, (long)S);
    const int blocks = (S + REC_SAVE - 1) / REC_SAVE;
    const int mine = (at.wave * REC_LT + at.tl) * R;           // this thread's first frame in a tile
    typedef typename VecOf<T, V>::type vec;
    vec nx[R], ng[R];
    auto fetch = [&](long t) {
        const RecFrames<R> fr(t + mine, t, TILE, t1, at.n, S, reverse);
#pragma unroll
        for (int j = 0; j < R; ++j) {
            nx[j] = load_vec<V>(x.at(at.b, fr.held(j)) + at.c);
            ng[j] = load_vec<V>(gate.at(at.b, fr.held(j)) + at.c);
        }
    };
    fetch(t0);
    float carry[V];
    rec_carry<false, V>(pl, agg, start, at.b, at.p, at.c, C, carry);
    int turn = 0;
    for (long t = t0; t < t1; t += TILE, turn ^= 1) {
        const RecFrames<R> fr(t + mine, t, TILE, t1, at.n, S, reverse);
        float a[R][V], f[R][V];
        Run<V> r, before, all;
        r.clear();
        if (!fr.all) {
#pragma unroll
            for (int j = 0; j < R; ++j)
                if (!fr.live(j) || fr.t + j >= t1) rec_shut<V, T>(ng[j]), nx[j] = 0;
        }
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float na;
                rec_gate<rec_fine<T>()>((float)ng[j][v], a[j][v], na);
                f[j][v] = na * (float)nx[j][v];
                r.b[v] = fmaf(a[j][v], r.b[v], f[j][v]);
                r.a[v] *= a[j][v];
            }
        if (t + TILE < t1) fetch(t + TILE);
        wave_scan<false, V>(r, at.tl, before, all);
        float hv[V];
        join_waves<false, V, W>(all, at.wave, at.tl, runs[turn], carry, hv);
        before.apply(hv);
        if (saved && fr.t % REC_SAVE == 0 && fr.t < t1)
            rec_store<V>(saved + ((long)at.b * blocks + fr.t / REC_SAVE) * C + at.c, at.own, hv);
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) f[j][v] = hv[v] = fmaf(a[j][v], hv[v], f[j][v]);
        if (fr.all && at.whole) {
#pragma unroll
            for (int j = 0; j < R; ++j) store_vec<V>(h.at(at.b, fr.s(j)) + at.c, f[j]);
        } else {
#pragma unroll
            for (int j = 0; j < R; ++j)
                if (fr.t + j < t1) {
#pragma unroll
                    for (int v = 0; v < V; ++v) f[j][v] = fr.live(j) ? f[j][v] : 0.f;
                    rec_store<V>(h.at(at.b, fr.s(j)) + at.c, at.own, f[j]);
                }
        }
    }
    if (last && t1 == S && at.wave == 0 && at.tl == 0) rec_store<V>(last + (long)at.b * C + at.c, at.own, carry);
}

template <class T, int V, int R, int W>
__global__ __launch_bounds__(64 * W) void rec_backward_kernel(Rows<const T> dh, Rows<const T> x, Rows<const T> gate, const float* saved,
                                                              const float* start, const int* lengths, Rows<T> dx, Rows<T> dgate,
                                                              float* dh0, const float* agg, RecPlan pl, int S, int C, int reverse) {
    constexpr int TILE = W * REC_LT * R;
    static_assert(REC_LT * R % REC_SAVE == 0, "a wave's frames begin at a saved state");
    __shared__ Run<V> runs[2][W][REC_LC];
    const RecPlace<V> at(pl, lengths, S, C);
    const long t0 = at.p * pl.piece, t1 = min(t0 + pl.piece, (long)S);
    const int blocks = (S + REC_SAVE - 1) / REC_SAVE;
    const int mine = (at.wave * REC_LT + at.tl) * R;
    typedef typename VecOf<T, V>::type vec;
    vec nd[R], nx[R], ng[R];
    float nh[V];
    auto fetch = [&](long t) {
        const RecFrames<R> fr(t + mine, t, TILE, t1, at.n, S, reverse);
#pragma unroll
        for (int j = 0; j < R; ++j) {
            nd[j] = load_vec<V>(dh.at(at.b, fr.held(j)) + at.c);
            nx[j] = load_vec<V>(x.at(at.b, fr.held(j)) + at.c);
            ng[j] = load_vec<V>(gate.at(at.b, fr.held(j)) + at.c);
        }
        const long block = min((t + at.wave * (REC_LT * R)) / REC_SAVE, (long)blocks - 1);      // the wave's first frame
        rec_read<V>(saved + ((long)at.b * blocks + block) * C + at.c, nh);
    };
    const long tiles = (t1 - t0 + TILE - 1) / TILE;
    fetch(t0 + (tiles - 1) * TILE);
    float carry[V];
    rec_carry<true, V>(pl, agg, start, at.b, at.p, at.c, C, carry);
    int turn = 0;
    for (long t = t0 + (tiles - 1) * TILE; t >= t0; t -= TILE, turn ^= 1) {
        const RecFrames<R> fr(t + mine, t, TILE, t1, at.n, S, reverse);
        float a[R][V], na[R][V], f[R][V], d[R][V], hv[V];
        Run<V> r, q, before, all;
        r.clear();
        if (!fr.all) {
#pragma unroll
            for (int j = 0; j < R; ++j)
                if (!fr.live(j) || fr.t + j >= t1) rec_shut<V, T>(ng[j]), nx[j] = 0, nd[j] = 0;
        }
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                rec_gate<rec_fine<T>()>((float)ng[j][v], a[j][v], na[j][v]);
                f[j][v] = (float)nx[j][v];
                d[j][v] = (float)nd[j][v];
                r.b[v] = fmaf(a[j][v], r.b[v], na[j][v] * f[j][v]);
                r.a[v] *= a[j][v];
            }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            hv[v] = nh[v];
            q.a[v] = r.a[v];
            q.b[v] = 0.f;
#pragma unroll
            for (int j = R - 1; j >= 0; --j) q.b[v] = a[j][v] * (d[j][v] + q.b[v]);
        }
        if (t > t0) fetch(t - TILE);
        wave_scan<false, V>(r, at.tl, before, all);
        before.apply(hv);
        // f becomes (1 - a_t) (h_{t-1} - x_t)
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float xv = f[j][v];
                f[j][v] = na[j][v] * (hv[v] - xv);
                hv[v] = fmaf(a[j][v], hv[v], na[j][v] * xv);
            }
        wave_scan<true, V>(q, at.tl, before, all);
        float e[V];
        join_waves<true, V, W>(all, at.wave, at.tl, runs[turn], carry, e);
        before.apply(e);
        // d becomes dx, f becomes dgate
#pragma unroll
        for (int j = R - 1; j >= 0; --j)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float dv = d[j][v] + e[v];
                d[j][v] = na[j][v] * dv;
                e[v] = a[j][v] * dv;
                f[j][v] *= e[v];
            }
        if (fr.all && at.whole) {
#pragma unroll
            for (int j = 0; j < R; ++j) {
                store_vec<V>(dx.at(at.b, fr.s(j)) + at.c, d[j]);
                store_vec<V>(dgate.at(at.b, fr.s(j)) + at.c, f[j]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < R; ++j)
                if (fr.t + j < t1) {
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        d[j][v] = fr.live(j) ? d[j][v] : 0.f;
                        f[j][v] = fr.live(j) ? f[j][v] : 0.f;
                    }
                    rec_store<V>(dx.at(at.b, fr.s(j)) + at.c, at.own, d[j]);
                    rec_store<V>(dgate.at(at.b, fr.s(j)) + at.c, at.own, f[j]);
                }
        }
    }
    if (dh0 && t0 == 0 && at.wave == 0 && at.tl == 0) rec_store<V>(dh0 + (long)at.b * C + at.c, at.own, carry);
}

constexpr int REC_V = 2;                                       // channels a lane
constexpr int rec_rows(int bytes, bool backward) { return backward || bytes == 4 ? 8 : 16; }     // frames a thread

// `rows` frames a thread; slices of REC_LC V channels; pieces until the chip is filled.
static inline RecPlan rec_plan(int B, int S, int C, int rows) {
    const int V = C >= REC_V ? REC_V : 1;
    RecPlan pl;
    pl.slices = (C + REC_LC * V - 1) / (REC_LC * V);
    pl.waves = S <= REC_LT * rows ? 1 : REC_WIDE;
    const long tile = (long)pl.waves * REC_LT * rows, tiles = (S + tile - 1) / tile, seqs = (long)B * pl.slices;
    const long want = seqs >= 192 ? 1 : std::min((512 + seqs - 1) / seqs, 64l);
    const long per = std::max(1l, tiles / std::min(want, tiles));
    pl.piece = per * tile;
    pl.pieces = (int)((tiles + per - 1) / per);
    return pl;
}
static inline size_t rec_ws_bytes(int B, int S, int C, int bytes, bool backward) {
    const RecPlan pl = rec_plan(B, S, C, rec_rows(bytes, backward));
    return pl.pieces == 1 ? 0 : align_up((size_t)B * pl.pieces * 2 * C * sizeof(float)) + align_up((size_t)B * C * sizeof(float));
}

// f(V, W) as integral constants
template <class F> static int rec_shape(int C, const RecPlan& pl, F f) {
    std::integral_constant<int, REC_V> v;
    std::integral_constant<int, 1> one;
    std::integral_constant<int, REC_WIDE> wide;
    if (C >= REC_V) return pl.waves == 1 ? f(v, one) : f(v, wide);
    return pl.waves == 1 ? f(one, one) : f(one, wide);
}

template <class T>
static int run_recurrence(Rows<const T> x, Rows<const T> gate, const float* h0, const int* lengths, Rows<T> h, float* last, float* saved,
                          int B, int S, int C, int reverse, void* ws, hipStream_t st) {
    constexpr int R = rec_rows(sizeof(T), false);
    const RecPlan pl = rec_plan(B, S, C, R);
    Arena arena(ws, ~(size_t)0);
    float* agg = pl.pieces > 1 ? arena.take<float>((size_t)B * pl.pieces * 2 * C) : nullptr;
    float* kept = pl.pieces > 1 ? arena.take<float>((size_t)B * C) : nullptr;
    const long grid = (long)B * pl.pieces * pl.slices;
    if (grid > 0x7fffffff) return MSF2_ERR_ARG;
    return rec_shape(C, pl, [&](auto v, auto w) {
        constexpr int V = decltype(v)::value, W = decltype(w)::value;
        if constexpr (W > 1)
            if (pl.pieces > 1) rec_piece_kernel<false, T, V, W><<<grid, 64 * W, 0, st>>>(x, gate, h0, lengths, agg, kept, pl, S, C, reverse);
        rec_forward_kernel<T, V, R, W><<<grid, 64 * W, 0, st>>>(x, gate, pl.pieces > 1 ? kept : h0, lengths, h, last, saved, agg, pl, S, C, reverse);
        return check_launch();
    });
}

template <class T>
static int run_recurrence_backward(Rows<const T> dh, Rows<const T> x, Rows<const T> gate, const float* saved, const float* dlast,
                                   const int* lengths, Rows<T> dx, Rows<T> dgate, float* dh0, int B, int S, int C, int reverse, void* ws,
                                   hipStream_t st) {
    constexpr int R = rec_rows(sizeof(T), true);
    const RecPlan pl = rec_plan(B, S, C, R);
    Arena arena(ws, ~(size_t)0);
    float* agg = pl.pieces > 1 ? arena.take<float>((size_t)B * pl.pieces * 2 * C) : nullptr;
    float* kept = pl.pieces > 1 ? arena.take<float>((size_t)B * C) : nullptr;
    const long grid = (long)B * pl.pieces * pl.slices;
    if (grid > 0x7fffffff) return MSF2_ERR_ARG;
    return rec_shape(C, pl, [&](auto v, auto w) {
        constexpr int V = decltype(v)::value, W = decltype(w)::value;
        if constexpr (W > 1)
            if (pl.pieces > 1) rec_piece_kernel<true, T, V, W><<<grid, 64 * W, 0, st>>>(dh, gate, dlast, lengths, agg, kept, pl, S, C, reverse);
        rec_backward_kernel<T, V, R, W><<<grid, 64 * W, 0, st>>>(dh, x, gate, saved, pl.pieces > 1 ? kept : dlast, lengths, dx, dgate, dh0, agg,
                                                                 pl, S, C, reverse);
        return check_launch();
    });
}

}  // namespace msf2
