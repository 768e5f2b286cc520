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
constexpr int REC_LC = 8;                    // lanes side by side over channels; the other 8 of a wave follow one another in time
constexpr int REC_LT = 64 / REC_LC;
constexpr int REC_R = REC_SAVE / REC_LT;     // frames a thread: a wave's frames are those between two saved states
constexpr int REC_WIDE = 8;                  // waves of a workgroup where the sequence fills them (256 frames a tile)

// How the work is dealt out: `slices` of channels by `pieces` of `piece` frames by utterances.
struct RecPlan {
    int slices, pieces, waves;
    long piece;
};

// What a workgroup works on, and a thread's place in it.  The lane of the last channels is moved left to end with the
// row, so that every load is a whole vector; what it shares with its neighbour is computed twice and written once (`own` on).
template <int V> struct RecPlace {
    int b, slice, p, n, tl, wave, lane, c, own;
    __device__ RecPlace(const RecPlan& pl, const int* lengths, int S, int C) {
        slice = blockIdx.x % pl.slices;
        const unsigned rest = blockIdx.x / pl.slices;
        p = rest % pl.pieces;
        b = rest / pl.pieces;
        n = frames_of(lengths, b, S);
        lane = threadIdx.x & 63;
        wave = threadIdx.x >> 6;
        tl = lane / REC_LC;
        const int c0 = (slice * REC_LC + lane % REC_LC) * V;
        c = min(c0, C - V);
        own = c0 - c;                        // V and more: nothing is this lane's own
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

// From each time lane's run: `before`, the run of all earlier lanes of the wave, and `all`, the run of the whole wave.
// BACK: later lanes come first.
template <bool BACK, int V> __device__ __forceinline__ void wave_scan(Run<V> r, int tl, Run<V>& before, Run<V>& all) {
    const int at = BACK ? REC_LT - 1 - tl : tl;
    auto from = [&](const Run<V>& q, int d) {
        Run<V> o;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            o.a[v] = BACK ? __shfl_down(q.a[v], d * REC_LC, 64) : __shfl_up(q.a[v], d * REC_LC, 64);
            o.b[v] = BACK ? __shfl_down(q.b[v], d * REC_LC, 64) : __shfl_up(q.b[v], d * REC_LC, 64);
        }
        return o;
    };
#pragma unroll
    for (int d = 1; d < REC_LT; d *= 2) {
        const Run<V> o = from(r, d);
        if (at >= d) r.after(o);
    }
    before = from(r, 1);
    if (at == 0) before.clear();
    const int last = (BACK ? 0 : REC_LT - 1) * REC_LC + (threadIdx.x & (REC_LC - 1));
#pragma unroll
    for (int v = 0; v < V; ++v) {
        all.a[v] = __shfl(r.a[v], last, 64);
        all.b[v] = __shfl(r.b[v], last, 64);
    }
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

// a, 1 - a and x (or dh) of one vector; dead frames are a = 1 and nothing else, whatever memory holds there
template <int V, class T>
__device__ __forceinline__ void rec_gates(const typename VecOf<T, V>::type& g, bool live, float (&a)[V], float (&na)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
        sigmoid_pair((float)g[v], a[v], na[v]);
        a[v] = live ? a[v] : 1.f;
        na[v] = live ? na[v] : 0.f;
    }
}
template <int V, class T> __device__ __forceinline__ void rec_values(const typename VecOf<T, V>::type& x, bool live, float (&f)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = live ? (float)x[v] : 0.f;
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

// The run of one piece, for sequences too few to fill the chip: agg, and `start` copied to `kept`, because the pieces of the next launch
// read it while one of them may write the last state into the same memory.  u is x, or dh with BACK; a thread walks
// piece / (W REC_LT) frames on end.
template <bool BACK, class T, int V, int W>
__global__ __launch_bounds__(64 * W) void rec_piece_kernel(Rows<const T> u, Rows<const T> gate, const float* start, const int* lengths,
                                                           float* agg, float* kept, RecPlan pl, int S, int C, int reverse) {
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
    const int steps = (int)(pl.piece / (W * REC_LT));
    const long t0 = at.p * pl.piece + (long)(at.wave * REC_LT + at.tl) * steps;
    const int cap = max(at.n - 1, 0);
    Run<V> r;
    r.clear();
    for (int k = 0; k < steps; k += REC_R) {
        typename VecOf<T, V>::type uv[REC_R], gv[REC_R];
        bool live[REC_R];
#pragma unroll
        for (int j = 0; j < REC_R; ++j) {
            const long t = t0 + (BACK ? steps - 1 - (k + j) : k + j), s = reverse ? S - 1 - t : t;
            live[j] = t < S && s < at.n;
            const long sc = min(max(s, 0l), (long)cap);
            uv[j] = load_vec<V>(u.at(at.b, sc) + at.c);
            gv[j] = load_vec<V>(gate.at(at.b, sc) + at.c);
        }
#pragma unroll
        for (int j = 0; j < REC_R; ++j) {
            float a[V], na[V], f[V];
            rec_gates<V, T>(gv[j], live[j], a, na);
            rec_values<V, T>(uv[j], live[j], f);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                r.b[v] = BACK ? a[v] * (r.b[v] + f[v]) : fmaf(a[v], r.b[v], na[v] * f[v]);
                r.a[v] *= a[v];
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

template <class T, int V, int W>
__global__ __launch_bounds__(64 * W) void rec_forward_kernel(Rows<const T> x, Rows<const T> gate, const float* start, const int* lengths,
                                                             Rows<T> h, float* last, float* saved, const float* agg, RecPlan pl,
                                                             int S, int C, int reverse) {
    constexpr int TILE = W * REC_SAVE;
    __shared__ Run<V> runs[2][W][REC_LC];
    const RecPlace<V> at(pl, lengths, S, C);
    const long t0 = at.p * pl.piece, t1 = min(t0 + pl.piece, (long)S);
    const int cap = max(at.n - 1, 0), blocks = (S + REC_SAVE - 1) / REC_SAVE;
    const int mine = at.wave * REC_SAVE + at.tl * REC_R;        // this thread's first frame in a tile
    typedef typename VecOf<T, V>::type vec;
    vec nx[REC_R], ng[REC_R];
    auto fetch = [&](long t) {
#pragma unroll
        for (int j = 0; j < REC_R; ++j) {
            const long tt = t + mine + j, s = min(max(reverse ? S - 1 - tt : tt, 0l), (long)cap);
            nx[j] = load_vec<V>(x.at(at.b, s) + at.c);
            ng[j] = load_vec<V>(gate.at(at.b, s) + at.c);
        }
    };
    fetch(t0);
    float carry[V];
    rec_carry<false, V>(pl, agg, start, at.b, at.p, at.c, C, carry);
    int turn = 0;
    for (long t = t0; t < t1; t += TILE, turn ^= 1) {
        float a[REC_R][V], b[REC_R][V];
        Run<V> r, before, all;
        r.clear();
#pragma unroll
        for (int j = 0; j < REC_R; ++j) {
            const long tt = t + mine + j, s = reverse ? S - 1 - tt : tt;
            const bool live = tt < S && s < at.n;
            float na[V], f[V];
            rec_gates<V, T>(ng[j], live, a[j], na);
            rec_values<V, T>(nx[j], live, f);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                b[j][v] = na[v] * f[v];
                r.b[v] = fmaf(a[j][v], r.b[v], b[j][v]);
                r.a[v] *= a[j][v];
            }
        }
        if (t + TILE < t1) fetch(t + TILE);
        wave_scan<false, V>(r, at.tl, before, all);
        float hv[V];
        join_waves<false, V, W>(all, at.wave, at.tl, runs[turn], carry, hv);
        if (saved && at.tl == 0 && t + mine < S)
            rec_store<V>(saved + ((long)at.b * blocks + (t + mine) / REC_SAVE) * C + at.c, at.own, hv);
        before.apply(hv);
#pragma unroll
        for (int j = 0; j < REC_R; ++j) {
            const long tt = t + mine + j, s = reverse ? S - 1 - tt : tt;
            float out[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                hv[v] = fmaf(a[j][v], hv[v], b[j][v]);
                out[v] = s < at.n ? hv[v] : 0.f;
            }
            if (tt < S) rec_store<V>(h.at(at.b, s) + at.c, at.own, out);
        }
    }
    if (last && t1 == S && at.wave == 0 && at.tl == 0) rec_store<V>(last + (long)at.b * C + at.c, at.own, carry);
}

template <class T, int V, int W>
__global__ __launch_bounds__(64 * W) void rec_backward_kernel(Rows<const T> dh, Rows<const T> x, Rows<const T> gate, const float* saved,
                                                              const float* start, const int* lengths, Rows<T> dx, Rows<T> dgate,
                                                              float* dh0, const float* agg, RecPlan pl, int S, int C, int reverse) {
    constexpr int TILE = W * REC_SAVE;
    __shared__ Run<V> runs[2][W][REC_LC];
    const RecPlace<V> at(pl, lengths, S, C);
    const long t0 = at.p * pl.piece, t1 = min(t0 + pl.piece, (long)S);
    const int cap = max(at.n - 1, 0), blocks = (S + REC_SAVE - 1) / REC_SAVE;
    const int mine = at.wave * REC_SAVE + at.tl * REC_R;
    typedef typename VecOf<T, V>::type vec;
    vec nd[REC_R], nx[REC_R], ng[REC_R];
    float nh[V];
    auto fetch = [&](long t) {
#pragma unroll
        for (int j = 0; j < REC_R; ++j) {
            const long tt = t + mine + j, s = min(max(reverse ? S - 1 - tt : tt, 0l), (long)cap);
            nd[j] = load_vec<V>(dh.at(at.b, s) + at.c);
            nx[j] = load_vec<V>(x.at(at.b, s) + at.c);
            ng[j] = load_vec<V>(gate.at(at.b, s) + at.c);
        }
        rec_read<V>(saved + ((long)at.b * blocks + min((t + mine) / REC_SAVE, (long)blocks - 1)) * C + at.c, nh);
    };
    const long tiles = (t1 - t0 + TILE - 1) / TILE;
    fetch(t0 + (tiles - 1) * TILE);
    float carry[V];
    rec_carry<true, V>(pl, agg, start, at.b, at.p, at.c, C, carry);
    int turn = 0;
    for (long t = t0 + (tiles - 1) * TILE; t >= t0; t -= TILE, turn ^= 1) {
        float a[REC_R][V], na[REC_R][V], f[REC_R][V], d[REC_R][V], hv[V];
        Run<V> r, q, before, all;
        r.clear();
        q.clear();
#pragma unroll
        for (int j = 0; j < REC_R; ++j) {
            const long tt = t + mine + j, s = reverse ? S - 1 - tt : tt;
            const bool live = tt < S && s < at.n;
            rec_gates<V, T>(ng[j], live, a[j], na[j]);
            rec_values<V, T>(nx[j], live, f[j]);
            rec_values<V, T>(nd[j], live, d[j]);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                r.b[v] = fmaf(a[j][v], r.b[v], na[j][v] * f[j][v]);
                r.a[v] *= a[j][v];
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            hv[v] = nh[v];
            q.a[v] = r.a[v];
#pragma unroll
            for (int j = REC_R - 1; j >= 0; --j) q.b[v] = a[j][v] * (d[j][v] + q.b[v]);
        }
        if (t > t0) fetch(t - TILE);
        wave_scan<false, V>(r, at.tl, before, all);
        before.apply(hv);
        // f becomes h_{t-1} - x_t
#pragma unroll
        for (int j = 0; j < REC_R; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float xv = f[j][v];
                f[j][v] = hv[v] - xv;
                hv[v] = fmaf(a[j][v], hv[v], na[j][v] * xv);
            }
        wave_scan<true, V>(q, at.tl, before, all);
        float e[V];
        join_waves<true, V, W>(all, at.wave, at.tl, runs[turn], carry, e);
        before.apply(e);
#pragma unroll
        for (int j = REC_R - 1; j >= 0; --j) {
            const long tt = t + mine + j, s = reverse ? S - 1 - tt : tt;
            float gx[V], gg[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float dv = d[j][v] + e[v];
                gx[v] = na[j][v] * dv;
                e[v] = a[j][v] * dv;
                gg[v] = e[v] * na[j][v] * f[j][v];
            }
            if (tt < S) {
                rec_store<V>(dx.at(at.b, s) + at.c, at.own, gx);
                rec_store<V>(dgate.at(at.b, s) + at.c, at.own, gg);
            }
        }
    }
    if (dh0 && t0 == 0 && at.wave == 0 && at.tl == 0) rec_store<V>(dh0 + (long)at.b * C + at.c, at.own, carry);
}

constexpr int rec_vec(int bytes) { return 4; }        // channels a lane

// Rows of V C channels wide slices; pieces until the chip is filled.
static inline RecPlan rec_plan(int B, int S, int C, int bytes) {
    const int V = C >= rec_vec(bytes) ? rec_vec(bytes) : 1;
    RecPlan pl;
    pl.slices = (C + REC_LC * V - 1) / (REC_LC * V);
    pl.waves = S <= REC_SAVE ? 1 : REC_WIDE;
    const long tile = (long)pl.waves * REC_SAVE, tiles = (S + tile - 1) / tile, seqs = (long)B * pl.slices;
    const long want = seqs >= 192 ? 1 : std::min((512 + seqs - 1) / seqs, 64l);
    const long per = std::max(1l, tiles / std::min(want, tiles));
    pl.piece = per * tile;
    pl.pieces = (int)((tiles + per - 1) / per);
    return pl;
}
static inline size_t rec_ws_bytes(int B, int S, int C, int bytes) {
    const RecPlan pl = rec_plan(B, S, C, bytes);
    return pl.pieces == 1 ? 0 : align_up((size_t)B * pl.pieces * 2 * C * sizeof(float)) + align_up((size_t)B * C * sizeof(float));
}

// f(V, W) as integral constants
template <class T, class F> static int rec_shape(int C, const RecPlan& pl, F f) {
    constexpr int V = rec_vec(sizeof(T));
    std::integral_constant<int, V> v;
    std::integral_constant<int, 1> one;
    std::integral_constant<int, REC_WIDE> wide;
    if (C >= V) return pl.waves == 1 ? f(v, one) : f(v, wide);
    return pl.waves == 1 ? f(one, one) : f(one, wide);
}

template <class T>
static int run_recurrence(Rows<const T> x, Rows<const T> gate, const float* h0, const int* lengths, Rows<T> h, float* last, float* saved,
                          int B, int S, int C, int reverse, void* ws, hipStream_t st) {
    const RecPlan pl = rec_plan(B, S, C, sizeof(T));
    Arena arena(ws, ~(size_t)0);
    float* agg = pl.pieces > 1 ? arena.take<float>((size_t)B * pl.pieces * 2 * C) : nullptr;
    float* kept = pl.pieces > 1 ? arena.take<float>((size_t)B * C) : nullptr;
    const long grid = (long)B * pl.pieces * pl.slices;
    if (grid > 0x7fffffff) return MSF2_ERR_ARG;
    return rec_shape<T>(C, pl, [&](auto v, auto w) {
        constexpr int V = decltype(v)::value, W = decltype(w)::value;
        if (pl.pieces > 1)
            rec_piece_kernel<false, T, V, W><<<grid, 64 * W, 0, st>>>(x, gate, h0, lengths, agg, kept, pl, S, C, reverse);
        rec_forward_kernel<T, V, W><<<grid, 64 * W, 0, st>>>(x, gate, pl.pieces > 1 ? kept : h0, lengths, h, last, saved, agg, pl, S, C, reverse);
        return check_launch();
    });
}

template <class T>
static int run_recurrence_backward(Rows<const T> dh, Rows<const T> x, Rows<const T> gate, const float* saved, const float* dlast,
                                   const int* lengths, Rows<T> dx, Rows<T> dgate, float* dh0, int B, int S, int C, int reverse, void* ws,
                                   hipStream_t st) {
    const RecPlan pl = rec_plan(B, S, C, sizeof(T));
    Arena arena(ws, ~(size_t)0);
    float* agg = pl.pieces > 1 ? arena.take<float>((size_t)B * pl.pieces * 2 * C) : nullptr;
    float* kept = pl.pieces > 1 ? arena.take<float>((size_t)B * C) : nullptr;
    const long grid = (long)B * pl.pieces * pl.slices;
    if (grid > 0x7fffffff) return MSF2_ERR_ARG;
    return rec_shape<T>(C, pl, [&](auto v, auto w) {
        constexpr int V = decltype(v)::value, W = decltype(w)::value;
        if (pl.pieces > 1)
            rec_piece_kernel<true, T, V, W><<<grid, 64 * W, 0, st>>>(dh, gate, dlast, lengths, agg, kept, pl, S, C, reverse);
        rec_backward_kernel<T, V, W><<<grid, 64 * W, 0, st>>>(dh, x, gate, saved, pl.pieces > 1 ? kept : dlast, lengths, dx, dgate, dh0, agg,
                                                              pl, S, C, reverse);
        return check_launch();
    });
}

}  // namespace msf2
