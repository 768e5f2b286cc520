// Gated linear recurrence and its gradient: h_t = a_t h_{t-1} + (1 - a_t) x_t per channel, a = sigmoid(gate).
//
// A run of frames acts on the state as h -> A h + B, with A the product of its gates and B what it adds; runs join as
// (A, B) then (A', B') = (A A', A' B + B').  So a workgroup takes a tile of frames by channels into registers in one go: every
// thread joins its R frames, a scan over the time lanes gives each thread the state before its first frame, and a second walk
// over the registers gives every h_t.  x and gate are read once and h is written once.  The gradient is the same recurrence
// from the last frame back, E_t = a_t (dh_t + E_{t+1}); the h_{t-1} that dgate needs are scanned again within 32 frames from
// a state that the forward pass saved, which costs 1/32 of a row per frame instead of reading h, and keeps them in 32 bits.
// 1 - a comes from e^-gate, and h from a h + (1 - a) x: the shorter x + a (h - x) rounds at the size of x, which a gate near 1
// lets through to a state that is far smaller.
// Memory-bound with a busy vector unit (29 instructions a value forward, without its exponential and reciprocal just as fast):
// 64 x 3999 x 512 bf16 forward 156 us, backward 258 (5.0 and 5.2 TB/s), 16 x 3999 x 512 fp32 83 and 127 us (4.7 and 5.3), one sequence
// of 61499 x 512 bf16 in pieces 25 + 38 us.
// t counts frames in walking order; frame s is t, or S - 1 - t in reverse.  Frames past an utterance's end count as a = 1, B = 0.
#pragma once
#include <algorithm>
#include "msf2_rows.h"

namespace msf2 {

constexpr int REC_SAVE = MSF2_RECURRENCE_SAVE;
constexpr int REC_WIDE = 8;                  // waves of a workgroup, where a sequence is longer than the short form's frames

// How the work is dealt out: `slices` of channels by `pieces` of `piece` frames by utterances.
struct RecPlan {
    int vec, lanes, slices, pieces, waves, piece;
    bool near;                               // a tile's rows span less than 2^32 bytes in every operand
    bool past;                               // results go past the caches
};

// The lanes of a workgroup: LC side by side over V channels each, the LT = 64 / LC groups of a wave one after the other in time,
// R frames a thread, W waves.
template <class T_, int V_, int LC_, int R_, int W_> struct RecShape {
    typedef T_ T;
    typedef typename VecOf<T_, V_>::type vec;
    static constexpr int V = V_, LC = LC_, LT = 64 / LC_, R = R_, W = W_;
    static constexpr int WAVE = LT * R, TILE = WAVE * W;       // frames of a wave, of a workgroup
    static_assert(LC == 16 || LC == 32 || LC == 64, "the scans are over rows of 16 lanes or halves of a wave");
};

// What a workgroup works on, and a thread's place in it.  The lane of the last channels is moved left to end with the
// row, so that every load is a whole vector; what it shares with its neighbour is computed twice and written once (`own` on).
// Slices of the same frames share lines where rows are not aligned to them, and go to the same XCD one after the other: blocks are dealt
// to the 8 XCDs in turn, so block i of XCD k takes the i-th of the k-th eighth of the work.
template <class Q> struct RecPlace {
    int b, p, n, tl, cl, wave, c, own;
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
        tl = lane / Q::LC;
        cl = lane % Q::LC;
        const int c0 = (slice * Q::LC + cl) * Q::V;
        c = min(c0, C - Q::V);
        own = c0 - c;                        // V and more: nothing is this lane's own
    }
    __device__ __forceinline__ bool first() const { return wave == 0 && tl == 0; }
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

// One level of a scan over the lanes of a wave: every lane gets the run of the earlier (lo) and of the later (hi) half of its
// pair, rows of 16 lanes 2k and 2k + 1 with D = 16, the two halves of the wave with D = 32.  v_permlane*_swap exchanges the odd half
// of its first register with the even half of its second, so with the same value in both it leaves lo in the first, hi in the
// second.
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
template <bool BACK, int LC, int V> __device__ __forceinline__ void wave_scan(const Run<V>& r, int tl, Run<V>& before, Run<V>& all) {
    Run<V> lo, hi, part;
    auto pick = [&](bool on) {               // the run of the half that comes first, for the lanes of the other
        Run<V> o;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            o.a[v] = on ? (BACK ? hi : lo).a[v] : 1.f;
            o.b[v] = on ? (BACK ? hi : lo).b[v] : 0.f;
        }
        return o;
    };
    part = r;
    before.clear();
    if constexpr (LC == 64) {                // a wave is one frame wide
        all = r;
        return;
    }
    if constexpr (LC == 16) {
        halves<16, V>(part, lo, hi);
        before = pick(BACK ? !(tl & 1) : tl & 1);
        part = BACK ? lo : hi;
        part.after(BACK ? hi : lo);
    }
    halves<32, V>(part, lo, hi);
    const Run<V> skip = pick(BACK ? tl < 32 / LC : tl >= 32 / LC);
    if constexpr (LC == 16) before.after(skip);
    else before = skip;
    all = BACK ? lo : hi;
    all.after(BACK ? hi : lo);
}

// The waves of a workgroup in turn: h, the state before the tile, becomes the state after it, and `mine` the one before this
// wave's frames.  The runs lie in one of two buffers that tiles take in turn, so one barrier a tile is enough: who fills a
// buffer again has passed the barrier of the tile between, which nobody passes before having read it.
template <bool BACK, class Q>
__device__ __forceinline__ void join_waves(const Run<Q::V> (*runs)[Q::LC], int wave, int cl, float (&h)[Q::V], float (&mine)[Q::V]) {
#pragma unroll
    for (int k = 0; k < Q::W; ++k) {
        const int w = BACK ? Q::W - 1 - k : k;
        if (w == wave) {
#pragma unroll
            for (int v = 0; v < Q::V; ++v) mine[v] = h[v];
        }
        runs[w][cl].apply(h);
    }
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

// The state before piece p in every lane: `start` and the runs of the pieces before it (BACK: behind it), agg
// [b][pieces][2][C].  The time lanes and waves take a share of the pieces each, joined like the frames of a tile.
template <bool BACK, class Q>
__device__ __forceinline__ void rec_carry(const RecPlan& pl, const float* agg, const float* start, const RecPlace<Q>& at, int C,
                                          Run<Q::V> (*runs)[Q::LC], float (&h)[Q::V]) {
    constexpr int V = Q::V, SHARES = Q::W * Q::LT;
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = 0.f;
    if (start) rec_read<V>(start + (long)at.b * C + at.c, h);
    const int count = BACK ? pl.pieces - 1 - at.p : at.p;
    if (pl.pieces == 1 || count == 0) return;        // the same for the whole workgroup
    const int share = (count + SHARES - 1) / SHARES, place = at.wave * Q::LT + at.tl;
    const int from = BACK ? at.p + 1 : 0;            // BACK: the last piece comes first, and so does the last lane
    const int k0 = min(place * share, count), k1 = min(k0 + share, count);
    Run<V> r, before, all;
    r.clear();
#pragma unroll 4
    for (int i = 0; i < k1 - k0; ++i) {
        const float* q = agg + ((long)at.b * pl.pieces + from + (BACK ? k1 - 1 - i : k0 + i)) * 2 * C + at.c;
        Run<V> next;
        rec_read<V>(q, next.a);
        rec_read<V>(q + C, next.b);
        next.after(r);
        r = next;
    }
    wave_scan<BACK, Q::LC, V>(r, at.tl, before, all);
    if (at.tl == 0) runs[at.wave][at.cl] = all;
    __syncthreads();
    float mine[V];
    join_waves<BACK, Q>(runs, at.wave, at.cl, h, mine);
}

// Where a tile's frames lie.  `all`: every one of them is in the utterance, and then a thread's row j is at an address that is the same for
// the workgroup up to a 32-bit offset of the thread's own: the compiler keeps the one in scalar registers, and a load costs no vector
// arithmetic.  At the ends each row has its own address, held to the utterance (to memory, at least), and frames outside it are
// a = 1 and add nothing, whatever memory holds there.
template <class Q> struct RecFrames {
    int t, first, n, S, end;                 // the tile's and this thread's first frame walked; no frame from `end` on
    bool reverse, all;
    __device__ __forceinline__ RecFrames(int tile, int mine, int end_, int n_, int S_, bool reverse_, bool near)
        : t(tile), first(tile + mine), n(n_), S(S_), end(end_), reverse(reverse_) {
        all = near && tile + Q::TILE <= end && (reverse ? tile >= S - n : tile + Q::TILE <= n);
    }
    __device__ __forceinline__ int s(int j) const { return reverse ? S - 1 - first - j : first + j; }
    __device__ __forceinline__ bool live(int j) const { return first + j < end && s(j) < n; }
    __device__ __forceinline__ int held(int j) const { return min(max(s(j), 0), max(n - 1, 0)); }
};
// One operand's rows: utterance b, and this thread's offset in bytes within a tile.
template <class Q, class U> struct RecRows {
    U* p;
    long row;
    unsigned mine;
    int c;
    __device__ __forceinline__ RecRows(const Rows<U>& r, int b, int mine_, int c_, bool reverse) : p(r.p + b * r.batch), row(r.row), c(c_) {
        mine = (unsigned)(((long)(reverse ? Q::TILE - Q::R - mine_ : mine_) * r.row + c_) * (long)sizeof(U));
    }
    // the address of row j without this thread's offset, for a whole tile
    __device__ __forceinline__ U* base(const RecFrames<Q>& fr, int j) const {
        return p + (long)(fr.reverse ? fr.S - fr.t - Q::TILE + Q::R - 1 - j : fr.t + j) * row;
    }
    template <class B> static __device__ __forceinline__ B* off(B* q, unsigned bytes) {
        return reinterpret_cast<B*>(reinterpret_cast<std::conditional_t<std::is_const<B>::value, const char, char>*>(q) + bytes);
    }
    __device__ __forceinline__ void load(const RecFrames<Q>& fr, typename Q::vec (&v)[Q::R]) const {
        if (fr.all) {
#pragma unroll
            for (int j = 0; j < Q::R; ++j) v[j] = load_vec<Q::V>(off(base(fr, j), mine));
        } else {
#pragma unroll
            for (int j = 0; j < Q::R; ++j) v[j] = load_vec<Q::V>(p + (long)fr.held(j) * row + c);
        }
    }
    __device__ __forceinline__ void store(const RecFrames<Q>& fr, bool past, int own, float (&f)[Q::R][Q::V]) const {
        if (fr.all && own <= 0) {
            if (past) {                      // the empty statements keep the compiler from making one of the two
                asm volatile("");
#pragma unroll
                for (int j = 0; j < Q::R; ++j) store_vec<Q::V, true>(off(base(fr, j), mine), f[j]);
                asm volatile("");
            } else {
#pragma unroll
                for (int j = 0; j < Q::R; ++j) store_vec<Q::V>(off(base(fr, j), mine), f[j]);
            }
        } else if (fr.all) {
#pragma unroll
            for (int v = 1; v < Q::V; ++v)
                if (v >= own) {
#pragma unroll
                    for (int j = 0; j < Q::R; ++j) off(base(fr, j), mine)[v] = (U)f[j][v];
                }
        } else {
#pragma unroll
            for (int j = 0; j < Q::R; ++j)
                if (fr.first + j < fr.end) {
#pragma unroll
                    for (int v = 0; v < Q::V; ++v) f[j][v] = fr.live(j) ? f[j][v] : 0.f;
                    rec_store<Q::V>(p + (long)fr.s(j) * row + c, own, f[j]);
                }
        }
    }
};

// The run of one piece, for sequences too few to fill the chip: agg, and `start` copied to `kept`, because the pieces of the
// next launch read it while one of them may write the last state into the same memory.  u is x, or dh with BACK; a thread
// walks piece / (W LT) frames on end.
template <bool BACK, class Q>
__global__ __launch_bounds__(64 * Q::W) void rec_piece_kernel(Rows<const typename Q::T> u, Rows<const typename Q::T> gate, const float* start,
                                                              const int* lengths, float* agg, float* kept, RecPlan pl, int S, int C, bool reverse) {
    typedef typename Q::T T;
    constexpr int V = Q::V, R = Q::R;
    __shared__ Run<V> runs[Q::W][Q::LC];
    const RecPlace<Q> at(pl, lengths, S, C);
    if (at.p == (BACK ? pl.pieces - 1 : 0) && at.first()) {
        float h[V];
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = 0.f;
        if (start) rec_read<V>(start + (long)at.b * C + at.c, h);
        rec_store<V>(kept + (long)at.b * C + at.c, at.own, h);
    }
    if (at.p == (BACK ? 0 : pl.pieces - 1)) return;         // nothing follows it
    const int steps = pl.piece / (Q::W * Q::LT);            // a multiple of R
    const int t0 = at.p * pl.piece + (at.wave * Q::LT + at.tl) * steps, cap = max(at.n - 1, 0);
    const T *up = u.at(at.b, 0) + at.c, *gp = gate.at(at.b, 0) + at.c;
    Run<V> r;
    r.clear();
    for (int k = 0; k < steps; k += R) {
        typename Q::vec uv[R], gv[R];
        bool live[R];
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const int t = t0 + (BACK ? steps - 1 - k - j : k + j), s = reverse ? S - 1 - t : t, h = min(max(s, 0), cap);
            live[j] = t < S && s < at.n;
            uv[j] = load_vec<V>(up + (long)h * u.row);
            gv[j] = load_vec<V>(gp + (long)h * gate.row);
        }
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float a, na;
                sigmoid_pair<fine<T>()>(live[j] ? (float)gv[j][v] : 87.f, a, na);       // 87: a is 1
                const float f = live[j] ? (float)uv[j][v] : 0.f;
                r.b[v] = BACK ? a * (r.b[v] + f) : fmaf(a, r.b[v], na * f);
                r.a[v] *= a;
            }
    }
    Run<V> before, all;
    wave_scan<BACK, Q::LC, V>(r, at.tl, before, all);
    if (at.tl == 0) runs[at.wave][at.cl] = all;
    __syncthreads();
    if (at.first()) {
        r.clear();
        for (int k = 0; k < Q::W; ++k) {
            Run<V> next = runs[BACK ? Q::W - 1 - k : k][at.cl];
            next.after(r);
            r = next;
        }
        float* q = agg + ((long)at.b * pl.pieces + at.p) * 2 * C + at.c;
        rec_store<V>(q, at.own, r.a);
        rec_store<V>(q + C, at.own, r.b);
    }
}

// Frames outside the utterance: a gate of 87 is a = 1 exactly, and nothing is added.
template <class Q> __device__ __forceinline__ void rec_mask(const RecFrames<Q>& fr, typename Q::vec (&v)[Q::R], float with) {
#pragma unroll
    for (int j = 0; j < Q::R; ++j)
        if (!fr.live(j))
#pragma unroll
            for (int i = 0; i < Q::V; ++i) v[j][i] = (typename Q::T)with;
}

template <class Q>
__global__ __launch_bounds__(64 * Q::W) void rec_forward_kernel(Rows<const typename Q::T> x_, Rows<const typename Q::T> gate_, const float* start,
                                                                const int* lengths, Rows<typename Q::T> h_, float* last, float* saved,
                                                                const float* agg, RecPlan pl, int S, int C, bool reverse) {
    typedef typename Q::T T;
    constexpr int V = Q::V, R = Q::R;
    __shared__ Run<V> runs[2][Q::W][Q::LC];
    const RecPlace<Q> at(pl, lengths, S, C);
    const int t0 = at.p * pl.piece, t1 = min(t0 + pl.piece, S), blocks = (S + REC_SAVE - 1) / REC_SAVE;
    const int mine = at.wave * Q::WAVE + at.tl * R;            // this thread's first frame in a tile
    const RecRows<Q, const T> x(x_, at.b, mine, at.c, reverse), gate(gate_, at.b, mine, at.c, reverse);
    const RecRows<Q, T> h(h_, at.b, mine, at.c, reverse);
    typename Q::vec nx[R], ng[R];
    auto fetch = [&](int t) {
        const RecFrames<Q> fr(t, mine, t1, at.n, S, reverse, pl.near);
        x.load(fr, nx);
        gate.load(fr, ng);
    };
    fetch(t0);
    float carry[V];
    rec_carry<false, Q>(pl, agg, start, at, C, runs[0], carry);
    int turn = 1;
    for (int t = t0; t < t1; t += Q::TILE, turn ^= 1) {
        const RecFrames<Q> fr(t, mine, t1, at.n, S, reverse, pl.near);
        float a[R][V], f[R][V];
        Run<V> r, before, all;
        r.clear();
        if (!fr.all) rec_mask<Q>(fr, nx, 0.f), rec_mask<Q>(fr, ng, 87.f);
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float na;
                sigmoid_pair<fine<T>()>((float)ng[j][v], a[j][v], na);
                f[j][v] = na * (float)nx[j][v];
                r.b[v] = fmaf(a[j][v], r.b[v], f[j][v]);
                r.a[v] *= a[j][v];
            }
        if (t + Q::TILE < t1) fetch(t + Q::TILE);
        wave_scan<false, Q::LC, V>(r, at.tl, before, all);
        if (at.tl == 0) runs[turn][at.wave][at.cl] = all;
        __syncthreads();
        float hv[V];
        join_waves<false, Q>(runs[turn], at.wave, at.cl, carry, hv);
        before.apply(hv);
        if (saved && fr.first % REC_SAVE == 0 && fr.first < t1)
            rec_store<V>(saved + ((long)at.b * blocks + fr.first / REC_SAVE) * C + at.c, at.own, hv);
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) f[j][v] = hv[v] = fmaf(a[j][v], hv[v], f[j][v]);
        h.store(fr, pl.past, at.own, f);
    }
    if (last && t1 == S && at.first()) rec_store<V>(last + (long)at.b * C + at.c, at.own, carry);
}

template <class Q>
__global__ __launch_bounds__(64 * Q::W) void rec_backward_kernel(Rows<const typename Q::T> dh_, Rows<const typename Q::T> x_,
                                                                 Rows<const typename Q::T> gate_, const float* saved, const float* start,
                                                                 const int* lengths, Rows<typename Q::T> dx_, Rows<typename Q::T> dgate_, float* dh0,
                                                                 const float* agg, RecPlan pl, int S, int C, bool reverse) {
    typedef typename Q::T T;
    constexpr int V = Q::V, R = Q::R;
    constexpr int SHARE = Q::WAVE < REC_SAVE ? REC_SAVE / Q::WAVE : 1;       // waves that start from the same saved state
    static_assert(Q::TILE % REC_SAVE == 0 && (SHARE > 1 || Q::WAVE % REC_SAVE == 0), "a tile begins at a saved state");
    __shared__ Run<V> runs[2][Q::W][Q::LC], ahead[2][SHARE > 1 ? Q::W : 1][Q::LC];
    const RecPlace<Q> at(pl, lengths, S, C);
    const int t0 = at.p * pl.piece, t1 = min(t0 + pl.piece, S), blocks = (S + REC_SAVE - 1) / REC_SAVE;
    const int mine = at.wave * Q::WAVE + at.tl * R;
    const RecRows<Q, const T> dh(dh_, at.b, mine, at.c, reverse), x(x_, at.b, mine, at.c, reverse), gate(gate_, at.b, mine, at.c, reverse);
    const RecRows<Q, T> dx(dx_, at.b, mine, at.c, reverse), dgate(dgate_, at.b, mine, at.c, reverse);
    typename Q::vec nd[R], nx[R], ng[R];
    float nh[V];
    auto fetch = [&](int t) {
        const RecFrames<Q> fr(t, mine, t1, at.n, S, reverse, pl.near);
        dh.load(fr, nd);
        x.load(fr, nx);
        gate.load(fr, ng);
        const int block = min((t + at.wave * Q::WAVE) / REC_SAVE, blocks - 1);
        rec_read<V>(saved + ((long)at.b * blocks + block) * C + at.c, nh);
    };
    const int tiles = (t1 - t0 + Q::TILE - 1) / Q::TILE;
    fetch(t0 + (tiles - 1) * Q::TILE);
    float carry[V];
    rec_carry<true, Q>(pl, agg, start, at, C, runs[0], carry);
    int turn = 1;
    for (int t = t0 + (tiles - 1) * Q::TILE; t >= t0; t -= Q::TILE, turn ^= 1) {
        const RecFrames<Q> fr(t, mine, t1, at.n, S, reverse, pl.near);
        float a[R][V], na[R][V], f[R][V], d[R][V], hv[V], e[V];
        Run<V> r, q, before, behind, all;
        r.clear();
        if (!fr.all) rec_mask<Q>(fr, nd, 0.f), rec_mask<Q>(fr, nx, 0.f), rec_mask<Q>(fr, ng, 87.f);
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                sigmoid_pair<fine<T>()>((float)ng[j][v], a[j][v], na[j][v]);
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
        if (t > t0) fetch(t - Q::TILE);
        wave_scan<false, Q::LC, V>(r, at.tl, before, all);
        if (SHARE > 1 && at.tl == 0) ahead[turn][at.wave][at.cl] = all;
        wave_scan<true, Q::LC, V>(q, at.tl, behind, all);
        if (at.tl == 0) runs[turn][at.wave][at.cl] = all;
        __syncthreads();
        join_waves<true, Q>(runs[turn], at.wave, at.cl, carry, e);
        if constexpr (SHARE > 1) {
#pragma unroll
            for (int k = 1; k < SHARE; ++k)
                if (at.wave % SHARE >= k) ahead[turn][at.wave / SHARE * SHARE + k - 1][at.cl].apply(hv);
        }
        before.apply(hv);
        behind.apply(e);
        // f becomes (1 - a_t) (h_{t-1} - x_t)
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float xv = f[j][v];
                f[j][v] = na[j][v] * (hv[v] - xv);
                hv[v] = fmaf(a[j][v], hv[v], na[j][v] * xv);
            }
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
        dx.store(fr, pl.past, at.own, d);
        dgate.store(fr, pl.past, at.own, f);
    }
    if (dh0 && t0 == 0 && at.first()) rec_store<V>(dh0 + (long)at.b * C + at.c, at.own, carry);
}

// A thread takes 16 values: `vec` channels by 16 / vec frames, 8 bytes of a frame, except that the backward pass of the 16-bit types
// takes 4 of an even width (64 x 3999 x 512 bf16 backward, 4 and 8 bytes: 260 and 279 us; x 501, where every other row is off the
// 4-byte grid: 430 and 371; forward 163 and 159, 236 and 212).  By width and not by the operands' alignment, so that a slice of a wider
// tensor gives the same bits as its copy.
constexpr int REC_VALUES = 16;
static inline bool rec_pairs(int bytes, int C, bool backward) { return bytes == 2 && backward && C % 2 == 0; }
// the short form's waves: as many as reach from one saved state to the next
constexpr int rec_short(int lanes, int rows) { return std::max(1, REC_SAVE / (64 / lanes * rows)); }

// The division of the work that takes the least time by this count, in tiles that a CU works off:
//   whole sequences, workgroups / 256 CUs rounded up;
//   pieces, where the operands are read twice: 5 / 3 of that forward, or 1.5 with two workgroups on a CU at once, 7 / 5 backward (one
//   workgroup a CU, for its registers), and another launch, worth 1.5 tiles;
//   slices of 256 bytes of a frame 0.92 of those of 128 (two lines a row reach 4.9 TB/s, one 4.3).
// Measured: 16 x 4000 x 512 bf16 forward, 128 sequences, 74 us whole, 58 in 4 pieces, 64 in 2; backward 88 us in 512 workgroups, 81 in
// 256; 4 x 512 x 256 fp32, two tiles, 8.3 us whole and 9.5 in pieces, three tiles 10.8 and 9.6.
static inline RecPlan rec_plan(int B, int S, int C, int bytes, bool backward) {
    const int vec = rec_pairs(bytes, C, backward) ? 2 : 8 / bytes, V = C >= vec ? vec : 1, rows = REC_VALUES / vec;
    RecPlan best;
    double least = 0;
    for (int wide = 1; wide >= 0; --wide) {
        if (V == 1 && wide) continue;
        RecPlan pl;
        pl.vec = V;
        pl.lanes = (wide ? 256 : 128) / (vec * bytes);
        const int wave = 64 / pl.lanes * rows, few = rec_short(pl.lanes, rows);
        pl.slices = (C + pl.lanes * V - 1) / (pl.lanes * V);
        pl.waves = S <= few * wave ? few : REC_WIDE;
        const long tile = (long)pl.waves * wave, tiles = (S + tile - 1) / tile, seqs = (long)B * pl.slices;
        long before = 0;
        for (int fill = 0; fill <= 8; ++fill) {              // whole, then workgroups for up to 8 times the CUs
            const long want = fill ? std::min(256l * fill / seqs, tiles) : 1;
            if (want <= before) continue;
            before = want;
            const long per = (tiles + want - 1) / want, pieces = (tiles + per - 1) / per, groups = seqs * pieces;
            double cost = (double)((groups + 255) / 256 * per);
            if (pieces > 1) cost = cost * (backward ? 1.4 : groups >= 480 ? 1.5 : 1.67) + 1.5;
            if (wide) cost *= 0.92;
            if (least && cost >= least) continue;
            least = cost;
            pl.piece = (int)(per * tile);
            pl.pieces = (int)pieces;
            best = pl;
        }
    }
    best.near = best.past = true;
    return best;
}
static inline size_t rec_ws_bytes(int B, int S, int C, int bytes, bool backward) {
    const RecPlan pl = rec_plan(B, S, C, bytes, backward);
    return pl.pieces == 1 ? 0 : align_up((size_t)B * pl.pieces * 2 * C * sizeof(float)) + align_up((size_t)B * C * sizeof(float));
}

// f(RecShape) of the form that the plan names
template <class T, int V, int LC, int R, class F> static int rec_waves(const RecPlan& pl, F f) {
    return pl.waves == REC_WIDE ? f(RecShape<T, V, LC, R, REC_WIDE>()) : f(RecShape<T, V, LC, R, rec_short(LC, R)>());
}
template <class T, int VEC, class F> static int rec_lanes(const RecPlan& pl, F f) {
    constexpr int LC = 256 / (VEC * sizeof(T)), R = REC_VALUES / VEC;
    if constexpr (VEC * sizeof(T) == 8)      // 4-byte accesses are for even widths, which are never narrower
        if (pl.vec == 1) return rec_waves<T, 1, LC / 2, R>(pl, f);
    return pl.lanes == LC ? rec_waves<T, VEC, LC, R>(pl, f) : rec_waves<T, VEC, LC / 2, R>(pl, f);
}
template <class T, bool BACK, class F> static int rec_shape(const RecPlan& pl, int C, F f) {
    if constexpr (BACK && sizeof(T) == 2)
        if (rec_pairs(sizeof(T), C, true)) return rec_lanes<T, 2>(pl, f);
    return rec_lanes<T, 8 / sizeof(T)>(pl, f);
}
// whether a tile of an operand can be addressed by 32-bit offsets
template <class Q, class U> static bool rec_near(const Rows<U>& r, int C) {
    return r.row >= 0 && r.row < (1l << 31) / (Q::TILE * (long)sizeof(U)) && C < 1 << 28;
}
// Whether a result's rows are whole lines.  Past the caches those are 10 % faster (16 x 3999 x 512 fp32 forward 85 and 94 us), parts of
// lines, which only meet in a cache, up to 45 % slower (16 x 3999 x 501 fp32 backward 212 and 147 us).
template <class U> static bool rec_lines(const Rows<U>& r) {
    return ((uintptr_t)r.p | (r.row | r.batch) * sizeof(U)) % 128 == 0;
}

template <class T>
static int run_recurrence(Rows<const T> x, Rows<const T> gate, const float* h0, const int* lengths, Rows<T> h, float* last, float* saved,
                          int B, int S, int C, bool reverse, void* ws, hipStream_t st) {
    RecPlan pl = rec_plan(B, S, C, sizeof(T), false);
    Arena arena(ws, ~(size_t)0);
    float* agg = pl.pieces > 1 ? arena.take<float>((size_t)B * pl.pieces * 2 * C) : nullptr;
    float* kept = pl.pieces > 1 ? arena.take<float>((size_t)B * C) : nullptr;
    const long grid = (long)B * pl.pieces * pl.slices;
    if (!launch_ok(grid, 64 * pl.waves)) return MSF2_ERR_ARG;
    return rec_shape<T, false>(pl, C, [&](auto q) {
        typedef decltype(q) Q;
        pl.near = rec_near<Q>(x, C) && rec_near<Q>(gate, C) && rec_near<Q>(h, C);
        pl.past = rec_lines(h);
        if constexpr (Q::W == REC_WIDE)
            if (pl.pieces > 1) rec_piece_kernel<false, Q><<<grid, 64 * Q::W, 0, st>>>(x, gate, h0, lengths, agg, kept, pl, S, C, reverse);
        rec_forward_kernel<Q><<<grid, 64 * Q::W, 0, st>>>(x, gate, pl.pieces > 1 ? kept : h0, lengths, h, last, saved, agg, pl, S, C, reverse);
        return check_launch();
    });
}

template <class T>
static int run_recurrence_backward(Rows<const T> dh, Rows<const T> x, Rows<const T> gate, const float* saved, const float* dlast,
                                   const int* lengths, Rows<T> dx, Rows<T> dgate, float* dh0, int B, int S, int C, bool reverse, void* ws,
                                   hipStream_t st) {
    RecPlan pl = rec_plan(B, S, C, sizeof(T), true);
    Arena arena(ws, ~(size_t)0);
    float* agg = pl.pieces > 1 ? arena.take<float>((size_t)B * pl.pieces * 2 * C) : nullptr;
    float* kept = pl.pieces > 1 ? arena.take<float>((size_t)B * C) : nullptr;
    const long grid = (long)B * pl.pieces * pl.slices;
    if (!launch_ok(grid, 64 * pl.waves)) return MSF2_ERR_ARG;
    return rec_shape<T, true>(pl, C, [&](auto q) {
        typedef decltype(q) Q;
        pl.near = rec_near<Q>(dh, C) && rec_near<Q>(x, C) && rec_near<Q>(gate, C) && rec_near<Q>(dx, C) && rec_near<Q>(dgate, C);
        pl.past = rec_lines(dx) && rec_lines(dgate);
        if constexpr (Q::W == REC_WIDE)
            if (pl.pieces > 1) rec_piece_kernel<true, Q><<<grid, 64 * Q::W, 0, st>>>(dh, gate, dlast, lengths, agg, kept, pl, S, C, reverse);
        rec_backward_kernel<Q><<<grid, 64 * Q::W, 0, st>>>(dh, x, gate, saved, pl.pieces > 1 ? kept : dlast, lengths, dx, dgate, dh0, agg,
                                                           pl, S, C, reverse);
        return check_launch();
    });
}

}  // namespace msf2
