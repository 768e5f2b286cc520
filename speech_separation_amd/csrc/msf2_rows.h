// [B, S, C] tensors of the block operators: element types, strided rows, utterance lengths, activations.
#pragma once
#include <type_traits>
#include "msf2_common.h"

namespace msf2 {

typedef __bf16 bf16;
typedef _Float16 fp16;

// Calls f with a value of the element type that `type` names; MSF2_ERR_ARG for any other.
template <class F> static inline int by_type(int type, F f) {
    switch (type) {
        case MSF2_TYPE_FP32: return f(float());
        case MSF2_TYPE_BF16: return f(bf16());
        case MSF2_TYPE_FP16: return f(fp16());
        default: return MSF2_ERR_ARG;
    }
}

// One [B, S, C] operand: channels contiguous, strides in elements (64 bits: a long batch passes 2^31 of them).
template <class T> struct Rows {
    T* p;
    long batch, row;
    __host__ __device__ T* at(long b, long s) const { return p + b * batch + s * row; }
};

// V neighbouring elements at any address that suits one element: gfx950 loads and stores 16 bytes at any byte address, so odd
// widths and slices need no form of their own (an access that straddles two lines costs the second line).
template <class T, int V> struct VecOf {
    typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};
template <int V, class T> __device__ __forceinline__ typename VecOf<T, V>::type load_vec(const T* p) {
    return *reinterpret_cast<const typename VecOf<T, V>::type*>(p);
}
// the first n < V of them, zeros behind
template <int V, class T> __device__ __forceinline__ typename VecOf<T, V>::type load_some(const T* p, int n) {
    typename VecOf<T, V>::type v = {};
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (j < n) v[j] = p[j];
    return v;
}
// PAST: past the caches, for results that would only push the operands out of them.
template <int V, bool PAST = false, class T> __device__ __forceinline__ void store_vec(T* p, const float (&f)[V]) {
    typename VecOf<T, V>::type v;
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = (T)f[j];
    if constexpr (PAST) __builtin_nontemporal_store(v, reinterpret_cast<typename VecOf<T, V>::type*>(p));
    else *reinterpret_cast<typename VecOf<T, V>::type*>(p) = v;
}
template <int V, class T> __device__ __forceinline__ void store_some(T* p, int n, const float (&f)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (j < n) p[j] = (T)f[j];
}
// All from element n on, n the same for all lanes that come here: one access for each bit of V - n, V / 2 elements last.
template <int V, class T> __device__ __forceinline__ void store_last(T* p, int n, const float (&f)[V]) {
    auto bit = [&](auto width) {
        constexpr int W = decltype(width)::value;
        if constexpr (W < V) {
            if (n & W) {
                float g[W];
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    g[j] = 0.f;
#pragma unroll
                    for (int o = W; o < V; o += 2 * W) g[j] = n == o ? f[o + j] : g[j];
                }
                store_vec<W>(p + n, g);
                n += W;
            }
        }
    };
    bit(std::integral_constant<int, 1>());   // n is a multiple of 2 after this one, of 4 after the next
    bit(std::integral_constant<int, 2>());
    bit(std::integral_constant<int, 4>());
}

// n / d for n < 2^31 by one multiplication: with 2^(l-1) < d <= 2^l the factor m = 2^(31+l) / d + 1 is off by less than 1, so
// n m / 2^(31+l) is off by less than 1 / d and its whole part is right.
struct Divider {
    unsigned d, m, shift;
    explicit Divider(unsigned d_ = 1) : d(d_), shift(31) {
        while ((1ull << (shift - 31)) < d) ++shift;
        m = (unsigned)((1ull << shift) / d + 1);
    }
    __host__ __device__ __forceinline__ unsigned div(unsigned n) const { return (unsigned)((uint64_t)n * m >> shift); }
};

// Whether a launch of so many workgroups counts its threads in 32 bits, as the hardware does.
static inline bool launch_ok(long groups, int threads) { return groups * threads < 1l << 32; }

// Frames of utterance b: lengths[b] held to [0, S], all S without lengths.
__device__ __forceinline__ int frames_of(const int* lengths, int b, int S) {
    return lengths ? min(max(lengths[b], 0), S) : S;
}

// p = 1 / (1 + t) and q = 1 - p = t p, t = e^-v: neither cancels.  A rounding d of v log2 e is a relative error d ln 2 of t, which p takes
// q times and q takes p times: FINE (fp32 operands) adds the part that the product's rounding left out.  Without it the smaller of
// p and q is off by up to |v| 2^-24 of itself, 2^-18 at the most: far below the steps of the 16-bit operands that v comes from.  Values beyond 87 are
// held there (e^87 and its inverse are normal numbers; maximum and minimum keep NaN).
template <bool FINE> __device__ __forceinline__ void sigmoid_pair(float v, float& p, float& q) {
    constexpr float LOG2E = 1.44269504088896f, LN2 = 0.693147180559945f;
    v = __builtin_elementwise_maximum(v, -87.f);
    if constexpr (FINE) v = __builtin_elementwise_minimum(v, 87.f);
    const float u = -v * LOG2E;
    float t = __builtin_amdgcn_exp2f(u);
    if constexpr (FINE) t = fmaf(t * LN2, fmaf(-v, LOG2E, -u), t);
    p = __builtin_amdgcn_rcpf(1.f + t);
    q = t * p;
}
template <class T> constexpr bool fine() { return sizeof(T) == 4; }

// v p of v far below zero ends at -87 e^-87, -1e-36, where v itself would give a product of infinity and the least p
__device__ __forceinline__ float silu_of(float v, float p) { return __builtin_elementwise_maximum(v, -87.f) * p; }

template <int ACT, bool FINE> __device__ __forceinline__ float act_f(float v) {
    if constexpr (ACT == MSF2_ACT_RELU) return v < 0.f ? 0.f : v;       // keeps NaN
    if constexpr (ACT == MSF2_ACT_SILU || ACT == MSF2_ACT_SIGMOID) {
        float p, q;
        sigmoid_pair<FINE>(v, p, q);
        return ACT == MSF2_ACT_SILU ? silu_of(v, p) : p;
    }
    return v;
}
// act'(v)
template <int ACT, bool FINE> __device__ __forceinline__ float act_grad_f(float v) {
    if constexpr (ACT == MSF2_ACT_RELU) return v > 0.f ? 1.f : 0.f;
    if constexpr (ACT == MSF2_ACT_SILU || ACT == MSF2_ACT_SIGMOID) {
        float p, q;
        sigmoid_pair<FINE>(v, p, q);
        return ACT == MSF2_ACT_SILU ? p * fmaf(__builtin_elementwise_minimum(__builtin_elementwise_maximum(v, -87.f), 87.f), q, 1.f) : p * q;
    }
    return 1.f;
}
template <class F> static inline int by_act(int act, F f) {
    switch (act) {
        case MSF2_ACT_NONE: return f(std::integral_constant<int, MSF2_ACT_NONE>());
        case MSF2_ACT_SILU: return f(std::integral_constant<int, MSF2_ACT_SILU>());
        case MSF2_ACT_SIGMOID: return f(std::integral_constant<int, MSF2_ACT_SIGMOID>());
        case MSF2_ACT_RELU: return f(std::integral_constant<int, MSF2_ACT_RELU>());
        default: return MSF2_ERR_ARG;
    }
}

}  // namespace msf2
