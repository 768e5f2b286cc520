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
template <int V, class T> __device__ __forceinline__ void store_vec(T* p, const float (&f)[V]) {
    typename VecOf<T, V>::type v;
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = (T)f[j];
    *reinterpret_cast<typename VecOf<T, V>::type*>(p) = v;
}
template <int V, class T> __device__ __forceinline__ void store_some(T* p, int n, const float (&f)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (j < n) p[j] = (T)f[j];
}

// n / d for n < 2^31 by one multiplication: with 2^(l-1) < d <= 2^l the factor m = 2^(31+l) / d + 1 is off by less than 1, so
// n m / 2^(31+l) is off by less than 1 / d and its whole part is right.
struct Divider {
    unsigned d, m, shift;
    explicit Divider(unsigned d_) : d(d_), shift(31) {
        while ((1ull << (shift - 31)) < d) ++shift;
        m = (unsigned)((1ull << shift) / d + 1);
    }
    __device__ __forceinline__ unsigned div(unsigned n) const { return (unsigned)((uint64_t)n * m >> shift); }
};

// Frames of utterance b: lengths[b] held to [0, S], all S without lengths.
__device__ __forceinline__ int frames_of(const int* lengths, int b, int S) {
    return lengths ? min(max(lengths[b], 0), S) : S;
}

// 1 / (1 + e^-v) and its complement 1 / (1 + e^v) without cancellation: the exponential of -|v| only, so neither overflows.
// e^-|v| = 2^t (1 + r), t = -|v| log2 e rounded and r the part of the product that the rounding and the constant's own tail
// leave out: v_exp_f32 alone would carry |v| half-steps of error into a gate near 0 or 1.
__device__ __forceinline__ void sigmoid_pair(float v, float& p, float& q) {
    const float n = -fabsf(v), t = n * 1.44269504088896f;
    const float r = fmaf(n, 1.44269504088896f, -t) + n * 1.925963033e-8f;
    float e = __builtin_amdgcn_exp2f(t);
    e = fmaf(e, 0.693147180559945f * (t < -126.f ? 0.f : r), e);        // -infinity: t is, and r is not a number
    const float d = __builtin_amdgcn_rcpf(1.f + e), s = e * d;
    p = v < 0.f ? s : d;
    q = v < 0.f ? d : s;
}

template <int ACT> __device__ __forceinline__ float act_f(float v) {
    if constexpr (ACT == MSF2_ACT_RELU) return v < 0.f ? 0.f : v;       // keeps NaN
    if constexpr (ACT == MSF2_ACT_SILU || ACT == MSF2_ACT_SIGMOID) {
        float p, q;
        sigmoid_pair(v, p, q);
        return ACT == MSF2_ACT_SILU ? v * p : p;
    }
    return v;
}
// act'(v)
template <int ACT> __device__ __forceinline__ float act_grad_f(float v) {
    if constexpr (ACT == MSF2_ACT_RELU) return v > 0.f ? 1.f : 0.f;
    if constexpr (ACT == MSF2_ACT_SILU || ACT == MSF2_ACT_SIGMOID) {
        float p, q;
        sigmoid_pair(v, p, q);
        return ACT == MSF2_ACT_SILU ? p * fmaf(v, q, 1.f) : p * q;
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
