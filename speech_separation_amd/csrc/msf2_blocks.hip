// C-ABI entry points of the block operators: group norm with an activation, gated recurrence, dropout.  All work is
// enqueued on the caller's stream; nothing here allocates, synchronises or keeps state.
#include <algorithm>
#include <cmath>
#include "msf2_groupnorm.h"
#include "msf2_recurrence.h"
#include "msf2_dropout.h"

using namespace msf2;

// S and C below 2^30: indices of frames and channels, and the end of the tile that holds the last one, stay below 2^31
static inline bool sizes_ok(int B, int S, int C) {
    return B >= 1 && S >= 1 && S < 1 << 30 && C >= 1 && C < 1 << 30 && (long)B * S <= (1l << 46) / C;
}
static inline bool type_ok(int type) { return type == MSF2_TYPE_FP32 || type == MSF2_TYPE_BF16 || type == MSF2_TYPE_FP16; }
static inline int type_bytes(int type) { return type == MSF2_TYPE_FP32 ? 4 : 2; }
static inline bool norm_ok(int B, int S, int C, int groups, int type) {
    return sizes_ok(B, S, C) && groups >= 1 && C % groups == 0 && type_ok(type);
}

extern "C" {

size_t msf2_group_norm_act_ws_bytes(int B, int S, int C, int groups, int type) {
    return norm_ok(B, S, C, groups, type) ? gn_ws_bytes(B, S, C, groups, type_bytes(type), false) : 0;
}

int msf2_group_norm_act(const void* x, int64_t x_batch, int64_t x_row, const float* gamma, const float* beta,
                        const int32_t* lengths, void* y, int64_t y_batch, int64_t y_row, float* stats, int B, int S, int C,
                        int groups, float eps, int act, int act_first, int type, void* ws, size_t ws_bytes, void* stream) {
    if (!x || !y || !stats || !ws || !norm_ok(B, S, C, groups, type) || !(eps >= 0.f)) return MSF2_ERR_ARG;
    if (ws_bytes < msf2_group_norm_act_ws_bytes(B, S, C, groups, type)) return MSF2_ERR_WORKSPACE;
    return by_type(type, [&](auto t) {
        typedef decltype(t) T;
        return by_act(act, [&](auto a) {
            auto go = [&](auto pre, auto post) {
                return run_group_norm<T, decltype(pre)::value, decltype(post)::value>(
                    {(const T*)x, x_batch, x_row}, gamma, beta, lengths, {(T*)y, y_batch, y_row}, stats, B, S, C, groups, eps, ws, (hipStream_t)stream);
            };
            std::integral_constant<int, MSF2_ACT_NONE> none;
            return act_first ? go(a, none) : go(none, a);
        });
    });
}

size_t msf2_group_norm_act_backward_ws_bytes(int B, int S, int C, int groups, int type) {
    return norm_ok(B, S, C, groups, type) ? gn_ws_bytes(B, S, C, groups, type_bytes(type), true) : 0;
}

int msf2_group_norm_act_backward(const void* dy, int64_t dy_batch, int64_t dy_row, const void* x, int64_t x_batch,
                                 int64_t x_row, const float* gamma, const float* beta, const float* stats,
                                 const int32_t* lengths, void* dx, int64_t dx_batch, int64_t dx_row, float* dgamma,
                                 float* dbeta, int B, int S, int C, int groups, int act, int act_first, int type, void* ws,
                                 size_t ws_bytes, void* stream) {
    if (!dy || !x || !stats || !dx || !ws || !norm_ok(B, S, C, groups, type)) return MSF2_ERR_ARG;
    if (ws_bytes < msf2_group_norm_act_backward_ws_bytes(B, S, C, groups, type)) return MSF2_ERR_WORKSPACE;
    return by_type(type, [&](auto t) {
        typedef decltype(t) T;
        return by_act(act, [&](auto a) {
            auto go = [&](auto pre, auto post) {
                return run_group_norm_backward<T, decltype(pre)::value, decltype(post)::value>(
                    {(const T*)dy, dy_batch, dy_row}, {(const T*)x, x_batch, x_row}, gamma, beta, stats, lengths, {(T*)dx, dx_batch, dx_row}, dgamma,
                    dbeta, B, S, C, groups, ws, (hipStream_t)stream);
            };
            std::integral_constant<int, MSF2_ACT_NONE> none;
            return act_first ? go(a, none) : go(none, a);
        });
    });
}

size_t msf2_gated_recurrence_ws_bytes(int B, int S, int C, int type) {
    return sizes_ok(B, S, C) && type_ok(type) ? rec_ws_bytes(B, S, C, type_bytes(type), false) : 0;
}

int msf2_gated_recurrence(const void* x, int64_t x_batch, int64_t x_row, const void* gate, int64_t gate_batch,
                          int64_t gate_row, const float* h0, const int32_t* lengths, void* h, int64_t h_batch,
                          int64_t h_row, float* last, float* saved, int B, int S, int C, int reverse, int type, void* ws,
                          size_t ws_bytes, void* stream) {
    if (!x || !gate || !h || !sizes_ok(B, S, C)) return MSF2_ERR_ARG;
    const size_t need = msf2_gated_recurrence_ws_bytes(B, S, C, type);
    if (need && (!ws || ws_bytes < need)) return MSF2_ERR_WORKSPACE;
    return by_type(type, [&](auto t) {
        typedef decltype(t) T;
        return run_recurrence<T>({(const T*)x, x_batch, x_row}, {(const T*)gate, gate_batch, gate_row}, h0, lengths, {(T*)h, h_batch, h_row},
                                 last, saved, B, S, C, reverse != 0, ws, (hipStream_t)stream);
    });
}

size_t msf2_gated_recurrence_backward_ws_bytes(int B, int S, int C, int type) {
    return sizes_ok(B, S, C) && type_ok(type) ? rec_ws_bytes(B, S, C, type_bytes(type), true) : 0;
}

int msf2_gated_recurrence_backward(const void* dh, int64_t dh_batch, int64_t dh_row, const void* x, int64_t x_batch,
                                   int64_t x_row, const void* gate, int64_t gate_batch, int64_t gate_row,
                                   const float* saved, const float* dlast, const int32_t* lengths, void* dx,
                                   int64_t dx_batch, int64_t dx_row, void* dgate, int64_t dgate_batch, int64_t dgate_row,
                                   float* dh0, int B, int S, int C, int reverse, int type, void* ws, size_t ws_bytes,
                                   void* stream) {
    if (!dh || !x || !gate || !saved || !dx || !dgate || !sizes_ok(B, S, C)) return MSF2_ERR_ARG;
    const size_t need = msf2_gated_recurrence_backward_ws_bytes(B, S, C, type);
    if (need && (!ws || ws_bytes < need)) return MSF2_ERR_WORKSPACE;
    return by_type(type, [&](auto t) {
        typedef decltype(t) T;
        return run_recurrence_backward<T>({(const T*)dh, dh_batch, dh_row}, {(const T*)x, x_batch, x_row}, {(const T*)gate, gate_batch, gate_row},
                                          saved, dlast, lengths, {(T*)dx, dx_batch, dx_row}, {(T*)dgate, dgate_batch, dgate_row}, dh0, B, S, C,
                                          reverse != 0, ws, (hipStream_t)stream);
    });
}

int msf2_dropout(const void* x, int64_t x_batch, int64_t x_row, const void* residual, int64_t r_batch, int64_t r_row, void* y,
                 int64_t y_batch, int64_t y_row, const int64_t* rng, uint32_t site, double p, int B, int S, int C,
                 int x_type, int y_type, void* stream) {
    if (!x || !y || !rng || !sizes_ok(B, S, C) || !(p >= 0. && p <= 1.)) return MSF2_ERR_ARG;
    if (x_type != y_type && x_type != MSF2_TYPE_FP32 && y_type != MSF2_TYPE_FP32) return MSF2_ERR_ARG;
    const unsigned thr = (unsigned)std::floor(p * 65536. + 0.5);
    const float scale = thr < 65536u ? (float)(65536. / (65536. - thr)) : 0.f;
    return by_type(x_type, [&](auto tx) {
        return by_type(y_type, [&](auto ty) {
            typedef decltype(tx) TX;
            typedef decltype(ty) TY;
            if constexpr (std::is_same<TX, TY>::value || std::is_same<TX, float>::value || std::is_same<TY, float>::value) {
                return run_dropout<TX, TY>({(const TX*)x, x_batch, x_row}, {(const TY*)residual, r_batch, r_row}, {(TY*)y, y_batch, y_row}, rng, site,
                                           thr, scale, B, S, C, (hipStream_t)stream);
            }
            return MSF2_ERR_ARG;
        });
    });
}

}  // extern "C"
