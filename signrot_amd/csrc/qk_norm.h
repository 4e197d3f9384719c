// One head row of q or k through RMSNorm and the rotary embedding, in fp32
// from the fp16 input to one rounding at the end; shared by qk_norm_rope and
// the pass that also writes the int8 cache, so both give the same bits.
//
// A row of D = 8 G values is held by G consecutive lanes of a wave (8 values
// a lane, 16-byte accesses): the sum of squares is a reduction over those
// lanes, and rotate_half's partner of value i, i +- D / 2, is the same slot of
// lane l ^ (G / 2), so nothing goes through LDS.
#pragma once

#include "common.h"

template <int CTRL>
SRQ_DEV float qk_dpp(float x) {
    return __builtin_bit_cast(
        float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, true));
}

// The value of lane l ^ M: inside a row of 16 lanes by DPP moves, which cost
// one vector instruction, beyond it by a cross-lane read.
template <int M>
SRQ_DEV float qk_xor(float v) {
    if constexpr (M == 1) return qk_dpp<0xB1>(v);             // quad_perm [1, 0, 3, 2]
    else if constexpr (M == 2) return qk_dpp<0x4E>(v);        // quad_perm [2, 3, 0, 1]
    else if constexpr (M == 4) return qk_dpp<0x1B>(qk_dpp<0x141>(v));  // l ^ 7, then l ^ 3
    else if constexpr (M == 8) return qk_dpp<0x128>(v);       // row_ror:8
    else return __shfl_xor(v, M, 64);
}

template <int G, int M = 1>
SRQ_DEV float qk_row_sum(float v) {
    if constexpr (M < G) return qk_row_sum<G, 2 * M>(v + qk_xor<M>(v));
    else return v;
}

// x: this lane's 8 values; w: its weights (ones when there are none); c, s: its
// slice of the cos and sin rows; l: lane within the row.
// y = x / sqrt(mean(x^2) + eps) * w (x itself when norm is 0), then
// y * cos + rotate_half(y) * sin.  Every lane of the wave calls it.
template <int G>
SRQ_DEV v8h qk_norm_rope_row(const v8h &x, const v8h &w, const v8h &c, const v8h &s, int l,
                             float eps, int norm) {
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (float)x[e];
    if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(y[e], y[e], ss);
        ss = qk_row_sum<G>(ss);
        const float inv = 1.0f / __builtin_sqrtf(ss * (1.0f / (8 * G)) + eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = y[e] * inv * (float)w[e];
    }
    v8h o;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float p = qk_xor<G / 2>(y[e]);
        const float sn = l < G / 2 ? -(float)s[e] : (float)s[e];
        o[e] = (f16)__builtin_fmaf(p, sn, y[e] * (float)c[e]);
    }
    return o;
}
