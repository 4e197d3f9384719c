// Few fp16 tokens through a linear of 4-bit weights with a scale, and in the
// asymmetric form a zero point, for each group of input columns:
//   out[m, n] = sum_g s[n, g] sum_{k in g} x[m, k] (c[n, k] - z[n, g]) (+ bias)
// The weights' bytes bound it: they are read once, straight from HBM into
// registers, 16 output rows by 128 columns a wave at a time (16 bytes a lane),
// and become exact fp16 integers c - z in two operations a pair (a mask that
// also inserts the exponent of 1024, and an addition).  The products run on
// v_mfma_f32_16x16x32_f16 with the weights as the second operand: a lane's
// accumulators then all belong to one output row, so its group scale is one
// register, applied in fp32 to the group's sum.  The waves of a block split
// K and are joined through LDS.
#include "common.h"

namespace {

constexpr int kWavesK = 8;   // waves of a block, each with its part of K

struct W4Args {
    const f16 *x;          // [M, K]
    const uint8_t *w;      // [N, K / 2]
    const f16 *s;          // [N, groups]
    const uint8_t *z;      // [N, groups] or null
    const f16 *bias;       // [N] or null
    f16 *out;              // [M, N]
    int64_t M, N, K;
    int group, groups;
};

SRQ_DEV v4f mfma16(v8h a, v8h b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// 8 codes of a dword (element e in bits 4 e ..) as fp16 c - zero, in the order
// 0 4 1 5 2 6 3 7 of their places; zero2 holds -(1024 + zero) twice
SRQ_DEV v8h codes8(u32 w, v2h zero2) {
    v2h d[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        d[i] = __builtin_bit_cast(v2h, ((w >> (4 * i)) & 0x000F000Fu) | 0x64006400u) + zero2;
    return (v8h){d[0][0], d[0][1], d[1][0], d[1][1], d[2][0], d[2][1], d[3][0], d[3][1]};
}

// 8 consecutive values of x in the order of codes8
SRQ_DEV v8h ordered(const v8h &x) {
    return (v8h){x[0], x[4], x[1], x[5], x[2], x[6], x[3], x[7]};
}

// WIDE: groups are whole multiples of 128 columns, which one 16-byte load a
// lane covers (k = 128 b + 32 g + 8 s + e); otherwise of 32 columns, and step
// s of a 128-column block is columns 128 b + 32 s + 8 g + e.
template <bool WIDE>
__global__ __launch_bounds__(kWavesK * 64) void w4a16_kernel(W4Args a) {
    __shared__ float part[kWavesK][16][17];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 15, g = lane >> 4;
    const int64_t n = (int64_t)blockIdx.x * 16 + col, m = (int64_t)blockIdx.y * 16 + col;
    const int64_t nn = n < a.N ? n : a.N - 1, mm = m < a.M ? m : a.M - 1;
    const uint8_t *wr = a.w + nn * (a.K / 2);
    const f16 *xr = a.x + mm * a.K;
    const f16 *sr = a.s + nn * a.groups;
    const uint8_t *zr = a.z ? a.z + nn * a.groups : nullptr;
    const u32 flip = a.z ? 0u : 0x88888888u;   // two's complement -> code + 8
    const int blocks = (int)srq_cdiv(a.K, 128);
    v4f acc = (v4f)0.f;
    for (int b = wave; b < blocks; b += kWavesK) {
        if constexpr (WIDE) {
            const int64_t k0 = (int64_t)b * 128 + 32 * g;
            const v4i w = *reinterpret_cast<const v4i *>(wr + k0 / 2);
            const int gi = (int)((uint32_t)b * 128u / (uint32_t)a.group);
            const float sc = (float)sr[gi];
            const f16 zf = (f16)(-(float)(1024 + (zr ? zr[gi] : 8)));
            const v2h zz = {zf, zf};
            v4f t = (v4f)0.f;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const v8h xv = *reinterpret_cast<const v8h *>(xr + k0 + 8 * s);
                t = mfma16(ordered(xv), codes8((u32)w[s] ^ flip, zz), t);
            }
            acc += t * sc;
        } else {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int64_t kb = (int64_t)b * 128 + 32 * s;
                if (kb < a.K) {
                    const int64_t k0 = kb + 8 * g;
                    const u32 w = *reinterpret_cast<const u32 *>(wr + k0 / 2);
                    const int gi = (int)((uint32_t)kb / (uint32_t)a.group);
                    const float sc = (float)sr[gi];
                    const f16 zf = (f16)(-(float)(1024 + (zr ? zr[gi] : 8)));
                    const v8h xv = *reinterpret_cast<const v8h *>(xr + k0);
                    acc += mfma16(ordered(xv), codes8(w ^ flip, (v2h){zf, zf}), (v4f)0.f) * sc;
                }
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) part[wave][4 * g + e][col] = acc[e];
    __syncthreads();
    const int om = threadIdx.x >> 4, on = threadIdx.x & 15;
    if (om >= 16) return;
    const int64_t row = (int64_t)blockIdx.y * 16 + om, c = (int64_t)blockIdx.x * 16 + on;
    if (row >= a.M || c >= a.N) return;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWavesK; ++w) sum += part[w][om][on];
    if (a.bias) sum += (float)a.bias[c];
    a.out[row * a.N + c] = (f16)sum;
}

}  // namespace

extern "C" int srq_w4a16_linear(const void *x, const void *w, const void *scales,
                                const void *zeros, const void *bias, int64_t M, int64_t N,
                                int64_t K, int64_t group, void *out, void *stream) {
    SRQ_CHECK_ARG(M >= 0 && N >= 0 && K >= 0, "w4a16_linear: negative size");
    SRQ_CHECK_ARG(group > 0 && group % 32 == 0 && K % group == 0,
                  "w4a16_linear: group=%lld must be a multiple of 32 that divides K=%lld",
                  (long long)group, (long long)K);
    SRQ_CHECK_ARG(K <= 1 << 24 && N <= 1 << 28 && M <= 16 * 65535,
                  "w4a16_linear: shape out of range");
    if (M == 0 || N == 0) return SRQ_OK;
    SRQ_CHECK_ARG(out && (K == 0 || (x && w && scales)), "w4a16_linear: null pointer");
    SRQ_CHECK_ARG(srq_aligned(x, 16) && srq_aligned(w, 16),
                  "w4a16_linear: x and the weights must be 16-byte aligned");
    W4Args a;
    a.x = (const f16 *)x;
    a.w = (const uint8_t *)w;
    a.s = (const f16 *)scales;
    a.z = (const uint8_t *)zeros;
    a.bias = (const f16 *)bias;
    a.out = (f16 *)out;
    a.M = M;
    a.N = N;
    a.K = K;
    a.group = (int)group;
    a.groups = (int)(K / group);
    const dim3 grid((unsigned)srq_cdiv(N, 16), (unsigned)srq_cdiv(M, 16));
    hipStream_t st = (hipStream_t)stream;
    if (group % 128 == 0)
        w4a16_kernel<true><<<grid, kWavesK * 64, 0, st>>>(a);
    else
        w4a16_kernel<false><<<grid, kWavesK * 64, 0, st>>>(a);
    SRQ_LAUNCH_CHECK("w4a16_linear");
    return SRQ_OK;
}
