// Few fp16 tokens through a linear of 4-bit weights with a scale, and in the
// asymmetric form a zero point, for each group of input columns:
//   out[m, n] = sum_g s[n, g] sum_{k in g} x[m, k] (c[n, k] - z[n, g]) (+ bias)
// The weights' bytes bound it, and next to them the number of cache accesses.
// Weights go straight from HBM into registers, a wave taking 16 NT output rows by
// 128 columns at a time with R such blocks in flight; four neighbouring lanes read
// 64 bytes of one row (one access; in the order of the matrix operand, where
// neighbouring lanes are different rows, each lane's 16 bytes are an access of
// their own: M = 16, 8192 x 28672 took 70 us so, 38 now), and four lane permutes
// bring a dword of each row to its place.  x passes through a wave's own piece of
// LDS for the same reason, and scales through it 32 groups at a time.
// Codes become exact fp16 integers c - z in two operations a pair (a mask that also
// inserts an exponent, and an addition).  The products run on
// v_mfma_f32_16x16x32_f16 with the weights as the second operand: a lane's
// accumulators then all belong to one output row, so its group scale is one
// register, applied in fp32 to the group's sum, and the codes never meet a scale
// in 16 bits.  The waves of a block split K and are joined through LDS.
// M = 16, 8192 x 28672 with zero points, 124 MB: 37.3 us, 3.3 TB/s, bound by its
// instructions (32 us with the weights in cache); M = 1 29 us, 4.2 TB/s; M = 1, 4096 x
// 4096 5 us, a launch and one load round trip.
#include "common.h"

#include <type_traits>

namespace {

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
// 0 4 1 5 2 6 3 7 of their places; zero2 holds -(1024 + zero) twice.  A code is
// masked out where it stands, in the lowest bits of a number from 1024 on or four
// bits higher in one from 64 on, so that one shift serves all eight.
SRQ_DEV v8h codes8(u32 w, v2h zero2) {
    const v2h zero2s = zero2 + (v2h){960, 960};   // -(64 + zero)
    v2h d[4];
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const u32 x = w >> (4 * i);
        d[i] = __builtin_bit_cast(v2h, (x & 0x000F000Fu) | 0x64006400u) + zero2;
        d[i + 1] = __builtin_bit_cast(v2h, (x & 0x00F000F0u) | 0x54005400u) + zero2s;
    }
    return (v8h){d[0][0], d[0][1], d[1][0], d[1][1], d[2][0], d[2][1], d[3][0], d[3][1]};
}

// 8 consecutive values of x in the order of codes8
SRQ_DEV v8h ordered(const v8h &x) {
    return (v8h){x[0], x[4], x[1], x[5], x[2], x[6], x[3], x[7]};
}

// The 4 x 4 dwords of lanes l, l + 16, l + 32, l + 48 transposed: dword s of lane
// group g <-> dword g of lane group s.
SRQ_DEV v4i transpose_groups(v4i w) {
    const auto a = __builtin_amdgcn_permlane32_swap((u32)w[0], (u32)w[2], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap((u32)w[1], (u32)w[3], false, false);
    const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    return (v4i){(int)c[0], (int)c[1], (int)d[0], (int)d[1]};
}

// Groups of whole 128-column blocks (kWide: step s of lane group g takes columns
// 128 b + 32 g + 8 s .. + 7, four products are summed before the scale), of 64 or 32
// columns in rows of whole blocks, or any multiple of 32 (columns 128 b + 32 s + 8 g
// after a transposition across the lane groups, so that a product lies in one
// group; the scale is applied to each, or to each two).
enum { kWide, k64, k32, kAny };

constexpr int W = 8;           // waves of a block
constexpr int R = 2;           // blocks of 128 columns that a wave has in flight
constexpr int kUnit = 4;       // blocks in a turn of the loop
static_assert(R == 2 && kUnit % R == 0, "a turn refills its blocks in pairs");
constexpr int kXS = 128 + 8;   // stride of x rows in LDS (halves)
constexpr int kGroups = 32;    // scales of a row that a wave has in LDS at a time

SRQ_DEV u32 lane_move(int from4, u32 v) {
    return (u32)__builtin_amdgcn_ds_bpermute(from4, (int)v);
}

// Between the lanes of a wave: what one wrote to LDS, another reads.
SRQ_DEV void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// XI: x rows in fours (1 for M <= 4)
template <int NT, int XI>
struct Slot {
    v4i w[NT];
    v8h x[XI];
};

// A wave's own LDS.
template <int NT, int XI>
struct Own {
    f16 x[4 * XI * kXS];                  // a block's x rows
    u32 s[NT][16][kGroups + 1];           // scale in the low half, zero point above
};

template <int FORM, bool ASYM, int NT, int XI>
__global__ __launch_bounds__(W * 64) void w4a16_kernel(W4Args a) {
    constexpr int G = FORM == kWide ? 1 : FORM == k64 ? 2 : 4;   // scales of a block
    constexpr int SB = kGroups / G;                              // blocks that LDS has scales for
    union Lds {
        Own<NT, XI> own[W];
        float part[W][16][16 * NT + 1];
    };
    __shared__ __align__(16) Lds lds;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;      // place in the matrix operands
    const int row4 = lane >> 2, part4 = lane & 3;  // place in the weights' loads
    const int from = 4 * (4 * col + g);            // the lane that loaded what belongs here
    const int64_t n0 = (int64_t)blockIdx.x * 16 * NT, m0 = (int64_t)blockIdx.y * 16;
    Own<NT, XI> &own = lds.own[wave];
    const uint8_t *wr[NT];
    int64_t sr[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int64_t n = n0 + 16 * t + row4, nn = n < a.N ? n : a.N - 1;
        wr[t] = a.w + nn * (a.K / 2);
        sr[t] = nn * a.groups;
    }
    const f16 *xr[XI];
#pragma unroll
    for (int i = 0; i < XI; ++i) {
        const int64_t m = m0 + 4 * i + g;
        xr[i] = a.x + (m < a.M ? m : a.M - 1) * a.K;
    }
    // an even number of blocks a wave: rows are read in whole lines of 128 bytes
    const int blocks = (int)srq_cdiv(a.K, 128), per = (blocks + 2 * W - 1) / (2 * W) * 2;
    const int b_lo = wave * per, b_hi = min(blocks, b_lo + per);

    auto load = [&](Slot<NT, XI> &q, int b) __attribute__((always_inline)) {
        const int64_t kw = (int64_t)b * 128 + 32 * part4, kx = (int64_t)b * 128 + 8 * col;
        const bool okw = FORM != kAny || kw < a.K, okx = FORM != kAny || kx < a.K;
#pragma unroll
        for (int t = 0; t < NT; ++t)
            q.w[t] = *reinterpret_cast<const v4i *>(wr[t] + (okw ? kw / 2 : 0));
#pragma unroll
        for (int i = 0; i < XI; ++i) {
            q.x[i] = *reinterpret_cast<const v8h *>(xr[i] + (okx ? kx : 0));
            if (!okx) q.x[i] = (v8h)(f16)0;
        }
    };
    // the scales of SB blocks from b on: a lane takes every fourth group of a row
    struct Fetched {
        f16 s[NT][kGroups / 4];
        uint8_t z[NT][kGroups / 4];
    };
    auto fetch_scales = [&](Fetched &q, int b) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kGroups / 4; ++i) {
            if (4 * i >= (b_hi - b) * G) break;
            const uint32_t j = part4 + 4 * i;
            uint32_t gi;
            if constexpr (FORM == kWide) gi = (b + j) * 128u / (uint32_t)a.group;
            else if constexpr (FORM == kAny) gi = (4u * b + j) * 32u / (uint32_t)a.group;
            else gi = (uint32_t)G * b + j;
            gi = min(gi, (uint32_t)a.groups - 1);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                q.s[t][i] = a.s[sr[t] + gi];
                if constexpr (ASYM) q.z[t][i] = a.z[sr[t] + gi];
            }
        }
    };
    auto keep_scales = [&](const Fetched &q) __attribute__((always_inline)) {
        wave_fence();   // the last blocks' reads are done
#pragma unroll
        for (int i = 0; i < kGroups / 4; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const u32 z = ASYM ? (u32)q.z[t][i] : 8u;
                // -(1024 + z) as fp16 above: 0xE400 + z, exact
                own.s[t][row4][part4 + 4 * i] =
                    (u32)__builtin_bit_cast(uint16_t, q.s[t][i]) | (0xE400u + z) << 16;
            }
        wave_fence();
    };

    v4f acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = (v4f)0.f;
    // block j of those whose scales are in LDS
    auto step = [&](const Slot<NT, XI> &q, int j) __attribute__((always_inline)) {
        // x to its operand's order: written by rows, read by (row, columns)
#pragma unroll
        for (int i = 0; i < XI; ++i)
            *reinterpret_cast<v8h *>(own.x + (4 * i + g) * kXS + 8 * col) = q.x[i];
        wave_fence();
        v8h xv[4];
#pragma unroll
        for (int s = 0; s < 4; ++s)
            xv[s] = ordered(*reinterpret_cast<const v8h *>(
                own.x + (XI == 4 ? col : col & 3) * kXS +
                (FORM == kWide ? 32 * g + 8 * s : 32 * s + 8 * g)));
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            v4i w;
#pragma unroll
            for (int s = 0; s < 4; ++s) w[s] = (int)lane_move(from, (u32)q.w[t][s]);
            if constexpr (FORM != kWide) w = transpose_groups(w);
            v4f p = (v4f)0.f;
            u32 pair = 0;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                if (s * G % 4 == 0) pair = own.s[t][col][G * j + s * G / 4];
                const u32 zz = __builtin_amdgcn_perm(0u, pair, 0x03020302u);   // its zero twice
                const u32 c = ASYM ? (u32)w[s] : (u32)w[s] ^ 0x88888888u;      // signed: code + 8
                p = mfma16(xv[s], codes8(c, __builtin_bit_cast(v2h, zz)), p);
                if ((s + 1) * G % 4 == 0) {
                    const float k = (float)__builtin_bit_cast(f16, (uint16_t)pair);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[t][e] = __builtin_fmaf(p[e], k, acc[t][e]);
                    p = (v4f)0.f;
                }
            }
        }
        wave_fence();
    };

    if (b_lo < b_hi) {
        // R blocks in flight; behind the last one the last is read again, so that
        // no load stands under a condition (a wait behind one is for all loads)
        Slot<NT, XI> q[R];
        {
            Fetched f;
            fetch_scales(f, b_lo);
#pragma unroll
            for (int r = 0; r < R; ++r) load(q[r], min(b_lo + r, b_hi - 1));
            keep_scales(f);
        }
        int base = b_lo;   // the first block that LDS has scales for
        auto turn = [&](auto place, int b) __attribute__((always_inline)) {
            constexpr int u = decltype(place)::value;
            step(q[u % R], b + u - base);
            if (b + u + 1 >= b_hi) return true;
            // with many x rows in pairs (M = 16, 8192 x 28672 38.2 us against 38.9),
            // else at once (M = 1 29.5 against 30.8)
            if constexpr (XI == 1) {
                load(q[u % R], min(b + u + R, b_hi - 1));
            } else if constexpr (u % 2 == 1) {
                load(q[(u - 1) % R], min(b + u - 1 + R, b_hi - 1));
                load(q[u % R], min(b + u + R, b_hi - 1));
            }
            return false;
        };
        for (int b = b_lo;; b += kUnit) {
            if (b - base == SB) {
                base = b;
                Fetched f;
                fetch_scales(f, b);
                keep_scales(f);
            }
            if (turn(std::integral_constant<int, 0>(), b) ||
                turn(std::integral_constant<int, 1>(), b) ||
                turn(std::integral_constant<int, 2>(), b) ||
                turn(std::integral_constant<int, 3>(), b))
                break;
        }
    }
    __syncthreads();   // the waves' own parts of LDS are free
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) lds.part[wave][4 * g + e][16 * t + col] = acc[t][e];
    __syncthreads();
    for (int i = threadIdx.x; i < 256 * NT; i += W * 64) {
        const int om = i / (16 * NT), on = i % (16 * NT);
        const int64_t row = m0 + om, c = n0 + on;
        if (row >= a.M || c >= a.N) continue;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) sum += lds.part[w][om][on];
        if (a.bias) sum += (float)a.bias[c];
        a.out[row * a.N + c] = (f16)sum;
    }
}

template <int FORM, int NT, int XI>
void launch(const W4Args &a, hipStream_t st) {
    const dim3 grid((unsigned)srq_cdiv(a.N, 16 * NT), (unsigned)srq_cdiv(a.M, 16));
    if (a.z)
        w4a16_kernel<FORM, true, NT, XI><<<grid, W * 64, 0, st>>>(a);
    else
        w4a16_kernel<FORM, false, NT, XI><<<grid, W * 64, 0, st>>>(a);
}

template <int NT, int XI>
void launch(int form, const W4Args &a, hipStream_t st) {
    switch (form) {
    case kWide: return launch<kWide, NT, XI>(a, st);
    case k64: return launch<k64, NT, XI>(a, st);
    case k32: return launch<k32, NT, XI>(a, st);
    default: return launch<kAny, NT, XI>(a, st);
    }
}

}  // namespace

extern "C" int srq_w4a16_linear(const void *x, const void *w, const void *scales,
                                const void *zeros, const void *bias, int64_t M, int64_t N,
                                int64_t K, int64_t group, void *out, void *stream) {
    SRQ_CHECK_ARG(M >= 0 && N >= 0 && K >= 0, "w4a16_linear: negative size");
    SRQ_CHECK_ARG(group > 0 && group % 32 == 0 && K % group == 0,
                  "w4a16_linear: group=%lld must be a multiple of 32 that divides K=%lld",
                  (long long)group, (long long)K);
    SRQ_CHECK_ARG(K <= 1 << 24 && N <= 1 << 26 && M <= 16 * 65535,
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
    hipStream_t st = (hipStream_t)stream;
    const int form = group % 128 == 0 ? kWide : K % 128 ? kAny : group == 64 ? k64
                                                             : group == 32 ? k32 : kAny;
    // Two row tiles a wave, which halves what x costs, where that still gives a block
    // per CU (256).  us on one MI355X, one / two tiles: M = 16, 8192 x 28672 49.7 /
    // 37.7 (weights alone stream in 22, x adds 10: 235 MB from L2), M = 1 31.4 /
    // 30.7, M = 8, 8192 x 8192 12.5 / 11.9, M = 1, 28672 x 4096 16.5 / 16.5; 4096 x
    // 14336 10.7 / 15.7, M = 16, 4096 x 4096 6.1 / 6.8.
    const bool two = N >= 32 * 256;
    // Four x rows are a quarter of the loads and LDS traffic of sixteen: M = 4, 4 rows
    // / 16 rows, 4096 x 14336 11.0 / 13.3, 8192 x 8192 10.4 / 11.8, 8192 x 28672 31 / 35.
    // The forms of whole groups against kAny: M = 16, 8192 x 28672 in groups of 128 37.3
    // / 47.6, of 64 42.9 / 51.0; 8192 x 8192 in groups of 32 14.2 / 15.2.
    if (M <= 4)
        two ? launch<2, 1>(form, a, st) : launch<1, 1>(form, a, st);
    else
        two ? launch<2, 4>(form, a, st) : launch<1, 4>(form, a, st);
    SRQ_LAUNCH_CHECK("w4a16_linear");
    return SRQ_OK;
}
