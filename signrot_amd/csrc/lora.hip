// Low-rank adapters of many requests beside a projection that they share:
//   out[m] = fp16(y[m] + scaling[i] * (x[m] A_i^T) B_i^T),  i = ids[m]
// x, y, A, B fp16; A [L, S r, K], B [L, N, r]: a projection that is S in one (q/k/v) has
// r rows of A for each of its column slices, whose columns meet only those.  Tokens
// whose id lies outside [0, L) have no adapter: out = y.  Sums are fp32 throughout.
// Two launches: t = x A^T (fp32, in the workspace), then out = y + t B^T.  The adapters'
// bytes bound few tokens, those of x, y and out many.
//
// Few tokens: each by itself.  A wave takes one row of A for one token, whole lines at a
// time; then a thread takes one output column, whose row of B is r values, with t in
// fp32 from LDS.
//
// Many tokens: tiles of 64 consecutive ones, whose distinct adapters are found by ballots
// (lane i holds the id of token i) and taken one after the other, or shared out among the
// blocks in z; a request's tokens stand together, so a tile has one or two.  Rows of other
// adapters are computed and not kept: never multiplied by zero, since another request's
// infinities would then come through.  t is split over K where tiles are few, each part
// stored for itself, and added in order.  In the second product t is an fp16 number and
// the fp16 rest, scaled by a power of two of the token's largest: 22 bits.
#include "common.h"

namespace {

constexpr int kMaxSlices = 8;
constexpr int kMaxRank = 256;
constexpr uint32_t kOob = 0xFFFFFFF0u;

struct LoraArgs {
    const f16 *y, *x, *a, *b;
    const int32_t *ids;
    const float *scaling;    // [L] or null
    f16 *out;
    float *t;                // [splits, M, R]
    int64_t M, N, K;
    int64_t ys, xs, os;      // row strides
    int L, r, R;             // R = slices * r
    int slices, splits;
    int kc;                  // columns of K in a split (a multiple of 64)
    int col_end[kMaxSlices];    // of each slice
    int tile_end[kMaxSlices];   // its column tiles (second product of many tokens)
};

SRQ_DEV int adapter_of(const LoraArgs &a, int64_t m) {
    const int id = a.ids[m];
    return id >= 0 && id < a.L ? id : -1;
}

// ------------------------------------------------------------- few tokens

__global__ __launch_bounds__(256) void lora_shrink_few_kernel(LoraArgs a) {
    const int lane = threadIdx.x & 63;
    const int j = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int64_t m = blockIdx.y;
    const int id = __builtin_amdgcn_readfirstlane(adapter_of(a, m));
    if (j >= a.R || id < 0) return;
    const f16 *x = a.x + m * a.xs, *w = a.a + ((int64_t)id * a.R + j) * a.K;
    float acc[8] = {};
    auto add = [&](const v8h &p, const v8h &q) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = __builtin_fmaf((float)p[i], (float)q[i], acc[i]);
    };
    int64_t k = 8 * lane;
    constexpr int U = 4;
    for (; k + 512 * (U - 1) < a.K; k += 512 * U) {
        v8h p[U], q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            p[u] = *reinterpret_cast<const v8h *>(x + k + 512 * u);
            q[u] = *reinterpret_cast<const v8h *>(w + k + 512 * u);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) add(p[u], q[u]);
    }
    for (; k < a.K; k += 512)
        add(*reinterpret_cast<const v8h *>(x + k), *reinterpret_cast<const v8h *>(w + k));
    const float s = wave_sum(((acc[0] + acc[1]) + (acc[2] + acc[3])) +
                             ((acc[4] + acc[5]) + (acc[6] + acc[7])));
    if (lane == 0) a.t[m * a.R + j] = s;
}

__global__ __launch_bounds__(256) void lora_expand_few_kernel(LoraArgs a) {
    __shared__ float t[kMaxSlices * kMaxRank];
    const int64_t m = blockIdx.y;
    const int id = __builtin_amdgcn_readfirstlane(adapter_of(a, m));
    const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id < 0) {
        if (n < a.N && a.out != a.y) a.out[m * a.os + n] = a.y[m * a.ys + n];
        return;
    }
    const float f = a.scaling ? a.scaling[id] : 1.f;
    for (int i = threadIdx.x; i < a.R; i += 256) t[i] = a.t[m * a.R + i];
    __syncthreads();
    if (n >= a.N) return;
    int s = 0;
    while (n >= a.col_end[s]) ++s;   // col_end of the last slice is N
    const f16 *b = a.b + ((int64_t)id * a.N + n) * a.r;
    const float *ts = t + s * a.r;
    float acc = 0.f;
    for (int k = 0; k < a.r; k += 8) {
        const v8h v = *reinterpret_cast<const v8h *>(b + k);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc = __builtin_fmaf((float)v[i], ts[k + i], acc);
    }
    a.out[m * a.os + n] = f16_rn(__builtin_fmaf(acc, f, (float)a.y[m * a.ys + n]));
}

// ------------------------------------------------------------ many tokens

constexpr int kTok = 64;   // tokens of a tile: one a lane

// The distinct adapters of a tile, one at a time: those with j % nz == z are this block's.
struct Turns {
    uint64_t left, invalid;
    int id, j;
    SRQ_DEV Turns(const LoraArgs &a, int64_t m0, int lane) : j(0) {
        const int64_t m = m0 + lane;
        id = m < a.M ? adapter_of(a, m) : -1;
        left = __ballot(id >= 0);
        invalid = __ballot(m < a.M && id < 0);
    }
    // the next adapter of this block and the mask of its tokens, or -1
    SRQ_DEV int next(int z, int nz, uint64_t &same) {
        while (left) {
            const int first = __builtin_ctzll(left);
            const int cur = __builtin_amdgcn_readlane(id, first);
            same = __ballot(id == cur);
            left &= ~same;
            if (j++ % nz == z) return cur;
        }
        return -1;
    }
};

SRQ_DEV v4f mfma16(v8h a, v8h b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

SRQ_DEV v16f mfma32(v8h a, v8h b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// t of 64 tokens x 16 RT rows of A: four waves of 16 tokens, K in steps of 64 through a
// ring of four LDS stages (64 rows of x, 16 RT of A, 128 bytes each, the 16-byte chunks
// of a row exchanged by its number).
constexpr int kStages = 4;

template <int RT>
__global__ __launch_bounds__(256) void lora_shrink_kernel(LoraArgs a, int groups, int nz) {
    constexpr int kStage = (kTok + 16 * RT) * 128;
    constexpr int PER = 2 + RT / 2;   // loads of a wave in a stage
    static_assert(RT % 2 == 0 && 3 * PER < 64, "loads");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[kStages * kStage];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int64_t m0 = (int64_t)blockIdx.x * kTok;
    const int rg = (blockIdx.y % groups) * 16 * RT, split = blockIdx.y / groups;
    const int z = blockIdx.z;
    const int64_t k_lo = (int64_t)split * a.kc, k_hi = min(a.K, k_lo + a.kc);
    const int steps = (int)((k_hi - k_lo + 63) / 64);
    const int64_t rows = min((int64_t)kTok, a.M - m0);
    const uint32_t xbytes = (uint32_t)__builtin_amdgcn_readfirstlane(
        (int)(uint32_t)(2 * ((rows - 1) * a.xs + a.K)));
    const __amdgpu_buffer_rsrc_t xr = make_rsrc(a.x + m0 * a.xs, xbytes);
    const int arows = min(16 * RT, a.R - rg);
    const uint32_t ring0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)smem;
    const int r8 = lane >> 3, m = lane & 15, g = lane >> 4;
    const int ck = 8 * ((lane & 7) ^ r8);   // column of this lane's chunk in a step

    Turns turns(a, m0, lane);
    uint64_t same;
    for (int id; (id = turns.next(z, nz, same)) >= 0;) {
        const __amdgpu_buffer_rsrc_t wr =
            make_rsrc(a.a + ((int64_t)id * a.R + rg) * a.K, (int64_t)arows * a.K * 2);
        auto issue = [&](int s) __attribute__((always_inline)) {
            const uint32_t dst = ring0 + (s % kStages) * kStage;
            const int64_t k = k_lo + 64 * (int64_t)s + ck;
            // past K, and rows past the tile's last: zeros, on both sides
            const bool in = k < a.K;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int i = 2 * wave + q, row = 8 * i + r8;
                const uint32_t off = (uint32_t)(2 * (row * a.xs + k));
                dma16(xr, in && row < rows ? off : kOob, dst + i * 1024);
            }
#pragma unroll
            for (int q = 0; q < RT / 2; ++q) {
                const int i = (RT / 2) * wave + q, row = 8 * i + r8;
                const uint32_t off = (uint32_t)(2 * (row * a.K + k));
                dma16(wr, in && row < arows ? off : kOob, dst + kTok * 128 + i * 1024);
            }
        };
        v4f acc[RT];
#pragma unroll
        for (int f = 0; f < RT; ++f) acc[f] = (v4f)0.f;
#pragma unroll
        for (int p = 0; p < kStages - 1; ++p)
            if (p < steps) issue(p);
        for (int s = 0; s < steps; ++s) {
            const int ahead = min(kStages - 2, steps - 1 - s);
            if (ahead == 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * PER) : "memory");
            else if (ahead == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PER) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (s + kStages - 1 < steps) issue(s + kStages - 1);
            const uint8_t *xs = smem + (s % kStages) * kStage, *ws = xs + kTok * 128;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = 16 * ((4 * h + g) ^ (m & 7));
                const v8h xv = *reinterpret_cast<const v8h *>(xs + (16 * wave + m) * 128 + at);
#pragma unroll
                for (int f = 0; f < RT; ++f)
                    acc[f] = mfma16(xv, *reinterpret_cast<const v8h *>(ws + (16 * f + m) * 128 + at),
                                    acc[f]);
            }
        }
        // the ring is filled anew for the next adapter
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int row = 16 * wave + 4 * g + e;
            if (!(same >> row & 1)) continue;
            float *t = a.t + ((int64_t)split * a.M + m0 + row) * a.R + rg;
#pragma unroll
            for (int f = 0; f < RT; ++f)
                if (16 * f + m < arows) t[16 * f + m] = acc[f][e];
        }
    }
}

// out of 64 tokens x 128 columns of one slice: four waves of 32 x 64.
constexpr int kCols = 128;

__global__ __launch_bounds__(256) void lora_expand_kernel(LoraArgs a, int tiles_n, int nz) {
    // t as fp16 number and rest, rows of r values (zeros up to whole 16) and 8 to spare the banks
    __shared__ __attribute__((aligned(16))) f16 th[kTok * (kMaxRank + 8)];
    __shared__ __attribute__((aligned(16))) f16 tl[kTok * (kMaxRank + 8)];
    __shared__ float unit[kTok];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1, rr = lane & 31, g = lane >> 5;
    const int tile = blockIdx.x % tiles_n, z = blockIdx.y;
    const int64_t m0 = (int64_t)(blockIdx.x / tiles_n) * kTok;
    int s = 0;
    while (tile >= a.tile_end[s]) ++s;
    const int64_t n_lo = s ? a.col_end[s - 1] : 0, n_hi = a.col_end[s];
    const int64_t n0 = n_lo + (int64_t)(tile - (s ? a.tile_end[s - 1] : 0)) * kCols + 64 * wn;
    const int rp = (a.r + 15) & ~15, stride = rp + 8;

    Turns turns(a, m0, lane);
    // the rows that this block writes, and what is added to them
    uint64_t done = z == 0 && a.out != a.y ? turns.invalid : 0;
    v16f total[2] = {(v16f)0.f, (v16f)0.f};
    uint64_t same;
    for (int id; (id = turns.next(z, nz, same)) >= 0;) {
        done |= same;
        __syncthreads();   // the last adapter's reads of LDS are over
        {
            // four threads a token, each every fourth pair of values
            const int row = threadIdx.x >> 2, part = threadIdx.x & 3;
            const bool mine = same >> row & 1;
            const float *t = a.t + (m0 + row) * a.R + s * a.r;
            float top = 0.f;
            for (int k = 2 * part; k < rp; k += 8) {
                float v0 = 0.f, v1 = 0.f;
                if (mine && k < a.r)
                    for (int p = 0; p < a.splits; ++p) {
                        const float *q = t + (int64_t)p * a.M * a.R + k;
                        v0 += q[0];
                        v1 += q[1];
                    }
                top = fmaxf(top, fmaxf(fabsf(v0), fabsf(v1)));
                // kept as they are for the moment: hi and lo halves of the fp32 bits
                const u32 b0 = __builtin_bit_cast(u32, v0), b1 = __builtin_bit_cast(u32, v1);
                th[row * stride + k] = __builtin_bit_cast(f16, (uint16_t)(b0 >> 16));
                tl[row * stride + k] = __builtin_bit_cast(f16, (uint16_t)b0);
                th[row * stride + k + 1] = __builtin_bit_cast(f16, (uint16_t)(b1 >> 16));
                tl[row * stride + k + 1] = __builtin_bit_cast(f16, (uint16_t)b1);
            }
            top = group_max<4>(top);
            // a power of two that takes the largest to [2^10, 2^11): there the rest of
            // the fp16 number is one too, down to 2^-25 of the largest
            const int e = top > 0.f && top <= 3.4e38f ? 10 - (int)__builtin_amdgcn_frexp_expf(top) + 1
                                                      : 0;
            for (int k = 2 * part; k < rp; k += 8)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    f16 &h = th[row * stride + k + i], &l = tl[row * stride + k + i];
                    const u32 b = (u32)__builtin_bit_cast(uint16_t, h) << 16 |
                                  (u32)__builtin_bit_cast(uint16_t, l);
                    const float v = __builtin_amdgcn_ldexpf(__builtin_bit_cast(float, b), e);
                    h = (f16)v;
                    const float rest = v - (float)h;
                    l = fabsf(v) <= 65504.f ? (f16)rest : (f16)0.f;
                }
            if (part == 0)
                unit[row] = __builtin_amdgcn_ldexpf(a.scaling ? a.scaling[id] : 1.f, -e);
        }
        __syncthreads();
        v16f acc[2] = {(v16f)0.f, (v16f)0.f};
        const f16 *b = a.b + (int64_t)id * a.N * a.r;
        for (int k0 = 0; k0 < rp; k0 += 16) {
            const int k = k0 + 8 * g;
            const int at = (32 * wm + rr) * stride + k;
            const v8h h = *reinterpret_cast<const v8h *>(th + at);
            const v8h l = *reinterpret_cast<const v8h *>(tl + at);
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                const int64_t n = n0 + 32 * f + rr;
                v8h w = (v8h)(f16)0;
                if (n < n_hi && k < a.r) w = *reinterpret_cast<const v8h *>(b + n * a.r + k);
                acc[f] = mfma32(h, w, acc[f]);
                acc[f] = mfma32(l, w, acc[f]);
            }
        }
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            const int row = 32 * wm + 8 * (v / 4) + 4 * g + v % 4;
            const bool mine = same >> row & 1;
            const float u = unit[row];
#pragma unroll
            for (int f = 0; f < 2; ++f) total[f][v] = mine ? acc[f][v] * u : total[f][v];
        }
    }
#pragma unroll
    for (int v = 0; v < 16; ++v) {
        const int row = 32 * wm + 8 * (v / 4) + 4 * g + v % 4;
        if (!(done >> row & 1)) continue;
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            const int64_t n = n0 + 32 * f + rr;
            if (n >= n_hi) continue;
            const float y = (float)a.y[(m0 + row) * a.ys + n];
            a.out[(m0 + row) * a.os + n] = f16_rn(y + total[f][v]);
        }
    }
}

// Tokens up to which each is taken by itself.
constexpr int64_t kFew = 64;

struct Plan {
    int rt, groups, splits, kc;
};

Plan plan_of(int64_t M, int64_t R, int64_t K) {
    Plan p{0, 1, 1, 0};
    if (M <= kFew) return p;
    p.rt = R <= 32 ? 2 : 4;
    p.groups = (int)srq_cdiv(R, 16 * p.rt);
    // enough blocks for the 256 CUs, at least 8 steps each
    const int64_t blocks = srq_cdiv(M, kTok) * p.groups, steps = srq_cdiv(K, 64);
    int64_t s = srq_cdiv(512, blocks);
    if (s > steps / 8) s = steps / 8;
    if (s < 1) s = 1;
    if (s > 8) s = 8;
    const int64_t per = srq_cdiv(steps, s);
    p.kc = (int)(64 * per);
    p.splits = (int)srq_cdiv(steps, per);
    return p;
}

}  // namespace

extern "C" int srq_lora_workspace(int64_t M, int64_t K, int64_t rank, int64_t slices,
                                  int64_t *bytes) {
    SRQ_CHECK_ARG(bytes, "lora_add: null pointer");
    *bytes = 0;
    if (M <= 0 || K <= 0 || rank <= 0 || slices <= 0) return SRQ_OK;
    *bytes = 4 * M * rank * slices * plan_of(M, rank * slices, K).splits;
    return SRQ_OK;
}

extern "C" int srq_lora_add(const void *y, int64_t y_stride, const void *x, int64_t x_stride,
                            const void *lora_a, const void *lora_b, const int32_t *ids,
                            const float *scaling, int64_t M, int64_t K, int64_t adapters,
                            int64_t rank, int64_t slices, const int64_t *slice_cols, void *out,
                            int64_t out_stride, void *ws, int64_t ws_bytes, void *stream) {
    SRQ_CHECK_ARG(M >= 0 && K >= 0 && adapters >= 0, "lora_add: negative size");
    SRQ_CHECK_ARG(rank >= 8 && rank <= kMaxRank && rank % 8 == 0,
                  "lora_add: rank=%lld must be a multiple of 8 up to %d", (long long)rank, kMaxRank);
    SRQ_CHECK_ARG(slices >= 1 && slices <= kMaxSlices && slice_cols,
                  "lora_add: 1 to %d column slices", kMaxSlices);
    SRQ_CHECK_ARG(K > 0 && K % 8 == 0 && K <= 1 << 20,
                  "lora_add: K=%lld must be a multiple of 8 up to 2^20", (long long)K);
    SRQ_CHECK_ARG(M <= (int64_t)1 << 30 && adapters <= (int64_t)1 << 30,
                  "lora_add: shape out of range");
    LoraArgs a{};
    int64_t tiles = 0;
    for (int64_t i = 0; i < slices; ++i) {
        SRQ_CHECK_ARG(slice_cols[i] > 0 && slice_cols[i] <= 1 << 24, "lora_add: slice of %lld columns",
                      (long long)slice_cols[i]);
        a.N += slice_cols[i];
        tiles += srq_cdiv(slice_cols[i], kCols);
        a.col_end[i] = (int)a.N;
        a.tile_end[i] = (int)tiles;
    }
    if (M == 0) return SRQ_OK;
    SRQ_CHECK_ARG(y && x && ids && out && (adapters == 0 || (lora_a && lora_b)),
                  "lora_add: null pointer");
    SRQ_CHECK_ARG(srq_aligned(x, 16) && srq_aligned(lora_a, 16) && srq_aligned(lora_b, 16) &&
                      x_stride % 8 == 0,
                  "lora_add: x (its rows too) and the adapters must be 16-byte aligned");
    SRQ_CHECK_ARG(x_stride >= K && x_stride <= 1 << 24 && y_stride >= a.N && out_stride >= a.N,
                  "lora_add: row stride out of range");
    const Plan p = plan_of(M, rank * slices, K);
    SRQ_CHECK_ARG(ws && srq_aligned(ws, 16) && ws_bytes >= 4 * M * rank * slices * p.splits,
                  "lora_add: the workspace is missing or too small");
    SRQ_CHECK_ARG(srq_cdiv(M, kTok) * tiles <= 0x7FFFFFFF, "lora_add: shape out of range");
    a.y = (const f16 *)y;
    a.x = (const f16 *)x;
    a.a = (const f16 *)lora_a;
    a.b = (const f16 *)lora_b;
    a.ids = ids;
    a.scaling = scaling;
    a.out = (f16 *)out;
    a.t = (float *)ws;
    a.M = M;
    a.K = K;
    a.ys = y_stride;
    a.xs = x_stride;
    a.os = out_stride;
    a.L = (int)adapters;
    a.r = (int)rank;
    a.R = (int)(rank * slices);
    a.slices = (int)slices;
    a.splits = p.splits;
    a.kc = p.kc;
    hipStream_t st = (hipStream_t)stream;
    if (M <= kFew) {
        lora_shrink_few_kernel<<<dim3((unsigned)srq_cdiv(a.R, 4), (unsigned)M), 256, 0, st>>>(a);
        SRQ_LAUNCH_CHECK("lora_add");
        lora_expand_few_kernel<<<dim3((unsigned)srq_cdiv(a.N, 256), (unsigned)M), 256, 0, st>>>(a);
        SRQ_LAUNCH_CHECK("lora_add (second product)");
        return SRQ_OK;
    }
    // Blocks in z share out a tile's adapters: a tile of single-token requests has up to
    // 64, and few tiles then leave the CUs idle.
    auto shares = [&](int64_t blocks) {
        int64_t z = srq_cdiv(1024, blocks);
        const int64_t most = adapters < kTok ? (adapters > 0 ? adapters : 1) : kTok;
        return (unsigned)(z > most ? most : z);
    };
    const unsigned tm = (unsigned)srq_cdiv(M, kTok), gy = (unsigned)(p.groups * p.splits);
    const unsigned z1 = shares((int64_t)tm * gy), z2 = shares((int64_t)tm * tiles);
    if (p.rt == 2)
        lora_shrink_kernel<2><<<dim3(tm, gy, z1), 256, 0, st>>>(a, p.groups, (int)z1);
    else
        lora_shrink_kernel<4><<<dim3(tm, gy, z1), 256, 0, st>>>(a, p.groups, (int)z1);
    SRQ_LAUNCH_CHECK("lora_add");
    lora_expand_kernel<<<dim3((unsigned)(tm * tiles), z2), 256, 0, st>>>(a, (int)tiles, (int)z2);
    SRQ_LAUNCH_CHECK("lora_add (second product)");
    return SRQ_OK;
}
