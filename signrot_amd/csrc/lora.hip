// Low-rank adapters of many requests beside a projection that they share:
//   out[m] = fp16(y[m] + scaling[i] * (x[m] A_i^T) B_i^T),  i = ids[m]
// x, y, A, B fp16; A [L, S r, K], B [L, N, r]: a projection that is S in one (q/k/v) has
// r rows of A for each of its column slices, whose columns meet only those.  Tokens
// whose id lies outside [0, L) have no adapter: out = y.  Sums are fp32 throughout.
// t = x A^T (fp32, in the workspace), then out = y + t B^T, a launch each.  The adapters'
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
// stored for itself, and a launch between the two adds them in order.  In the second
// product t is an fp16 number and the fp16 rest, scaled by a power of two of the token's
// largest: 22 bits.
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
    f16 *th, *tl;            // many tokens: [M, R], t as a number and a rest
    float *unit;             // [M, slices], what those are multiplied by
    int64_t M, N, K;
    int64_t ys, xs, os;      // row strides
    int L, r, R;             // R = slices * r
    int slices, splits;
    int kc;                  // columns of K in a split (a multiple of 64)
    int col_end[kMaxSlices];    // of each slice
    int tile_end[kMaxSlices];   // its column tiles (second product of many tokens)
};

SRQ_DEV uint32_t uni(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }

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

// Block b runs on XCD b % 8: its place in the work such that each XCD, with its own L2,
// has a run of neighbouring token tiles, which share their adapters.
SRQ_DEV uint32_t place_of_block() {
    const uint32_t x = blockIdx.x % 8, per = gridDim.x / 8, rem = gridDim.x % 8;
    return x * per + min(x, rem) + blockIdx.x / 8;
}

// t of 64 tokens x 16 RT rows of A, K in steps of 64 through a ring of four LDS stages
// (64 rows of x, 16 RT of A, 128 bytes each, the 16-byte chunks of a row exchanged by its
// number).  A block takes as many rows of A as there are, up to 192: x then crosses the
// fabric once.  The waves share the rows of A out first, and the tokens where those are
// fewer than four fragments.
constexpr int kStages = 4;

template <int RT>
__global__ __launch_bounds__(256) void lora_shrink_kernel(LoraArgs a, int groups, int nz) {
    constexpr int kStage = (kTok + 16 * RT) * 128;
    constexpr int PER = 2 + RT / 2;   // loads of a wave in a stage
    constexpr int WR = RT < 4 ? RT : 4, WT = 4 / WR, FT = 4 / WT, FR = RT / WR;
    static_assert(RT % 2 == 0 && WR * FR == RT && WR * WT == 4 && 2 * PER < 64, "waves");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[kStages * kStage];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const uint32_t at = place_of_block(), zs = uni(at / (uint32_t)nz);
    const int z = (int)(at - zs * nz);
    const uint32_t gy = groups * a.splits, tile = uni(zs / gy), part = zs - tile * gy;
    const int split = (int)uni(part / (uint32_t)groups), rg = (int)(part - split * groups) * 16 * RT;
    const int64_t m0 = (int64_t)tile * kTok;
    const int K = (int)a.K, k_lo = split * a.kc;
    const int steps = (int)uni((uint32_t)((min(K, k_lo + a.kc) - k_lo + 63) / 64));
    const int64_t rows = min((int64_t)kTok, a.M - m0);
    const uint32_t xbytes = uni((uint32_t)(2 * ((rows - 1) * a.xs + a.K)));
    const __amdgpu_buffer_rsrc_t xr = make_rsrc(a.x + m0 * a.xs, xbytes);
    const int arows = min(16 * RT, a.R - rg);
    const uint32_t ring0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)smem;
    const int r8 = lane >> 3, m = lane & 15, g = lane >> 4;
    const int wr = wave % WR, wt = wave / WR;

    // byte offsets of this lane's chunks in step 0 of the split; rows past the last lie
    // outside the buffers and read zeros
    uint32_t xo[2], ao[RT / 2];
    int xk[2], ak[RT / 2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int row = 8 * (2 * wave + q) + r8;
        xk[q] = k_lo + 8 * ((lane & 7) ^ (row >> 1 & 7));
        xo[q] = (uint32_t)(2 * (row * a.xs + xk[q]));
    }
#pragma unroll
    for (int q = 0; q < RT / 2; ++q) {
        const int row = 8 * (RT / 2 * wave + q) + r8;
        ak[q] = k_lo + 8 * ((lane & 7) ^ (row >> 1 & 7));
        ao[q] = (uint32_t)(2 * (row * a.K + ak[q]));
    }

    Turns turns(a, m0, lane);
    uint64_t same;
    for (int id; (id = turns.next(z, nz, same)) >= 0;) {
        const __amdgpu_buffer_rsrc_t ar =
            make_rsrc(a.a + ((int64_t)id * a.R + rg) * a.K, (int64_t)arows * a.K * 2);
        auto issue = [&](int s) __attribute__((always_inline)) {
            const uint32_t dst = ring0 + (s % kStages) * kStage;
            const int left = K - 64 * s;   // past K: zeros, on both sides
#pragma unroll
            for (int q = 0; q < 2; ++q)
                dma16(xr, xk[q] < left ? xo[q] + 128 * s : kOob, dst + (2 * wave + q) * 1024);
#pragma unroll
            for (int q = 0; q < RT / 2; ++q)
                dma16(ar, ak[q] < left ? ao[q] + 128 * s : kOob,
                      dst + kTok * 128 + (RT / 2 * wave + q) * 1024);
        };
        v4f acc[FT][FR];
#pragma unroll
        for (int i = 0; i < FT; ++i)
#pragma unroll
            for (int f = 0; f < FR; ++f) acc[i][f] = (v4f)0.f;
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
            const uint8_t *xs = smem + (s % kStages) * kStage, *as = xs + kTok * 128;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int c = 16 * ((4 * h + g) ^ (m >> 1));
                v8h xv[FT], av[FR];
#pragma unroll
                for (int i = 0; i < FT; ++i)
                    xv[i] = *reinterpret_cast<const v8h *>(xs + (16 * (FT * wt + i) + m) * 128 + c);
#pragma unroll
                for (int f = 0; f < FR; ++f)
                    av[f] = *reinterpret_cast<const v8h *>(as + (16 * (FR * wr + f) + m) * 128 + c);
#pragma unroll
                for (int i = 0; i < FT; ++i)
#pragma unroll
                    for (int f = 0; f < FR; ++f) acc[i][f] = mfma16(xv[i], av[f], acc[i][f]);
            }
        }
        // the ring is filled anew for the next adapter
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 0; i < FT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = 16 * (FT * wt + i) + 4 * g + e;
                if (!(same >> row & 1)) continue;
                float *t = a.t + ((int64_t)split * a.M + m0 + row) * a.R + rg;
#pragma unroll
                for (int f = 0; f < FR; ++f) {
                    const int j = 16 * (FR * wr + f) + m;
                    if (j < arows) t[j] = acc[i][f][e];
                }
            }
    }
}

// The splits' parts of t added in order, as an fp16 number, the fp16 rest and a factor
// for each token and slice: a wave each.
__global__ __launch_bounds__(256) void lora_join_kernel(LoraArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t m = w / a.slices;
    if (m >= a.M) return;
    const int s = (int)(w - m * a.slices);
    const int id = adapter_of(a, m);
    if (id < 0) return;   // never read
    const int64_t at = m * a.R + s * a.r;
    constexpr int V = kMaxRank / 64;
    float v[V], top = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int k = 64 * i + lane;
        v[i] = 0.f;
        if (k < a.r)
            for (int p = 0; p < a.splits; ++p) v[i] += a.t[(int64_t)p * a.M * a.R + at + k];
        top = fmaxf(top, fabsf(v[i]));
    }
    top = wave_max(top);
    // a power of two that takes the largest to [2^10, 2^11): there the rest of the fp16
    // number is one too, down to 2^-25 of the largest
    const int e = top > 0.f && top <= 3.4e38f ? 11 - (int)__builtin_amdgcn_frexp_expf(top) : 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int k = 64 * i + lane;
        if (k >= a.r) continue;
        const float x = __builtin_amdgcn_ldexpf(v[i], e);
        const f16 h = (f16)x;
        a.th[at + k] = h;
        a.tl[at + k] = fabsf(x) <= 65504.f ? (f16)(x - (float)h) : (f16)0.f;
    }
    if (lane == 0)
        a.unit[m * a.slices + s] = __builtin_amdgcn_ldexpf(a.scaling ? a.scaling[id] : 1.f, -e);
}

struct __attribute__((packed, aligned(2))) U8h { v8h v; };

// out of 64 tokens x 128 columns of one slice: four waves of 32 x 64.  t (both halves) and
// B pass through LDS, KW ranks at a time: in operand order neighbouring lanes are
// different rows, each an access of its own.  The products go through the wave's own rows
// of B's place, so that y and out move in 16 bytes a lane; y is loaded ahead.
constexpr int kCols = 128;

template <int KW>
__global__ __launch_bounds__(256, KW == 64 ? 3 : 4) void lora_expand_kernel(LoraArgs a, int tiles_n, int nz) {
    constexpr int C = KW / 8, RPD = 64 / C;        // chunks of a row, rows of a load
    constexpr int kT = kTok * 2 * KW, kB = kCols * 2 * KW;
    constexpr int kW = 64 + 4, kP = 4 * 16 * kW * 4;   // 16 rows of products a wave
    __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * kT + (kB > kP ? kB : kP)];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1, rr = lane & 31, g = lane >> 5;
    const uint32_t at = place_of_block();
    const uint32_t zt = uni(at / (uint32_t)nz);
    const int z = (int)(at - zt * nz);
    const uint32_t tm = uni(zt / (uint32_t)tiles_n);
    const int tile = (int)(zt - tm * tiles_n);
    const int64_t m0 = (int64_t)tm * kTok;
    int s = 0;
    while (tile >= a.tile_end[s]) ++s;
    const int n_hi = a.col_end[s];
    const int nb = (s ? a.col_end[s - 1] : 0) + (tile - (s ? a.tile_end[s - 1] : 0)) * kCols;
    // place in the row-wise pass: 8 rows of 64 columns an instruction
    const int pr = 32 * wm + (lane >> 3), pn = nb + 64 * wn + 8 * (lane & 7);
    const bool full = pn + 8 <= n_hi;
    // 32-bit offsets from the tile's first row
    const f16 *y0 = a.y + m0 * a.ys;
    f16 *o0 = a.out + m0 * a.os;
    const float *u0 = a.unit + m0 * a.slices + s;
    const uint32_t ys = (uint32_t)a.ys, os = (uint32_t)a.os;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)smem;
    // the 16-byte chunks of a row exchanged by its number: 16 rows of one chunk then lie
    // in all banks
    auto swz = [](int row, int c) __attribute__((always_inline)) {
        return c ^ (row / (256 / (2 * KW)) & (C - 1));
    };
    const int64_t rows = min((int64_t)kTok, a.M - m0);
    const uint32_t tbytes = uni((uint32_t)(2 * ((rows - 1) * a.R + a.r)));
    const int64_t t0 = m0 * a.R + s * a.r;
    const __amdgpu_buffer_rsrc_t hr = make_rsrc(a.th + t0, tbytes);
    const __amdgpu_buffer_rsrc_t lr = make_rsrc(a.tl + t0, tbytes);
    const uint32_t bbytes = uni((uint32_t)(2 * min(kCols, n_hi - nb) * a.r));

    Turns turns(a, m0, lane);
    uint64_t same;
    for (int id; (id = turns.next(z, nz, same)) >= 0;) {
        const __amdgpu_buffer_rsrc_t br = make_rsrc(a.b + ((int64_t)id * a.N + nb) * a.r, bbytes);
        v16f acc[2] = {(v16f)0.f, (v16f)0.f};
        v8h yv[4];
        float unit[4];
#pragma unroll 1
        for (int k0 = 0; k0 < a.r; k0 += KW) {
            __syncthreads();   // LDS is free
            constexpr int DT = kT / 4096 ? kT / 4096 : 1, DB = kB / 4096;
#pragma unroll
            for (int q = 0; q < DT; ++q) {
                const int i = DT * wave + q, row = RPD * i + lane / C;
                const int k = k0 + 8 * swz(row, lane % C);
                if (i * 1024 >= kT) break;         // narrow rows: two waves' loads are enough
                const uint32_t off = k < a.r ? (uint32_t)(2 * (row * a.R + k)) : kOob;
                dma16(hr, off, lds0 + i * 1024);
                dma16(lr, off, lds0 + kT + i * 1024);
            }
#pragma unroll
            for (int q = 0; q < DB; ++q) {
                const int i = DB * wave + q, row = RPD * i + lane / C;
                const int k = k0 + 8 * swz(row, lane % C);
                dma16(br, k < a.r ? (uint32_t)(2 * (row * a.r + k)) : kOob, lds0 + 2 * kT + i * 1024);
            }
            if (k0 == 0) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t row = pr + 8 * q;
                    if (!(same >> row & 1)) continue;
                    unit[q] = u0[row * a.slices];
                    if (full) yv[q] = reinterpret_cast<const U8h *>(y0 + (row * ys + pn))->v;
                }
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
#pragma unroll
            for (int st = 0; st < KW / 16; ++st) {
                const int row = 32 * wm + rr, c = row * 2 * KW + 16 * swz(row, 2 * st + g);
                const v8h h = *reinterpret_cast<const v8h *>(smem + c);
                const v8h l = *reinterpret_cast<const v8h *>(smem + kT + c);
#pragma unroll
                for (int f = 0; f < 2; ++f) {
                    const int col = 64 * wn + 32 * f + rr;
                    const v8h w = *reinterpret_cast<const v8h *>(smem + 2 * kT + col * 2 * KW +
                                                                 16 * swz(col, 2 * st + g));
                    acc[f] = mfma32(h, w, acc[f]);
                    acc[f] = mfma32(l, w, acc[f]);
                }
            }
        }
        __syncthreads();   // B's place is free
        float *mine = reinterpret_cast<float *>(smem + 2 * kT) + wave * 16 * kW;
#pragma unroll
        for (int i = 0; i < 2; ++i) {   // 16 rows at a time
#pragma unroll
            for (int v = 0; v < 8; ++v)
#pragma unroll
                for (int f = 0; f < 2; ++f)
                    mine[(8 * (v / 4) + 4 * g + v % 4) * kW + 32 * f + rr] = acc[f][8 * i + v];
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const uint32_t row = pr + 16 * i + 8 * q;
                const float u = unit[2 * i + q];
                const float *p = mine + (8 * q + (lane >> 3)) * kW + 8 * (lane & 7);
                const v4f lo = *reinterpret_cast<const v4f *>(p);
                const v4f hi = *reinterpret_cast<const v4f *>(p + 4);
                if (!(same >> row & 1)) continue;
                f16 *o = o0 + (row * os + pn);
                if (full) {
                    v8h v = yv[2 * i + q];
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        v[k] = f16_rn(__builtin_fmaf(k < 4 ? lo[k & 3] : hi[k & 3], u, (float)v[k]));
                    reinterpret_cast<U8h *>(o)->v = v;
                } else {
                    const f16 *y = y0 + (row * ys + pn);
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (pn + k < n_hi)
                            o[k] = f16_rn(
                                __builtin_fmaf(k < 4 ? lo[k & 3] : hi[k & 3], u, (float)y[k]));
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
    }
    // tokens without an adapter
    if (z == 0 && a.out != a.y && turns.invalid && pn < n_hi)
        for (int q = 0; q < 4; ++q) {
            const uint32_t row = pr + 8 * q;
            if (!(turns.invalid >> row & 1)) continue;
            const f16 *y = y0 + (row * ys + pn);
            f16 *o = o0 + (row * os + pn);
            if (full) {
                reinterpret_cast<U8h *>(o)->v = reinterpret_cast<const U8h *>(y)->v;
            } else {
                for (int k = 0; k < 8; ++k)
                    if (pn + k < n_hi) o[k] = y[k];
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
    p.rt = R <= 32 ? 2 : R <= 64 ? 4 : R <= 128 ? 8 : 12;
    p.groups = (int)srq_cdiv(R, 16 * p.rt);
    // a block for each place on the 256 CUs (two of the small ones fit one), of at least
    // 8 steps
    const int64_t blocks = srq_cdiv(M, kTok) * p.groups, steps = srq_cdiv(K, 64);
    int64_t s = (p.rt <= 4 ? 512 : 256) / blocks;
    if (s > steps / 8) s = steps / 8;
    if (s > 16) s = 16;
    if (s < 1) s = 1;
    const int64_t per = srq_cdiv(steps, s);
    p.kc = (int)(64 * per);
    p.splits = (int)srq_cdiv(steps, per);
    return p;
}

// t, and with many tokens its two halves and factors
int64_t workspace(const Plan &p, int64_t M, int64_t R, int64_t slices) {
    return 4 * M * R * p.splits + (p.rt ? 4 * M * R + 4 * M * slices : 0);
}

}  // namespace

extern "C" int srq_lora_workspace(int64_t M, int64_t K, int64_t rank, int64_t slices,
                                  int64_t *bytes) {
    SRQ_CHECK_ARG(bytes, "lora_add: null pointer");
    *bytes = 0;
    if (M <= 0 || K <= 0 || rank <= 0 || slices <= 0) return SRQ_OK;
    *bytes = workspace(plan_of(M, rank * slices, K), M, rank * slices, slices);
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
    SRQ_CHECK_ARG(x_stride >= K && x_stride <= 1 << 24 && y_stride >= a.N && out_stride >= a.N &&
                      y_stride <= 1 << 25 && out_stride <= 1 << 25,
                  "lora_add: row stride out of range");
    const Plan p = plan_of(M, rank * slices, K);
    SRQ_CHECK_ARG(ws && srq_aligned(ws, 16) && ws_bytes >= workspace(p, M, rank * slices, slices),
                  "lora_add: the workspace is missing or too small");
    // a launch has fewer than 2^32 threads in x
    SRQ_CHECK_ARG(srq_cdiv(M, kTok) * tiles < 1 << 24 && M * slices < 1 << 26,
                  "lora_add: shape out of range");
    a.y = (const f16 *)y;
    a.x = (const f16 *)x;
    a.a = (const f16 *)lora_a;
    a.b = (const f16 *)lora_b;
    a.ids = ids;
    a.scaling = scaling;
    a.out = (f16 *)out;
    a.t = (float *)ws;
    a.th = (f16 *)(a.t + p.splits * M * rank * slices);
    a.tl = a.th + M * rank * slices;
    a.unit = (float *)(a.tl + M * rank * slices);
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
    // Neighbouring blocks share out a tile's adapters: a tile of single-token requests has
    // up to 64, and few tiles then leave the CUs idle; and where one of many tiles has two
    // adapters, the second does not wait for the first.
    auto shares = [&](int64_t blocks) {
        int64_t z = srq_cdiv(1024, blocks), most = adapters < kTok ? adapters : kTok;
        if (z > most) z = most;
        return (int)(z < 1 ? 1 : z);
    };
    const unsigned tm = (unsigned)srq_cdiv(M, kTok), gy = (unsigned)(p.groups * p.splits);
    const int z1 = shares((int64_t)tm * gy), z2 = shares((int64_t)tm * tiles);
    SRQ_CHECK_ARG((int64_t)tm * tiles * z2 < 1 << 24 && (int64_t)tm * gy * z1 < 1 << 24,
                  "lora_add: shape out of range");
    const unsigned grid = tm * gy * z1;
    switch (p.rt) {
    case 2: lora_shrink_kernel<2><<<grid, 256, 0, st>>>(a, p.groups, z1); break;
    case 4: lora_shrink_kernel<4><<<grid, 256, 0, st>>>(a, p.groups, z1); break;
    case 8: lora_shrink_kernel<8><<<grid, 256, 0, st>>>(a, p.groups, z1); break;
    default: lora_shrink_kernel<12><<<grid, 256, 0, st>>>(a, p.groups, z1); break;
    }
    SRQ_LAUNCH_CHECK("lora_add");
    lora_join_kernel<<<(unsigned)srq_cdiv(M * slices, 4), 256, 0, st>>>(a);
    SRQ_LAUNCH_CHECK("lora_add (join)");
    const unsigned blocks = (unsigned)(tm * tiles * z2);
    if (rank <= 16)
        lora_expand_kernel<16><<<blocks, 256, 0, st>>>(a, (int)tiles, z2);
    else if (rank <= 32)
        lora_expand_kernel<32><<<blocks, 256, 0, st>>>(a, (int)tiles, z2);
    else
        lora_expand_kernel<64><<<blocks, 256, 0, st>>>(a, (int)tiles, z2);
    SRQ_LAUNCH_CHECK("lora_add (second product)");
    return SRQ_OK;
}
