// Attention over the paged int8 cache: the last n tokens of each request (one
// in a decode step, a piece of a prompt otherwise) against everything that its
// pages hold, causal, grouped-query.
//
// A row is one (query token, query head) of a KV head's group; rows of a group
// share every byte of K and V, so they are packed into the 16 columns of the
// matrix instruction and the cache is read once per row tile.  Everything is
// computed transposed, S^T = K Q^T and O^T += V^T P^T (v_mfma_f32_16x16x32_f16):
// a lane then holds scores of one row (column l % 16), the running maximum and
// sum are in-lane, and P^T is the second product's operand straight from the
// registers it was computed in, when the 32 k-slots of that product are given
// to tokens in the order of the first one's output (slot 8 g + j <-> token
// 16 (j / 4) + 4 g + j % 4 for lane group g = l / 16).
//
// K and V go from HBM to registers, never through LDS.  A lane's K bytes are
// 2 x 16 of a token's row (which dims they are does not matter as long as q
// is read alike).  Its V bytes are dims 8 (l % 16) .. + 7 of the 8 tokens in
// its slots; two byte permutes pair tokens, which is the transposition the
// product needs, and give fp16 numbers 1024 + c, from which an addition leaves
// the code itself, exactly.  Scales never touch the codes: K's multiplies the
// scores of its block of 16 tokens, and V's goes into the exponent,
//   p' = exp2(s ks c + log2 vs - m),   O = sum p' code,   l = sum p' / vs,
// so out = O / l with codes as integers throughout.  m (the running maximum of
// the exponent) moves only when a score exceeds it by more than 8, so p' <= 2^8.
// p' is rounded to fp16 for the second product, the one rounding to 16 bits before
// the output's: 2.4e-4 to 2.9e-4 from 64 bits where the output's alone leaves
// 2.1e-4.  The rest of p' as a second fp16 operand would leave 2.1e-4 too; it
// doubles that product, 45.2 -> 46.4 us for the decode batch below and 181 -> 233 us
// for pieces of a prompt, and was not taken.  (Scores are summed over codes + 128,
// whose part 128 sum(q) is taken out in fp32: far below either.)
//
// The waves of a block take 32-token tiles in turn and are joined through LDS;
// a request is split over blocks (chunks) when there are few, whose partial
// (O, m, l) a second kernel joins.  HBM bounds decode: 32 requests of up to 4096
// tokens, 32 / 8 heads, 204 MB: 45.2 us, 4.5 TB/s (loads alone 41, products alone
// 30 to 33).
#include "kv_i8.h"

#include <math.h>

#include <algorithm>
#include <type_traits>

namespace {

constexpr int kTileTok = 32;
constexpr int kWaves = 4;
constexpr float kSlack = 8.f;
constexpr int kRec = kI8D + 4;   // floats of a partial state: O, m, l and padding

struct AttnI8Args {
    const f16 *q;                 // [rows, hq, 128]
    f16 *o;
    const int32_t *q_indptr;      // [B + 1] or null
    float *tmp;                   // [rows, hq, chunks, kRec]
    int64_t rows;
    int hq, group, chunks, tiles; // tiles: row tiles in the grid
    float c, qmul;                // |scale| log2 e, and its sign
};

SRQ_DEV v4f mfma16(v8h a, v8h b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// two unsigned codes in bytes 0 and 2 of fp16 patterns 0x64cc (1024 + code +
// 128) -> the signed codes
SRQ_DEV v2h unbias(u32 w) { return __builtin_bit_cast(v2h, w) - (v2h){1152, 1152}; }

// 8 int8 codes -> fp16 subnormals (code + 128) 2^-24, in order: a byte below a
// zero byte, exact.  The 128 and the 2^-24 are taken out of the fp32 scores.
SRQ_DEV v8h codes8(u32 a, u32 b) {
    const u32 x = a ^ 0x80808080u, y = b ^ 0x80808080u;
    const v2h p0 = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0u, x, 0x0c010c00u));
    const v2h p1 = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0u, x, 0x0c030c02u));
    const v2h p2 = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0u, y, 0x0c010c00u));
    const v2h p3 = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0u, y, 0x0c030c02u));
    return (v8h){p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
}

// 8 int8 codes -> fp16, in order
SRQ_DEV v8h signed8(u32 a, u32 b) {
    const u32 x = a ^ 0x80808080u, y = b ^ 0x80808080u, k = 0x64646464u;
    const v2h p0 = unbias(__builtin_amdgcn_perm(k, x, 0x04010400u));
    const v2h p1 = unbias(__builtin_amdgcn_perm(k, x, 0x04030402u));
    const v2h p2 = unbias(__builtin_amdgcn_perm(k, y, 0x04010400u));
    const v2h p3 = unbias(__builtin_amdgcn_perm(k, y, 0x04030402u));
    return (v8h){p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
}

// dwords of tokens a and b (4 dims each): fp16 pairs (a, b) of the 4 dims
SRQ_DEV void pair_dims(u32 a, u32 b, v2h (&d)[4]) {
    const u32 x = a ^ 0x80808080u, y = b ^ 0x80808080u, k = 0x64646464u;
    const u32 lo = __builtin_amdgcn_perm(y, x, 0x05010400u);   // a0 b0 a1 b1
    const u32 hi = __builtin_amdgcn_perm(y, x, 0x07030602u);   // a2 b2 a3 b3
    d[0] = unbias(__builtin_amdgcn_perm(k, lo, 0x04010400u));
    d[1] = unbias(__builtin_amdgcn_perm(k, lo, 0x04030402u));
    d[2] = unbias(__builtin_amdgcn_perm(k, hi, 0x04010400u));
    d[3] = unbias(__builtin_amdgcn_perm(k, hi, 0x04030402u));
}

// log2 and inverse of a V scale.  A block of zeros (scale 0) adds to l alone: it
// counts as one of scale 2^-60, under the least that fp16 values have (2^-31), so
// that m follows the blocks that do add values and p' keeps its bits for them.
SRQ_DEV float log_scale(float v) { return v != 0.f ? __builtin_amdgcn_logf(v) : -60.f; }
SRQ_DEV float inv_scale(float v) { return v != 0.f ? 1.f / v : 0x1p60f; }

struct Tile {
    v4i k[2][2];   // [block][half of the dims]
    uint2 v[8];    // tokens of the lane's slots
};

SRQ_DEV int read_lane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
SRQ_DEV float read_lane(float v, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// RT row tiles of 16 rows per block.  With one, a wave has two tiles in flight (the
// registers of two waves per SIMD).
template <int RT>
__global__ __launch_bounds__(kWaves * 64, 2) void attn_i8_kernel(AttnI8Args a, PagedI8 p) {
    constexpr int DEPTH = RT == 1 ? 2 : 1;
    __shared__ float so[kWaves][16][kI8D + 4];
    __shared__ float sm[kWaves][16], sl[kWaves][16];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int hk = blockIdx.y;
    const int64_t b = blockIdx.z;
    const int chunk = blockIdx.x % a.chunks;
    int64_t s0, n;
    i8_new_rows(a.q_indptr, b, a.rows, s0, n);
    const I8Request rq = i8_request(p, b);
    const int64_t nrows = n * a.group;
    for (int64_t r0 = (int64_t)(blockIdx.x / a.chunks) * 16 * RT; r0 < nrows;
         r0 += (int64_t)a.tiles * 16 * RT) {
        // this lane's rows: query token, head, first token that it does not see
        v8h qf[RT][4];
        float qsum[RT];
        int lim[RT];
        int64_t orow[RT];
        int lo = 0x7fffffff, hi = 0;   // least and largest limit of the block's rows
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int64_t r = r0 + 16 * t + col;
            const bool ok = r < nrows;
            const int64_t i = ok ? (uint32_t)r / (uint32_t)a.group : 0;
            const int h = hk * a.group + (ok ? (int)(r - i * a.group) : 0);
            orow[t] = ok ? (s0 + i) * a.hq + h : -1;
            const int64_t pos = rq.len - n + i + 1;
            lim[t] = ok && pos > 0 ? (int)pos : 0;
            const f16 *src = a.q + (ok ? orow[t] : 0) * kI8D + 16 * g;
            float sum = 0.f;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                qf[t][s] = *reinterpret_cast<const v8h *>(src + 64 * (s >> 1) + 8 * (s & 1)) *
                           (f16)a.qmul;
#pragma unroll
                for (int e = 0; e < 8; ++e) sum += (float)qf[t][s][e];
            }
            sum += __shfl_xor(sum, 16, 64);
            sum += __shfl_xor(sum, 32, 64);
            qsum[t] = sum * -0x1p-17f;   // -128 sum(q) 2^-24
        }
        {
            const int64_t last = r0 + 16 * RT < nrows ? r0 + 16 * RT : nrows;
            const int64_t f = rq.len - n + (uint32_t)r0 / (uint32_t)a.group + 1;
            const int64_t e = rq.len - n + (uint32_t)(last - 1) / (uint32_t)a.group + 1;
            lo = f > 0 ? (int)f : 0;
            hi = e > 0 ? (int)e : 0;
        }
        // this chunk's tiles
        const int ntile = (hi + kTileTok - 1) / kTileTok;
        const int per = (ntile + a.chunks - 1) / a.chunks;
        const int t_lo = chunk * per, t_hi = min(ntile, t_lo + per);

        v4f o[RT][8];
        float m[RT], l[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            m[t] = -INFINITY;
            l[t] = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) o[t][i] = (v4f)0.f;
        }

        const int64_t v_part = (int64_t)p.H * p.page * kI8D;
        const uint32_t k_lane = col * kI8D + 16 * g, v_lane = 4 * g * kI8D + 8 * col;
        // The wave's tiles are t_lo + wave, + kWaves, ...; lane j looks up the
        // page and the scales of block j of the next 64 (32 tiles).
        for (int base = t_lo + wave; base < t_hi; base += 32 * kWaves) {
            const int mine = base + (lane >> 1) * kWaves;
            const int blk = 2 * mine + (lane & 1);
            int pg = -1;
            float ks = 0.f, vs = 0.f, lv, rv;
            int64_t at = 0;   // its K codes; any block where there is none
            if (mine < t_hi && blk * kI8Block < hi) {
                pg = (int)i8_page(p, rq.first, blk);
                if (pg >= 0) {
                    const int64_t si =
                        i8_scale_index(p, pg, hk, (uint32_t)blk % (uint32_t)p.bpp);
                    at = si * (kI8Block * kI8D);
                    ks = p.scale[si];
                    vs = p.scale[si + (int64_t)p.H * p.bpp];
                }
            }
            const int at_lo = (int)at, at_hi = (int)(at >> 32);
            auto block_of = [&](int j, int bk) __attribute__((always_inline)) {
                const uint32_t lo32 = (uint32_t)read_lane(at_lo, 2 * j + bk);
                const int hi32 = read_lane(at_hi, 2 * j + bk);
                return p.data + ((int64_t)hi32 << 32 | lo32);
            };
            auto load_k = [&](Tile &x, int j) __attribute__((always_inline)) {
#pragma unroll
                for (int bk = 0; bk < 2; ++bk) {
                    const int8_t *kb = block_of(j, bk) + k_lane;
                    x.k[bk][0] = *reinterpret_cast<const v4i *>(kb);
                    x.k[bk][1] = *reinterpret_cast<const v4i *>(kb + 64);
                }
            };
            auto load_v = [&](Tile &x, int j) __attribute__((always_inline)) {
#pragma unroll
                for (int bk = 0; bk < 2; ++bk) {
                    const int8_t *vb = block_of(j, bk) + v_part + v_lane;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        x.v[4 * bk + e] = *reinterpret_cast<const uint2 *>(vb + e * kI8D);
                }
            };
            auto step = [&](Tile &x, int j, auto more) __attribute__((always_inline)) {
                const int tok = (base + j * kWaves) * kTileTok;
                v8h pb[RT];
                v4f s[RT][2];
#pragma unroll
                for (int t = 0; t < RT; ++t) s[t][0] = s[t][1] = (v4f)qsum[t];
#pragma unroll
                for (int bk = 0; bk < 2; ++bk)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const v4i w = x.k[bk][q >> 1];
                        const v8h kf = codes8((u32)w[2 * (q & 1)], (u32)w[2 * (q & 1) + 1]);
#pragma unroll
                        for (int t = 0; t < RT; ++t) s[t][bk] = mfma16(kf, qf[t][q], s[t][bk]);
                    }
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (more.value) load_k(x, j + DEPTH);
                const bool full = tok + kTileTok <= lo && read_lane(pg, 2 * j) >= 0 &&
                                  read_lane(pg, 2 * j + 1) >= 0;
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    float mx = -INFINITY;
#pragma unroll
                    for (int bk = 0; bk < 2; ++bk) {
                        const float kc = read_lane(ks, 2 * j + bk), add = read_lane(lv, 2 * j + bk);
                        const bool there = read_lane(pg, 2 * j + bk) >= 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float y = __builtin_fmaf(s[t][bk][e], kc, add);
                            if (!full && (!there || tok + 16 * bk + 4 * g + e >= lim[t]))
                                y = -INFINITY;
                            s[t][bk][e] = y;
                            mx = fmaxf(mx, y);
                        }
                    }
                    const bool grow = mx > m[t] + kSlack;
                    if (__builtin_amdgcn_ballot_w64(grow)) {
                        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
                        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                        const float to = fmaxf(m[t], mx);
                        const float f = m[t] == to ? 1.f : __builtin_amdgcn_exp2f(m[t] - to);
                        m[t] = to;
                        l[t] *= f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) o[t][i] *= f;
                    }
                    const float sub = m[t] == -INFINITY ? 0.f : m[t];
#pragma unroll
                    for (int bk = 0; bk < 2; ++bk) {
                        float sum = 0.f;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float pr = __builtin_amdgcn_exp2f(s[t][bk][e] - sub);
                            sum += pr;
                            pb[t][4 * bk + e] = (f16)pr;
                        }
                        // a block that this row does not see may hold any scale
                        if (sum != 0.f) l[t] = __builtin_fmaf(sum, read_lane(rv, 2 * j + bk), l[t]);
                    }
                }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    v2h d[4][4];   // [token pair][dim]
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        pair_dims(half ? x.v[2 * e].y : x.v[2 * e].x,
                                  half ? x.v[2 * e + 1].y : x.v[2 * e + 1].x, d[e]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const v8h vf = {d[0][i][0], d[0][i][1], d[1][i][0], d[1][i][1],
                                        d[2][i][0], d[2][i][1], d[3][i][0], d[3][i][1]};
#pragma unroll
                        for (int t = 0; t < RT; ++t)
                            o[t][4 * half + i] = mfma16(vf, pb[t], o[t][4 * half + i]);
                    }
                    // half the converted codes at a time in registers
                    __builtin_amdgcn_sched_barrier(0);
                }
                if constexpr (more.value) load_v(x, j + DEPTH);
            };
            const int cnt = min(32, (t_hi - base + kWaves - 1) / kWaves);
            // the next tile's K is loaded as soon as this one's scores have
            // taken its registers, its V after the second product; the first
            // tile's loads come before its scales are used
            Tile x;
            load_k(x, 0);
            __builtin_amdgcn_sched_barrier(0);   // K first: its wait leaves V in flight
            load_v(x, 0);
            __builtin_amdgcn_sched_barrier(0);
            lv = log_scale(vs);
            rv = inv_scale(vs);
            ks *= a.c * 0x1p24f;
            // (the last tiles apart: with their loads under a condition every wait
            // would be for all that are in flight)
            if constexpr (DEPTH == 1) {
                for (int j = 0; j + 1 < cnt; ++j) step(x, j, std::true_type());
                step(x, cnt - 1, std::false_type());
            } else {
                Tile y;
                load_k(y, cnt > 1 ? 1 : 0);
                __builtin_amdgcn_sched_barrier(0);
                load_v(y, cnt > 1 ? 1 : 0);
                __builtin_amdgcn_sched_barrier(0);
                int j = 0;
                for (; j + 3 < cnt; j += 2) {
                    step(x, j, std::true_type());
                    step(y, j + 1, std::true_type());
                }
                if (j + 2 < cnt) {
                    step(x, j, std::true_type());
                    step(y, j + 1, std::false_type());
                    step(x, j + 2, std::false_type());
                } else {
                    step(x, j, std::false_type());
                    if (j + 1 < cnt) step(y, j + 1, std::false_type());
                }
            }
        }

        // join the waves: one row tile at a time through LDS
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            l[t] += __shfl_xor(l[t], 16, 64);
            l[t] += __shfl_xor(l[t], 32, 64);
            __syncthreads();   // the previous row tile's readers are done
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                // dims 8 (4 g + e) + 0 .. 7
                float *to = &so[wave][col][8 * (4 * g + e)];
#pragma unroll
                for (int i = 0; i < 8; ++i) to[i] = o[t][i][e];
            }
            if (g == 0) {
                sm[wave][col] = m[t];
                sl[wave][col] = l[t];
            }
            __syncthreads();
            // thread -> row threadIdx.x / 16, dims 8 (threadIdx.x % 16) .. + 7
            const int rr = threadIdx.x >> 4, d0 = 8 * (threadIdx.x & 15);
            const int64_t r = r0 + 16 * t + rr;
            if (rr < 16 && r < nrows) {
                const int64_t i = (uint32_t)r / (uint32_t)a.group;
                const int64_t row = (s0 + i) * a.hq + hk * a.group + (r - i * a.group);
                float mx = sm[0][rr];
#pragma unroll
                for (int w = 1; w < kWaves; ++w) mx = fmaxf(mx, sm[w][rr]);
                float acc[8] = {}, sum = 0.f;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) {
                    const float f =
                        sm[w][rr] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm[w][rr] - mx);
                    sum = __builtin_fmaf(sl[w][rr], f, sum);
#pragma unroll
                    for (int d = 0; d < 8; ++d)
                        acc[d] = __builtin_fmaf(so[w][rr][d0 + d], f, acc[d]);
                }
                if (a.chunks == 1) {
                    const float inv = sum == 0.f ? 0.f : 1.f / sum;
                    v8h out;
#pragma unroll
                    for (int d = 0; d < 8; ++d) out[d] = (f16)(acc[d] * inv);
                    *reinterpret_cast<v8h *>(a.o + row * kI8D + d0) = out;
                } else {
                    float *rec = a.tmp + (row * a.chunks + chunk) * kRec;
#pragma unroll
                    for (int d = 0; d < 8; d += 4)
                        *reinterpret_cast<v4f *>(rec + d0 + d) =
                            (v4f){acc[d], acc[d + 1], acc[d + 2], acc[d + 3]};
                    if (d0 == 0) {
                        rec[kI8D] = mx;
                        rec[kI8D + 1] = sum;
                    }
                }
            }
        }
        __syncthreads();
    }
}

// ----------------------------------------------------------- many query rows
// The same attention for pieces of a prompt, where the products bound it and
// not the cache's bytes: four waves of 32 rows each (v_mfma_f32_32x32x16_f16)
// share tiles of 64 keys in LDS, double-buffered, with codes converted to
// fp16 once per block on the way in.  A lane owns one row (column l % 32 of the
// transposed scores); register v of a 32-key block is key 8 (v / 4) + 4 (l / 32) +
// v % 4, so registers 0-7 and 8-15 each belong to one block of 16 keys, whose
// scales reach the scores as above, and P^T is the second product's operand
// straight from registers.  V's operand comes from the transposing LDS read.
// 3125 to 5000 cached and 320 to 512 new tokens of 4 requests, 32 / 8 heads, 120
// GFLOP: 180 us, 0.66 PFLOP/s, bound by the instructions of a wave (535 a tile: 2290
// of its 4750 cycles issue one, 1440 wait to) and by uneven requests.
constexpr int KT = 64;
constexpr int kRowsBlock = 32 * kWaves;
constexpr int KS = kI8D + 8;     // row strides in halves: 16-byte reads of K and the
constexpr int VR = kI8D + 16;    // transposing reads of V fall on distinct banks
typedef short v4s __attribute__((vector_size(8)));

SRQ_DEV v16f mfma32(v8h a, v8h b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// what a tile's scores need of a block of 16 keys
struct BlockScale {
    float kc, lv, rv, pad;
};

// A wave per SIMD from each of the two blocks that fit a CU.
__global__ __launch_bounds__(kWaves * 64, 2) void attn_i8_rows_kernel(AttnI8Args a, PagedI8 p) {
    constexpr int NT = kWaves * 64, RB = kRowsBlock;
    constexpr int KR = NT / KT, KB = kI8D / KR;     // threads per key row, bytes of each
    static_assert(KR * kI8Block == 64, "a wave stages a block of keys");
    __shared__ __align__(16) f16 Ks_[2][KT * KS];
    __shared__ __align__(16) f16 Vs_[2][KT * VR];
    __shared__ BlockScale Bs_[2][KT / kI8Block];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 5, ln = lane & 31;
    const int hk = blockIdx.y;
    const int64_t b = blockIdx.z;
    int64_t s0, n;
    i8_new_rows(a.q_indptr, b, a.rows, s0, n);
    const I8Request rq = i8_request(p, b);
    const int64_t nrows = n * a.group;
    const int64_t rtiles = (nrows + RB - 1) / RB;
    // the last rows see most keys: their tiles come first
    for (int64_t rt = rtiles - 1 - (int64_t)blockIdx.x; rt >= 0; rt -= a.tiles) {
        const int64_t r0 = rt * RB, r = r0 + 32 * wave + ln;
        const bool ok = r < nrows;
        const int64_t qi = ok ? (uint32_t)r / (uint32_t)a.group : 0;
        const int64_t orow = (s0 + qi) * a.hq + hk * a.group + (ok ? (int)(r - qi * a.group) : 0);
        const int64_t past = rq.len - n;
        int lim = ok && past + qi + 1 > 0 ? (int)(past + qi + 1) : 0;
        // limits of the wave's first row and of the block's last one
        const int64_t wrow = r0 + 32 * wave < nrows ? r0 + 32 * wave : nrows - 1;
        const int64_t brow = r0 + RB < nrows ? r0 + RB - 1 : nrows - 1;
        const int64_t wlast = wrow + 31 < nrows ? wrow + 31 : nrows - 1;
        const int64_t lo64 = past + (uint32_t)wrow / (uint32_t)a.group + 1;
        const int64_t wh64 = past + (uint32_t)wlast / (uint32_t)a.group + 1;
        const int64_t hi64 = past + (uint32_t)brow / (uint32_t)a.group + 1;
        const int lo = lo64 > 0 ? (int)lo64 : 0, hi = hi64 > 0 ? (int)hi64 : 0;
        const int wave_hi = r0 + 32 * wave < nrows && wh64 > 0 ? (int)wh64 : 0;
        const int ntile = (hi + KT - 1) / KT;

        v8h qf[kI8D / 16];
        float qs = 0.f;
        {
            const f16 *src = a.q + (ok ? orow : 0) * kI8D + 8 * g;
#pragma unroll
            for (int kk = 0; kk < kI8D / 16; ++kk) {
                const v8h x = *reinterpret_cast<const v8h *>(src + 16 * kk);
                qf[kk] = lim > 0 ? x * (f16)a.qmul : (v8h)(f16)0;
#pragma unroll
                for (int e = 0; e < 8; ++e) qs += (float)qf[kk][e];
            }
            qs += __shfl_xor(qs, 32);
            qs *= -0x1p-17f;   // -128 sum(q) 2^-24, what K's codes + 128 add to a score
        }
        v16f o[kI8D / 32];
#pragma unroll
        for (int i = 0; i < kI8D / 32; ++i) o[i] = (v16f)0.f;
        float m = -INFINITY, l = 0.f;

        // staging: wave w -> the tile's w-th block of 16 keys, KB bytes of a row's K
        // and V codes a lane; the block's place is the same for the whole wave, so
        // its arithmetic is scalar
        const int kr = tid / KR, kd = (tid % KR) * KB;
        const int64_t v_part = (int64_t)p.H * p.page * kI8D;
        const uint32_t in_block = (kr & (kI8Block - 1)) * kI8D + kd;
        v4i kx[KB / 16], vx[KB / 16];
        float ksc = 0.f, vsc = 0.f;
        bool there = false;
        int page_next = -1;                          // in every lane
        int slot = wave / p.bpp, in_page = wave - slot * p.bpp, in_next = 0;
        // the page of the wave's block of tile t, looked up in order of t
        auto find = [&](int t) __attribute__((always_inline)) {
            const bool in = t < ntile && (t * (KT / kI8Block) + wave) * kI8Block < hi;
            page_next = in ? p.indices[rq.first + slot] : -1;
            in_next = in_page;
            in_page += KT / kI8Block;
            while (in_page >= p.bpp) {
                in_page -= p.bpp;
                ++slot;
            }
        };
        auto load_tile = [&]() __attribute__((always_inline)) {
            const int64_t pg = __builtin_amdgcn_readfirstlane(page_next);
            there = pg >= 0 && pg < p.pages;
            const int64_t at = there ? i8_scale_index(p, pg, hk, in_next) : 0;
            const int8_t *kb = p.data + at * (kI8Block * kI8D) + in_block;
            const int8_t *vb = kb + v_part;
#pragma unroll
            for (int i = 0; i < KB / 16; ++i) {
                kx[i] = *reinterpret_cast<const v4i *>(kb + 16 * i);
                vx[i] = *reinterpret_cast<const v4i *>(vb + 16 * i);
            }
            ksc = p.scale[at];
            vsc = p.scale[at + (int64_t)p.H * p.bpp];
        };
        auto store_tile = [&](int buf) __attribute__((always_inline)) {
            f16 *kd_ = &Ks_[buf][kr * KS + kd], *vd_ = &Vs_[buf][kr * VR + kd];
#pragma unroll
            for (int i = 0; i < KB / 16; ++i) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    *reinterpret_cast<v8h *>(kd_ + 16 * i + 8 * h) =
                        codes8((u32)kx[i][2 * h], (u32)kx[i][2 * h + 1]);
                    *reinterpret_cast<v8h *>(vd_ + 16 * i + 8 * h) =
                        signed8((u32)vx[i][2 * h], (u32)vx[i][2 * h + 1]);
                }
            }
            if (lane == 0) {
                BlockScale s;
                // (a block of zeros: any factor, but -inf * 0 would not be -inf)
                s.kc = there ? (ksc != 0.f ? ksc : 0x1p-100f) * a.c * 0x1p24f : 0.f;
                s.lv = there ? log_scale(vsc) : -INFINITY;
                s.rv = there ? inv_scale(vsc) : 0.f;
                s.pad = 0.f;
                Bs_[buf][wave] = s;
            }
        };

        if (ntile > 0) {
            find(0);
            load_tile();
            find(1);
            store_tile(0);
        }
        __syncthreads();
        for (int t = 0; t < ntile; ++t) {
            const int k0 = t * KT, buf = t & 1;
            const f16 *Ks = Ks_[buf];
            const f16 *Vs = Vs_[buf];
            if (t + 1 < ntile) {
                load_tile();    // in flight during this tile's products
                find(t + 2);
            }
            [&]() __attribute__((always_inline)) {
                if (k0 >= wave_hi) return;      // no key of this tile is visible
                v16f s[2];
#pragma unroll
                for (int sb = 0; sb < 2; ++sb) {
                    s[sb] = (v16f)0.f;
                    const f16 *row = &Ks[(32 * sb + ln) * KS + 8 * g];
#pragma unroll
                    for (int kk = 0; kk < kI8D / 16; ++kk) {
                        const v8h kf = *reinterpret_cast<const v8h *>(row + 16 * kk);
                        s[sb] = mfma32(kf, qf[kk], s[sb]);
                    }
                }
                // the K operand reads run 4 ahead of the products that take them
                __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
                for (int i = 0; i < 12; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
                BlockScale bs[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) bs[i] = Bs_[buf][i];
                if (k0 + KT > lo) {
                    // A block that this row does not see, or that is not there,
                    // may hold any scale: its exponents become 0 * 0 - inf.
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool seen = k0 + 16 * i < lim && bs[i].lv != -INFINITY;
                        const float out = seen ? -INFINITY : 0.f;
                        bs[i].kc = seen ? bs[i].kc : 0.f;
                        bs[i].lv = seen ? bs[i].lv : -INFINITY;
#pragma unroll
                        for (int v = 0; v < 8; ++v) {
                            const int key = k0 + 16 * i + 8 * (v / 4) + 4 * g + (v % 4);
                            const int at = 8 * (i % 2) + v;
                            s[i / 2][at] = seen && key < lim ? s[i / 2][at] : out;
                        }
                    }
                }
                // the largest exponent: scales are positive, so a block's largest
                // score is its largest exponent
                float mt = -INFINITY;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float mb = -INFINITY;
#pragma unroll
                    for (int v = 0; v < 8; ++v) mb = fmaxf(mb, s[i / 2][8 * (i % 2) + v]);
                    mt = fmaxf(mt, __builtin_fmaf(mb + qs, bs[i].kc, bs[i].lv));
                }
                mt = fmaxf(mt, __shfl_xor(mt, 32));
                const bool grow = mt > m + kSlack;
                if (__builtin_amdgcn_ballot_w64(grow)) {
                    const float f = grow ? __builtin_amdgcn_exp2f(m - mt) : 1.f;
                    m = grow ? mt : m;
                    l *= f;
#pragma unroll
                    for (int i = 0; i < kI8D / 32; ++i) o[i] *= f;
                }
                const float sub = m == -INFINITY ? 0.f : m;
                v8h pb[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float kc = bs[i].kc, add = __builtin_fmaf(qs, kc, bs[i].lv - sub);
                    float ps0 = 0.f, ps1 = 0.f;
#pragma unroll
                    for (int v = 0; v < 8; ++v) {
                        const float x = s[i / 2][8 * (i % 2) + v];
                        const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(x, kc, add));
                        if (v & 1) ps1 += pr; else ps0 += pr;
                        pb[i][v] = (f16)pr;
                    }
                    const float sum = ps0 + ps1;
                    if (sum != 0.f) l = __builtin_fmaf(sum, bs[i].rv, l);
                }
#pragma unroll
                for (int st = 0; st < 4; ++st)
#pragma unroll
                    for (int db = 0; db < kI8D / 32; ++db) {
                        const f16 *vr = &Vs[(16 * st + 4 * g + ((lane & 15) >> 2)) * VR + 32 * db +
                                            16 * ((lane >> 4) & 1) + 4 * (lane & 3)];
                        v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) v4s *)vr);
                        v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) v4s *)(vr + 8 * VR));
                        const v4h xh = __builtin_bit_cast(v4h, x), yh = __builtin_bit_cast(v4h, y);
                        const v8h av = {xh[0], xh[1], xh[2], xh[3], yh[0], yh[1], yh[2], yh[3]};
                        o[db] = mfma32(av, pb[st], o[db]);
                    }
            }();
            if (t + 1 < ntile) store_tile(buf ^ 1);
            __syncthreads();
        }
        l += __shfl_xor(l, 32);
        if (ok) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            f16 *to = a.o + orow * kI8D;
#pragma unroll
            for (int db = 0; db < kI8D / 32; ++db)
#pragma unroll
                for (int grp = 0; grp < 4; ++grp) {
                    v4h x;
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = (f16)(o[db][4 * grp + i] * inv);
                    *reinterpret_cast<v4h *>(to + 32 * db + 8 * grp + 4 * g) = x;
                }
        }
    }
}

// Join of the chunks: a block of 4 waves per (row, head), each wave a quarter of
// the chunks, two dims per lane.  Lane c of a wave holds chunk c's maximum and
// sum, so the weights need one reduction; the records are then read with all
// loads in flight.
SRQ_DEV void merge_row(const AttnI8Args &a, int64_t row, float (&sx)[4][kI8D], float (&sm)[4],
                       float (&ss)[4]) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const float *rec = a.tmp + row * a.chunks * kRec;
    float m = -INFINITY, x = 0.f, y = 0.f, sum = 0.f;
    const int per = (a.chunks + 3) / 4, end = min(a.chunks, (wave + 1) * per);
    for (int c0 = wave * per; c0 < end; c0 += 64) {
        const int c = c0 + lane;
        float mc = -INFINITY, lc = 0.f;
        if (c < end) {
            const float2 v = *reinterpret_cast<const float2 *>(rec + (int64_t)c * kRec + kI8D);
            mc = v.x;
            lc = v.y;
        }
        const float to = fmaxf(m, wave_max(mc));
        const float f = m == to ? 1.f : __builtin_amdgcn_exp2f(m - to);
        // an empty chunk's record is zeros; NaN stays NaN
        const float w = mc == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mc - to);
        m = to;
        sum = __builtin_fmaf(sum, f, wave_sum(lc * w));
        x *= f;
        y *= f;
        const int n = min(64, end - c0);
        const float *r = rec + (int64_t)c0 * kRec + 2 * lane;
        for (int i0 = 0; i0 < n; i0 += 8) {
            float2 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)   // past the end: the last record, weight 0
                v[i] = *reinterpret_cast<const float2 *>(r + (int64_t)min(i0 + i, n - 1) * kRec);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float wi = i0 + i < n ? read_lane(w, i0 + i) : 0.f;
                x = __builtin_fmaf(v[i].x, wi, x);
                y = __builtin_fmaf(v[i].y, wi, y);
            }
        }
    }
    sx[wave][2 * lane] = x;
    sx[wave][2 * lane + 1] = y;
    if (lane == 0) {
        sm[wave] = m;
        ss[wave] = sum;
    }
    __syncthreads();
    if (wave) return;   // to the caller's barrier
    const float mx = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    x = y = sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float f = sm[w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm[w] - mx);
        sum = __builtin_fmaf(ss[w], f, sum);
        x = __builtin_fmaf(sx[w][2 * lane], f, x);
        y = __builtin_fmaf(sx[w][2 * lane + 1], f, y);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    reinterpret_cast<v2h *>(a.o + row * kI8D)[lane] = (v2h){(f16)(x * inv), (f16)(y * inv)};
}

constexpr int64_t kMergeBlocks = 1 << 20;

__global__ __launch_bounds__(256) void attn_i8_merge_kernel(AttnI8Args a, int64_t batch) {
    __shared__ float sx[4][kI8D], sm[4], ss[4];
    int64_t lo = 0, hi = a.rows;   // rows of the requests
    if (a.q_indptr) {
        lo = a.q_indptr[0];
        lo = lo < 0 ? 0 : lo;
        hi = a.q_indptr[batch];
        hi = hi > a.rows ? a.rows : hi;
    }
    for (int64_t row = lo * a.hq + blockIdx.x; row < hi * a.hq; row += gridDim.x) {
        merge_row(a, row, sx, sm, ss);
        __syncthreads();   // before the next row's parts
    }
}

// Kernel, row tiles and chunks of a request, from the sizes alone.  us on one
// MI355X, B x (cached + new tokens), query / KV heads; "rows" are new tokens x
// group.
//  * Up to 16 rows, attn_i8_kernel<1>; a request and KV head is split until there
//    is a block per CU (256), into pieces of 512 tokens or more: 8 x 2048 tokens
//    over 8 heads in 1 / 2 / 4 / 8 chunks 19.8 / 15.9 / 13.9 / 15.1, 1 x 4096 33.8 /
//    22.3 / 15.3 / 12.7, 1 x 60000 in 16 / 24 / 32 / 48 / 64 chunks 41 / 34 / 37 / 45 /
//    45; 32 x 4096 (256 blocks) unsplit 45.2, in two 45.9.
//  * Where blocks of 128 rows fill the CUs, attn_i8_rows_kernel, unsplit: 4 x (5000 + 512),
//    32 / 8 heads, 182 against 267 for the next form; 1 x 2048 new 79 against 102; at
//    256 blocks, 2 x (1000 + 256) of 64 / 8 heads, 37.5 against 44.8.
//  * Otherwise attn_i8_kernel<2>, four times as many blocks: 1 x (5000 + 512) 90
//    against 158 (94 with the 128-row form in 4 chunks), 2 x (2000 + 128) of 64 / 8
//    heads 34 against 65; split below 256 blocks until there are 512: 4 x (8000 + 8)
//    in 2 / 4 / 8 / 16 chunks 55 / 35 / 28 / 37, 8 x (3000 + 8) 31 / 28.5 / 34 in 2 / 4 / 8
//    (256 blocks, 2 x (1000 + 128) over 32 heads: unsplit 20.4, in two 28.6).
constexpr int64_t kMaxBlocks = 1 << 18;
enum { kRows16, kRows32, kRows128 };
struct Plan {
    int form, tiles, chunks;
};

Plan plan_of(int64_t n_rows, int64_t batch, int64_t group, int64_t H, int64_t max_q,
             int64_t max_kv) {
    constexpr int64_t kCUs = 256;
    // (the largest request has at least the mean and at most all, whatever the
    // caller says)
    const int64_t rows = std::max(std::min(max_q, n_rows), srq_cdiv(n_rows, batch)) * group;
    Plan pl;
    pl.form = rows <= 16 ? kRows16
              : batch * H * srq_cdiv(rows, kRowsBlock) >= kCUs ? kRows128 : kRows32;
    int64_t tiles = srq_cdiv(rows, pl.form == kRows16 ? 16 : pl.form == kRows32 ? 32 : kRowsBlock);
    // no swarm of empty blocks where many uneven requests come without a hint; the
    // kernels' loops reach the rest
    tiles = std::min(tiles, std::max<int64_t>(64, kMaxBlocks / (batch * H)));
    const int64_t blocks = batch * H * tiles;
    int64_t chunks = 1;
    if (blocks < kCUs) {
        chunks = srq_cdiv(pl.form == kRows16 ? kCUs : 2 * kCUs, blocks);
        const int64_t most = max_kv / 512 < 1 ? 1 : max_kv / 512;
        if (chunks > most) chunks = most;
    }
    pl.tiles = (int)tiles;
    pl.chunks = (int)chunks;
    return pl;
}

}  // namespace

extern "C" int srq_batch_attention_i8_workspace(int64_t rows, int64_t batch, int64_t n_q_heads,
                                               int64_t n_kv_heads, int64_t max_q_len,
                                               int64_t max_kv_len, int64_t *bytes) {
    SRQ_CHECK_ARG(bytes, "batch_attention_i8_workspace: null pointer");
    SRQ_CHECK_ARG(rows >= 0 && batch >= 0 && n_kv_heads > 0 && n_q_heads > 0 &&
                      n_q_heads % n_kv_heads == 0,
                  "batch_attention_i8: %lld query heads for %lld KV heads", (long long)n_q_heads,
                  (long long)n_kv_heads);
    *bytes = 0;
    if (rows == 0 || batch == 0) return SRQ_OK;
    const Plan pl =
        plan_of(rows, batch, n_q_heads / n_kv_heads, n_kv_heads, max_q_len, max_kv_len);
    if (pl.chunks > 1) *bytes = rows * n_q_heads * pl.chunks * kRec * 4;
    return SRQ_OK;
}

extern "C" int srq_batch_attention_i8(
    void *o, const void *q, int64_t rows, int64_t n_q_heads, const void *kv_data,
    const void *kv_scale, const int32_t *kv_indptr, const int32_t *kv_indices,
    const int32_t *last_page_offset, int64_t pages, int64_t n_indices, int64_t batch,
    int64_t num_layers, int64_t layer_idx, int64_t num_kv_heads, int64_t page_size,
    int64_t head_dim, const int32_t *q_indptr, int64_t max_q_len, int64_t max_kv_len,
    float sm_scale, void *ws, int64_t ws_bytes, void *stream) {
    PagedI8 p{};
    const int rc = i8_check("batch_attention_i8", kv_data, kv_scale, kv_indptr, kv_indices,
                            last_page_offset, pages, n_indices, batch, num_layers, layer_idx,
                            num_kv_heads, page_size, head_dim, p);
    if (rc != SRQ_OK) return rc;
    SRQ_CHECK_ARG(n_q_heads > 0 && n_q_heads <= 65536 && n_q_heads % num_kv_heads == 0,
                  "batch_attention_i8: %lld query heads for %lld KV heads", (long long)n_q_heads,
                  (long long)num_kv_heads);
    SRQ_CHECK_ARG(rows >= 0 && (q_indptr || rows == batch),
                  "batch_attention_i8: %lld rows for %lld requests", (long long)rows,
                  (long long)batch);
    SRQ_CHECK_ARG(rows <= 0x7fffffff / n_q_heads, "batch_attention_i8: rows x heads >= 2^31");
    // (its products with a block's scale, 2^24 and 2^-100 stay normal numbers)
    SRQ_CHECK_ARG(sm_scale == 0.f || (fabsf(sm_scale) >= 0x1p-20f && fabsf(sm_scale) <= 0x1p60f),
                  "batch_attention_i8: sm_scale=%g is not a finite scale: 0, or 2^-20 to 2^60",
                  (double)sm_scale);
    if (batch == 0 || rows == 0) return SRQ_OK;
    SRQ_CHECK_ARG(o && q, "batch_attention_i8: null pointer");
    SRQ_CHECK_ARG(srq_aligned(o, 16) && srq_aligned(q, 16),
                  "batch_attention_i8: o and q must be 16-byte aligned");
    const int64_t group = n_q_heads / num_kv_heads;
    const Plan pl = plan_of(rows, batch, group, num_kv_heads, max_q_len, max_kv_len);
    int64_t need = 0;
    if (pl.chunks > 1) need = rows * n_q_heads * pl.chunks * kRec * 4;
    SRQ_CHECK_ARG(need == 0 || (ws && ws_bytes >= need && srq_aligned(ws, 16)),
                  "batch_attention_i8: workspace of %lld bytes, 16-byte aligned, is needed",
                  (long long)need);
    AttnI8Args a{};
    a.q = (const f16 *)q;
    a.o = (f16 *)o;
    a.q_indptr = q_indptr;
    a.tmp = (float *)ws;
    a.rows = rows;
    a.hq = (int)n_q_heads;
    a.group = (int)group;
    a.chunks = pl.chunks;
    a.tiles = pl.tiles;
    // the sign of the scale goes into q, so that a larger product is a larger score
    a.c = (sm_scale == 0.f ? 1.f : fabsf(sm_scale)) * 1.4426950408889634f;
    a.qmul = sm_scale > 0.f ? 1.f : sm_scale < 0.f ? -1.f : 0.f;
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)(pl.chunks * pl.tiles), (unsigned)num_kv_heads, (unsigned)batch);
    switch (pl.form) {
    case kRows16: attn_i8_kernel<1><<<grid, kWaves * 64, 0, st>>>(a, p); break;
    case kRows32: attn_i8_kernel<2><<<grid, kWaves * 64, 0, st>>>(a, p); break;
    default: attn_i8_rows_kernel<<<grid, kWaves * 64, 0, st>>>(a, p); break;
    }
    if (pl.chunks > 1)
        attn_i8_merge_kernel<<<(unsigned)std::min(rows * n_q_heads, kMergeBlocks), 256, 0, st>>>(
            a, batch);
    SRQ_LAUNCH_CHECK("batch_attention_i8");
    return SRQ_OK;
}
