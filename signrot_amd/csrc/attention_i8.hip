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
// so out = O / l with codes as integers throughout.  p' is rounded to fp16 for
// the product; m (the running maximum of the exponent) moves only when a score
// exceeds it by more than 8, so p' <= 2^8.
//
// The waves of a block take 32-token tiles in turn and are joined through LDS;
// a request is split over blocks (chunks) when there are few, whose partial
// (O, m, l) a second kernel joins.
#include "kv_i8.h"

#include <math.h>

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

// 8 int8 codes -> fp16, in order
SRQ_DEV v8h codes8(u32 a, u32 b) {
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

struct Tile {
    v4i k[2][2];   // [block][half of the dims]
    uint2 v[8];    // tokens of the lane's slots
};

SRQ_DEV int read_lane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
SRQ_DEV float read_lane(float v, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// RT row tiles of 16 rows per block
template <int RT>
__global__ __launch_bounds__(kWaves * 64) void attn_i8_kernel(AttnI8Args a, PagedI8 p) {
    __shared__ float so[kWaves][16][kI8D + 4];
    __shared__ float sm[kWaves][16], sl[kWaves][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
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
#pragma unroll
            for (int s = 0; s < 4; ++s)
                qf[t][s] = *reinterpret_cast<const v8h *>(src + 64 * (s >> 1) + 8 * (s & 1)) *
                           (f16)a.qmul;
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

        // The wave's tiles are t_lo + wave, + kWaves, ...; lane j looks up the
        // page and the scales of block j of the next 64 (32 tiles).
        for (int base = t_lo + wave; base < t_hi; base += 32 * kWaves) {
            const int mine = base + (lane >> 1) * kWaves;
            const int blk = 2 * mine + (lane & 1);
            int pg = -1;
            float ks = 0.f, vs = 0.f;
            uint32_t in_page = 0;
            if (mine < t_hi && blk * kI8Block < hi) {
                pg = (int)i8_page(p, rq.first, blk);
                in_page = (uint32_t)blk % (uint32_t)p.bpp;
                if (pg >= 0) {
                    const int64_t si = i8_scale_index(p, pg, hk, in_page);
                    ks = p.scale[si];
                    vs = p.scale[si + (int64_t)p.H * p.bpp];
                }
            }
            const float lv = vs != 0.f ? __builtin_amdgcn_logf(vs) : 0.f;
            const float rv = vs != 0.f ? 1.f / vs : 1.f;
            ks *= a.c;

            auto load = [&](Tile &x, int j) __attribute__((always_inline)) {
#pragma unroll
                for (int bk = 0; bk < 2; ++bk) {
                    const int pgj = read_lane(pg, 2 * j + bk);
                    const uint32_t in = (uint32_t)read_lane((int)in_page, 2 * j + bk);
                    const int8_t *kb =
                        p.data + i8_scale_index(p, pgj < 0 ? 0 : pgj, hk, in) * (kI8Block * kI8D);
                    const int8_t *vb = kb + (int64_t)p.H * p.page * kI8D;
                    const int8_t *kr = kb + col * kI8D + 16 * g;
                    x.k[bk][0] = *reinterpret_cast<const v4i *>(kr);
                    x.k[bk][1] = *reinterpret_cast<const v4i *>(kr + 64);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        x.v[4 * bk + e] =
                            *reinterpret_cast<const uint2 *>(vb + (4 * g + e) * kI8D + 8 * col);
                }
            };
            auto step = [&](const Tile &x, int j) __attribute__((always_inline)) {
                const int tok = (base + j * kWaves) * kTileTok;
                v8h pb[RT];
                v4f s[RT][2];
#pragma unroll
                for (int t = 0; t < RT; ++t) s[t][0] = s[t][1] = (v4f)0.f;
#pragma unroll
                for (int bk = 0; bk < 2; ++bk)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const v4i w = x.k[bk][q >> 1];
                        const v8h kf = codes8((u32)w[2 * (q & 1)], (u32)w[2 * (q & 1) + 1]);
#pragma unroll
                        for (int t = 0; t < RT; ++t) s[t][bk] = mfma16(kf, qf[t][q], s[t][bk]);
                    }
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
                }
            };
            const int cnt = min(32, (t_hi - base + kWaves - 1) / kWaves);
            for (int j = 0; j < cnt; ++j) {
                Tile x;
                load(x, j);
                step(x, j);
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
            if (r < nrows) {
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

// Join of the chunks: a wave per (row, head), two dims per lane.
__global__ __launch_bounds__(256) void attn_i8_merge_kernel(AttnI8Args a, int64_t batch) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    int64_t lo = 0, hi = a.rows;   // rows of the requests
    if (a.q_indptr) {
        lo = a.q_indptr[0];
        hi = a.q_indptr[batch];
        hi = hi > a.rows ? a.rows : hi;
    }
    if (row < lo * a.hq || row >= hi * a.hq) return;
    const float *rec = a.tmp + row * a.chunks * kRec;
    float mx = -INFINITY;
    for (int c = 0; c < a.chunks; ++c) mx = fmaxf(mx, rec[(int64_t)c * kRec + kI8D]);
    float x = 0.f, y = 0.f, sum = 0.f;
    for (int c = 0; c < a.chunks; ++c) {
        const float *r = rec + (int64_t)c * kRec;
        const float mc = r[kI8D];
        const float f = mc == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mc - mx);
        sum = __builtin_fmaf(r[kI8D + 1], f, sum);
        x = __builtin_fmaf(r[2 * lane], f, x);
        y = __builtin_fmaf(r[2 * lane + 1], f, y);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    reinterpret_cast<v2h *>(a.o + row * kI8D)[lane] = (v2h){(f16)(x * inv), (f16)(y * inv)};
}

// Row tiles per block and chunks of a request.
struct Plan {
    int rt, tiles, chunks;
};

Plan plan_of(int64_t batch, int64_t group, int64_t H, int64_t max_q, int64_t max_kv) {
    const int64_t rows = (max_q < 1 ? 1 : max_q) * group;
    Plan pl;
    pl.rt = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    int64_t tiles = srq_cdiv(rows, 16 * pl.rt);
    if (tiles > 65536) tiles = 65536;
    pl.tiles = (int)tiles;
    const int64_t blocks = batch * H * tiles;
    int64_t chunks = 1;
    if (blocks < 256) {
        chunks = srq_cdiv(512, blocks);
        const int64_t most = max_kv / 256 < 1 ? 1 : max_kv / 256;
        if (chunks > most) chunks = most;
    }
    pl.chunks = (int)chunks;
    return pl;
}

}  // namespace

extern "C" int srq_batch_attention_i8_ws_bytes(int64_t rows, int64_t batch, int64_t n_q_heads,
                                               int64_t n_kv_heads, int64_t max_q_len,
                                               int64_t max_kv_len, int64_t *bytes) {
    SRQ_CHECK_ARG(bytes, "batch_attention_i8_ws_bytes: null pointer");
    SRQ_CHECK_ARG(rows >= 0 && batch >= 0 && n_kv_heads > 0 && n_q_heads > 0 &&
                      n_q_heads % n_kv_heads == 0,
                  "batch_attention_i8: %lld query heads for %lld KV heads", (long long)n_q_heads,
                  (long long)n_kv_heads);
    *bytes = 0;
    if (rows == 0 || batch == 0) return SRQ_OK;
    const Plan pl = plan_of(batch, n_q_heads / n_kv_heads, n_kv_heads, max_q_len, max_kv_len);
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
    SRQ_CHECK_ARG(__builtin_isfinite(sm_scale), "batch_attention_i8: sm_scale is not finite");
    if (batch == 0 || rows == 0) return SRQ_OK;
    SRQ_CHECK_ARG(o && q, "batch_attention_i8: null pointer");
    SRQ_CHECK_ARG(srq_aligned(o, 16) && srq_aligned(q, 16),
                  "batch_attention_i8: o and q must be 16-byte aligned");
    const int64_t group = n_q_heads / num_kv_heads;
    const Plan pl = plan_of(batch, group, num_kv_heads, max_q_len, max_kv_len);
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
    switch (pl.rt) {
    case 1: attn_i8_kernel<1><<<grid, kWaves * 64, 0, st>>>(a, p); break;
    case 2: attn_i8_kernel<2><<<grid, kWaves * 64, 0, st>>>(a, p); break;
    default: attn_i8_kernel<4><<<grid, kWaves * 64, 0, st>>>(a, p); break;
    }
    if (pl.chunks > 1)
        attn_i8_merge_kernel<<<(unsigned)srq_cdiv(rows * n_q_heads, 4), 256, 0, st>>>(a, batch);
    SRQ_LAUNCH_CHECK("batch_attention_i8");
    return SRQ_OK;
}
