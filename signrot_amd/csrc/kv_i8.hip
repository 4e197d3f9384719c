// Writing the paged int8 KV cache: new keys and values, one token per request
// or any number, with the q/k norm and the rotary embedding in the same pass
// where they come straight from the projection.
//
// A block of 16 tokens of one head shares a scale, so its tokens cannot be
// quantized one by one: a wave takes one block of one head (of K or of V), 16
// lanes per token row and 8 values per lane, reduces the new tokens' largest
// magnitude over the wave and needs no LDS and no other wave.  With
//   s = max(s_old, fp32(max|new| * fp32(1 / 127)))   s_old = 0 for a block without
// older tokens, new codes are rne(x / s), and where s grew the older codes
// follow, c -> rne(c s_old / s), instead of being clipped.  Each growth rounds them
// anew, by up to half a step of that time: a token is off by half a step when its
// block came in one piece and by up to half a step more for every growth behind it,
// 8 in the worst order of 16 single tokens.  Normal values one token at a time: 2.5
// growths a block, its largest error 1.2 steps on average (2.4 in 400 blocks), its
// rms error 25% above that of one piece; where one channel grows by 1% a token, codes
// below 50 stand still and so grow with the scale, 6.5 steps.  A NaN or an infinity among the
// new values makes the scale NaN: the block reads as NaN until it is started
// anew.
//
// Roundings are decided as in exact arithmetic: the fp32 quotient is off by
// under 2^-15 here (|quotient| <= 127), so only one that lies closer than
// 2^-14 to a half is divided again in 64 bits, where the quotient of an
// 8-bit code or an fp16 value times a 24-bit scale is never that close
// without being a tie.
//
// A wave's chain of dependent loads bounds it (row index, table, block, scale), and
// with many tokens HBM: 6500 tokens of 8 heads, 40 MB, 12.6 us, 3.2 TB/s; one token
// for each of 32 requests 4.5 us, of 16 with norm and rotation 5.6; 2048 tokens
// with them and 32 query heads, 49 MB, 13.6 us, 3.6 TB/s.
#include "kv_i8.h"
#include "qk_norm.h"

#include <algorithm>

namespace {

struct AppendArgs {
    const f16 *k, *v;              // [rows, H, 128] with these token strides (elements)
    int64_t k_tok, v_tok, rows;
    const int32_t *new_indptr;     // [B + 1] or null: one row per request
    int kv_blocks;                 // grid.x of the K / V part
    // the fused form
    const f16 *q;                  // [rows, hq, 128], token stride k_tok
    f16 *q_out;                    // dense
    const f16 *cs, *sn;            // [rows or 1, 128]
    const f16 *qw, *kw;
    int hq, cos_one, norm;
    float eps;
};

// rne(f num / den) of eight values, |f num / den| <= 127 (and under 128 with the
// fp32 quotient's error), packed; r = num / den in fp32.  Adding 1.5 2^23 rounds to
// nearest and leaves the code in the low byte; what the quotient then is off its
// code tells the ones that lie near a half.
SRQ_DEV uint2 codes_row(const float (&f)[8], float r, double num, double den) {
    constexpr float kMagic = 12582912.f, kNear = 0.5f - 0x1p-14f;
    float y[8];
    bool near = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float t = f[e] * r;
        y[e] = t + kMagic;
        near |= fabsf(t - (y[e] - kMagic)) > kNear;
    }
    if (__builtin_amdgcn_ballot_w64(near)) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (fabsf(f[e] * r - (y[e] - kMagic)) > kNear)
                y[e] = (float)__builtin_rint(f[e] * num / den) + kMagic;
    }
    u32 w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        u32 u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = __builtin_bit_cast(u32, y[4 * h + e]);
        const u32 lo = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u);
        const u32 hi = __builtin_amdgcn_perm(u[3], u[2], 0x04000c0cu);
        w[h] = lo | hi;
    }
    return make_uint2(w[0], w[1]);
}

template <bool FUSED>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a, PagedI8 p) {
    const int64_t b = blockIdx.y;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int l = lane & 15, r4 = lane >> 4;
    int64_t s0, n;
    i8_new_rows(a.new_indptr, b, a.rows, s0, n);
    if constexpr (FUSED) {
        if ((int)blockIdx.x >= a.kv_blocks) {
            // q rows: a block per token at a time, 16 rows at once
            v8h one;
#pragma unroll
            for (int e = 0; e < 8; ++e) one[e] = (f16)1.f;
            const v8h w = a.qw ? *reinterpret_cast<const v8h *>(a.qw + 8 * l) : one;
            const int64_t step = gridDim.x - a.kv_blocks;
            for (int64_t i = blockIdx.x - a.kv_blocks; i < n; i += step) {
                const int64_t row = s0 + i, ct = (a.cos_one ? 0 : row) * kI8D + 8 * l;
                const v8h c = *reinterpret_cast<const v8h *>(a.cs + ct);
                const v8h s = *reinterpret_cast<const v8h *>(a.sn + ct);
                for (int h0 = 0; h0 < a.hq; h0 += 16) {
                    const int h = h0 + (threadIdx.x >> 4);
                    v8h x = {};
                    if (h < a.hq)
                        x = *reinterpret_cast<const v8h *>(a.q + row * a.k_tok + h * kI8D + 8 * l);
                    x = qk_norm_rope_row<16>(x, w, c, s, l, a.eps, a.norm);
                    if (h < a.hq)
                        *reinterpret_cast<v8h *>(a.q_out + (row * a.hq + h) * kI8D + 8 * l) = x;
                }
            }
            return;
        }
    }
    if (n == 0) return;
    const I8Request rq = i8_request(p, b);
    const int64_t old = rq.len - n;                    // tokens held before (below 0: no room)
    const int64_t j0 = (old > 0 ? old : 0) / kI8Block;
    const int64_t items = (srq_cdiv(rq.len, kI8Block) - j0) * 2 * p.H;
    for (int64_t it = (int64_t)blockIdx.x * 4 + wave; it < items; it += (int64_t)a.kv_blocks * 4) {
        const int64_t jj = (uint32_t)it / (uint32_t)(2 * p.H);
        const int hv = (int)(it - jj * 2 * p.H), kv = hv / p.H, h = hv - kv * p.H;
        const int64_t j = j0 + jj, t0 = j * kI8Block;
        const int held = (int)(old > t0 ? old - t0 : 0);   // older tokens of the block
        const int fill = (int)(rq.len - t0 < kI8Block ? rq.len - t0 : kI8Block);
        const f16 *src = kv ? a.v : a.k;
        const int64_t tok = kv ? a.v_tok : a.k_tok;
        // the new rows first: the table's dependent reads overlap them (a row that is
        // not new reads the block's first one that is)
        v8h x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = 4 * i + r4;                       // row of the block
            const int64_t row = s0 + t0 + (e >= held && e < fill ? e : held) - old;
            x[i] = *reinterpret_cast<const v8h *>(src + row * tok + h * kI8D + 8 * l);
        }
        const int64_t pg = i8_page(p, rq.first, j);
        if (pg < 0) continue;
        const int64_t si = i8_scale_index(p, pg, h, (uint32_t)j % (uint32_t)p.bpp) +
                           (int64_t)kv * p.H * p.bpp;
        int8_t *codes = p.data + si * (kI8Block * kI8D);   // a block's rows are consecutive
        const float was = held > 0 ? p.scale[si] : 0.f;
        float amax = 0.f;
        bool bad = !(was <= 3e38f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = 4 * i + r4;
            const bool fresh = e >= held && e < fill;
            const int64_t row = s0 + t0 + e - old;
            if (!fresh) x[i] = (v8h){};
            if (FUSED && kv == 0) {
                const int64_t ct = (a.cos_one || !fresh ? 0 : row) * kI8D + 8 * l;
                const v8h c = *reinterpret_cast<const v8h *>(a.cs + ct);
                const v8h s = *reinterpret_cast<const v8h *>(a.sn + ct);
                v8h w;
#pragma unroll
                for (int d = 0; d < 8; ++d) w[d] = (f16)1.f;
                if (a.kw) w = *reinterpret_cast<const v8h *>(a.kw + 8 * l);
                const v8h y = qk_norm_rope_row<16>(x[i], w, c, s, l, a.eps, a.norm);
                if (fresh) x[i] = y;
            }
            amax = absmax8_flag(x[i], amax, bad);
        }
        amax = wave_max(amax);
        float now = fmaxf(was, amax * (1.f / 127.f));
        if (__builtin_amdgcn_ballot_w64(bad)) now = __builtin_nanf("");
        const bool live = now > 0.f;                        // false for NaN: codes 0
        const float rs = live ? 1.0f / now : 0.f;
        const float ratio = live ? was / now : 0.f;
        const bool moved = held > 0 && now != was;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = 4 * i + r4;
            uint2 *at = reinterpret_cast<uint2 *>(codes + e * kI8D + 8 * l);
            float f[8];
            if (e >= held && e < fill) {
#pragma unroll
                for (int d = 0; d < 8; ++d) f[d] = live ? (float)x[i][d] : 0.f;
                *at = codes_row(f, rs, 1.0, now);
            } else if (moved && e < held) {
                const uint2 o = *at;
#pragma unroll
                for (int d = 0; d < 8; ++d) {
                    const u32 w = d < 4 ? o.x : o.y;
                    f[d] = live ? (float)(int)(int8_t)(w >> (8 * (d & 3))) : 0.f;
                }
                *at = codes_row(f, ratio, was, now);
            }
        }
        if (lane == 0 && (held == 0 || now != was)) p.scale[si] = now;
    }
}

int launch_append(const char *name, bool fused, AppendArgs a, const PagedI8 &p, int64_t batch,
                  int64_t max_new, void *stream) {
    // a block is touched once by each of its heads' K and V waves; blocks
    // behind the hint are reached by the loop, and so are those behind a limit
    // that keeps many requests without a hint from a swarm of empty blocks
    const int64_t hint = std::max<int64_t>(1, std::min(max_new, a.rows));
    const int64_t most = std::max<int64_t>(64, (1 << 18) / batch);
    int64_t kvb = srq_cdiv((srq_cdiv(hint - 1, kI8Block) + 1) * 2 * p.H, 4);
    int64_t qb = fused ? hint : 0;
    kvb = std::min(kvb, most);
    qb = std::min(qb, most);
    a.kv_blocks = (int)kvb;
    const dim3 grid((unsigned)(kvb + qb), (unsigned)batch);
    if (fused)
        append_kernel<true><<<grid, 256, 0, (hipStream_t)stream>>>(a, p);
    else
        append_kernel<false><<<grid, 256, 0, (hipStream_t)stream>>>(a, p);
    SRQ_LAUNCH_CHECK(name);
    return SRQ_OK;
}

}  // namespace

extern "C" int srq_append_kv_i8(void *kv_data, void *kv_scale, const int32_t *kv_indptr,
                                const int32_t *kv_indices, const int32_t *last_page_offset,
                                int64_t pages, int64_t n_indices, int64_t batch,
                                int64_t num_layers, int64_t layer_idx, int64_t num_kv_heads,
                                int64_t page_size, int64_t head_dim, const void *k, const void *v,
                                int64_t k_tok_stride, int64_t v_tok_stride, int64_t rows,
                                const int32_t *new_indptr, int64_t max_new, void *stream) {
    PagedI8 p{};
    const int rc = i8_check("append_kv_i8", kv_data, kv_scale, kv_indptr, kv_indices,
                            last_page_offset, pages, n_indices, batch, num_layers, layer_idx,
                            num_kv_heads, page_size, head_dim, p);
    if (rc != SRQ_OK) return rc;
    SRQ_CHECK_ARG(rows >= 0 && rows <= 0x7fffffff && (new_indptr || rows == batch),
                  "append_kv_i8: %lld rows for %lld requests", (long long)rows, (long long)batch);
    if (batch == 0 || rows == 0) return SRQ_OK;
    SRQ_CHECK_ARG(k && v, "append_kv_i8: null pointer");
    SRQ_CHECK_ARG(k_tok_stride >= num_kv_heads * kI8D && v_tok_stride >= num_kv_heads * kI8D &&
                      k_tok_stride % 8 == 0 && v_tok_stride % 8 == 0,
                  "append_kv_i8: token strides must hold the heads and be multiples of 8");
    SRQ_CHECK_ARG(srq_aligned(k, 16) && srq_aligned(v, 16),
                  "append_kv_i8: k and v must be 16-byte aligned");
    AppendArgs a{};
    a.k = (const f16 *)k;
    a.v = (const f16 *)v;
    a.k_tok = k_tok_stride;
    a.v_tok = v_tok_stride;
    a.rows = rows;
    a.new_indptr = new_indptr;
    return launch_append("append_kv_i8", false, a, p, batch, max_new, stream);
}

extern "C" int srq_qkv_norm_rope_append_i8(
    void *kv_data, void *kv_scale, const int32_t *kv_indptr, const int32_t *kv_indices,
    const int32_t *last_page_offset, int64_t pages, int64_t n_indices, int64_t batch,
    int64_t num_layers, int64_t layer_idx, int64_t num_kv_heads, int64_t page_size,
    int64_t head_dim, const void *qkv, int64_t tok_stride, int64_t rows, const void *cos,
    const void *sin, int64_t cos_rows, int64_t n_q_heads, const void *q_weight,
    const void *k_weight, float eps, int norm, const int32_t *new_indptr, int64_t max_new,
    void *q_out, void *stream) {
    const char *name = "qkv_norm_rope_append_i8";
    PagedI8 p{};
    const int rc = i8_check(name, kv_data, kv_scale, kv_indptr, kv_indices, last_page_offset, pages,
                            n_indices, batch, num_layers, layer_idx, num_kv_heads, page_size,
                            head_dim, p);
    if (rc != SRQ_OK) return rc;
    SRQ_CHECK_ARG(rows >= 0 && rows <= 0x7fffffff && (new_indptr || rows == batch),
                  "%s: %lld rows for %lld requests", name, (long long)rows, (long long)batch);
    SRQ_CHECK_ARG(n_q_heads >= 0 && n_q_heads <= 65536, "%s: bad number of query heads", name);
    SRQ_CHECK_ARG(!norm || (eps >= 0.f && __builtin_isfinite(eps)),
                  "%s: eps must be finite and not negative", name);
    SRQ_CHECK_ARG(norm || (!q_weight && !k_weight), "%s: weights without a norm", name);
    SRQ_CHECK_ARG(cos_rows == 1 || cos_rows == rows, "%s: cos/sin must have 1 or %lld rows", name,
                  (long long)rows);
    if (batch == 0 || rows == 0) return SRQ_OK;
    SRQ_CHECK_ARG(qkv && cos && sin && (q_out || n_q_heads == 0), "%s: null pointer", name);
    SRQ_CHECK_ARG(tok_stride >= (n_q_heads + 2 * num_kv_heads) * kI8D && tok_stride % 8 == 0,
                  "%s: the token stride must hold the heads and be a multiple of 8", name);
    SRQ_CHECK_ARG(srq_aligned(qkv, 16) && srq_aligned(cos, 16) && srq_aligned(sin, 16) &&
                      srq_aligned(q_weight, 16) && srq_aligned(k_weight, 16) &&
                      srq_aligned(q_out, 16),
                  "%s: tensors must be 16-byte aligned", name);
    AppendArgs a{};
    a.q = (const f16 *)qkv;
    a.k = a.q + n_q_heads * kI8D;
    a.v = a.k + num_kv_heads * kI8D;
    a.k_tok = a.v_tok = tok_stride;
    a.rows = rows;
    a.new_indptr = new_indptr;
    a.q_out = (f16 *)q_out;
    a.cs = (const f16 *)cos;
    a.sn = (const f16 *)sin;
    a.qw = (const f16 *)q_weight;
    a.kw = (const f16 *)k_weight;
    a.hq = (int)n_q_heads;
    a.cos_one = cos_rows == 1;
    a.norm = norm ? 1 : 0;
    a.eps = eps;
    return launch_append(name, true, a, p, batch, max_new, stream);
}
