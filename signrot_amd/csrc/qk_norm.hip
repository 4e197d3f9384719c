// RMSNorm of each query and key head with the rotary embedding in the same
// pass, from the strided q / k columns of a projection output into dense
// outputs: every value is read once and written once, in place of a norm pass
// and a rotation pass (and the copies that make the columns dense).  HBM bounds it
// at many tokens (2048 of 64 + 8 heads of 128, 76.5 MB: 14.2 us, 5.4 TB/s), one load
// round trip and a row's reduction at few (32 tokens: 2.3 us in a graph).
#include "qk_norm.h"

namespace {

struct QkArgs {
    const f16 *q, *k;                     // [B, T, H, D], token and sequence strides below
    const f16 *cs, *sn;                   // [cos_batch, T, D]
    const f16 *qw, *kw;                   // [D] or null
    f16 *qo, *ko;                         // dense [B, T, H, D]
    int64_t q_tok, q_seq, k_tok, k_seq;   // strides in elements
    int64_t T;
    int cos_batch, hq, hk, norm;
    float eps;
};

// A block works on one token: its cos and sin slices and the weights stay in
// registers over the token's heads, and the divisions are done once.
template <int G>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(QkArgs a) {
    constexpr int D = 8 * G, R = 256 / G;   // rows at a time
    const int l = threadIdx.x % G, r = threadIdx.x / G;
    const int64_t tok = blockIdx.x;
    const int64_t b = tok / a.T, t = tok - b * a.T;
    const int64_t ct = (a.cos_batch == 1 ? t : tok) * D + 8 * l;
    const v8h c = *reinterpret_cast<const v8h *>(a.cs + ct);
    const v8h s = *reinterpret_cast<const v8h *>(a.sn + ct);
    v8h one;
#pragma unroll
    for (int e = 0; e < 8; ++e) one[e] = (f16)1.f;
    const v8h qw = a.qw ? *reinterpret_cast<const v8h *>(a.qw + 8 * l) : one;
    const v8h kw = a.kw ? *reinterpret_cast<const v8h *>(a.kw + 8 * l) : one;
    const f16 *qr = a.q + b * a.q_seq + t * a.q_tok + 8 * l;
    const f16 *kr = a.k + b * a.k_seq + t * a.k_tok + 8 * l;
    f16 *qo = a.qo + tok * a.hq * D + 8 * l;
    f16 *ko = a.ko + tok * a.hk * D + 8 * l;
    const int hs = a.hq + a.hk;
    for (int h0 = R * blockIdx.y; h0 < hs; h0 += R * gridDim.y) {
        const int h = h0 + r;
        const bool is_q = h < a.hq, valid = h < hs;
        const int hh = is_q ? h : h - a.hq;
        v8h x = {};
        if (valid) x = *reinterpret_cast<const v8h *>((is_q ? qr : kr) + (int64_t)hh * D);
        const v8h o = qk_norm_rope_row<G>(x, is_q ? qw : kw, c, s, l, a.eps, a.norm);
        if (valid) *reinterpret_cast<v8h *>((is_q ? qo : ko) + (int64_t)hh * D) = o;
    }
}

}  // namespace

extern "C" int srq_qk_norm_rope(const void *q, const void *k, const void *cos, const void *sin,
                                int64_t cos_batch, const void *q_weight, const void *k_weight,
                                float eps, int norm, int64_t batch, int64_t seq_len,
                                int64_t n_q_heads, int64_t n_kv_heads, int64_t head_dim,
                                int64_t q_tok_stride, int64_t q_seq_stride, int64_t k_tok_stride,
                                int64_t k_seq_stride, void *q_out, void *k_out, void *stream) {
    SRQ_CHECK_ARG(batch >= 0 && seq_len >= 0 && n_q_heads >= 0 && n_kv_heads >= 0,
                  "qk_norm_rope: bad shape");
    SRQ_CHECK_ARG(head_dim == 64 || head_dim == 128 || head_dim == 256,
                  "qk_norm_rope: head_dim=%lld, 64, 128 or 256 is supported", (long long)head_dim);
    SRQ_CHECK_ARG(cos_batch == 1 || cos_batch == batch,
                  "qk_norm_rope: cos/sin batch must be 1 or the batch");
    SRQ_CHECK_ARG(!norm || (eps >= 0.f && __builtin_isfinite(eps)),
                  "qk_norm_rope: eps must be finite and not negative");
    SRQ_CHECK_ARG(norm || (!q_weight && !k_weight), "qk_norm_rope: weights without a norm");
    if (batch == 0 || seq_len == 0 || n_q_heads + n_kv_heads == 0) return SRQ_OK;
    SRQ_CHECK_ARG(cos && sin && (n_q_heads == 0 || (q && q_out)) &&
                      (n_kv_heads == 0 || (k && k_out)),
                  "qk_norm_rope: null pointer");
    SRQ_CHECK_ARG(n_q_heads + n_kv_heads <= 65536, "qk_norm_rope: too many heads");
    // a block of 256 threads per token, and fewer than 2^32 threads a launch
    SRQ_CHECK_ARG(batch <= 0xffffff / seq_len, "qk_norm_rope: batch x seq_len >= 2^24");
    SRQ_CHECK_ARG(q_tok_stride >= n_q_heads * head_dim && k_tok_stride >= n_kv_heads * head_dim &&
                      q_seq_stride >= 0 && k_seq_stride >= 0,
                  "qk_norm_rope: strides smaller than the [H, D] extent");
    SRQ_CHECK_ARG(q_tok_stride % 8 == 0 && k_tok_stride % 8 == 0 && q_seq_stride % 8 == 0 &&
                      k_seq_stride % 8 == 0,
                  "qk_norm_rope: strides must be multiples of 8 elements");
    SRQ_CHECK_ARG(srq_aligned(q, 16) && srq_aligned(k, 16) && srq_aligned(cos, 16) &&
                      srq_aligned(sin, 16) && srq_aligned(q_weight, 16) &&
                      srq_aligned(k_weight, 16) && srq_aligned(q_out, 16) &&
                      srq_aligned(k_out, 16),
                  "qk_norm_rope: tensors must be 16-byte aligned");
    QkArgs a;
    a.q = (const f16 *)q;
    a.k = (const f16 *)k;
    a.cs = (const f16 *)cos;
    a.sn = (const f16 *)sin;
    a.qw = (const f16 *)q_weight;
    a.kw = (const f16 *)k_weight;
    a.qo = (f16 *)q_out;
    a.ko = (f16 *)k_out;
    a.q_tok = q_tok_stride;
    a.q_seq = q_seq_stride;
    a.k_tok = k_tok_stride;
    a.k_seq = k_seq_stride;
    a.T = seq_len;
    a.cos_batch = (int)(cos_batch == 1 ? 1 : 2);
    a.hq = (int)n_q_heads;
    a.hk = (int)n_kv_heads;
    a.norm = norm ? 1 : 0;
    a.eps = eps;
    const int64_t tokens = batch * seq_len, hs = n_q_heads + n_kv_heads;
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](auto kern, int rows) {
        // Few tokens: a block for every group of rows, else one that keeps the
        // token's cos, sin and weights for all of them.  us on one MI355X in a
        // graph, by groups / one block: 64 + 8 heads of 128, 1 token 2.2 / 3.8, 128 3.1 /
        // 4.3, 512 5.9 / 6.0, 768 7.8 / 7.7, 1024 9.9 / 9.3, 4096 36 / 28; 32 + 8 heads
        // of 64, 128 2.4 / 2.8, 512 3.4 / 3.4, 1024 4.8 / 4.5.
        const int64_t groups = srq_cdiv(hs, rows);
        const int64_t y = tokens > 512 ? 1 : groups;
        kern<<<dim3((unsigned)tokens, (unsigned)y), 256, 0, st>>>(a);
    };
    switch (head_dim) {
    case 64: go(qk_norm_rope_kernel<8>, 32); break;
    case 128: go(qk_norm_rope_kernel<16>, 16); break;
    default: go(qk_norm_rope_kernel<32>, 8); break;
    }
    SRQ_LAUNCH_CHECK("qk_norm_rope");
    return SRQ_OK;
}
