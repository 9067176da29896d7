// Attention of whole prompts, packed one after the other: causal within each sequence, grouped heads.
//
// Query i of a sequence with nq queries and nk keys stands at key i + (nk - nq) and sees the keys up to there:
//   out_i = sum_j softmax_j(scale * q_i . k_j) v_j,   j <= i + nk - nq.
// A query that sees no key gives zeros.  Operands are F16 (the cache's and the mat-mul's type for the contracted
// operand), sums and the soft-max are f32.
#include "kv_cache_q8.cuh"

namespace {

struct rows16 {  // an F16 {head_dim, heads, tokens} operand
    const __half* p;
    int64_t head, tok;
};

// One query row by one warp: a lane holds HD / 32 numbers.
template <int HD, typename T>
__device__ __forceinline__ void prompt_row(const rows16& q, const rows16& k, const rows16& v, int t, int k0, int n, int h, int kh, float scale, T* out) {
    constexpr int E = HD / 32;
    const int lane = threadIdx.x & 31;
    float qr[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) qr[e] = __half2float(q.p[h * q.head + t * q.tok + lane * E + e]) * scale, o[e] = 0.0f;
    for (int j = 0; j < n; j++) {
        const __half* kr = k.p + kh * k.head + (int64_t)(k0 + j) * k.tok + lane * E;
        const __half* vr = v.p + kh * v.head + (int64_t)(k0 + j) * v.tok + lane * E;
        float x = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) x = fmaf(qr[e], __half2float(kr[e]), x);
        x = gb_warp_sum(x);
        const float top = fmaxf(m, x), keep = m == -INFINITY ? 0.0f : expf(m - top), p = x == -INFINITY ? 0.0f : expf(x - top);
        m = top;
        l = l * keep + p;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = fmaf(p, __half2float(vr[e]), o[e] * keep);
    }
#pragma unroll
    for (int e = 0; e < E; e++) {
        const float x = l == 0.0f ? 0.0f : o[e] / l;
        if constexpr (sizeof(T) == 4) out[lane * E + e] = x;
        else out[lane * E + e] = __float2half_rn(x);
    }
}

template <int HD, typename T>
__global__ void __launch_bounds__(128) prompt_attention_kernel(rows16 q, rows16 k, rows16 v, const int32_t* __restrict__ q_starts,
                                                               const int32_t* __restrict__ k_starts, int nseq, int tq, int tk, int group, float scale,
                                                               T* __restrict__ out, int64_t o_head, int64_t o_tok, int* __restrict__ status) {
    gb_pdl_entry();
    const int t = blockIdx.x * 4 + (threadIdx.x >> 5), h = blockIdx.y;
    if (t >= tq) return;
    const int s = gb_find_seq(q_starts, nseq, t);
    if (s >= nseq) return;  // behind the last sequence
    const int q0 = q_starts[s], q1 = q_starts[s + 1], k0 = k_starts[s], k1 = k_starts[s + 1];
    if (q0 < 0 || q0 > t || q1 <= t || q1 > tq || k0 < 0 || k1 < k0 || k1 > tk) {
        if ((threadIdx.x & 31) == 0) *status = GALOIS_B200_E_BADARG;
        return;
    }
    const int n = (t - q0) + (k1 - k0) - (q1 - q0) + 1;
    prompt_row<HD, T>(q, k, v, t, k0, n, h, h / group, scale, out + h * o_head + t * o_tok);
}

int check_rows16(galois_b200_ctx* ctx, const char* name, const void* p, const galois_dim* d, size_t elem) {
    if (!d) return gb_fail(ctx, GALOIS_B200_E_BADARG, "prompt_attention: null dim of %s", name);
    for (int i = 0; i < 4; i++)
        if (d->ne[i] < 0 || d->nb[i] < 0) return gb_fail(ctx, GALOIS_B200_E_BADARG, "prompt_attention: negative extent or stride of %s", name);
    if (d->ne[0] != 64 && d->ne[0] != 128) return gb_fail(ctx, GALOIS_B200_E_UNSUPPORTED, "prompt_attention: head_dim %lld (64 and 128 are built)", (long long)d->ne[0]);
    if (d->ne[3] != 1 || d->ne[1] > 65535 || d->ne[2] > 0x3fffffff) return gb_fail(ctx, GALOIS_B200_E_SHAPE, "prompt_attention: %s must be {head_dim, heads, tokens}", name);
    if (!p && gb_span(d, 1)) return gb_fail(ctx, GALOIS_B200_E_BADARG, "prompt_attention: null pointer");
    if (d->nb[0] != 1 || (uintptr_t)p % 16 || (d->ne[1] > 1 && d->nb[1] * elem % 16) || (d->ne[2] > 1 && d->nb[2] * elem % 16))
        return gb_fail(ctx, GALOIS_B200_E_LAYOUT, "prompt_attention: rows of %s must be contiguous and 16-byte aligned", name);
    return 0;
}

template <typename T>
int prompt_attention(galois_b200_ctx* ctx, const void* q, const galois_dim* qd, const void* k, const galois_dim* kd, const void* v, const galois_dim* vd,
                     const int32_t* q_starts, const int32_t* k_starts, int nseq, T* dst, const galois_dim* dd, float scale) {
    GB_CHECK_CTX(ctx);
    int rc = check_rows16(ctx, "q", q, qd, 2);
    if (rc == 0) rc = check_rows16(ctx, "k", k, kd, 2);
    if (rc == 0) rc = check_rows16(ctx, "v", v, vd, 2);
    if (rc == 0) rc = check_rows16(ctx, "dst", dst, dd, sizeof(T));
    if (rc) return rc;
    if (!gb_same_shape(qd, dd) || !gb_same_shape(kd, vd) || qd->ne[0] != kd->ne[0])
        return gb_fail(ctx, GALOIS_B200_E_SHAPE, "prompt_attention: q and dst, k and v must be of one shape each, all of one head_dim");
    const int heads = (int)qd->ne[1], kv_heads = (int)kd->ne[1], tq = (int)qd->ne[2], tk = (int)kd->ne[2];
    if (heads && (kv_heads == 0 || heads % kv_heads)) return gb_fail(ctx, GALOIS_B200_E_BROADCAST, "prompt_attention: %d heads over %d key/value heads", heads, kv_heads);
    if (nseq < 0 || nseq > 0xfffff) return gb_fail(ctx, GALOIS_B200_E_BADARG, "prompt_attention: %d sequences", nseq);
    if (heads == 0 || tq == 0 || nseq == 0) return 0;
    if (!q_starts || !k_starts) return gb_fail(ctx, GALOIS_B200_E_BADARG, "prompt_attention: null pointer");
    if ((uintptr_t)q_starts % 4 || (uintptr_t)k_starts % 4) return gb_fail(ctx, GALOIS_B200_E_LAYOUT, "prompt_attention: misaligned starts");
    if (!gb_injective(dd)) return gb_fail(ctx, GALOIS_B200_E_DST, "prompt_attention: rows of dst overlap");
    const size_t dn = gb_span(dd, sizeof(T)), sn = 4 * ((size_t)nseq + 1);
    if (gb_overlap(dst, dn, q, gb_span(qd, 2)) || gb_overlap(dst, dn, k, gb_span(kd, 2)) || gb_overlap(dst, dn, v, gb_span(vd, 2)) ||
        gb_overlap(dst, dn, q_starts, sn) || gb_overlap(dst, dn, k_starts, sn))
        return gb_fail(ctx, GALOIS_B200_E_DST, "prompt_attention: dst overlaps an operand");
    gb_on_device on(ctx);
    const rows16 qr{(const __half*)q, qd->nb[1], qd->nb[2]}, kr{(const __half*)k, kd->nb[1], kd->nb[2]}, vr{(const __half*)v, vd->nb[1], vd->nb[2]};
    auto kern = qd->ne[0] == 64 ? prompt_attention_kernel<64, T> : prompt_attention_kernel<128, T>;
    GB_CUDA(ctx, gb_launch(ctx, kern, dim3((unsigned)((tq + 3) / 4), (unsigned)heads), dim3(128), 0, qr, kr, vr, q_starts, k_starts, nseq, tq, tk,
                           heads / kv_heads, scale, dst, dd->nb[1], dd->nb[2], ctx->dev_status));
    GB_LAUNCHED(ctx, "prompt_attention");
    return 0;
}

}  // namespace

extern "C" int galois_b200_prompt_attention_f16(galois_b200_ctx* ctx, const void* q, const galois_dim* qd, const void* k, const galois_dim* kd, const void* v,
                                                const galois_dim* vd, const int32_t* q_starts, const int32_t* k_starts, int nseq, void* dst,
                                                const galois_dim* dd, float scale) {
    return prompt_attention<__half>(ctx, q, qd, k, kd, v, vd, q_starts, k_starts, nseq, (__half*)dst, dd, scale);
}
extern "C" int galois_b200_prompt_attention_f16_f32(galois_b200_ctx* ctx, const void* q, const galois_dim* qd, const void* k, const galois_dim* kd,
                                                    const void* v, const galois_dim* vd, const int32_t* q_starts, const int32_t* k_starts, int nseq,
                                                    float* dst, const galois_dim* dd, float scale) {
    return prompt_attention<float>(ctx, q, qd, k, kd, v, vd, q_starts, k_starts, nseq, dst, dd, scale);
}
