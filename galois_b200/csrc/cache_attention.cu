// Attention of one new token per sequence over the 8-bit key/value cache.
//
//   s_j = scale * (q . k_j),  p_j = exp(s_j - max) / sum,  out = sum_j p_j v_j      over the cache rows j < len
//
// with grouped heads: heads / kv_heads consecutive query heads read the same key/value head.  A sequence of length
// 0 gives zeros.  With `weights`, weights_out[j] = weights[j] + the sum of p_j over the heads of the group.
#include "kv_cache_q8.cuh"

namespace {

// One CTA per (head, sequence); a warp takes every fourth row, a lane HD / 32 numbers of it.
template <int HD>
__global__ void __launch_bounds__(128) cache_attention_kernel(const float* __restrict__ q, int64_t q_head, int64_t q_seq, gb_cache_view c,
                                                              const int32_t* __restrict__ lens, float* __restrict__ out, int64_t o_head, int64_t o_seq,
                                                              int heads, float scale, float* __restrict__ stats, float* __restrict__ scores,
                                                              int* __restrict__ status) {
    gb_pdl_entry();
    constexpr int E = HD / 32;
    __shared__ float sm[4], sl[4], so[4][HD];
    const int h = blockIdx.x, s = blockIdx.y, kh = h / (heads / c.kv_heads), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int n = lens[s];
    if (n < 0 || n > c.ctx) {
        if (threadIdx.x == 0) *status = GALOIS_B200_E_BADARG;
        n = 0;
    }
    float qr[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) qr[e] = q[h * q_head + s * q_seq + lane * E + e] * scale, o[e] = 0.0f;
    for (int j = warp; j < n; j += 4) {
        const int64_t at = kh * c.head + s * c.seq + j * c.tok + lane * E, sat = kh * c.s_head + s * c.s_seq + j / GB_CACHE_BLOCK;
        float x = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) x = fmaf(qr[e], (float)c.k[at + e], x);
        x = gb_warp_sum(x) * c.ks[sat];
        if (scores && lane == 0) scores[((int64_t)s * heads + h) * c.ctx + j] = x;
        const float top = fmaxf(m, x), keep = m == -INFINITY ? 0.0f : expf(m - top), p = x == -INFINITY ? 0.0f : expf(x - top);
        m = top;
        l = l * keep + p;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = fmaf(p * c.vs[sat], (float)c.v[at + e], o[e] * keep);
    }
    if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
    for (int e = 0; e < E; e++) so[warp][lane * E + e] = o[e];
    __syncthreads();
    const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    float f[4], total = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) f[w] = sm[w] == -INFINITY ? 0.0f : expf(sm[w] - top), total += f[w] * sl[w];
    if (stats && threadIdx.x == 0) stats[2 * ((int64_t)s * heads + h)] = top, stats[2 * ((int64_t)s * heads + h) + 1] = total;
    for (int e = threadIdx.x; e < HD; e += 128) {
        float x = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++)
            if (f[w] != 0.0f) x += f[w] * so[w][e];
        out[h * o_head + s * o_seq + e] = total == 0.0f ? 0.0f : x / total;
    }
}

__global__ void __launch_bounds__(256) cache_weights_kernel(const int32_t* __restrict__ lens, const float* __restrict__ stats, const float* __restrict__ scores,
                                                            const float* weights, int64_t w_head, int64_t w_seq, float* weights_out, int64_t wo_head,
                                                            int64_t wo_seq, int heads, int kv_heads, int ctx) {
    gb_pdl_entry();
    const int j = blockIdx.x * 256 + threadIdx.x, kh = blockIdx.y, s = blockIdx.z, group = heads / kv_heads;
    const int n = lens[s];
    if (n < 0 || n > ctx || j >= n) return;
    float x = 0.0f;
    for (int g = 0; g < group; g++) {
        const int64_t at = (int64_t)s * heads + kh * group + g;
        const float m = stats[2 * at], l = stats[2 * at + 1], sc = scores[at * ctx + j];
        if (sc != -INFINITY) x += expf(sc - m) / l;
    }
    weights_out[kh * wo_head + s * wo_seq + j] = weights[kh * w_head + s * w_seq + j] + x;
}

size_t workspace_floats(const gb_cache_view& c, int heads, bool weights) {
    return 4 + (weights ? (size_t)c.seqs * heads * (2 + (size_t)c.ctx) : 0);
}

}  // namespace

extern "C" int galois_b200_cache_attention_workspace_bytes(galois_b200_ctx* ctx, const galois_b200_cache_q8* cache, int heads, int with_weights,
                                                           size_t* out_bytes) {
    GB_CHECK_CTX(ctx);
    gb_cache_view c;
    const int rc = gb_check_cache(ctx, "cache_attention_workspace_bytes", cache, &c);
    if (rc) return rc;
    if (!out_bytes) return gb_fail(ctx, GALOIS_B200_E_BADARG, "cache_attention_workspace_bytes: null pointer");
    if (heads < 0 || (heads && (c.kv_heads == 0 || heads % c.kv_heads)) || heads > 65535)
        return gb_fail(ctx, GALOIS_B200_E_BROADCAST, "cache_attention_workspace_bytes: %d heads over %d key/value heads", heads, c.kv_heads);
    *out_bytes = workspace_floats(c, heads, with_weights != 0) * sizeof(float);
    return 0;
}

extern "C" int galois_b200_cache_attention_f32(galois_b200_ctx* ctx, const float* q, const galois_dim* qd, const galois_b200_cache_q8* cache,
                                               const int32_t* lens, float* dst, const galois_dim* dd, float scale, const float* weights,
                                               const galois_dim* wd, float* weights_out, const galois_dim* wod, void* workspace, size_t workspace_bytes) {
    GB_CHECK_CTX(ctx);
    gb_cache_view c;
    const char* what = "cache_attention";
    const int rc = gb_check_cache(ctx, what, cache, &c);
    if (rc) return rc;
    if (!qd || !dd || (weights && !wd) || (weights_out && !wod)) return gb_fail(ctx, GALOIS_B200_E_BADARG, "%s: null dim", what);
    if ((weights != nullptr) != (weights_out != nullptr)) return gb_fail(ctx, GALOIS_B200_E_BADARG, "%s: weights and weights_out come together", what);
    for (int i = 0; i < 4; i++)
        if (qd->ne[i] < 0 || qd->nb[i] < 0 || dd->ne[i] < 0 || dd->nb[i] < 0) return gb_fail(ctx, GALOIS_B200_E_BADARG, "%s: negative extent or stride", what);
    const int64_t heads = qd->ne[1];
    if (qd->ne[0] != c.head_dim || qd->ne[2] != c.seqs || qd->ne[3] != 1 || !gb_same_shape(qd, dd))
        return gb_fail(ctx, GALOIS_B200_E_SHAPE, "%s: q and dst must be {head_dim, heads, sequences} of the cache", what);
    if (heads > 65535 || (heads && (c.kv_heads == 0 || heads % c.kv_heads)))
        return gb_fail(ctx, GALOIS_B200_E_BROADCAST, "%s: %lld heads over %d key/value heads", what, (long long)heads, c.kv_heads);
    if (heads == 0 || c.seqs == 0) return 0;
    if (!q || !lens || !dst || !workspace) return gb_fail(ctx, GALOIS_B200_E_BADARG, "%s: null pointer", what);
    if (qd->nb[0] != 1 || dd->nb[0] != 1 || (uintptr_t)q % 16 || (uintptr_t)dst % 16 || (heads > 1 && (qd->nb[1] % 4 || dd->nb[1] % 4)) ||
        (c.seqs > 1 && (qd->nb[2] % 4 || dd->nb[2] % 4)) || (uintptr_t)lens % 4 || (uintptr_t)workspace % 16)
        return gb_fail(ctx, GALOIS_B200_E_LAYOUT, "%s: rows of q and dst must be contiguous, they and the workspace 16-byte aligned", what);
    if (!gb_injective(dd)) return gb_fail(ctx, GALOIS_B200_E_DST, "%s: rows of dst overlap", what);
    const size_t qn = gb_span(qd, 4), dn = gb_span(dd, 4), ln = 4 * (size_t)c.seqs, need = workspace_floats(c, (int)heads, weights != nullptr) * sizeof(float);
    if (workspace_bytes < need) return gb_fail(ctx, GALOIS_B200_E_NOMEM, "%s: workspace of %zu bytes, %zu are needed", what, workspace_bytes, need);
    size_t wn = 0, won = 0;
    if (weights) {
        for (const galois_dim* d : {wd, wod}) {
            for (int i = 0; i < 4; i++)
                if (d->nb[i] < 0) return gb_fail(ctx, GALOIS_B200_E_BADARG, "%s: negative stride of the weights", what);
            if (d->ne[0] != c.ctx || d->ne[1] != c.kv_heads || d->ne[2] != c.seqs || d->ne[3] != 1)
                return gb_fail(ctx, GALOIS_B200_E_SHAPE, "%s: weights must be {ctx, kv_heads, sequences} of the cache", what);
            if (d->nb[0] != 1) return gb_fail(ctx, GALOIS_B200_E_LAYOUT, "%s: rows of the weights must be contiguous", what);
        }
        if ((uintptr_t)weights % 4 || (uintptr_t)weights_out % 4) return gb_fail(ctx, GALOIS_B200_E_LAYOUT, "%s: misaligned weights", what);
        if (!gb_injective(wod)) return gb_fail(ctx, GALOIS_B200_E_DST, "%s: rows of weights_out overlap", what);
        wn = gb_span(wd, 4), won = gb_span(wod, 4);
        // in place (the very same tensor) is fine: every element is read by the thread that writes it
        const bool same = weights == weights_out && memcmp(wd->nb, wod->nb, sizeof(wd->nb)) == 0;
        if (!same && gb_overlap(weights, wn, weights_out, won)) return gb_fail(ctx, GALOIS_B200_E_DST, "%s: weights and weights_out overlap", what);
    }
    const size_t cn = gb_span(&cache->qd, 1), sn = gb_span(&cache->sd, 4);
    const struct { const void* p; size_t n; } get[6] = {{q, qn}, {lens, ln}, {c.k, cn}, {c.v, cn}, {c.ks, sn}, {c.vs, sn}}, put[3] = {{dst, dn}, {workspace, need}, {weights_out, won}};
    for (int i = 0; i < 3; i++) {
        bool bad = i < 2 && gb_overlap(put[i].p, put[i].n, weights, wn);
        for (const auto& g : get) bad = bad || gb_overlap(put[i].p, put[i].n, g.p, g.n);
        for (int j = 0; j < i; j++) bad = bad || gb_overlap(put[i].p, put[i].n, put[j].p, put[j].n);
        if (bad) return gb_fail(ctx, GALOIS_B200_E_DST, "%s: dst, workspace or weights_out overlap each other or an operand", what);
    }
    gb_on_device on(ctx);
    float* stats = weights ? (float*)workspace + 4 : nullptr;
    float* scores = weights ? stats + 2 * (size_t)c.seqs * heads : nullptr;
    auto kern = c.head_dim == 64 ? cache_attention_kernel<64> : cache_attention_kernel<128>;
    GB_CUDA(ctx, gb_launch(ctx, kern, dim3((unsigned)heads, (unsigned)c.seqs), dim3(128), 0, q, qd->nb[1], qd->nb[2], c, lens, dst, dd->nb[1], dd->nb[2],
                           (int)heads, scale, stats, scores, ctx->dev_status));
    GB_LAUNCHED(ctx, what);
    if (weights && c.ctx) {
        GB_CUDA(ctx, gb_launch(ctx, cache_weights_kernel, dim3((unsigned)((c.ctx + 255) / 256), (unsigned)c.kv_heads, (unsigned)c.seqs), dim3(256), 0, lens, stats,
                               scores, weights, wd->nb[1], wd->nb[2], weights_out, wod->nb[1], wod->nb[2], (int)heads, c.kv_heads, c.ctx));
        GB_LAUNCHED(ctx, "cache_weights");
    }
    return 0;
}
