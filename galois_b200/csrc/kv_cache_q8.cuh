// The 8-bit key/value cache: what its operators share (argument checks on the host, the rounding to whole
// numbers and the look-up of packed rows on the device).
#pragma once
#include "common.cuh"

#define GB_CACHE_BLOCK 32  // tokens of one head that share a scale

// Makes the context's device current for the calls of one entry point and puts the caller's back.
struct gb_on_device {
    int before = -1;
    explicit gb_on_device(const galois_b200_ctx* ctx) {
        if (cudaGetDevice(&before) == cudaSuccess && before != ctx->ordinal)
            cudaSetDevice(ctx->ordinal);
        else
            before = -1;
    }
    ~gb_on_device() {
        if (before >= 0) cudaSetDevice(before);
    }
};

// Bytes from the first to behind the last element of a tensor (0 if it has none).
static inline size_t gb_span(const galois_dim* d, size_t elem) {
    size_t last = 0;
    for (int i = 0; i < 4; i++) {
        if (d->ne[i] <= 0) return 0;
        last += (size_t)(d->ne[i] - 1) * (size_t)d->nb[i];
    }
    return (last + 1) * elem;
}
static inline bool gb_overlap(const void* a, size_t an, const void* b, size_t bn) {
    return an && bn && (uintptr_t)a < (uintptr_t)b + bn && (uintptr_t)b < (uintptr_t)a + an;
}
// No two elements at one address: sorted by stride, each dimension steps over all of the smaller ones.
static inline bool gb_injective(const galois_dim* d) {
    if (gb_span(d, 1) == 0) return true;
    int64_t span = 1;
    bool used[4] = {false, false, false, false};
    for (int k = 0; k < 4; k++) {
        int at = -1;
        for (int i = 0; i < 4; i++)
            if (!used[i] && d->ne[i] > 1 && (at < 0 || d->nb[i] < d->nb[at])) at = i;
        if (at < 0) return true;
        used[at] = true;
        if (d->nb[at] < span) return false;
        span = (d->ne[at] - 1) * d->nb[at] + span;
    }
    return true;
}

// Strides of a {head_dim, heads, tokens} operand and of the cache, in elements.
struct gb_cache_view {
    int8_t *k, *v;
    float *ks, *vs;
    int64_t tok, head, seq;     // strides of k and v
    int64_t s_head, s_seq;      // strides of the scales
    int ctx, kv_heads, seqs, head_dim;
};
// Sets the shared-memory limits of the attention kernels on the current device.
int gb_cache_attention_init(galois_b200_ctx* ctx);
int gb_prompt_attention_init(galois_b200_ctx* ctx);
// 0 and *out filled, or a failure of `what`.
int gb_check_cache(galois_b200_ctx* ctx, const char* what, const galois_b200_cache_q8* cache, gb_cache_view* out);

#ifdef __CUDACC__
// The sequence that packed row t belongs to: the first that ends behind t, n if there is none.  Where starts descend, that
// sequence and all behind it have no rows (they could be others' too).  Called by a whole warp; the loads of a warp are
// independent of each other, so a batch of 32 sequences costs one trip to memory where a binary search costs five.
__device__ __forceinline__ int gb_find_seq(const int32_t* __restrict__ starts, int n, int t) {
    unsigned first = (unsigned)n, descent = (unsigned)n;
    for (int i = threadIdx.x & 31; i < n; i += 32) {
        const int begin = starts[i], end = starts[i + 1];
        if (end > t) first = min(first, (unsigned)i);
        if (end < begin) descent = min(descent, (unsigned)i);
    }
    first = __reduce_min_sync(0xffffffffu, first);
    return first < __reduce_min_sync(0xffffffffu, descent) ? (int)first : n;
}

// Whether packed rows begin .. end can be rows p0.. of a slot.  The position of a sequence without rows does not matter.
__device__ __forceinline__ bool gb_packed_ok(int begin, int end, int p0, int tokens, int ctx) {
    return begin >= 0 && end >= begin && end <= tokens && (end == begin || (p0 >= 0 && p0 <= ctx - (end - begin)));
}
// By one CTA of its own, which nothing waits for: says so if a sequence is out of range, whether or not a token lies in it.
__device__ __forceinline__ void gb_report_packed(const int32_t* __restrict__ starts, const int32_t* __restrict__ pos, int nseq, int tokens, int ctx,
                                                 int* __restrict__ status) {
    for (int i = threadIdx.x; i < nseq; i += blockDim.x)
        if (!gb_packed_ok(starts[i], starts[i + 1], pos[i], tokens, ctx)) *status = GALOIS_B200_E_BADARG;
}

// A quotient x / d is rounded to a whole number (half to even) by adding 1.5 * 2^23 to x * (1 / d): the sum's last bits are
// the number.  1 / d is not exact, so it is taken a little too small and a little too large: where both give the same
// number it is the exact quotient's, else a border k + 1/2 lies next to it and is compared with in full.
#define GB_ROUND 12582912.0f
struct gb_around {
    float lo, hi;
};
__device__ __forceinline__ gb_around gb_make_around(float r) { return gb_around{__fmul_rn(r, 1.0f - 0x1p-22f), __fmul_rn(r, 1.0f + 0x1p-22f)}; }
__device__ __forceinline__ uint32_t gb_low_bytes(float a, float b, float c, float d) {
    return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040), __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040), 0x5410);
}
__device__ __forceinline__ uint32_t gb_bytes_of(float4 x, float r) {
    return gb_low_bytes(fmaf(x.x, r, GB_ROUND), fmaf(x.y, r, GB_ROUND), fmaf(x.z, r, GB_ROUND), fmaf(x.w, r, GB_ROUND));
}
// The whole number next to q that is nearest to x / d, by the signs of x - (q -+ 1/2) d, which one fused multiply-add gives
// exactly (d is not below 2^-100).
__device__ __forceinline__ float gb_q8_border(float x, float d, float r) {
    float q = rintf(__fmul_rn(x, r));
    const float lo = fmaf(-(q - 0.5f), d, x), hi = fmaf(-(q + 0.5f), d, x);
    const bool odd = ((int)q) & 1;
    if (lo < 0.0f || (lo == 0.0f && odd)) q -= 1.0f;
    else if (hi > 0.0f || (hi == 0.0f && odd)) q += 1.0f;
    return fminf(fmaxf(q, -127.0f), 127.0f) + GB_ROUND;
}
// Four numbers as bytes; r: around 1 / d, |x| at most 127.5 d.
__device__ __forceinline__ uint32_t gb_q8_round4(float4 x, float d, const gb_around& r) {
    const uint32_t a = gb_bytes_of(x, r.lo);
    if (a == gb_bytes_of(x, r.hi)) return a;
    return gb_low_bytes(gb_q8_border(x.x, d, r.lo), gb_q8_border(x.y, d, r.lo), gb_q8_border(x.z, d, r.lo), gb_q8_border(x.w, d, r.lo));
}
// The bytes of w as f32.
__device__ __forceinline__ float4 gb_q8_float4(uint32_t w) {
    w ^= 0x80808080u;  // 0..255, as the last bits of 2^23 + it
    return make_float4(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440)) - 8388736.0f, __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7441)) - 8388736.0f,
                       __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7442)) - 8388736.0f, __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7443)) - 8388736.0f);
}
// The same of q0 * d0 / d for four whole numbers that move to a larger scale; r: around d0 / d.  The product has 32 bits, so
// next to a border the two sides are compared in 64 bits, where both are exact.
__device__ __forceinline__ float gb_q8_border64(float q0, float d0, float d, float r) {
    float q = rintf(__fmul_rn(q0, r));
    const double x = (double)q0 * (double)d0, lo = x - ((double)q - 0.5) * (double)d, hi = x - ((double)q + 0.5) * (double)d;
    const bool odd = ((int)q) & 1;
    if (lo < 0.0 || (lo == 0.0 && odd)) q -= 1.0f;
    else if (hi > 0.0 || (hi == 0.0 && odd)) q += 1.0f;
    return fminf(fmaxf(q, -127.0f), 127.0f) + GB_ROUND;
}
__device__ __forceinline__ uint32_t gb_q8_rescale4(uint32_t w, float d0, float d, const gb_around& r) {
    const float4 x = gb_q8_float4(w);
    const uint32_t a = gb_bytes_of(x, r.lo);
    if (a == gb_bytes_of(x, r.hi)) return a;
    return gb_low_bytes(gb_q8_border64(x.x, d0, d, r.lo), gb_q8_border64(x.y, d0, d, r.lo), gb_q8_border64(x.z, d0, d, r.lo), gb_q8_border64(x.w, d0, d, r.lo));
}
#endif
