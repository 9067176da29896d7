// The 8-bit key/value cache of a decoder layer: append, read, eviction.
//
// A cache holds, for each of its sequences and key/value heads, `ctx` rows of head_dim whole numbers -127..127 for
// the keys and for the values, and one f32 scale d for each 32 consecutive rows of a head; a row stands for q * d.
// The scale of a block is f32(max|x| / 127) over all it was given, so that it only grows while the block fills; when
// it grows the rows already held are brought to the new scale, q' = round(q d_held / d).  Both roundings are exact
// (half to even), which makes the contents a function of the numbers alone, whatever the order or split of the calls'
// work.  All move bytes and are meant to be bound by HBM (B200, 6.55 TB/s measured copy rate): 50 000 rows of 8 heads x 128
// are read into F16 in 53 us (5.8 TB/s); 8 000 F16 tokens appended in 15.4 us where they lie in L2 and 19.3 from HBM (49 MB, 2.5
// TB/s; 0.71 of the issue slots, for the rounding, and each CTA's chain of look-up, load, maximum and store); 16 sequences of up
// to 8192 rows cut to 2048 in 42 us (134 MB of rows), some of it the selection, whose passes over the digits wait for one
// another.  Few rows cost a launch.
#include "kv_cache_q8.cuh"

#include <type_traits>

namespace {

constexpr float Q8_TINY = 0x1p-100f;  // a smaller scale stands for a block of zeros (its quotients could underflow)
constexpr float Q8_MAX = 3.402823466e38f;
// 127 times a larger scale is rounded to infinity.  Append makes one such scale, f32(Q8_MAX / 127), for what it stores as Q8_MAX.
constexpr float Q8_SAFE = 0x1.020406p+121f;

__device__ __forceinline__ float finite(float x) { return fminf(fmaxf(x, -Q8_MAX), Q8_MAX); }
__device__ __forceinline__ float tame(float x) { return x != x ? 0.0f : finite(x); }

// 16 bytes of a row of new numbers: 4 f32 or 8 F16.
template <typename T>
struct piece;
template <>
struct piece<float> {
    static constexpr int N = 4;
    uint4 w;
    // the largest magnitude's bits; 0x7f800000 and above: not finite
    __device__ __forceinline__ uint32_t top() const { return max(max(w.x & 0x7fffffffu, w.y & 0x7fffffffu), max(w.z & 0x7fffffffu, w.w & 0x7fffffffu)); }
    __device__ __forceinline__ float4 get(int) const { return make_float4(__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w)); }
    static __device__ __forceinline__ float magnitude(uint32_t t) { return __uint_as_float(t); }
};
template <>
struct piece<__half> {
    static constexpr int N = 8;
    uint4 w;
    __device__ __forceinline__ uint32_t top() const {
        const uint32_t m = __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
        return max(m & 0xffffu, m >> 16);
    }
    __device__ __forceinline__ float4 get(int i) const {
        const uint32_t u = i ? w.z : w.x, v = i ? w.w : w.y;
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u)), b = __half22float2(*reinterpret_cast<const __half2*>(&v));
        return make_float4(a.x, a.y, b.x, b.y);
    }
    static __device__ __forceinline__ float magnitude(uint32_t t) { return __half2float(__ushort_as_half((unsigned short)t)); }
};

// ---------------------------------------------------------------- append
// A CTA of 128 threads looks at `tile` packed tokens of one head, of the keys (z = 0) or the values (z = 1).  Each
// token there that is the first new one of its block leads the block: the CTA takes all new rows of that block into
// registers (16 bytes of a row a lane), finds the largest magnitude, settles the scale and writes.  A block has one
// leader, so no two CTAs write the same rows or scale.  Sequences out of range are left out as a whole; the last column of the
// grid reports them.
template <typename T, int HD>
__global__ void __launch_bounds__(128) cache_append_kernel(const T* __restrict__ k, int64_t k_head, int64_t k_tok, const T* __restrict__ v,
                                                           int64_t v_head, int64_t v_tok, const int32_t* __restrict__ starts,
                                                           const int32_t* __restrict__ pos, int nseq, int tokens, int tile, gb_cache_view c,
                                                           int* __restrict__ status) {
    gb_pdl_entry();
    if (blockIdx.x == gridDim.x - 1) {
        if (blockIdx.y + blockIdx.z == 0) gb_report_packed(starts, pos, nseq, tokens, c.ctx, status);
        return;
    }
    constexpr int V = piece<T>::N, W = V / 4, LPR = HD / V, RPP = 128 / LPR, N = GB_CACHE_BLOCK / RPP;  // numbers and words a lane, lanes a row, rows a pass, passes
    __shared__ uint32_t red[4];
    const int head = blockIdx.y, warp = threadIdx.x >> 5;
    const int row0 = threadIdx.x / LPR, col = (threadIdx.x % LPR) * V;
    const T* x = (blockIdx.z ? v + head * v_head : k + head * k_head) + col;
    const int64_t x_tok = blockIdx.z ? v_tok : k_tok;
    int8_t* q = (blockIdx.z ? c.v : c.k) + head * c.head + col;
    float* scales = (blockIdx.z ? c.vs : c.ks) + head * c.s_head;
    const int t1 = min(tokens, ((int)blockIdx.x + 1) * tile);
    for (int t = (int)blockIdx.x * tile; t < t1;) {
        const int s = gb_find_seq(starts, nseq, t);
        if (s >= nseq) break;  // behind the last sequence
        const int begin = starts[s], end = starts[s + 1], p0 = pos[s];
        if (s == 0 && begin > t && end >= begin && end <= tokens) {  // in front of the first sequence
            t = begin;
            continue;
        }
        if (begin > t || end <= t || !gb_packed_ok(begin, end, p0, tokens, c.ctx)) {
            t = end > t ? end : t + 1;
            continue;
        }
        const int p = p0 + (t - begin), block = p / GB_CACHE_BLOCK, next = t + GB_CACHE_BLOCK - p % GB_CACHE_BLOCK;
        if (t != begin && p % GB_CACHE_BLOCK != 0) {  // led by an earlier token
            t = min(next, end);
            continue;
        }
        const int lo = p % GB_CACHE_BLOCK, hi = min(GB_CACHE_BLOCK, lo + end - t);
        piece<T> r[N];
        const T* from = x + (int64_t)(t + row0 - lo) * x_tok;
#pragma unroll
        for (int i = 0; i < N; i++, from += RPP * x_tok) {
            r[i].w = make_uint4(0, 0, 0, 0);
            if (row0 + i * RPP >= lo && row0 + i * RPP < hi) r[i].w = *reinterpret_cast<const uint4*>(from);
        }
        float* scale = scales + s * c.s_seq + block;
        const float held = lo > 0 ? *scale : 0.0f;
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < N; i++) bits = max(bits, r[i].top());
        bits = __reduce_max_sync(0xffffffffu, bits);
        __syncthreads();  // the last block's maxima have been read
        if ((threadIdx.x & 31) == 0) red[warp] = bits;
        __syncthreads();  // also: every thread has read the held scale
        float top = piece<T>::magnitude(max(max(red[0], red[1]), max(red[2], red[3])));
        const bool odd = !(top <= Q8_MAX);  // something is not finite: infinities count as the largest number, NaN as 0
        if (odd) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < N; i++)
#pragma unroll
                for (int j = 0; j < W; j++) {
                    const float4 f = r[i].get(j);
                    m = fmaxf(m, fmaxf(fmaxf(fabsf(tame(f.x)), fabsf(tame(f.y))), fmaxf(fabsf(tame(f.z)), fabsf(tame(f.w)))));
                }
            const uint32_t u = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
            __syncthreads();
            if ((threadIdx.x & 31) == 0) red[warp] = u;
            __syncthreads();
            top = __uint_as_float(max(max(red[0], red[1]), max(red[2], red[3])));
        }
        float d = fmaxf(__fdiv_rn(top, 127.0f), held);
        if (!(d >= Q8_TINY)) d = 0.0f;
        if (threadIdx.x == 0) *scale = d;
        int8_t* const to = q + s * c.seq + (int64_t)(block * GB_CACHE_BLOCK + row0) * c.tok;
        const gb_around by = gb_make_around(d > 0.0f ? __fdiv_rn(1.0f, d) : 0.0f);  // 0: everything becomes 0
        auto store = [&](int i, const uint32_t(&w)[W]) {
            if constexpr (W == 1) *reinterpret_cast<uint32_t*>(to + i * RPP * c.tok) = w[0];
            else *reinterpret_cast<uint2*>(to + i * RPP * c.tok) = make_uint2(w[0], w[1]);
        };
        auto put = [&](auto with_odd) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                if (row0 + i * RPP < lo || row0 + i * RPP >= hi) continue;
                uint32_t w[W];
#pragma unroll
                for (int j = 0; j < W; j++) {
                    float4 f = r[i].get(j);
                    if constexpr (decltype(with_odd)::value) f = make_float4(tame(f.x), tame(f.y), tame(f.z), tame(f.w));
                    w[j] = gb_q8_round4(f, d, by);
                }
                store(i, w);
            }
        };
        if (odd) put(std::true_type());
        else put(std::false_type());
        if (lo > 0 && d != held) {  // the rows there are, to the larger scale
            const gb_around ratio = gb_make_around(d > 0.0f ? __fdiv_rn(held, d) : 0.0f);
#pragma unroll
            for (int i = 0; i < N; i++) {
                if (row0 + i * RPP >= lo) continue;
                uint32_t w[W];
#pragma unroll
                for (int j = 0; j < W; j++) w[j] = gb_q8_rescale4(reinterpret_cast<const uint32_t*>(to + i * RPP * c.tok)[j], held, d, ratio);
                store(i, w);
            }
        }
        t = min(next, end);
    }
}

// ---------------------------------------------------------------- read
// A CTA of 128 threads gives back 32 packed rows of one head: a lane turns 4 bytes of a row into 4 f32, or 8 into 8 F16, so
// that a warp's stores are whole lines.
constexpr int READ_ROWS = 32;
template <typename T, int HD>
__global__ void __launch_bounds__(128) cache_read_kernel(gb_cache_view c, const int32_t* __restrict__ starts, const int32_t* __restrict__ pos, int nseq,
                                                         int tokens, T* __restrict__ k, int64_t k_head, int64_t k_tok, T* __restrict__ v,
                                                         int64_t v_head, int64_t v_tok, int* __restrict__ status) {
    gb_pdl_entry();
    if (blockIdx.x == gridDim.x - 1) {
        if (blockIdx.y + blockIdx.z == 0) gb_report_packed(starts, pos, nseq, tokens, c.ctx, status);
        return;
    }
    constexpr int V = 16 / sizeof(T), W = V / 4, LPR = HD / V, RPP = 128 / LPR, N = READ_ROWS / RPP;
    const int head = blockIdx.y, col = (threadIdx.x % LPR) * V;
    const int8_t* q = (blockIdx.z ? c.v : c.k) + head * c.head + col;
    const float* scales = (blockIdx.z ? c.vs : c.ks) + head * c.s_head;
    T* y = (blockIdx.z ? v + head * v_head : k + head * k_head) + col;
    const int64_t y_tok = blockIdx.z ? v_tok : k_tok;
    const int tile = (int)blockIdx.x * READ_ROWS, t0 = tile + threadIdx.x / LPR;
    int s = gb_find_seq(starts, nseq, tile);
    int begin = 0, end = 0, p0 = 0;
    if (s < nseq) begin = starts[s], end = starts[s + 1], p0 = pos[s];
    uint32_t w[N][W];
    float d[N];
    bool live[N];
    if (s < nseq && begin <= tile && end >= tile + READ_ROWS && gb_packed_ok(begin, end, p0, tokens, c.ctx)) {
        // all rows of one sequence
        const int p = p0 + (t0 - begin);
        const int8_t* from = q + s * c.seq + p * c.tok;
        const float* scale = scales + s * c.s_seq;
#pragma unroll
        for (int i = 0; i < N; i++, from += RPP * c.tok) {
            live[i] = true;
            if constexpr (W == 1) {
                w[i][0] = *reinterpret_cast<const uint32_t*>(from);
            } else {
                const uint2 u = *reinterpret_cast<const uint2*>(from);
                w[i][0] = u.x, w[i][1] = u.y;
            }
            d[i] = scale[(p + i * RPP) / GB_CACHE_BLOCK];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int t = t0 + i * RPP;
            live[i] = false;
            while (s < nseq && end <= t) {
                if (++s < nseq) begin = end, end = starts[s + 1], p0 = pos[s];
                if (end < begin) s = nseq;  // as gb_find_seq has it
            }
            if (t < tokens && s < nseq && begin <= t && gb_packed_ok(begin, end, p0, tokens, c.ctx)) {
                const int p = p0 + (t - begin);
                live[i] = true;
                const int8_t* from = q + s * c.seq + p * c.tok;
                if constexpr (W == 1) {
                    w[i][0] = *reinterpret_cast<const uint32_t*>(from);
                } else {
                    const uint2 u = *reinterpret_cast<const uint2*>(from);
                    w[i][0] = u.x, w[i][1] = u.y;
                }
                d[i] = scales[s * c.s_seq + p / GB_CACHE_BLOCK];
            }
        }
    }
    T* to = y + (int64_t)t0 * y_tok;
#pragma unroll
    for (int i = 0; i < N; i++, to += RPP * y_tok) {
        if (!live[i]) continue;
        float4 f[W];
#pragma unroll
        for (int j = 0; j < W; j++) {
            f[j] = gb_q8_float4(w[i][j]);
            f[j] = make_float4(__fmul_rn(f[j].x, d[i]), __fmul_rn(f[j].y, d[i]), __fmul_rn(f[j].z, d[i]), __fmul_rn(f[j].w, d[i]));
        }
        if constexpr (W == 1) {
            *reinterpret_cast<float4*>(to) = f[0];
        } else {
            __half2 h[4] = {__floats2half2_rn(f[0].x, f[0].y), __floats2half2_rn(f[0].z, f[0].w), __floats2half2_rn(f[W - 1].x, f[W - 1].y), __floats2half2_rn(f[W - 1].z, f[W - 1].w)};
            *reinterpret_cast<uint4*>(to) = *reinterpret_cast<uint4*>(h);
        }
    }
    if constexpr (sizeof(T) == 4) {
        bool loud = false;
#pragma unroll
        for (int i = 0; i < N; i++) loud = loud || (live[i] && d[i] > Q8_SAFE);
        if (loud) {  // once more, for the rows that hold f32's largest number
#pragma unroll
            for (int i = 0; i < N; i++) {
                if (!live[i] || !(d[i] > Q8_SAFE)) continue;
                const float4 f = gb_q8_float4(w[i][0]);
                *reinterpret_cast<float4*>(y + (int64_t)(t0 + i * RPP) * y_tok) =
                    make_float4(finite(__fmul_rn(f.x, d[i])), finite(__fmul_rn(f.y, d[i])), finite(__fmul_rn(f.z, d[i])), finite(__fmul_rn(f.w, d[i])));
            }
        }
    }
}

// ---------------------------------------------------------------- eviction: selection
// One CTA per (sequence, head).  m = min(len, budget) tokens stay: the last r = min(recent, m) and, of the others, the
// m - r of largest weight, equal weights from the lowest index.  Weights are compared as whole numbers that order like
// them (NaN below all); the m - r th largest is found digit by digit, 8 bits at a time, from histograms in shared
// memory; a prefix sum over the CTA then gives every kept token its row, so that the order of the tokens stays.
constexpr int EV_THREADS = 1024;
__device__ __forceinline__ uint32_t order_key(float w) {
    const uint32_t u = __float_as_uint(w);
    if (w != w) return 0u;
    const uint32_t k = (u & 0x80000000u) ? ~u : u | 0x80000000u;
    return w == 0.0f ? 0x80000000u : k;  // -0 and 0 are equal
}
// Inclusive sum over the CTA's threads; *total receives the sum of all.  `part`: 32 words of shared memory that are free
// again after the caller's next __syncthreads.
__device__ __forceinline__ uint32_t cta_scan(uint32_t x, uint32_t* part, uint32_t* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) part[warp] = x;
    __syncthreads();
    uint32_t y = part[lane];  // every warp sums the warps' sums
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t z = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) y += z;
    }
    *total = __shfl_sync(0xffffffffu, y, 31);
    const uint32_t in_front = __shfl_sync(0xffffffffu, y, (warp + 31) & 31);
    return warp ? x + in_front : x;
}
// A thread holds EV_EACH consecutive weights of a chunk, so that one sum over the CTA orders the whole chunk; a row of up to
// 8192 tokens is one chunk and is read once.
constexpr int EV_EACH = 8, EV_CHUNK = EV_THREADS * EV_EACH;
__device__ __forceinline__ void load_keys(const float* __restrict__ w, int i0, int n, float (&x)[EV_EACH], uint32_t (&key)[EV_EACH]) {
    if (i0 + EV_EACH <= n && (uintptr_t)(w + i0) % 16 == 0) {
        const float4 a = *reinterpret_cast<const float4*>(w + i0), b = *reinterpret_cast<const float4*>(w + i0 + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
#pragma unroll
        for (int e = 0; e < EV_EACH; e++) x[e] = i0 + e < n ? w[i0 + e] : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < EV_EACH; e++) key[e] = order_key(x[e]);
}
__global__ void __launch_bounds__(EV_THREADS) cache_select_kernel(const int32_t* __restrict__ lens, const float* __restrict__ weights, int64_t w_head,
                                                                  int64_t w_seq, int ctx, int budget, int recent, int32_t* __restrict__ out_lens,
                                                                  float* __restrict__ out_weights, int64_t ow_head, int64_t ow_seq,
                                                                  int32_t* __restrict__ index, int64_t i_head, int64_t i_seq, int* __restrict__ status) {
    gb_pdl_entry();
    // the weights of a row lie close together, most of them in a few digits: eight counts of each, dealt by warp
    __shared__ int hist[8][256];
    __shared__ uint32_t part[32];
    __shared__ int pick[2];
    const int head = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
    int n = lens[s];
    if (n < 0 || n > ctx) {
        if (tid == 0) *status = GALOIS_B200_E_BADARG;
        n = 0;  // nothing is kept of this sequence
    }
    const float* w = weights + head * w_head + s * w_seq;
    float* ow = out_weights + head * ow_head + s * ow_seq;
    int32_t* idx = index + head * i_head + s * i_seq;
    const int m = min(n, budget), r = min(recent, m), cand = n - r, need = m - r;
    if (head == 0 && tid == 0) out_lens[s] = m;
    float x[EV_EACH];
    uint32_t key[EV_EACH];
    const bool once = n <= EV_CHUNK, choose = need > 0 && need < cand;
    if (once) load_keys(w, tid * EV_EACH, n, x, key);
    // the need-th largest key among the first `cand`: `limit`, and how many of those equal to it are kept
    uint32_t limit = 0;
    int left = need;
    if (choose) {
        uint32_t mask = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 8 * 256; i += EV_THREADS) (&hist[0][0])[i] = 0;
            __syncthreads();
            for (int c0 = 0; c0 < cand; c0 += EV_CHUNK) {
                const int i0 = c0 + tid * EV_EACH;
                if (!once) load_keys(w, i0, n, x, key);
#pragma unroll
                for (int e = 0; e < EV_EACH; e++)
                    if (i0 + e < cand && (key[e] & mask) == limit) atomicAdd(&hist[(tid >> 5) & 7][(key[e] >> shift) & 255u], 1);
            }
            __syncthreads();
            // thread t looks at digit 255 - t: the first whose count of keys at or above reaches `left`
            uint32_t total;
            int c = 0;
            if (tid < 256) {
#pragma unroll
                for (int i = 0; i < 8; i++) c += hist[i][255 - tid];
            }
            const int upto = (int)cta_scan((uint32_t)c, part, &total);
            if (tid < 256 && upto >= left && upto - c < left) pick[0] = 255 - tid, pick[1] = left - (upto - c);
            __syncthreads();
            limit |= (uint32_t)pick[0] << shift;
            left = pick[1];
            mask |= 255u << shift;
        }
    }
    // rows of the kept tokens, in order: in front of a token are all above the limit and, of those equal to it, `left` at most
    int above_front = 0, equal_front = 0;
    for (int c0 = 0; c0 < n; c0 += EV_CHUNK) {
        const int i0 = c0 + tid * EV_EACH;
        if (!once) load_keys(w, i0, n, x, key);
        uint32_t above = 0, equal = 0;  // bit e: token i0 + e
#pragma unroll
        for (int e = 0; e < EV_EACH; e++) {
            const int i = i0 + e;
            if (i >= n) continue;
            if (i >= cand || (need > 0 && !choose) || (choose && key[e] > limit)) above |= 1u << e;
            else if (choose && key[e] == limit) equal |= 1u << e;
        }
        uint32_t total;
        const uint32_t mine = (uint32_t)__popc(above) | ((uint32_t)__popc(equal) << 16);  // both sums are below 2^14
        const uint32_t front = cta_scan(mine, part, &total) - mine;
        int a = above_front + (int)(front & 0xffffu), q = equal_front + (int)(front >> 16);
#pragma unroll
        for (int e = 0; e < EV_EACH; e++) {
            const bool is = (above >> e) & 1, tie = (equal >> e) & 1;
            if (is || (tie && q < left)) {
                const int at = a + min(q, left);
                idx[at] = i0 + e;
                ow[at] = x[e];
            }
            a += is, q += tie;
        }
        above_front += (int)(total & 0xffffu), equal_front += (int)(total >> 16);
        __syncthreads();
    }
}

// ---------------------------------------------------------------- eviction: the kept rows
// A CTA of 128 threads makes one block of 32 rows of the new cache: rows from up to 32 blocks of the old one, brought
// to the largest of their scales.
template <int HD>
__global__ void __launch_bounds__(128) cache_gather_kernel(gb_cache_view c, gb_cache_view o, const int32_t* __restrict__ out_lens,
                                                           const int32_t* __restrict__ index, int64_t i_head, int64_t i_seq) {
    gb_pdl_entry();
    constexpr int LPR = HD / 16, RPP = 128 / LPR, N = (GB_CACHE_BLOCK + RPP - 1) / RPP;
    const int block = blockIdx.x, head = blockIdx.y >> 1, s = blockIdx.z, lane = threadIdx.x & 31;
    const bool values = blockIdx.y & 1;
    const int m = min(out_lens[s] - block * GB_CACHE_BLOCK, GB_CACHE_BLOCK);
    if (m <= 0) return;
    const int32_t* idx = index + head * i_head + s * i_seq + block * GB_CACHE_BLOCK;
    const float* scales = (values ? c.vs : c.ks) + head * c.s_head + s * c.s_seq;
    const int8_t* q = (values ? c.v : c.k) + head * c.head + s * c.seq;
    int8_t* out = (values ? o.v : o.k) + head * o.head + s * o.seq + (int64_t)block * GB_CACHE_BLOCK * o.tok;
    const int src = lane < m ? idx[lane] : 0;  // every warp holds all 32
    const int col = (threadIdx.x % LPR) * 16;
    uint4 w[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int row = threadIdx.x / LPR + i * RPP;
        const int from = __shfl_sync(0xffffffffu, src, row & 31);
        w[i] = make_uint4(0, 0, 0, 0);
        if (row < m) w[i] = *reinterpret_cast<const uint4*>(q + from * c.tok + col);
    }
    const float ds = lane < m ? scales[src / GB_CACHE_BLOCK] : 0.0f;
    float d = gb_warp_max(ds);
    if (!(d >= Q8_TINY)) d = 0.0f;
    if (threadIdx.x == 0) ((values ? o.vs : o.ks) + head * o.s_head + s * o.s_seq)[block] = d;
    const float ratio = d > 0.0f ? __fdiv_rn(ds, d) : 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int row = threadIdx.x / LPR + i * RPP;
        const float d0 = __shfl_sync(0xffffffffu, ds, row & 31);
        const gb_around r = gb_make_around(__shfl_sync(0xffffffffu, ratio, row & 31));
        if (row >= m) continue;
        if (d0 != d) {
            if (d > 0.0f) w[i] = make_uint4(gb_q8_rescale4(w[i].x, d0, d, r), gb_q8_rescale4(w[i].y, d0, d, r), gb_q8_rescale4(w[i].z, d0, d, r), gb_q8_rescale4(w[i].w, d0, d, r));
            else w[i] = make_uint4(0, 0, 0, 0);
        }
        *reinterpret_cast<uint4*>(out + row * o.tok + col) = w[i];
    }
}

// {head_dim, kv_heads, tokens} operand beside a cache: rows contiguous, 16-byte aligned.
int check_rows(galois_b200_ctx* ctx, const char* what, const void* p, const galois_dim* d, const gb_cache_view& c, size_t elem, bool written) {
    if (!d) return gb_fail(ctx, GALOIS_B200_E_BADARG, "%s: null dim", what);
    for (int i = 0; i < 4; i++)
        if (d->ne[i] < 0 || d->nb[i] < 0) return gb_fail(ctx, GALOIS_B200_E_BADARG, "%s: negative extent or stride", what);
    if (d->ne[0] != c.head_dim || d->ne[1] != c.kv_heads || d->ne[3] != 1)
        return gb_fail(ctx, GALOIS_B200_E_SHAPE, "%s: rows must be {head_dim, kv_heads, tokens} of the cache", what);
    if (d->ne[2] > 0x3fffffff) return gb_fail(ctx, GALOIS_B200_E_SHAPE, "%s: too many tokens", what);
    if (d->ne[2] == 0) return 0;
    if (!p) return gb_fail(ctx, GALOIS_B200_E_BADARG, "%s: null pointer", what);
    if (d->nb[0] != 1 || (uintptr_t)p % 16 || (d->ne[1] > 1 && d->nb[1] * elem % 16) || (d->ne[2] > 1 && d->nb[2] * elem % 16))
        return gb_fail(ctx, GALOIS_B200_E_LAYOUT, "%s: rows must be contiguous and 16-byte aligned", what);
    if (written && !gb_injective(d)) return gb_fail(ctx, GALOIS_B200_E_DST, "%s: rows of the destination overlap", what);
    return 0;
}
int check_packed(galois_b200_ctx* ctx, const char* what, const int32_t* starts, const int32_t* pos, int nseq, const gb_cache_view& c) {
    if (nseq < 0 || nseq > c.seqs) return gb_fail(ctx, GALOIS_B200_E_SHAPE, "%s: %d sequences, the cache holds %d", what, nseq, c.seqs);
    if (nseq && (!starts || !pos)) return gb_fail(ctx, GALOIS_B200_E_BADARG, "%s: null pointer", what);
    if ((uintptr_t)starts % 4 || (uintptr_t)pos % 4) return gb_fail(ctx, GALOIS_B200_E_LAYOUT, "%s: misaligned starts or positions", what);
    return 0;
}
bool touches(const gb_cache_view& c, const galois_b200_cache_q8* h, const void* p, size_t bytes) {
    const size_t qn = gb_span(&h->qd, 1), sn = gb_span(&h->sd, 4);
    return gb_overlap(p, bytes, c.k, qn) || gb_overlap(p, bytes, c.v, qn) || gb_overlap(p, bytes, c.ks, sn) || gb_overlap(p, bytes, c.vs, sn);
}

template <typename T>
int append(galois_b200_ctx* ctx, const char* what, const galois_b200_cache_q8* cache, const T* k, const galois_dim* kd, const T* v, const galois_dim* vd,
           const int32_t* starts, const int32_t* pos, int nseq) {
    GB_CHECK_CTX(ctx);
    gb_cache_view c;
    int rc = gb_check_cache(ctx, what, cache, &c);
    if (rc == 0) rc = check_rows(ctx, what, k, kd, c, sizeof(T), false);
    if (rc == 0) rc = check_rows(ctx, what, v, vd, c, sizeof(T), false);
    if (rc == 0) rc = check_packed(ctx, what, starts, pos, nseq, c);
    if (rc) return rc;
    if (kd->ne[2] != vd->ne[2]) return gb_fail(ctx, GALOIS_B200_E_SHAPE, "%s: k and v hold different numbers of tokens", what);
    if (touches(c, cache, k, gb_span(kd, sizeof(T))) || touches(c, cache, v, gb_span(vd, sizeof(T))) || touches(c, cache, starts, 4 * ((size_t)nseq + 1)) ||
        touches(c, cache, pos, 4 * (size_t)nseq))
        return gb_fail(ctx, GALOIS_B200_E_BADARG, "%s: the operands lie in the cache", what);
    const int tokens = (int)kd->ne[2];
    if (tokens == 0 || nseq == 0 || c.kv_heads == 0) return 0;
    gb_on_device on(ctx);
    // A CTA per token where most tokens lead a block of their own (single tokens of many sequences), else per 32.  One and 32
    // tokens a CTA: a token each of 48 sequences 5.8 and 36 us, 8 000 tokens of prompts 135 and 15.4 us.  The host knows only the
    // mean, which misleads where many single tokens come with one long prompt: 47 of them with one of 512 take 11.8 and 37.5 us,
    // and the rule takes the second.
    const int tile = (int64_t)nseq * 8 >= tokens ? 1 : GB_CACHE_BLOCK;
    const dim3 grid((unsigned)((tokens + tile - 1) / tile + 1), (unsigned)c.kv_heads, 2);  // and a column that reports
    auto kern = c.head_dim == 64 ? cache_append_kernel<T, 64> : cache_append_kernel<T, 128>;
    GB_CUDA(ctx, gb_launch(ctx, kern, grid, dim3(128), 0, k, kd->nb[1], kd->nb[2], v, vd->nb[1], vd->nb[2], starts, pos, nseq, tokens, tile, c, ctx->dev_status));
    GB_LAUNCHED(ctx, what);
    return 0;
}
template <typename T>
int read_rows(galois_b200_ctx* ctx, const char* what, const galois_b200_cache_q8* cache, const int32_t* starts, const int32_t* pos, int nseq, T* k,
              const galois_dim* kd, T* v, const galois_dim* vd) {
    GB_CHECK_CTX(ctx);
    gb_cache_view c;
    int rc = gb_check_cache(ctx, what, cache, &c);
    if (rc == 0) rc = check_rows(ctx, what, k, kd, c, sizeof(T), true);
    if (rc == 0) rc = check_rows(ctx, what, v, vd, c, sizeof(T), true);
    if (rc == 0) rc = check_packed(ctx, what, starts, pos, nseq, c);
    if (rc) return rc;
    if (kd->ne[2] != vd->ne[2]) return gb_fail(ctx, GALOIS_B200_E_SHAPE, "%s: k and v hold different numbers of tokens", what);
    const size_t kn = gb_span(kd, sizeof(T)), vn = gb_span(vd, sizeof(T));
    const size_t sn = 4 * ((size_t)nseq + 1), pn = 4 * (size_t)nseq;
    if (touches(c, cache, k, kn) || touches(c, cache, v, vn) || gb_overlap(k, kn, v, vn) || gb_overlap(k, kn, starts, sn) || gb_overlap(k, kn, pos, pn) ||
        gb_overlap(v, vn, starts, sn) || gb_overlap(v, vn, pos, pn))
        return gb_fail(ctx, GALOIS_B200_E_DST, "%s: the destinations overlap each other or the operands", what);
    const int tokens = (int)kd->ne[2];
    if (tokens == 0 || nseq == 0 || c.kv_heads == 0) return 0;
    gb_on_device on(ctx);
    const dim3 grid((unsigned)((tokens + READ_ROWS - 1) / READ_ROWS + 1), (unsigned)c.kv_heads, 2);  // and a column that reports
    auto kern = c.head_dim == 64 ? cache_read_kernel<T, 64> : cache_read_kernel<T, 128>;
    GB_CUDA(ctx, gb_launch(ctx, kern, grid, dim3(128), 0, c, starts, pos, nseq, tokens, k, kd->nb[1], kd->nb[2], v, vd->nb[1], vd->nb[2], ctx->dev_status));
    GB_LAUNCHED(ctx, what);
    return 0;
}

}  // namespace

int gb_check_cache(galois_b200_ctx* ctx, const char* what, const galois_b200_cache_q8* h, gb_cache_view* out) {
    if (!h) return gb_fail(ctx, GALOIS_B200_E_BADARG, "%s: null cache", what);
    const galois_dim *q = &h->qd, *s = &h->sd;
    for (int i = 0; i < 4; i++)
        if (q->ne[i] < 0 || s->ne[i] < 0 || q->nb[i] < 0 || s->nb[i] < 0) return gb_fail(ctx, GALOIS_B200_E_BADARG, "%s: negative extent or stride of the cache", what);
    if (q->ne[0] != 64 && q->ne[0] != 128) return gb_fail(ctx, GALOIS_B200_E_UNSUPPORTED, "%s: head_dim %lld (64 and 128 are built)", what, (long long)q->ne[0]);
    if (q->ne[1] > 0x3fffffff || q->ne[2] > 32767 || q->ne[3] > 65535) return gb_fail(ctx, GALOIS_B200_E_SHAPE, "%s: the cache is too large", what);
    if (s->ne[0] != (q->ne[1] + GB_CACHE_BLOCK - 1) / GB_CACHE_BLOCK || s->ne[1] != q->ne[2] || s->ne[2] != q->ne[3] || s->ne[3] != 1)
        return gb_fail(ctx, GALOIS_B200_E_SHAPE, "%s: scales must be {ceil(ctx / 32), kv_heads, sequences}", what);
    if (gb_span(q, 1) && (!h->k || !h->v || !h->k_scale || !h->v_scale)) return gb_fail(ctx, GALOIS_B200_E_BADARG, "%s: null pointer in the cache", what);
    if (q->nb[0] != 1 || s->nb[0] != 1 || (uintptr_t)h->k % 16 || (uintptr_t)h->v % 16 || (uintptr_t)h->k_scale % 4 || (uintptr_t)h->v_scale % 4)
        return gb_fail(ctx, GALOIS_B200_E_LAYOUT, "%s: rows of the cache must be contiguous and 16-byte aligned", what);
    for (int i = 1; i < 4; i++)
        if (q->ne[i] > 1 && q->nb[i] % 16) return gb_fail(ctx, GALOIS_B200_E_LAYOUT, "%s: strides of the cache must be multiples of 16", what);
    if (!gb_injective(q) || !gb_injective(s)) return gb_fail(ctx, GALOIS_B200_E_LAYOUT, "%s: rows of the cache overlap", what);
    const size_t qn = gb_span(q, 1), sn = gb_span(s, 4);
    const void* part[4] = {h->k, h->v, h->k_scale, h->v_scale};
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < i; j++)
            if (gb_overlap(part[i], i < 2 ? qn : sn, part[j], j < 2 ? qn : sn)) return gb_fail(ctx, GALOIS_B200_E_LAYOUT, "%s: parts of the cache overlap", what);
    out->k = (int8_t*)h->k, out->v = (int8_t*)h->v, out->ks = h->k_scale, out->vs = h->v_scale;
    out->tok = q->nb[1], out->head = q->nb[2], out->seq = q->nb[3], out->s_head = s->nb[1], out->s_seq = s->nb[2];
    out->head_dim = (int)q->ne[0], out->ctx = (int)q->ne[1], out->kv_heads = (int)q->ne[2], out->seqs = (int)q->ne[3];
    return 0;
}

extern "C" int galois_b200_cache_append_f32(galois_b200_ctx* ctx, const galois_b200_cache_q8* cache, const float* k, const galois_dim* kd, const float* v,
                                            const galois_dim* vd, const int32_t* starts, const int32_t* pos, int nseq) {
    return append<float>(ctx, "cache_append", cache, k, kd, v, vd, starts, pos, nseq);
}
extern "C" int galois_b200_cache_append_f16(galois_b200_ctx* ctx, const galois_b200_cache_q8* cache, const void* k, const galois_dim* kd, const void* v,
                                            const galois_dim* vd, const int32_t* starts, const int32_t* pos, int nseq) {
    return append<__half>(ctx, "cache_append", cache, (const __half*)k, kd, (const __half*)v, vd, starts, pos, nseq);
}
extern "C" int galois_b200_cache_read_f32(galois_b200_ctx* ctx, const galois_b200_cache_q8* cache, const int32_t* starts, const int32_t* pos, int nseq,
                                          float* k, const galois_dim* kd, float* v, const galois_dim* vd) {
    return read_rows<float>(ctx, "cache_read", cache, starts, pos, nseq, k, kd, v, vd);
}
extern "C" int galois_b200_cache_read_f16(galois_b200_ctx* ctx, const galois_b200_cache_q8* cache, const int32_t* starts, const int32_t* pos, int nseq,
                                          void* k, const galois_dim* kd, void* v, const galois_dim* vd) {
    return read_rows<__half>(ctx, "cache_read", cache, starts, pos, nseq, (__half*)k, kd, (__half*)v, vd);
}

extern "C" int galois_b200_cache_evict(galois_b200_ctx* ctx, const galois_b200_cache_q8* cache, const int32_t* lens, const float* weights,
                                       const galois_dim* wd, int recent, const galois_b200_cache_q8* out, int32_t* out_lens, float* out_weights,
                                       const galois_dim* owd, int32_t* index, const galois_dim* id) {
    GB_CHECK_CTX(ctx);
    gb_cache_view c, o;
    int rc = gb_check_cache(ctx, "cache_evict", cache, &c);
    if (rc == 0) rc = gb_check_cache(ctx, "cache_evict", out, &o);
    if (rc) return rc;
    if (!wd || !owd || !id) return gb_fail(ctx, GALOIS_B200_E_BADARG, "cache_evict: null dim");
    if (recent < 0) return gb_fail(ctx, GALOIS_B200_E_BADARG, "cache_evict: negative count of recent tokens");
    if (c.head_dim != o.head_dim || c.kv_heads != o.kv_heads || c.seqs != o.seqs)
        return gb_fail(ctx, GALOIS_B200_E_SHAPE, "cache_evict: the caches differ in head_dim, kv_heads or sequences");
    const struct { const galois_dim* d; int n; const char* name; } t[3] = {{wd, c.ctx, "weights"}, {owd, o.ctx, "out_weights"}, {id, o.ctx, "index"}};
    for (const auto& x : t) {
        for (int i = 0; i < 4; i++)
            if (x.d->nb[i] < 0) return gb_fail(ctx, GALOIS_B200_E_BADARG, "cache_evict: negative stride of %s", x.name);
        if (x.d->ne[0] != x.n || x.d->ne[1] != c.kv_heads || x.d->ne[2] != c.seqs || x.d->ne[3] != 1)
            return gb_fail(ctx, GALOIS_B200_E_SHAPE, "cache_evict: %s must be {ctx, kv_heads, sequences} of its cache", x.name);
        if (x.d->nb[0] != 1) return gb_fail(ctx, GALOIS_B200_E_LAYOUT, "cache_evict: rows of %s must be contiguous", x.name);
    }
    if (!gb_injective(owd) || !gb_injective(id)) return gb_fail(ctx, GALOIS_B200_E_DST, "cache_evict: rows of a destination overlap");
    if (c.seqs == 0 || c.kv_heads == 0) return 0;
    if (!lens || !out_lens || (c.ctx && !weights) || (o.ctx && (!out_weights || !index))) return gb_fail(ctx, GALOIS_B200_E_BADARG, "cache_evict: null pointer");
    if ((uintptr_t)lens % 4 || (uintptr_t)out_lens % 4 || (uintptr_t)weights % 4 || (uintptr_t)out_weights % 4 || (uintptr_t)index % 4)
        return gb_fail(ctx, GALOIS_B200_E_LAYOUT, "cache_evict: misaligned pointer");
    // everything written is apart from everything else: rows move while others are still read
    const size_t qn = gb_span(&out->qd, 1), sn = gb_span(&out->sd, 4), ln = 4 * (size_t)c.seqs;
    const struct { const void* p; size_t n; } put[7] = {{o.k, qn}, {o.v, qn}, {o.ks, sn}, {o.vs, sn}, {out_lens, ln}, {out_weights, gb_span(owd, 4)}, {index, gb_span(id, 4)}};
    for (int i = 0; i < 7; i++) {
        bool bad = touches(c, cache, put[i].p, put[i].n) || gb_overlap(put[i].p, put[i].n, lens, ln) || gb_overlap(put[i].p, put[i].n, weights, gb_span(wd, 4));
        for (int j = 0; j < i; j++) bad = bad || gb_overlap(put[i].p, put[i].n, put[j].p, put[j].n);
        if (bad) return gb_fail(ctx, GALOIS_B200_E_DST, "cache_evict: the destinations overlap each other or the operands");
    }
    gb_on_device on(ctx);
    GB_CUDA(ctx, gb_launch(ctx, cache_select_kernel, dim3((unsigned)c.kv_heads, (unsigned)c.seqs), dim3(EV_THREADS), 0, lens, weights, wd->nb[1], wd->nb[2],
                           c.ctx, o.ctx, recent, out_lens, out_weights, owd->nb[1], owd->nb[2], index, id->nb[1], id->nb[2], ctx->dev_status));
    GB_LAUNCHED(ctx, "cache_select");
    if (o.ctx == 0) return 0;
    const dim3 grid((unsigned)((o.ctx + GB_CACHE_BLOCK - 1) / GB_CACHE_BLOCK), (unsigned)c.kv_heads * 2, (unsigned)c.seqs);
    auto kern = c.head_dim == 64 ? cache_gather_kernel<64> : cache_gather_kernel<128>;
    GB_CUDA(ctx, gb_launch(ctx, kern, grid, dim3(128), 0, c, o, out_lens, index, id->nb[1], id->nb[2]));
    GB_LAUNCHED(ctx, "cache_gather");
    return 0;
}
