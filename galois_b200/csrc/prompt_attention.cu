// Attention of whole prompts, packed one after the other: causal within each sequence, grouped heads.
//
// Query i of a sequence with nq queries and nk keys stands at key i + (nk - nq) and sees the keys up to there:
//   out_i = sum_j softmax_j(scale * q_i . k_j) v_j,   j <= i + nk - nq.
// A query that sees no key gives zeros.  Operands are F16 (the cache's and the mat-mul's type for the contracted
// operand), sums and the soft-max are f32.
//
// 4 head_dim flops a pair of query and key against 4 bytes a token: bound by the tensor cores, and next to them by the
// exponentials (16 a cycle and SM against 32 pairs a cycle that the tensor cores get through).
//
//   warps 0-3, 4-7  soft-max of query tile 0, 1 (128 rows each, a thread per row)
//   warp 8          loader: TMA copies of the query tiles, then keys and values, 128 rows at a time, through four slots
//   warp 9          issues the tensor-core products and owns the tensor memory
//   warp 10         (of 10, 11) looks at the values of tiles that some query does not see whole
//
// The two query tiles of a CTA share the keys: two heads of a group over the same tokens where the group is even (their
// masks agree), else two runs of tokens of one head.  While one tile's logits are in the soft-max, the tensor cores work
// for the other.  Tensor memory: logits 2 x 128 columns, results 2 x head_dim; the probabilities (F16) overwrite the first
// half of their logits and are the second product's operand from there.  The running maximum that probabilities refer to is
// raised only when a row's maximum passes it by 2^8 (F16 holds what that leaves), so that the results in tensor memory
// are rarely rescaled; the logits' barrier also says that the products before them are done, so the rescaling needs no other.
//
// A probability of 0 does not hide a value that is not finite.  So warp 10 clears the values behind a sequence's end
// and, should the last tiles hold any number that is not finite, has the CTA's rows formed again by the plain loop below.
#include "kv_cache_q8.cuh"

#include "tcgen05.cuh"
#include "tma.cuh"

#include <algorithm>

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

constexpr int PT = 128;      // rows of a tile of queries, of keys, of values
constexpr int SLOTS = 4;     // tiles of keys and values in shared memory
constexpr int THREADS = 11 * 32;
template <int HD>
struct plan {
    static constexpr uint32_t TILE = PT * HD * 2, HALF = PT * 128;  // bytes of a tile; of its first 64 columns
    static constexpr uint32_t Q = 0, KV = 2 * TILE, BARS = KV + SLOTS * TILE, TOTAL = 1024 + BARS + 256;
};
struct prompt_args {
    rows16 q, k, v;
    const int32_t *q_starts, *k_starts;
    int nseq, tq, tk, heads, group;
    float scale;
    void* out;
    int64_t o_head, o_tok;
    int* status;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float f2_low(uint64_t a) { return __uint_as_float((uint32_t)a); }
__device__ __forceinline__ float f2_high(uint64_t a) { return __uint_as_float((uint32_t)(a >> 32)); }

// What of a sequence's starts can be used: queries [q0, q0 + nq), keys [k0, k0 + nk); false if they are out of range.
__device__ __forceinline__ bool sequence(const prompt_args& p, int s, int& q0, int& nq, int& k0, int& nk) {
    q0 = p.q_starts[s], k0 = p.k_starts[s];
    const int q1 = p.q_starts[s + 1], k1 = p.k_starts[s + 1];
    const bool ok = q0 >= 0 && q1 >= q0 && q1 <= p.tq && k0 >= 0 && k1 >= k0 && k1 <= p.tk;
    nq = ok ? q1 - q0 : 0, nk = ok ? k1 - k0 : 0;
    return ok;
}

template <int HD, typename T>
__global__ void __launch_bounds__(THREADS, 1)
    prompt_attention_kernel(const prompt_args p, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                            const __grid_constant__ CUtensorMap v_map) {
    using L = plan<HD>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BARS);
    uint64_t *q_full = bars, *full = bars + 1, *empty = full + SLOTS, *s_full = empty + SLOTS, *p_ready = s_full + 2, *o_done = p_ready + 2, *v_raw = o_done + 2;
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(v_raw + 2);
    volatile int* odd = reinterpret_cast<int*>(tmem_at + 1);  // a value that is not finite was seen
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        tma_prefetch_map(&q_map), tma_prefetch_map(&k_map), tma_prefetch_map(&v_map);
        mbar_init(q_full, 1);
        for (int i = 0; i < SLOTS; i++) mbar_init(full + i, 1), mbar_init(empty + i, 1);
        for (int i = 0; i < 2; i++) mbar_init(s_full + i, 1), mbar_init(p_ready + i, 4), mbar_init(o_done + i, 1), mbar_init(v_raw + i, 1);
        fence_mbarrier_init_cluster();
        *odd = 0;
    }
    if (warp == 9) {
        tc_alloc(tmem_at, 512);
        tc_relinquish();
    }
    tc_before_sync();
    __syncthreads();
    tc_after_sync();
    const uint32_t tmem = *tmem_at;
    gb_pdl_entry();

    // ---- the CTA's queries: heads vary fastest, and the last tokens of a sequence, which see the most keys, come first
    const bool two_heads = p.group % 2 == 0;
    const int units = two_heads ? p.heads / 2 : p.heads, span = two_heads ? PT : 2 * PT;
    const int unit = (int)(blockIdx.x % (unsigned)units), want = (int)(blockIdx.x / (unsigned)units);
    int seq = -1, tile = 0, q0 = 0, nq = 0, k0 = 0, nk = 0;
    for (int s0 = 0, before = 0; s0 < p.nseq; s0 += 32) {
        int a, n = 0, c, d;
        if (s0 + lane < p.nseq && !sequence(p, s0 + lane, a, n, c, d) && blockIdx.x == 0 && warp == 0) *p.status = GALOIS_B200_E_BADARG;
        const int mine = (n + span - 1) / span;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, before + upto > want);
        if (past && seq < 0) {
            const int l = __ffs(past) - 1, tiles = __shfl_sync(0xffffffffu, mine, l);
            seq = s0 + l;
            tile = tiles - 1 - (want - before - (__shfl_sync(0xffffffffu, upto, l) - tiles));
            if (blockIdx.x != 0) break;  // the first CTA looks at all starts
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (seq >= 0) sequence(p, seq, q0, nq, k0, nk);
    // per query tile s: its first token (within the sequence), its head, its valid rows, its key tiles
    const int head0 = two_heads ? 2 * unit : unit, kh = head0 / p.group;
    int n_tiles[2];
#pragma unroll
    for (int s = 0; s < 2; s++) {
        const int first = tile * span + (two_heads ? 0 : s * PT), rows = seq < 0 ? 0 : max(0, min(PT, nq - first));
        n_tiles[s] = rows > 0 ? (max(0, first + rows + nk - nq) + PT - 1) / PT : 0;
    }
    const int n = max(n_tiles[0], n_tiles[1]);
    const int whole = max(0, tile * span + nk - nq + 1) / PT;  // key tiles that every query sees whole
    bool fine = true;

    if (warp == 8) {
        if (lane == 0 && n > 0) {
            mbar_expect_tx(q_full, 2 * L::TILE);
            for (int s = 0; s < 2; s++)
                for (int h = 0; h < HD / 64; h++)
                    tma_load_3d(smem_u32(smem + L::Q) + s * L::TILE + h * L::HALF, &q_map, 64 * h, q0 + tile * span + (two_heads ? 0 : s * PT),
                                two_heads ? head0 + s : head0, q_full);
            int i = 0;
            for (; i < 2 * n; i++) {
                const int slot = i % SLOTS;
                if (i >= SLOTS && !mbar_wait_bounded(empty + slot, (i / SLOTS - 1) & 1)) {
                    fine = false;
                    break;
                }
                // values that warp 10 looks at arrive at a barrier of its own; it passes them on
                uint64_t* bar = (i & 1) && (i >> 1) >= whole ? v_raw + (((i >> 1) - whole) & 1) : full + slot;
                mbar_expect_tx(bar, L::TILE);
                for (int h = 0; h < HD / 64; h++)
                    tma_load_3d(smem_u32(smem + L::KV) + slot * L::TILE + h * L::HALF, (i & 1) ? &v_map : &k_map, 64 * h, k0 + (i >> 1) * PT, kh, bar);
            }
            if (!fine) {  // leave no copy of its own in flight
                mbar_wait_bounded(q_full, 0);
                for (int j = max(0, i - SLOTS); j < i; j++) mbar_wait_bounded(full + j % SLOTS, (j / SLOTS) & 1);
            }
        }
        __syncwarp();
    } else if (warp == 9) {
        if (lane == 0 && n > 0) {
            // f32 sums, F16 operands; logits: keys as they are; results: values with the contraction along their rows
            const uint32_t idesc_s = (1u << 4) | ((uint32_t)(PT >> 3) << 17) | ((uint32_t)(PT >> 4) << 24);
            const uint32_t idesc_o = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(PT >> 4) << 24);
            const uint32_t q_at = smem_u32(smem + L::Q), kv_at = smem_u32(smem + L::KV);
            auto logits = [&](int s, int j) {
                const uint32_t k_at = kv_at + (uint32_t)((2 * j) % SLOTS) * L::TILE;
#pragma unroll
                for (int kk = 0; kk < HD / 16; kk++) {
                    const uint32_t off = (kk / 4) * L::HALF + (kk % 4) * 32;
                    tc_mma_f16_ss(tmem + s * PT, tc_desc(q_at + s * L::TILE + off, 16, 1024, 128), tc_desc(k_at + off, 16, 1024, 128), idesc_s, kk > 0);
                }
                tc_commit(s_full + s);
            };
            fine = mbar_wait_bounded(q_full, 0) && mbar_wait_bounded(full, 0);
            if (fine) {
                for (int s = 0; s < 2; s++)
                    if (n_tiles[s] > 0) logits(s, 0);
                tc_commit(empty);
            }
            for (int j = 0; j < n && fine; j++) {
                const int vs = (2 * j + 1) % SLOTS, ks = (2 * j + 2) % SLOTS;
                fine = mbar_wait_bounded(full + vs, ((2 * j + 1) / SLOTS) & 1) && (j + 1 >= n || mbar_wait_bounded(full + ks, ((2 * j + 2) / SLOTS) & 1));
                for (int s = 0; s < 2 && fine; s++) {
                    if (j >= n_tiles[s]) continue;
                    fine = mbar_wait_bounded(p_ready + s, j & 1);
                    if (!fine) break;
                    tc_after_sync();
#pragma unroll
                    for (int kk = 0; kk < PT / 16; kk++)
                        tc_mma_f16_ts(tmem + 2 * PT + s * HD, tmem + s * PT + kk * 8, tc_desc(kv_at + vs * L::TILE + kk * 2048, L::HALF, 1024, 128), idesc_o, j > 0 || kk > 0);
                    if (j + 1 < n_tiles[s]) logits(s, j + 1);
                    else tc_commit(o_done + s);
                }
                if (fine) {
                    tc_commit(empty + vs);
                    if (j + 1 < n) tc_commit(empty + ks);
                }
            }
        }
        __syncwarp();
    } else if (warp == 10) {
        for (int j = whole; j < n && fine; j++) {
            const int slot = (2 * j + 1) % SLOTS, valid = min(PT, nk - j * PT);
            fine = __all_sync(0xffffffffu, mbar_wait_bounded(v_raw + ((j - whole) & 1), ((j - whole) >> 1) & 1));
            if (!fine) break;
            uint4* v = reinterpret_cast<uint4*>(smem + L::KV + slot * L::TILE);  // [half][row][8 pieces]
            uint32_t bad = 0;
#pragma unroll 8
            for (int x = lane; x < (int)L::TILE / 16; x += 32) {
                if ((x >> 3) % PT < valid) {
                    const uint4 w = v[x];
                    // an exponent of all ones carries into the sign's place
                    bad |= ((w.x & 0x7c007c00u) + 0x04000400u) | ((w.y & 0x7c007c00u) + 0x04000400u) | ((w.z & 0x7c007c00u) + 0x04000400u) |
                           ((w.w & 0x7c007c00u) + 0x04000400u);
                } else {
                    v[x] = make_uint4(0, 0, 0, 0);
                }
            }
            if (__any_sync(0xffffffffu, (bad & 0x80008000u) != 0) && lane == 0) *odd = 1;
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(full + slot);
        }
    } else if (warp < 8) {
        // ---- soft-max: thread = row
        const int s = warp >> 2, row = threadIdx.x & 127;
        const int first = tile * span + (two_heads ? 0 : s * PT), at = first + row, mine = n_tiles[s];
        const int last = min(at + nk - nq, nk - 1);  // the last key that this row sees
        const uint32_t s_at = tmem + s * PT + ((uint32_t)(warp & 3) << 21), o_at = tmem + 2 * PT + s * HD + ((uint32_t)(warp & 3) << 21);
        const float c = fmaxf(fabsf(p.scale) * 1.4426950408889634f, 1e-30f);  // not 0: a masked logit stays below all others
        const bool flip = p.scale < 0.0f;
        float top = -INFINITY, l = 0.0f;  // what the probabilities refer to, their sum
        for (int j = 0; j < mine; j++) {
            fine = __all_sync(0xffffffffu, mbar_wait_bounded(s_full + s, j & 1));
            if (!fine) break;
            tc_after_sync();
            // The logits are read twice, 32 at a time: 128 of them would not stay in registers.
            const int see = j >= whole ? last - j * PT : PT;
            float m0 = top, m1 = -INFINITY;
            float x[2][32];
            tc_ld32(s_at, reinterpret_cast<uint32_t*>(x[0]));
#pragma unroll
            for (int i = 0; i < PT / 32; i++) {
                float* y = x[i & 1];
                tc_wait_ld(reinterpret_cast<uint32_t*>(y));
                tc_ld32(s_at + (i + 1) % (PT / 32) * 32, reinterpret_cast<uint32_t*>(x[(i + 1) & 1]));
                if (flip || see < PT) {
#pragma unroll
                    for (int e = 0; e < 32; e++) y[e] = 32 * i + e <= see ? (flip ? -y[e] : y[e]) : -INFINITY;
                }
#pragma unroll
                for (int e = 0; e < 32; e += 4) m0 = max3(m0, y[e], y[e + 1]), m1 = max3(m1, y[e + 2], y[e + 3]);
            }
            m0 = fmaxf(m0, m1);
            const bool raise = (m0 - top) * c > 8.0f;  // also the first maximum of a row
            if (__any_sync(0xffffffffu, raise)) {
                const float to = raise ? m0 : top, keep = raise ? ex2((top - to) * c) : 1.0f;
                top = to;
                l *= keep;
                if (j > 0) {
#pragma unroll
                    for (int i = 0; i < HD / 32; i++) {
                        uint32_t o[32];
                        tc_ld32(o_at + i * 32, o);
                        tc_wait_ld(o);
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                        tc_st32(o_at + i * 32, o);
                    }
                }
            }
            const float shift = top == -INFINITY ? 0.0f : -top * c;
            const uint64_t cc = f2_pack(c, c), sh = f2_pack(shift, shift);
            uint64_t sum[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < PT / 32; i++) {
                float* y = x[i & 1];  // the first 32 were asked for above
                tc_wait_ld(reinterpret_cast<uint32_t*>(y));
                if (i + 1 < PT / 32) tc_ld32(s_at + (i + 1) * 32, reinterpret_cast<uint32_t*>(x[(i + 1) & 1]));
                if (flip || see < PT) {
#pragma unroll
                    for (int e = 0; e < 32; e++) y[e] = 32 * i + e <= see ? (flip ? -y[e] : y[e]) : -INFINITY;
                }
                uint32_t pk[16];
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const uint64_t z = f2_fma(f2_pack(y[2 * e], y[2 * e + 1]), cc, sh);
                    const float p0 = ex2(f2_low(z)), p1 = ex2(f2_high(z));
                    sum[e & 1] = f2_add(sum[e & 1], f2_pack(p0, p1));
                    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(pk[e]) : "f"(p1), "f"(p0));
                }
                tc_st16(s_at + i * 16, pk);
            }
            sum[0] = f2_add(sum[0], sum[1]);
            l += f2_low(sum[0]) + f2_high(sum[0]);
            tc_wait_st();
            tc_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_ready + s);
        }
        // ---- results
        if (fine && mine > 0) {
            fine = __all_sync(0xffffffffu, mbar_wait_bounded(o_done + s, 0));
            tc_after_sync();
        }
        if (fine) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            T* to = reinterpret_cast<T*>(p.out) + (int64_t)(two_heads ? head0 + s : head0) * p.o_head + (int64_t)(q0 + at) * p.o_tok;
#pragma unroll
            for (int i = 0; i < HD / 32; i++) {
                uint32_t o[32];
#pragma unroll
                for (int e = 0; e < 32; e++) o[e] = 0;
                if (mine > 0) {
                    tc_ld32(o_at + i * 32, o);
                    tc_wait_ld(o);
                }
                if (seq >= 0 && at < nq) {
                    if constexpr (sizeof(T) == 4) {
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            reinterpret_cast<float4*>(to)[i * 8 + e] = l == 0.0f ? make_float4(0.f, 0.f, 0.f, 0.f)
                                                                                 : make_float4(__uint_as_float(o[4 * e]) * inv, __uint_as_float(o[4 * e + 1]) * inv,
                                                                                               __uint_as_float(o[4 * e + 2]) * inv, __uint_as_float(o[4 * e + 3]) * inv);
                    } else {
                        uint32_t h[16];
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            const float a = l == 0.0f ? 0.0f : __uint_as_float(o[2 * e]) * inv, b = l == 0.0f ? 0.0f : __uint_as_float(o[2 * e + 1]) * inv;
                            asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(h[e]) : "f"(b), "f"(a));
                        }
#pragma unroll
                        for (int e = 0; e < 4; e++) reinterpret_cast<uint4*>(to)[i * 4 + e] = make_uint4(h[4 * e], h[4 * e + 1], h[4 * e + 2], h[4 * e + 3]);
                    }
                }
            }
        }
    }
    if (!fine && lane == 0) *p.status = GALOIS_B200_E_TIMEOUT;
    tc_before_sync();
    __syncthreads();
    if (warp == 9) tc_dealloc(tmem, 512);
    if (*odd) {
        for (int r = warp; r < 2 * PT; r += THREADS / 32) {
            const int s = r / PT, at = tile * span + (two_heads ? 0 : s * PT) + r % PT, h = two_heads ? head0 + s : head0;
            if (at >= nq) continue;
            prompt_row<HD, T>(p.q, p.k, p.v, q0 + at, k0, at + nk - nq + 1, h, kh, p.scale, reinterpret_cast<T*>(p.out) + h * p.o_head + (int64_t)(q0 + at) * p.o_tok);
        }
    }
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
    const int group = heads / kv_heads, units = group % 2 == 0 ? heads / 2 : heads, span = group % 2 == 0 ? PT : 2 * PT;
    // as many tiles as any lengths need: each sequence has at most one that is not full
    const int64_t ctas = ((int64_t)tq / span + std::min(nseq, tq)) * units;
    if (ctas > 0x7fffffff) return gb_fail(ctx, GALOIS_B200_E_SHAPE, "prompt_attention: too many tokens");
    const prompt_args a{qr, kr, vr, q_starts, k_starts, nseq, tq, tk, heads, group, scale, dst, dd->nb[1], dd->nb[2], ctx->dev_status};
    CUtensorMap maps[3];
    const rows16* rows[3] = {&qr, &kr, &vr};
    const galois_dim* dims[3] = {qd, kd, vd};
    for (int i = 0; i < 3; i++) {
        // a tensor without tokens is not read; a dimension of one element has any stride
        const uint64_t size[3] = {(uint64_t)qd->ne[0], (uint64_t)std::max<int64_t>(1, dims[i]->ne[2]), (uint64_t)dims[i]->ne[1]};
        const uint64_t stride[2] = {dims[i]->ne[2] > 1 ? (uint64_t)rows[i]->tok * 2 : 256, dims[i]->ne[1] > 1 ? (uint64_t)rows[i]->head * 2 : 256};
        const uint32_t box[3] = {64, PT, 1};
        const void* base = dims[i]->ne[2] > 0 ? (const void*)rows[i]->p : q;
        rc = gb_tensor_map(ctx, maps + i, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, base, size, stride, box, 128);
        if (rc) return rc;
    }
    auto kern = qd->ne[0] == 64 ? prompt_attention_kernel<64, T> : prompt_attention_kernel<128, T>;
    GB_CUDA(ctx, gb_launch(ctx, kern, dim3((unsigned)ctas), dim3(THREADS), qd->ne[0] == 64 ? plan<64>::TOTAL : plan<128>::TOTAL, a, maps[0], maps[1], maps[2]));
    GB_LAUNCHED(ctx, "prompt_attention");
    return 0;
}

}  // namespace

int gb_prompt_attention_init(galois_b200_ctx* ctx) {
    GB_CUDA(ctx, cudaFuncSetAttribute(prompt_attention_kernel<64, __half>, cudaFuncAttributeMaxDynamicSharedMemorySize, plan<64>::TOTAL));
    GB_CUDA(ctx, cudaFuncSetAttribute(prompt_attention_kernel<64, float>, cudaFuncAttributeMaxDynamicSharedMemorySize, plan<64>::TOTAL));
    GB_CUDA(ctx, cudaFuncSetAttribute(prompt_attention_kernel<128, __half>, cudaFuncAttributeMaxDynamicSharedMemorySize, plan<128>::TOTAL));
    GB_CUDA(ctx, cudaFuncSetAttribute(prompt_attention_kernel<128, float>, cudaFuncAttributeMaxDynamicSharedMemorySize, plan<128>::TOTAL));
    return 0;
}

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
