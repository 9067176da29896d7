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
//   warp 8          loader: TMA copies of the query tiles, then keys and values, 64 rows at a time, through a ring; a slot of it
//                   holds what one step takes, values j and keys j + 2 (the first: keys 0 and 1)
//   warp 9          issues the tensor-core products and owns the tensor memory
//   warp 10         clears what lies behind a sequence's end in its last tile of values
//
// One CTA per SM goes through units of two query tiles (those that see most keys first), and every role runs ahead on its
// own: keys of the next unit are loaded, and its first logits formed, while the results of this one are written.  The two
// query tiles share the keys: two heads of a group over the same tokens where the group is even (their masks agree), else
// two runs of tokens of one head.  Tensor memory: for each query tile two buffers of logits, 2 x 64 columns, so that the
// tensor cores form the next logits while the soft-max has these, and the results, head_dim columns; the probabilities (F16)
// overwrite the first half of their logits and are the second product's operand from there.  The running maximum that
// probabilities refer to is raised only when a row's maximum passes it by 2^7, so that the results in tensor memory are
// rarely rescaled; probabilities are held times 2^7, 2^14 at most, so that F16 keeps 11 bits of them down to 2^-21 of the row's
// largest and is off by 2^-32 of it below (their sum is f32's, and many small ones may count beside a large one).
//
// Measured (B200): 8192 tokens in three prompts, 32 heads over 8 x 128: 366 to 374 us, 0.49 to 0.50 of the measured matrix rate;
// 2048 tokens, 32 heads x 128: 52 to 53 us.  A step (two query tiles x 64 keys) takes some 1960 cycles: the products alone 1240
// of them (logits of 64 keys take 48 cycles an MMA, of 128 keys 64), the issuing warp's loop all of them, a tile's soft-max 1700.
// Tiles of 128 keys with one buffer of logits and tiles of 64 with two, before values and keys shared slots: 378 and 383 us
// on the first, 54.1 and 52.9 on the second, 10.2 and 8.8 on 300 tokens; 64 were taken for the shorter ones.  The shared slots: 375.
//
// A probability of 0 does not hide a value that is not finite: where a result is not finite (or has left F16's range), its rows
// are formed again by the plain loop below, which reads nothing that a query does not see.  That is a warp a row and a step a
// key, for the queries behind a value that is not finite and those whose last tile of keys holds it: one infinite value of one
// head among the 8192 tokens costs 109 ms if it is the first prompt's first, 28 ms if it is the last.
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
__device__ __noinline__ void prompt_row(const rows16& q, const rows16& k, const rows16& v, int t, int k0, int n, int h, int kh, float scale, T* out) {
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
        const float top = x > m || x != x ? x : m, keep = m == -INFINITY ? 0.0f : expf(m - top), p = x == -INFINITY ? 0.0f : expf(x - top);
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

constexpr int PT = 128;  // rows of a tile of queries
constexpr int KT = 64;   // rows of a tile of keys, of values
constexpr int LOADER = 8, ISSUER = 9, CLEARER = 10;  // warps behind the soft-max's
constexpr int THREADS = 11 * 32;
template <int HD>
struct plan {
    static constexpr uint32_t Q_TILE = PT * HD * 2, Q_HALF = PT * 128;  // bytes of a tile; of its first 64 columns
    static constexpr uint32_t TILE = KT * HD * 2, HALF = KT * 128;
    static constexpr int SLOTS = HD == 128 ? 5 : 10;                    // pairs of tiles of keys and values in shared memory
    static constexpr uint32_t Q = 0, KV = 2 * Q_TILE, BARS = KV + SLOTS * 2 * TILE, TOTAL = BARS + 512;
    static_assert(TOTAL <= 227 * 1024, "shared memory");
};
struct prompt_args {
    rows16 q, k, v;
    const int32_t *q_starts, *k_starts;
    int nseq, tq, tk, heads, group;
    float scale;
    void* out;
    int64_t o_head, o_tok;
    bool wide;  // rows of `out` begin at multiples of 32 bytes
    int* status;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void store32(void* to, const uint32_t* x) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7]) : "memory");
}
// N words of a row.  32 bytes at a time fill a sector of memory, 16 half of one: results of 8192 tokens in 372 us and 379, of 2048 in
// 52.8 and 53.3.
template <int N>
__device__ __forceinline__ void store_words(void* to, const uint32_t (&x)[N], bool wide) {
    if (wide) {
#pragma unroll
        for (int e = 0; e < N / 8; e++) store32((uint4*)to + 2 * e, x + 8 * e);
    } else {
#pragma unroll
        for (int e = 0; e < N / 4; e++) ((uint4*)to)[e] = make_uint4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
    }
}
// The largest, or NaN if one of them is: a logit that is not a number has to reach the result.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float f2_low(uint64_t a) { return __uint_as_float((uint32_t)a); }
__device__ __forceinline__ float f2_high(uint64_t a) { return __uint_as_float((uint32_t)(a >> 32)); }

// Bounded wait.  How long another role may rightly take is the length of the prompt's matter (a unit of a million keys, rows
// formed by the plain loop), so the limit is on time in which nobody reports progress: the issuer now and then, the plain
// loop after each row.
__device__ __forceinline__ bool arrived(uint64_t* bar, uint32_t parity, const volatile uint32_t* progress) {
    if (mbar_try(bar, parity)) return true;
    uint32_t seen = *progress;
    long long t0 = clock64();
    while (!mbar_try(bar, parity)) {
        if (clock64() - t0 <= (1ll << 32)) continue;
        if (*progress == seen) return false;
        seen = *progress, t0 = clock64();
    }
    return true;
}

// What of a sequence's starts can be used: queries [q0, q0 + nq), keys [k0, k0 + nk); false if they are out of range.
__device__ __forceinline__ bool sequence(const prompt_args& p, int s, int& q0, int& nq, int& k0, int& nk, bool& descends) {
    q0 = p.q_starts[s], k0 = p.k_starts[s];
    const int q1 = p.q_starts[s + 1], k1 = p.k_starts[s + 1];
    descends = q1 < q0 || k1 < k0;
    const bool ok = q0 >= 0 && q1 <= p.tq && k0 >= 0 && k1 <= p.tk && !descends;
    nq = ok ? q1 - q0 : 0, nk = ok ? k1 - k0 : 0;
    return ok;
}

// Where the CTA's units lie.  Units are counted with the heads fastest and, within a sequence, the tiles that see most keys
// first.  A warp keeps 32 sequences, a lane each, and goes forward.  Where starts descend, that sequence and all behind it are left
// out: their rows could be others' too, and would be written by two CTAs.
struct unit_finder {
    int s0, before, mine, upto, q0, nq, k0, nk;  // first sequence held, tiles before it; this lane's sequence
    __device__ __forceinline__ void load(const prompt_args& p, int span) {
        const int s = s0 + (threadIdx.x & 31);
        bool descends = false;
        q0 = nq = k0 = nk = 0;
        if (s < p.nseq) sequence(p, s, q0, nq, k0, nk, descends);
        const uint32_t descents = __ballot_sync(0xffffffffu, descends);
        if (descents << (31 - (threadIdx.x & 31))) nq = nk = 0;  // here or in a lower lane
        if (descents) s0 = p.nseq;                               // no more are loaded
        mine = upto = (nq + span - 1) / span;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, o);
            if ((int)(threadIdx.x & 31) >= o) upto += y;
        }
    }
    __device__ __forceinline__ void start(const prompt_args& p, int span) {
        s0 = before = 0;
        load(p, span);
    }
};
// The CTA's unit of a round: forwards, then backwards, so that who had one of the larger units gets one of the smaller.
__device__ __forceinline__ int64_t unit_of_round(int r) { return (int64_t)r * gridDim.x + ((r & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x); }
struct prompt_unit {
    int first, q0, nq, k0, nk;  // the first query's place within the sequence; the sequence
    int head0, kh;
    int tiles0, tiles1, n;      // key tiles of the two query tiles, the larger
    // unit `u` of this launch, or false behind the last
    __device__ __forceinline__ bool find(const prompt_args& p, unit_finder& f, int64_t u, int units, int span, bool two_heads) {
        const int unit = (int)(u % units), want = (int)(u / units);
        uint32_t past;
        while ((past = __ballot_sync(0xffffffffu, f.before + f.upto > want)) == 0) {
            if (f.s0 + 32 >= p.nseq) return false;
            f.before += __shfl_sync(0xffffffffu, f.upto, 31);
            f.s0 += 32;
            f.load(p, span);
        }
        const int l = __ffs(past) - 1;
        first = (f.before + __shfl_sync(0xffffffffu, f.upto, l) - 1 - want) * span;
        q0 = __shfl_sync(0xffffffffu, f.q0, l), nq = __shfl_sync(0xffffffffu, f.nq, l);
        k0 = __shfl_sync(0xffffffffu, f.k0, l), nk = __shfl_sync(0xffffffffu, f.nk, l);
        head0 = two_heads ? 2 * unit : unit;
        kh = head0 / p.group;
        tiles0 = tiles(0);
        tiles1 = two_heads ? tiles0 : tiles(PT);
        n = max(tiles0, tiles1);
        return true;
    }
    __device__ __forceinline__ int tiles(int off) const {
        const int rows = min(PT, nq - first - off);
        return rows > 0 ? (max(0, first + off + rows + nk - nq) + KT - 1) / KT : 0;
    }
    // the last tile of values reaches behind the sequence's end
    __device__ __forceinline__ bool ragged() const { return n > 0 && n * KT > nk; }
};

template <int HD, typename T>
__global__ void __launch_bounds__(THREADS, 1)
    prompt_attention_kernel(const prompt_args p, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                            const __grid_constant__ CUtensorMap v_map) {
    using L = plan<HD>;
    constexpr int SLOTS = L::SLOTS;
    extern __shared__ __align__(1024) uint8_t smem[];  // swizzled tiles start at multiples of 1024
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BARS);
    uint64_t *q_full = bars, *q_free = bars + 1, *full = bars + 2, *empty = full + SLOTS, *s_full = empty + SLOTS, *p_ready = s_full + 4, *pv_done = p_ready + 4,
             *v_raw = pv_done + 4;  // [query tile][buffer]; pv_done: [query tile][last but one, last tile of a unit]; v_raw: the units that are ragged in turn
    uint32_t *tmem_at = reinterpret_cast<uint32_t*>(v_raw + 2), *progress = tmem_at + 1;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        *progress = 0;
        tma_prefetch_map(&q_map), tma_prefetch_map(&k_map), tma_prefetch_map(&v_map);
        mbar_init(q_full, 1), mbar_init(q_free, 1), mbar_init(v_raw, 1), mbar_init(v_raw + 1, 1);
        for (int i = 0; i < SLOTS; i++) mbar_init(full + i, 1), mbar_init(empty + i, 1);
        for (int i = 0; i < 4; i++) mbar_init(s_full + i, 1), mbar_init(p_ready + i, 4), mbar_init(pv_done + i, 1);
        fence_mbarrier_init_cluster();
    }
    if (warp == ISSUER) {
        tc_alloc(tmem_at, 512);
        tc_relinquish();
    }
    tc_before_sync();
    __syncthreads();
    tc_after_sync();
    const uint32_t tmem = *tmem_at;
    gb_pdl_entry();

    const bool two_heads = p.group % 2 == 0;
    const int units = two_heads ? p.heads / 2 : p.heads, span = two_heads ? PT : 2 * PT;
    unit_finder f;
    if (warp >= LOADER) f.start(p, span);
    prompt_unit x;
    bool fine = true;

    if (warp == LOADER) {
        int it = 0, nu = 0, nr = 0;  // slots filled so far, units with any keys, ragged ones
        for (int r = 0; fine && x.find(p, f, unit_of_round(r), units, span, two_heads); r++) {
            if (x.n == 0) continue;
            if (lane == 0) {
                if (nu > 0) fine = arrived(q_free, (nu - 1) & 1, progress);
                if (fine) {
                    mbar_expect_tx(q_full, 2 * L::Q_TILE);
                    for (int s = 0; s < 2; s++)
                        for (int h = 0; h < HD / 64; h++)
                            tma_load_3d(smem_u32(smem + L::Q) + s * L::Q_TILE + h * L::Q_HALF, &q_map, 64 * h, x.q0 + x.first + (two_heads ? 0 : s * PT),
                                        two_heads ? x.head0 + s : x.head0, q_full);
                }
                for (int i = 0; i <= x.n && fine; i++, it++) {
                    const int slot = it % SLOTS;
                    if (it >= SLOTS) fine = arrived(empty + slot, (it / SLOTS - 1) & 1, progress);
                    if (!fine) break;
                    // A last tile of values that warp 10 has to clear arrives at a barrier of its own, and warp 10 passes the tile on.
                    // Two such tiles can be under way: this unit's and the one's before, whose values are not waited for here.
                    // The one's before that has been passed on, as its products came before the logits that q_free speaks for.
                    uint64_t* bar = i == x.n && x.ragged() ? v_raw + (nr & 1) : full + slot;
                    const bool second = i + 1 < x.n;  // keys i + 1 exist
                    mbar_expect_tx(bar, second ? 2 * L::TILE : L::TILE);
                    const uint32_t to = smem_u32(smem + L::KV) + slot * 2 * L::TILE;
                    for (int h = 0; h < HD / 64; h++) {
                        tma_load_3d(to + h * L::HALF, i == 0 ? &k_map : &v_map, 64 * h, x.k0 + (i == 0 ? 0 : i - 1) * KT, x.kh, bar);
                        if (second) tma_load_3d(to + L::TILE + h * L::HALF, &k_map, 64 * h, x.k0 + (i + 1) * KT, x.kh, bar);
                    }
                }
            }
            nu++;
            nr += x.ragged();
            fine = __shfl_sync(0xffffffffu, (int)fine, 0);
        }
        // no arrival and no copy is left under way: the last tiles have been used (or, after a time-out, have had time to land)
        if (lane == 0) {
            for (int i = max(0, it - SLOTS); i < it; i++) {
                if (fine) fine = arrived(empty + i % SLOTS, (i / SLOTS) & 1, progress);
                else arrived(full + i % SLOTS, (i / SLOTS) & 1, progress);
            }
            if (fine && nu > 0) fine = arrived(q_free, (nu - 1) & 1, progress);
        }
    } else if (warp == ISSUER) {
        // f32 sums, F16 operands; logits: keys as they are; results: values with the contraction along their rows
        const uint32_t idesc_s = (1u << 4) | ((uint32_t)(KT >> 3) << 17) | ((uint32_t)(PT >> 4) << 24);
        const uint32_t idesc_o = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(PT >> 4) << 24);
        // The whole warp goes through this, and one thread of it issues (see tc_elect).
        const uint32_t lead = tc_elect();
        const uint64_t q_desc = tc_desc(smem_u32(smem + L::Q), 16, 1024, 128), k_desc = tc_desc(smem_u32(smem + L::KV), 16, 1024, 128),
                       v_desc = tc_desc(smem_u32(smem + L::KV), L::HALF, 1024, 128);
        int slot = 0;
        uint32_t parity = 0, q_parity = 0;  // of the ring's round, of the next queries
        uint32_t ready = 0;                 // bit 2 s + b: of the next probabilities of query tile s in buffer b
        auto next = [&]() {
            if (++slot == SLOTS) slot = 0, parity ^= 1;
        };
        auto wait = [&](uint64_t* bar, uint32_t phase) { return __all_sync(0xffffffffu, arrived(bar, phase, progress)) != 0; };
        auto logits = [&](int s, int b, uint64_t k) {  // of the keys at k, into buffer b
            const uint64_t q = q_desc + (uint32_t)(s * (L::Q_TILE >> 4));
#pragma unroll
            for (int kk = 0; kk < HD / 16; kk++) {
                constexpr uint32_t QH = L::Q_HALF >> 4, KH = L::HALF >> 4;
                tc_mma_f16_ss(tmem + s * PT + b * KT, q + (kk / 4 * QH + kk % 4 * 2), k + (kk / 4 * KH + kk % 4 * 2), idesc_s, kk > 0, lead);
            }
            tc_commit(s_full + 2 * s + b, lead);
        };
        for (int r = 0; fine && x.find(p, f, unit_of_round(r), units, span, two_heads); r++) {
            if (x.n == 0) continue;
            fine = wait(q_full, q_parity) && wait(full + slot, parity);
            q_parity ^= 1;
            if (!fine) break;
            // both buffers of one query tile, then of the other (the other order takes as long)
            const uint64_t k0 = k_desc + (uint32_t)(2 * slot * (L::TILE >> 4)), k1 = k0 + (L::TILE >> 4);
            if (x.tiles0 > 0) logits(0, 0, k0);
            if (x.tiles0 > 1) logits(0, 1, k1);
            if (x.tiles1 > 0) logits(1, 0, k0);
            if (x.tiles1 > 1) logits(1, 1, k1);
            tc_commit(empty + slot, lead);
            next();
            if (x.n <= 2) tc_commit(q_free, lead);  // the queries have been used for the last time
            for (int j = 0; j < x.n; j++) {
                const int b = j & 1;
                const uint64_t v = v_desc + (uint32_t)(2 * slot * (L::TILE >> 4)), k = k_desc + (uint32_t)((2 * slot + 1) * (L::TILE >> 4));
                fine = wait(full + slot, parity);
                if ((j & 1023) == 0 && lead) atomicAdd(progress, 1u);
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    const int tiles = s ? x.tiles1 : x.tiles0;
                    if (j >= tiles || !fine) continue;
                    fine = wait(p_ready + 2 * s + b, (ready >> (2 * s + b)) & 1);
                    ready ^= 1u << (2 * s + b);
                    if (!fine) continue;
                    tc_after_sync();
#pragma unroll
                    for (int kk = 0; kk < KT / 16; kk++)
                        tc_mma_f16_ts(tmem + 2 * PT + s * HD, tmem + s * PT + b * KT + kk * 8, v + kk * (2048 >> 4), idesc_o, j > 0 || kk > 0, lead);
                    // logits j + 2 come after these products, so their barrier speaks for both
                    if (j + 2 < tiles) logits(s, b, k);
                    else tc_commit(pv_done + 2 * s + (j + 1 == tiles), lead);
                }
                if (!fine) break;
                tc_commit(empty + slot, lead);
                next();
                if (j + 3 == x.n) tc_commit(q_free, lead);
            }
        }
    } else if (warp == CLEARER) {
        if (blockIdx.x == 0) {
            int a, b, c, d;
            bool e;
            for (int s = lane; s < p.nseq; s += 32)
                if (!sequence(p, s, a, b, c, d, e)) *p.status = GALOIS_B200_E_BADARG;
        }
        int it = 0, nr = 0;
        for (int r = 0; fine && x.find(p, f, unit_of_round(r), units, span, two_heads); r++) {
            it += x.n > 0 ? x.n + 1 : 0;
            if (!x.ragged()) continue;
            fine = __all_sync(0xffffffffu, arrived(v_raw + (nr & 1), (nr >> 1) & 1, progress));
            nr++;
            if (!fine) break;
            const int slot = (it - 1) % SLOTS, valid = x.nk - (x.n - 1) * KT;
            uint4* v = reinterpret_cast<uint4*>(smem + L::KV + slot * 2 * L::TILE);  // [half][row][8 pieces]
            for (int h = 0; h < HD / 64; h++)
                for (int i = valid * 8 + lane; i < KT * 8; i += 32) v[h * KT * 8 + i] = make_uint4(0, 0, 0, 0);
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(full + slot);
        }
    } else {
        // ---- soft-max: thread = row
        const int s = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;
        const uint32_t s_at = tmem + s * PT + lanes, o_at = tmem + 2 * PT + s * HD + lanes;
        const float c = fmaxf(fabsf(p.scale) * 1.4426950408889634f, 1e-30f);  // not 0: a masked logit stays below all others
        const bool flip = p.scale < 0.0f;
        uint32_t nt = 0, done = 0;  // bit b: parity of the next logits in buffer b; the next last but one, the next last products
        for (int r = 0; fine; r++) {  // a wait that ran out ends it: the other roles' waits on this one then run out once each
            const int64_t u = unit_of_round(r);
            // The unit is looked up here and again for the results: what describes it does not stay in registers.
            f.start(p, span);
            if (!x.find(p, f, u, units, span, two_heads)) break;
            const int mine = s ? x.tiles1 : x.tiles0;
            const int last = min(x.first + (two_heads ? 0 : s * PT) + row + x.nk - x.nq, x.nk - 1);  // the last key that this row sees
            const int whole = max(0, x.first + (two_heads ? 0 : s * PT) + x.nk - x.nq + 1) / KT;    // key tiles that the first row, and so all, see whole
            float top = -INFINITY, l = 0.0f;  // what the probabilities refer to, their sum
            for (int j = 0; j < mine; j++) {
                const uint32_t b = j & 1, b_at = s_at + b * KT;
                fine = __all_sync(0xffffffffu, arrived(s_full + 2 * s + b, (nt >> b) & 1, progress));
                if (!fine) break;
                nt ^= 1u << b;
                tc_after_sync();
                float y[KT];
#pragma unroll
                for (int i = 0; i < KT / 32; i++) tc_ld32(b_at + i * 32, reinterpret_cast<uint32_t*>(y) + i * 32);
#pragma unroll
                for (int i = 0; i < KT / 32; i++) tc_wait_ld(reinterpret_cast<uint32_t*>(y) + i * 32);
                if (flip) {
#pragma unroll
                    for (int e = 0; e < KT; e++) y[e] = -y[e];
                }
                if (j >= whole) {
                    const int see = last - j * KT;
#pragma unroll
                    for (int e = 0; e < KT; e++) y[e] = e <= see ? y[e] : -INFINITY;
                }
                uint32_t pk[KT / 2];  // probabilities, pairs of F16
                uint64_t sums[2];
                auto exponentials = [&]() {
                    const float shift = top == -INFINITY ? 0.0f : fmaf(-top, c, 7.0f);
                    const uint64_t cc = f2_pack(c, c), sh = f2_pack(shift, shift);
                    sums[0] = sums[1] = 0;
#pragma unroll
                    for (int e = 0; e < KT / 2; e++) {
                        const uint64_t w = f2_fma(f2_pack(y[2 * e], y[2 * e + 1]), cc, sh);
                        const float p0 = ex2(f2_low(w)), p1 = ex2(f2_high(w));
                        sums[e & 1] = f2_add(sums[e & 1], f2_pack(p0, p1));
                        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(pk[e]) : "f"(p1), "f"(p0));
                    }
                };
                float m[4] = {top, top, top, top};
#pragma unroll
                for (int e = 0; e < KT; e += 2) m[(e >> 1) & 3] = max3(m[(e >> 1) & 3], y[e], y[e + 1]);
                const float most = max3(max3(m[0], m[1], m[2]), m[3], m[3]);
                // Behind the first tile the maximum that probabilities refer to hardly ever moves, so they are formed with the
                // one there is, beside the search for the tile's own; should it have to move after all, they are formed again.
                if (j > 0) exponentials();
                const bool raise = (most - top) * c > 7.0f || (most != most && top == top);  // also the first maximum of a row
                if (j == 0 || __any_sync(0xffffffffu, raise)) {
                    const float keep = raise ? ex2((top - most) * c) : 1.0f;
                    if (raise) top = most;
                    l *= keep;
                    if (j > 0) {
                        // products j - 1 are done: logits j + 1 come after them, or else a barrier of their own says so
                        const bool ok = j + 1 < mine ? arrived(s_full + 2 * s + (b ^ 1), (nt >> (b ^ 1)) & 1, progress) : arrived(pv_done + 2 * s, done & 1, progress);
                        fine = __all_sync(0xffffffffu, ok);
                        if (!fine) break;
                        tc_after_sync();
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
                    exponentials();
                }
                tc_st32(b_at, pk);
                sums[0] = f2_add(sums[0], sums[1]);
                l += f2_low(sums[0]) + f2_high(sums[0]);
                tc_wait_st();
                tc_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_ready + 2 * s + b);
            }
            // ---- results
            if (!fine) break;
            f.start(p, span);
            x.find(p, f, u, units, span, two_heads);
            const int at = x.first + (two_heads ? 0 : s * PT) + row;
            if (mine > 0) fine = __all_sync(0xffffffffu, arrived(pv_done + 2 * s + 1, done >> 1, progress));
            done ^= mine > 1 ? 3u : mine > 0 ? 2u : 0u;
            tc_after_sync();
            const bool none = top == -INFINITY, live = fine && at < x.nq;  // no key, or none that counts
            const float inv = none ? 0.0f : 1.0f / l;
            const int head = two_heads ? x.head0 + s : x.head0;
            T* out = reinterpret_cast<T*>(p.out) + (int64_t)head * p.o_head + (int64_t)(x.q0 + at - row) * p.o_tok;  // row 0's
            T* to = out + (int64_t)row * p.o_tok;
            // The sign bit of `odd`: a result is not finite, or beyond what F16 rounds to its largest number.  (Means of F16 numbers lie
            // within their range, but probabilities that were rounded up can pass their sum's 1.)
            constexpr uint32_t END = sizeof(T) == 4 ? 0x7f800000u : 0x477ff000u;
            uint32_t odd = 0;
#pragma unroll
            for (int i = 0; i < HD / 32; i++) {
                uint32_t o[32];
                tc_ld32(o_at + i * 32, o);
                tc_wait_ld(o);
#pragma unroll
                for (int e = 0; e < 32; e++) {
                    o[e] = none ? 0u : __float_as_uint(__uint_as_float(o[e]) * inv);
                    odd |= (o[e] & 0x7fffffffu) + (0x80000000u - END);
                }
                if (!live) continue;
                if constexpr (sizeof(T) == 4) {
                    store_words(reinterpret_cast<uint4*>(to) + i * 8, o, p.wide);
                } else {
                    uint32_t h[16];
#pragma unroll
                    for (int e = 0; e < 16; e++) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(h[e]) : "f"(__uint_as_float(o[2 * e + 1])), "f"(__uint_as_float(o[2 * e])));
                    store_words(reinterpret_cast<uint4*>(to) + i * 4, h, p.wide);
                }
            }
            tc_before_sync();
            // such rows by the plain loop
            for (uint32_t rows = __ballot_sync(0xffffffffu, live && (odd >> 31)); rows; rows &= rows - 1) {
                const int w = __ffs(rows) - 1, i = at - lane + w, key = i + x.nk - x.nq + 1;
                prompt_row<HD, T>(p.q, p.k, p.v, x.q0 + i, x.k0, key, head, x.kh, p.scale, out + (int64_t)(row - lane + w) * p.o_tok);
                if (lane == 0) atomicAdd(progress, 1u);
            }
        }
    }
    if (!fine && lane == 0) *p.status = GALOIS_B200_E_TIMEOUT;
    tc_before_sync();
    __syncthreads();
    if (warp == ISSUER) tc_dealloc(tmem, 512);
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
    if (!isfinite(scale)) return gb_fail(ctx, GALOIS_B200_E_BADARG, "prompt_attention: scale is not finite");
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
    // units as any lengths need, at most: each sequence has one tile at most that is not full
    const int64_t ctas = ((int64_t)tq / span + std::min(nseq, tq)) * units;
    if (ctas > 0x7fffffff) return gb_fail(ctx, GALOIS_B200_E_SHAPE, "prompt_attention: too many tokens");
    const bool wide = (uintptr_t)dst % 32 == 0 && (heads == 1 || dd->nb[1] * sizeof(T) % 32 == 0) && (tq == 1 || dd->nb[2] * sizeof(T) % 32 == 0);
    const prompt_args a{qr, kr, vr, q_starts, k_starts, nseq, tq, tk, heads, group, scale, dst, dd->nb[1], dd->nb[2], wide, ctx->dev_status};
    CUtensorMap maps[3];
    const rows16* rows[3] = {&qr, &kr, &vr};
    const galois_dim* dims[3] = {qd, kd, vd};
    for (int i = 0; i < 3; i++) {
        // a tensor without tokens is not read; a dimension of one element has any stride
        const uint64_t size[3] = {(uint64_t)qd->ne[0], (uint64_t)std::max<int64_t>(1, dims[i]->ne[2]), (uint64_t)dims[i]->ne[1]};
        const uint64_t stride[2] = {dims[i]->ne[2] > 1 ? (uint64_t)rows[i]->tok * 2 : 256, dims[i]->ne[1] > 1 && dims[i]->ne[2] > 0 ? (uint64_t)rows[i]->head * 2 : 256};
        const uint32_t box[3] = {64, (uint32_t)(i == 0 ? PT : KT), 1};
        const void* base = dims[i]->ne[2] > 0 ? (const void*)rows[i]->p : q;
        rc = gb_tensor_map(ctx, maps + i, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, base, size, stride, box, 128);
        if (rc) return rc;
    }
    auto kern = qd->ne[0] == 64 ? prompt_attention_kernel<64, T> : prompt_attention_kernel<128, T>;
    GB_CUDA(ctx, gb_launch(ctx, kern, dim3((unsigned)std::min<int64_t>(ctas, ctx->sm_count)), dim3(THREADS), qd->ne[0] == 64 ? plan<64>::TOTAL : plan<128>::TOTAL, a, maps[0], maps[1], maps[2]));
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
