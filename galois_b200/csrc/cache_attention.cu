// Attention of one new token per sequence over the 8-bit key/value cache.
//
//   s_j = scale * (q . k_j),  p_j = exp(s_j - max) / sum,  out = sum_j p_j v_j      over the cache rows j < len
//
// with grouped heads: heads / kv_heads consecutive query heads read the same key/value head.  A sequence of length
// 0 gives zeros.  With `weights`, weights_out[j] = weights[j] + the sum of p_j over the heads of the group.
#include "kv_cache_q8.cuh"

#include "ptx.cuh"
#include "tma.cuh"

#include <math.h>

namespace {

// What has to be read is 2 HD bytes a row and head (the arithmetic, 4 HD flops a row and query head, is far below
// the machine's), so the kernel is built to keep HBM busy whatever the lengths are:
//
//  * The rows of all (sequence, key/value head) pairs form one list of 32-row blocks, which is dealt evenly to all
//    warps of the device, each a contiguous part; a part may begin and end inside a pair.  No length is known on the
//    host, and none makes a warp wait for another: a warp writes what it has of a pair as one piece (maximum, sum, HD
//    halved means per head), and a second launch joins the pieces.
//  * Each warp streams its blocks through a ring of its own in shared memory, across the borders of pairs: one TMA copy
//    for the keys of a block and one for its values; nothing synchronises the CTA.  The logits of the next block are
//    formed between the soft-max and the products of this one, so that a warp always has independent work to issue.
//  * The whole numbers are exact in F16, so both products run on mma.sync m16n8k16 with f32 sums: the 16 rows are up
//    to 8 heads of the group twice, once with the upper and once with the lower 11 bits of the f32 operand.  The query is
//    scaled to 2^14..2^15, a block's probabilities so that their largest is 2^15, and lower bits are kept times 2^12: numbers
//    down to 2^-30 of the largest keep 22 bits, smaller ones are off by 2^-52 of it.  The order of a contraction is free, so
//    fragments are taken as a lane's 16-byte loads give them: of the keys, lane (g, t) has numbers 16 t.. of one row; of
//    the values, CW numbers of four rows, whose bytes are paired by permutes.  Which row and which chunk g and t stand
//    for is chosen so that the eight lanes of a load's phase meet no bank of the swizzled tile twice.
//
// Measured (B200): 64 sequences of up to 8192 rows, 8 key/value heads x 128, groups of 4: 664 MB in 140 to 151 us (one build, different
// cards), 4.4 to 4.7 TB/s, 0.67 to 0.72 of the copy rate; one sequence of 2048 rows, 32 heads: 13.9 us with the joining launch; 16
// sequences of up to 4096 rows with weights 39.4 us.  No unit is full (issue 0.53, ALU 0.40, FMA 0.32, tensor cores 0.30): an MMA with
// the conversion of its operand takes 13 to 16 cycles of a scheduler, the bare one 8.6.  Probabilities relative to each block, with
// lower halves of their own power of two, cost 2.4 % of the batch (143.4 us beside 146.8) over ones relative to the piece, which were off by
// 2^-25 of the largest.  Eight warps or twelve with shorter rings, in one run of an earlier build: the batch 145 and 141 us, one
// sequence 13.9 and 15.5, 16 sequences with weights 37.7 and 38.5; eight lose 2.5 % on the first and gain on the others.
constexpr int WARPS = 8;
constexpr int BLK = GB_CACHE_BLOCK;
template <int HD>
struct ring {
    static constexpr int HALF = BLK * HD;    // bytes of a block's keys (or values)
    static constexpr int DEPTH = HD == 128 ? 3 : 6;   // tiles of keys, and as many of values
    static constexpr int BARS = 1024 + WARPS * 2 * DEPTH * HALF;  // offset of the barriers; 1024 to align the tiles
    static constexpr int TOTAL = BARS + WARPS * 2 * DEPTH * 8;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float low(uint64_t a) { return __uint_as_float((uint32_t)a); }
__device__ __forceinline__ float high(uint64_t a) { return __uint_as_float((uint32_t)(a >> 32)); }
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
// Two numbers, at most 2^15, as F16 pairs: the nearest, and what is left of each (at most 2^3) times 2^12.  Without that factor the
// lower halves of numbers below 2^-3 would fall below F16's normal range.
constexpr float LOW = 0x1p-12f, F32_MAX = 3.402823466e38f;
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = pack_half2(a, b);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    lo = pack_half2((a - f.x) * (1.0f / LOW), (b - f.y) * (1.0f / LOW));
}
__device__ __forceinline__ uint32_t minus_1152(uint32_t h) {  // 1024 + (q + 128) -> q, exact
    const __half2 r = __hadd2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half((unsigned short)0xe480)));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
    return v;
}
// Where 16-byte chunk c of a block's row lies: TMA's swizzle over rows of 128 or 64 bytes.
template <int HD>
__device__ __forceinline__ uint32_t tile_at(int row, int c) {
    return HD == 128 ? (uint32_t)(row * 128 + ((c ^ (row & 7)) << 4)) : (uint32_t)(row * 64 + ((c ^ ((row >> 1) & 3)) << 4));
}
// The row of a block that column n of the n-tile j of logits stands for.
template <int HD>
__device__ __forceinline__ int row_of(int j, int n) {
    return 8 * j + (HD == 128 ? (n >> 1) + 4 * (n & 1) : n);
}

__device__ __forceinline__ int checked_len(int n, int ctx) { return n < 0 || n > ctx ? 0 : n; }
// By one warp of the first kernel that a call launches.
__device__ __forceinline__ void report_lens(const int32_t* __restrict__ lens, int n, int ctx, int* __restrict__ status) {
    for (int i = threadIdx.x & 31; i < n; i += 32)
        if (lens[i] < 0 || lens[i] > ctx) *status = GALOIS_B200_E_BADARG;
}

// How the list of blocks is dealt: `total` blocks over `warps` contiguous parts, none of them empty.
struct deal {
    int64_t total;
    int warps;
    __device__ deal(int64_t n, int most) : total(n), warps((int)min(n, (int64_t)most)) {}
    __device__ int64_t begin(int w) const { return (int64_t)w * total / warps; }
    __device__ int owner(int64_t b) const { return (int)(((b + 1) * warps - 1) / total); }
};

// Sum over the warp of `per` x the blocks of sequences [0, n).
__device__ __forceinline__ int64_t count_blocks(const int32_t* __restrict__ lens, int n, int ctx, int per) {
    int64_t c = 0;
    for (int i = threadIdx.x & 31; i < n; i += 32) c += (checked_len(lens[i], ctx) + BLK - 1) / BLK;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
    return c * per;
}

// A place in the list: block `blk` of a pair, with `left` rows from its first to the end.
struct place {
    int seq, kh, tile, blk, left, len;
    // true where a new pair begins
    __device__ __forceinline__ bool advance(const int32_t* __restrict__ lens, const gb_cache_view& c, int tiles) {
        blk++, left -= BLK;
        if (left > 0) return false;
        blk = 0;
        if (++tile == tiles) {
            tile = 0;
            if (++kh == c.kv_heads) {
                kh = 0;
                do {
                    seq++;
                    len = seq < c.seqs ? checked_len(lens[seq], c.ctx) : 1;
                } while (len == 0);
            }
        }
        left = len;
        return true;
    }
};

struct step_args {
    const float* q;
    int64_t q_head, q_seq;
    gb_cache_view c;
    const int32_t* lens;
    int group, tiles;  // query heads per key/value head; tiles of 8 of them
    int rows;          // min(8, group): heads that a piece holds
    float scale;       // scale * log2(e) / 2^scale_exp, 1/2 to 1
    int scale_exp;
    float *acc, *stats;  // pieces: [piece][rows][HD], [piece][rows][2]
    float* scores;       // [seq][heads][ctx] base-2 logits, or null
    int* status;
};

template <int HD>
__global__ void __launch_bounds__(WARPS * 32, 1)
    cache_attention_kernel(const step_args p, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int CW = HD / 8, NW = CW / 4, KS = HD / 16;  // bytes of a value row per lane, words of them, steps over head_dim
    constexpr int DEPTH = ring<HD>::DEPTH;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + ring<HD>::BARS) + warp * 2 * DEPTH;  // of the keys' tiles, then of the values'
    if (lane == 0) {
        tma_prefetch_map(&k_map);
        tma_prefetch_map(&v_map);
        for (int i = 0; i < 2 * DEPTH; i++) mbar_init(bars + i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    gb_pdl_entry();
    const gb_cache_view& c = p.c;
    const int per = c.kv_heads * p.tiles, heads = c.kv_heads * p.group;
    const deal D(count_blocks(p.lens, c.seqs, c.ctx, per), (int)gridDim.x * WARPS);
    if (blockIdx.x == 0 && warp == 0) report_lens(p.lens, c.seqs, c.ctx, p.status);
    const int w = warp * (int)gridDim.x + (int)blockIdx.x;  // parts of neighbours lie on different SMs
    if (w >= D.warps) return;
    const int64_t b0 = D.begin(w);
    const int count = (int)(D.begin(w + 1) - b0);
    // the place of block b0
    place at{};
    {
        int64_t before = 0;
        for (int s0 = 0;; s0 += 32) {
            const int n = s0 + lane < c.seqs ? checked_len(p.lens[s0 + lane], c.ctx) : 0;
            int64_t mine = (int64_t)((n + BLK - 1) / BLK) * per, upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, before + upto > b0);
            if (past) {
                const int l = __ffs(past) - 1;
                const int64_t off = b0 - before - (__shfl_sync(0xffffffffu, upto, l) - __shfl_sync(0xffffffffu, mine, l));
                at.seq = s0 + l;
                at.len = __shfl_sync(0xffffffffu, n, l);
                const int blocks = (at.len + BLK - 1) / BLK, inner = (int)(off / blocks);
                at.blk = (int)(off % blocks);
                at.left = at.len - at.blk * BLK;
                at.kh = inner / p.tiles, at.tile = inner % p.tiles;
                break;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    const uint32_t base = ((smem_u32(smem) + 1023u) & ~1023u) + (uint32_t)(warp * 2 * DEPTH * ring<HD>::HALF);
    // Keys are wanted one block earlier than values: the place of the newest keys is kept for the values' next copy.
    place ahead = at;
    int last_row = 0, last_kh = 0, last_seq = 0, to_fetch = count;  // blocks whose keys have not been asked for
    int64_t scale_at = ahead.kh * c.s_head + ahead.seq * c.s_seq;
    // the scales of the blocks from the current one on, in the ring's order
    float2 scales[DEPTH + 1];
    auto fetch_keys = [&](int slot) -> float2 {
        last_row = ahead.blk * BLK, last_kh = ahead.kh, last_seq = ahead.seq;
        const float2 sc = make_float2(c.ks[scale_at + ahead.blk], c.vs[scale_at + ahead.blk]);
        if (lane == 0) {
            mbar_expect_tx(bars + slot, ring<HD>::HALF);
            tma_load_4d(base + (uint32_t)(slot * ring<HD>::HALF), &k_map, 0, last_row, last_kh, last_seq, bars + slot);
        }
        if (ahead.advance(p.lens, c, p.tiles)) scale_at = ahead.kh * c.s_head + ahead.seq * c.s_seq;
        to_fetch--;
        return sc;
    };
    auto fetch_values = [&](int slot) {
        if (lane == 0) {
            mbar_expect_tx(bars + DEPTH + slot, ring<HD>::HALF);
            tma_load_4d(base + (uint32_t)((DEPTH + slot) * ring<HD>::HALF), &v_map, 0, last_row, last_kh, last_seq, bars + DEPTH + slot);
        }
    };
#pragma unroll
    for (int i = 0; i < DEPTH; i++) {
        scales[i] = make_float2(0.f, 0.f);
        if (to_fetch > 0) scales[i] = fetch_keys(i), fetch_values(i);
    }
    scales[DEPTH] = make_float2(0.f, 0.f);
    uint32_t phases = 0;  // bit i: parity that barrier i completes next
    auto wait = [&](int bar) {
        const bool ok = mbar_wait_bounded(bars + bar, (phases >> bar) & 1);
        phases ^= 1u << bar;
        return __all_sync(0xffffffffu, ok);
    };

    uint32_t qa[KS][4];
    float factor = 0.0f, factor2 = 0.0f;  // their product turns a key scale into the base-2 logit of a product of whole numbers
    bool live = false;       // this lane's head exists
    float* scores = nullptr;  // its logits' row, where they are wanted
    // The query of the pair at `at`: lane (g, t) holds numbers 16 (t + 4 i) + 4 j.. of head g, times the power of two that
    // brings the largest to 2^14..2^15, as two F16 each.
    auto load_query = [&]() {
        const int head = at.kh * p.group + at.tile * 8 + g;
        live = g < p.group - at.tile * 8;
        float4 f[KS];
        float top = 0.0f;
        const float* qh = p.q + (int64_t)head * p.q_head + (int64_t)at.seq * p.q_seq;
        scores = live && p.scores ? p.scores + ((int64_t)at.seq * heads + head) * c.ctx : nullptr;
#pragma unroll
        for (int i = 0; i < KS; i++) {
            f[i] = live ? *reinterpret_cast<const float4*>(qh + 16 * (t + 4 * (i / 4)) + 4 * (i % 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
            top = fmaxf(top, fmaxf(fmaxf(fabsf(f[i].x), fabsf(f[i].y)), fmaxf(fabsf(f[i].z), fabsf(f[i].w))));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = max(-110, (int)(__float_as_uint(top) >> 23) - 127);
        const float up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
        // The scale, the query's power of two and the key's scale may each be near an end of f32's range, and only their product an
        // ordinary number: the powers of two come in as two halves, so that nothing is lost unless the product itself is.
        const int pow2 = max(-252, e - 14 + p.scale_exp), half = pow2 >> 1;
        factor = p.scale * __uint_as_float((uint32_t)(127 + half) << 23);
        factor2 = __uint_as_float((uint32_t)(127 + pow2 - half) << 23);
#pragma unroll
        for (int i = 0; i < KS; i++) {
            split2(f[i].x * up, f[i].y * up, qa[i][0], qa[i][1]);
            split2(f[i].z * up, f[i].w * up, qa[i][2], qa[i][3]);
        }
    };
    // Base-2 logits of a block's 32 rows: lane (g, t) gets those of head g and rows row_of(j, 2 t), row_of(j, 2 t + 1).
    auto logits = [&](int slot, float k_scale, float (&x)[4][2]) {
        const uint32_t ks = base + (uint32_t)(slot * ring<HD>::HALF);
        float f = k_scale * factor * factor2;
        if (fabsf(f) > F32_MAX) f = copysignf(F32_MAX, f);  // a product of 0 is a logit of 0 all the same
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float s[KS / 4][4];
#pragma unroll
            for (int cc = 0; cc < KS / 4; cc++) {
                s[cc][0] = s[cc][1] = s[cc][2] = s[cc][3] = 0.0f;
                const uint4 kw = lds128(ks + tile_at<HD>(row_of<HD>(j, g), t + 4 * cc));
                const uint32_t word[4] = {kw.x, kw.y, kw.z, kw.w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t u = word[i] ^ 0x80808080u;
                    mma16816(s[cc], qa[4 * cc + i][0], qa[4 * cc + i][1], qa[4 * cc + i][2], qa[4 * cc + i][3],
                             minus_1152(__byte_perm(u, 0x64646464u, 0x4140)), minus_1152(__byte_perm(u, 0x64646464u, 0x4342)));
                }
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float hi = s[0][e], lo = s[0][e + 2];
                if constexpr (KS == 8) hi += s[1][e], lo += s[1][e + 2];
                x[j][e] = fmaf(lo, LOW, hi) * f;
            }
        }
    };

    uint64_t o[NW * 4];  // pairs of f32
#pragma unroll
    for (int i = 0; i < NW * 4; i++) o[i] = 0;
    // `l`, the sum of the piece's probabilities, is in units of 2^m, `o` in units of 2^(o_ref + o_exp).  Both are raised when a block passes
    // them by more than 2^SLACK, which f32 has room for, so that sums are rarely rescaled.
    constexpr float SLACK = 8.0f;
    float m = -INFINITY, l = 0.0f, o_ref = -INFINITY;
    int o_exp = 0;
    float x[4][2], xn[4][2];
    load_query();
    int slot = 0;
    bool fine = wait(0);
    logits(0, scales[0].x, x);
    __syncwarp();
    bool more = to_fetch > 0;  // the block behind the ring exists: its keys now, its values when this block's are used
    if (more) scales[DEPTH] = fetch_keys(0);
    for (int todo = count; todo > 0 && fine; todo--) {
        const int next = slot + 1 == DEPTH ? 0 : slot + 1;
        if (todo > 1) fine = wait(next);
        logits(next, scales[1].x, xn);  // formed again below if a new pair begins there; of no use behind the last block
        fine = fine && wait(DEPTH + slot);
        const uint32_t vs = base + (uint32_t)((DEPTH + slot) * ring<HD>::HALF);
        if (at.left < BLK) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (row_of<HD>(j, 2 * t) >= at.left) x[j][0] = -INFINITY;
                if (row_of<HD>(j, 2 * t + 1) >= at.left) x[j][1] = -INFINITY;
            }
        }
        if (scores) {
            float* to = scores + at.blk * BLK;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (row_of<HD>(j, 2 * t) < at.left) to[row_of<HD>(j, 2 * t)] = x[j][0];
                if (row_of<HD>(j, 2 * t + 1) < at.left) to[row_of<HD>(j, 2 * t + 1)] = x[j][1];
            }
        }
        float top = fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[1][0], x[1][1])), fmaxf(fmaxf(x[2][0], x[2][1]), fmaxf(x[3][0], x[3][1])));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float ref = top == -INFINITY ? 0.0f : top, v_scale = scales[0].y;
        // v_scale = v_part 2^v_exp, 1/2 <= |v_part| < 1 (or what 0, the smallest numbers and NaN leave)
        const uint32_t v_bits = __float_as_uint(v_scale);
        const int v_exp = (int)((v_bits >> 23) & 255u) - 126;
        const float v_part = (uint32_t)(v_exp + 125) < 254u ? __uint_as_float((v_bits & 0x807fffffu) | 0x3f000000u) : v_scale * 0x1p126f;
        // Results are summed in units of the largest probability x value scale there was: a block whose values are loud counts
        // only as far as its probabilities do.
        float rise = (top - o_ref) + (float)(v_exp - o_exp);  // log2 of the block's unit over that of `o`
        const bool higher = top > -INFINITY && !(rise <= SLACK), louder = top > m + SLACK;  // also the first finite logit
        if (__any_sync(0xffffffffu, louder || higher)) {
            const float keep_o = higher ? ex2(-rise) : 1.0f;
#pragma unroll
            for (int i = 0; i < NW * 4; i++) o[i] = f2_mul(o[i], f2_pack(keep_o, keep_o));
            if (higher) o_ref = top, o_exp = v_exp, rise = 0.0f;
            if (louder) l *= ex2(m - top), m = top;
        }
        // what the block's sums count in the piece: of values, of probabilities
        const float vw = top == -INFINITY ? 0.0f : ex2(rise) * v_part, lw = top == -INFINITY ? 0.0f : ex2(top - m);
        // Probabilities are relative to the block's largest, so that F16 halves hold its small ones beside it.  Rows of a last
        // block that lie behind the length have probability 0, and whole numbers as values, whatever they are.
        uint32_t ph[4], pl[4];
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float p0 = ex2(x[j][0] - ref), p1 = ex2(x[j][1] - ref);
            sum += p0 + p1;
            split2(p0 * 0x1p15f, p1 * 0x1p15f, ph[j], pl[j]);
        }
        l = fmaf(sum, lw, l);
        const uint64_t w_hi = f2_pack(vw * 0x1p-15f, vw * 0x1p-15f), w_lo = f2_pack(vw * (0x1p-15f * LOW), vw * (0x1p-15f * LOW));
        uint32_t r[2][4][NW];  // [half of the block][row][word]
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int row = row_of<HD>(2 * h + (i >> 1), 2 * t + (i & 1));
                if constexpr (HD == 128) {
                    const uint4 v = lds128(vs + tile_at<HD>(row, (g >> 1) + 4 * (g & 1)));
                    r[h][i][0] = v.x ^ 0x80808080u, r[h][i][1] = v.y ^ 0x80808080u, r[h][i][2] = v.z ^ 0x80808080u, r[h][i][3] = v.w ^ 0x80808080u;
                } else {
                    const uint2 v = lds64(vs + tile_at<HD>(row, g >> 1) + ((g & 1) << 3));
                    r[h][i][0] = v.x ^ 0x80808080u, r[h][i][1] = v.y ^ 0x80808080u;
                }
            }
        // The tensor cores cut their sums off instead of rounding them, which over thousands of rows would add up to one
        // side: a block's sum is formed there and added to the running one by ordinary additions.
#pragma unroll
        for (int n = 0; n < NW; n++) {
            float y[4][4];
#pragma unroll
            for (int j = 0; j < 4; j++) y[j][0] = y[j][1] = y[j][2] = y[j][3] = 0.0f;
#pragma unroll
            for (int h = 0; h < 2; h++) {  // 16 rows a step: bytes of two rows side by side, then as pairs of F16
                const uint32_t a0 = __byte_perm(r[h][0][n], r[h][1][n], 0x5140), a1 = __byte_perm(r[h][0][n], r[h][1][n], 0x7362);
                const uint32_t c0 = __byte_perm(r[h][2][n], r[h][3][n], 0x5140), c1 = __byte_perm(r[h][2][n], r[h][3][n], 0x7362);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t sel = (j & 1) ? 0x4342 : 0x4140;
                    mma16816(y[j], ph[2 * h], pl[2 * h], ph[2 * h + 1], pl[2 * h + 1], minus_1152(__byte_perm(j < 2 ? a0 : a1, 0x64646464u, sel)),
                             minus_1152(__byte_perm(j < 2 ? c0 : c1, 0x64646464u, sel)));
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j++) o[n * 4 + j] = f2_fma(f2_pack(y[j][2], y[j][3]), w_lo, f2_fma(f2_pack(y[j][0], y[j][1]), w_hi, o[n * 4 + j]));
        }
        __syncwarp();
        if (more) fetch_values(slot);
#pragma unroll
        for (int i = 0; i < DEPTH; i++) scales[i] = scales[i + 1];
        const int64_t item = (int64_t)at.seq * per + at.kh * p.tiles + at.tile;
        slot = next;
        if (at.advance(p.lens, c, p.tiles) || todo == 1) {  // this warp's piece of the pair
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            if (live) {
                const int64_t row = (w + item) * p.rows + g;
                if (t == 0) *reinterpret_cast<float2*>(p.stats + 2 * row) = make_float2(m, l);
                // column 2 t of an n-tile stands for chunk t of a 128-byte row (column 2 t + 1 for chunk t + 4), or bytes 16 t (+ 8) of a 64-byte one
                float* to = p.acc + row * HD + 16 * t;
                // As means: a sum of the largest values would leave f32's range, and so may the unit of `o`, in two factors therefore.  As
                // half of them: 127 times the largest scale that append makes is rounded to infinity, which no share of 0 would hide.
                const float unit = (o_ref - m) + (float)o_exp, far = unit > 0.0f ? 0x1p15f : 0.5f;
                const float mean = l == 0.0f ? 0.0f : ex2(unit > 0.0f ? unit - 16.0f : unit) / l;
                const uint64_t by = f2_pack(mean, mean), by2 = f2_pack(far, far);
#pragma unroll
                for (int n = 0; n < NW; n++) {
                    uint64_t on[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) on[e] = f2_mul(f2_mul(o[n * 4 + e], by), by2);
                    *reinterpret_cast<float4*>(to + 4 * n) = make_float4(low(on[0]), low(on[1]), low(on[2]), low(on[3]));
                    *reinterpret_cast<float4*>(to + (HD == 128 ? 64 : 8) + 4 * n) = make_float4(high(on[0]), high(on[1]), high(on[2]), high(on[3]));
                }
            }
#pragma unroll
            for (int i = 0; i < NW * 4; i++) o[i] = 0;
            m = -INFINITY, l = 0.0f, o_ref = -INFINITY, o_exp = 0;
            if (todo > 1) {
                load_query();
                logits(next, scales[0].x, xn);
            }
        }
        __syncwarp();
        more = to_fetch > 0;
        if (more) scales[DEPTH] = fetch_keys(next);
#pragma unroll
        for (int j = 0; j < 4; j++) x[j][0] = xn[j][0], x[j][1] = xn[j][1];
    }
    if (!fine) {  // a copy that does not arrive: reported, and the others are waited for, each with its limit
        if (lane == 0) *p.status = GALOIS_B200_E_TIMEOUT;
        for (int i = 0; i < 2 * DEPTH; i++) wait(i);
    }
}

// Joins the pieces of one head of one sequence, in their order.  W warps share a head's pieces: one where there are many
// heads (a head then has a few pieces), eight where there are few and each has up to one from every warp.
template <int HD, int W>
__global__ void __launch_bounds__(256) cache_join_kernel(const int32_t* __restrict__ lens, int nseq, int ctx, int kv_heads, int group, int tiles, int rows,
                                                         int warps, const float* __restrict__ acc, const float* __restrict__ stats,
                                                         float* __restrict__ out, int64_t o_head, int64_t o_seq, float* __restrict__ final_stats,
                                                         int* __restrict__ status) {
    gb_pdl_entry();
    if (ctx == 0 && blockIdx.x + blockIdx.y == 0 && threadIdx.x < 32) report_lens(lens, nseq, ctx, status);
    constexpr int E = HD / 32, PER_CTA = 8 / W;
    __shared__ float part[8][HD];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wr = warp % W;
    const int heads = kv_heads * group, head = blockIdx.x * PER_CTA + warp / W, s = blockIdx.y;
    const int per = kv_heads * tiles, inner = head / group * tiles + head % group / 8, r = head % group % 8;
    const int blocks = (checked_len(lens[s], ctx) + BLK - 1) / BLK;
    const bool live = head < heads;
    float* to = out + head * o_head + s * o_seq + lane * E;
    float l = 0.0f, use = 0.0f, x[E];
#pragma unroll
    for (int e = 0; e < E; e++) x[e] = 0.0f;
    if (live && blocks > 0) {
        int64_t before = 0, total = 0;  // blocks of the sequences before s, of all
        for (int i = lane; i < nseq; i += 32) {
            const int n = (checked_len(lens[i], ctx) + BLK - 1) / BLK;
            total += n;
            if (i < s) before += n;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o), before += __shfl_xor_sync(0xffffffffu, before, o);
        const deal D(total * per, warps);
        const int64_t first = before * per + (int64_t)inner * blocks;
        const int w0 = D.owner(first), n = D.owner(first + blocks - 1) - w0 + 1;
        const int64_t row0 = (w0 + (int64_t)s * per + inner) * rows + r;
        // a lane holds what the pieces lane, lane + 32, .. say of themselves; the first 128 stay in registers
        float2 st[4];
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            st[i] = make_float2(-INFINITY, 0.0f);
            if (lane + 32 * i < n) st[i] = *reinterpret_cast<const float2*>(stats + 2 * (row0 + (int64_t)(lane + 32 * i) * rows));
        }
#pragma unroll
        for (int i = 0; i < 4; i++) m = fmaxf(m, st[i].x);
        for (int i = lane + 128; i < n; i += 32) m = fmaxf(m, stats[2 * (row0 + (int64_t)i * rows)]);
        m = gb_warp_max(m);
        use = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            st[i].y *= ex2(st[i].x - use);
            l += st[i].y;
        }
        for (int i = lane + 128; i < n; i += 32) {
            const float2 s2 = *reinterpret_cast<const float2*>(stats + 2 * (row0 + (int64_t)i * rows));
            l += s2.y * ex2(s2.x - use);
        }
        l = gb_warp_sum(l);
        const float by = l == 0.0f ? 0.0f : 1.0f / l;  // a piece's share of the result: its sum over all
        const float* a = acc + row0 * HD + lane * E;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int end = min(n, 32 * (k + 1));
#pragma unroll 8
            for (int i = 32 * k + wr; i < end; i += W) {
                const float f = __shfl_sync(0xffffffffu, st[k].y, i & 31) * by;
#pragma unroll
                for (int e = 0; e < E; e++) x[e] = fmaf(a[(int64_t)i * rows * HD + e], f, x[e]);
            }
        }
        for (int i = 128 + wr; i < n; i += W) {
            const float2 s2 = *reinterpret_cast<const float2*>(stats + 2 * (row0 + (int64_t)i * rows));
            const float f = s2.y * ex2(s2.x - use) * by;
#pragma unroll
            for (int e = 0; e < E; e++) x[e] = fmaf(a[(int64_t)i * rows * HD + e], f, x[e]);
        }
    }
    if constexpr (W > 1) {
#pragma unroll
        for (int e = 0; e < E; e++) part[warp][lane * E + e] = x[e];
        __syncthreads();
        if (wr == 0) {
#pragma unroll
            for (int i = 1; i < W; i++)
#pragma unroll
                for (int e = 0; e < E; e++) x[e] += part[warp + i][lane * E + e];
        }
    }
    if (live && wr == 0) {
#pragma unroll
        for (int e = 0; e < E; e++) {  // pieces hold half of their means; what that takes beyond f32 was stored as its largest number
            const float y = 2.0f * x[e];
            to[e] = fabsf(y) > F32_MAX ? copysignf(F32_MAX, y) : y;
        }
        if (final_stats && lane == 0) *reinterpret_cast<float2*>(final_stats + 2 * ((int64_t)s * heads + head)) = make_float2(use, l);
    }
}

__global__ void __launch_bounds__(256) cache_weights_kernel(const int32_t* __restrict__ lens, const float* __restrict__ stats, const float* __restrict__ scores,
                                                            const float* weights, int64_t w_head, int64_t w_seq, float* weights_out, int64_t wo_head,
                                                            int64_t wo_seq, int heads, int kv_heads, int nseq, int ctx, int* __restrict__ status) {
    gb_pdl_entry();
    if (heads == 0 && blockIdx.x + blockIdx.y + blockIdx.z == 0 && threadIdx.x < 32) report_lens(lens, nseq, ctx, status);
    const int j = blockIdx.x * 256 + threadIdx.x, kh = blockIdx.y, s = blockIdx.z, group = heads / kv_heads;
    if (j >= checked_len(lens[s], ctx)) return;
    float x = 0.0f;
    for (int g = 0; g < group; g++) {
        const int64_t at = (int64_t)s * heads + kh * group + g;
        const float2 ml = *reinterpret_cast<const float2*>(stats + 2 * at);
        if (ml.y != 0.0f) x += ex2(scores[at * ctx + j] - ml.x) / ml.y;
    }
    weights_out[kh * wo_head + s * wo_seq + j] = weights[kh * w_head + s * w_seq + j] + x;
}

// Floats of the workspace's parts, each a multiple of 4.
struct layout {
    size_t acc, stats, final_stats, scores, total;
    layout(const galois_b200_ctx* ctx, const gb_cache_view& c, int heads, bool weights) {
        const int group = c.kv_heads ? heads / c.kv_heads : 0, rows = group < 8 ? group : 8, tiles = (group + 7) / 8;
        const size_t pieces = (size_t)ctx->sm_count * WARPS + (size_t)c.seqs * c.kv_heads * tiles;
        acc = 0;
        stats = acc + pieces * rows * c.head_dim;
        final_stats = stats + (pieces * rows * 2 + 3) / 4 * 4;
        scores = final_stats + (weights ? ((size_t)c.seqs * heads * 2 + 3) / 4 * 4 : 0);
        total = scores + (weights ? (size_t)c.seqs * heads * c.ctx : 0) + 4;
    }
};

}  // namespace

int gb_cache_attention_init(galois_b200_ctx* ctx) {
    GB_CUDA(ctx, cudaFuncSetAttribute(cache_attention_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, ring<64>::TOTAL));
    GB_CUDA(ctx, cudaFuncSetAttribute(cache_attention_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, ring<128>::TOTAL));
    return 0;
}

extern "C" int galois_b200_cache_attention_workspace_bytes(galois_b200_ctx* ctx, const galois_b200_cache_q8* cache, int heads, int with_weights,
                                                           size_t* out_bytes) {
    GB_CHECK_CTX(ctx);
    gb_cache_view c;
    const int rc = gb_check_cache(ctx, "cache_attention_workspace_bytes", cache, &c);
    if (rc) return rc;
    if (!out_bytes) return gb_fail(ctx, GALOIS_B200_E_BADARG, "cache_attention_workspace_bytes: null pointer");
    if (heads < 0 || (heads && (c.kv_heads == 0 || heads % c.kv_heads)) || heads > 65535)
        return gb_fail(ctx, GALOIS_B200_E_BROADCAST, "cache_attention_workspace_bytes: %d heads over %d key/value heads", heads, c.kv_heads);
    *out_bytes = layout(ctx, c, heads, with_weights != 0).total * sizeof(float);
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
    if (!isfinite(scale)) return gb_fail(ctx, GALOIS_B200_E_BADARG, "%s: scale is not finite", what);
    if (c.seqs == 0 || (heads == 0 && !(weights && c.kv_heads))) return 0;
    if (!lens || (heads && (!q || !dst || !workspace))) return gb_fail(ctx, GALOIS_B200_E_BADARG, "%s: null pointer", what);
    if (qd->nb[0] != 1 || dd->nb[0] != 1 || (uintptr_t)q % 16 || (uintptr_t)dst % 16 || (heads > 1 && (qd->nb[1] % 4 || dd->nb[1] % 4)) ||
        (c.seqs > 1 && (qd->nb[2] % 4 || dd->nb[2] % 4)) || (uintptr_t)lens % 4 || (uintptr_t)workspace % 16)
        return gb_fail(ctx, GALOIS_B200_E_LAYOUT, "%s: rows of q and dst must be contiguous, they and the workspace 16-byte aligned", what);
    if (!gb_injective(dd)) return gb_fail(ctx, GALOIS_B200_E_DST, "%s: rows of dst overlap", what);
    const size_t qn = gb_span(qd, 4), dn = gb_span(dd, 4), ln = 4 * (size_t)c.seqs, need = heads ? layout(ctx, c, (int)heads, weights != nullptr).total * sizeof(float) : 0;
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
    const layout L(ctx, c, (int)heads, weights != nullptr);
    float* ws = (float*)workspace;
    float *final_stats = weights ? ws + L.final_stats : nullptr, *scores = weights ? ws + L.scores : nullptr;  // not used without heads
    const int group = (int)heads / c.kv_heads, tiles = (group + 7) / 8, rows = group < 8 ? group : 8;
    if (heads > 0 && c.ctx > 0) {  // else every length is 0
        CUtensorMap k_map, v_map;
        const uint64_t size[4] = {(uint64_t)c.head_dim, (uint64_t)c.ctx, (uint64_t)c.kv_heads, (uint64_t)c.seqs};
        // the stride of a dimension of one element means nothing, but has to be a valid one
        const uint64_t stride[3] = {c.ctx > 1 ? (uint64_t)c.tok : 128, c.kv_heads > 1 ? (uint64_t)c.head : 128, c.seqs > 1 ? (uint64_t)c.seq : 128};
        const uint32_t box[4] = {(uint32_t)c.head_dim, BLK, 1, 1};
        int r = gb_tensor_map(ctx, &k_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, c.k, size, stride, box, c.head_dim);
        if (r == 0) r = gb_tensor_map(ctx, &v_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, c.v, size, stride, box, c.head_dim);
        if (r) return r;
        int scale_exp = 0;
        const double part = frexp((double)scale * 1.4426950408889634, &scale_exp);
        const step_args a{q, qd->nb[1], qd->nb[2], c, lens, group, tiles, rows, (float)part, scale_exp, ws + L.acc, ws + L.stats, scores, ctx->dev_status};
        GB_CUDA(ctx, gb_launch(ctx, c.head_dim == 64 ? cache_attention_kernel<64> : cache_attention_kernel<128>, dim3((unsigned)ctx->sm_count),
                               dim3(WARPS * 32), c.head_dim == 64 ? ring<64>::TOTAL : ring<128>::TOTAL, a, k_map, v_map));
        GB_LAUNCHED(ctx, what);
    }
    // one sequence of 32 heads: 13.9 us with eight warps a head, 23.0 with one; 64 sequences of 32: 145.4 and 141.4
    const bool few = (int64_t)heads * c.seqs < 4 * ctx->sm_count;
    if (heads > 0) {
        auto join = c.head_dim == 64 ? (few ? cache_join_kernel<64, 8> : cache_join_kernel<64, 1>) : (few ? cache_join_kernel<128, 8> : cache_join_kernel<128, 1>);
        GB_CUDA(ctx, gb_launch(ctx, join, dim3((unsigned)(few ? heads : (heads + 7) / 8), (unsigned)c.seqs), dim3(256), 0, lens, c.seqs, c.ctx, c.kv_heads, group,
                               tiles, rows, ctx->sm_count * WARPS, ws + L.acc, ws + L.stats, dst, dd->nb[1], dd->nb[2], final_stats, ctx->dev_status));
        GB_LAUNCHED(ctx, "cache_join");
    }
    if (weights && c.ctx) {
        GB_CUDA(ctx, gb_launch(ctx, cache_weights_kernel, dim3((unsigned)((c.ctx + 255) / 256), (unsigned)c.kv_heads, (unsigned)c.seqs), dim3(256), 0, lens, final_stats,
                               scores, weights, wd->nb[1], wd->nb[2], weights_out, wod->nb[1], wod->nb[2], (int)heads, c.kv_heads, c.seqs, c.ctx, ctx->dev_status));
        GB_LAUNCHED(ctx, "cache_weights");
    }
    return 0;
}
