"""How exact attention over the 8-bit cache and prompt attention are, on inputs made so that little else than the operators'
own roundings is left: logits that f32 holds exactly, so that a tolerance can be a small multiple of sum_j p_j |v_j|."""
import numpy as np
import pytest

import galois_b200 as gb
from galois_b200 import GGmlType
from test_cache import put, upload

pytestmark = pytest.mark.gpu

F32 = GGmlType.F32
WARPS = 148 * 8  # parts that the list of blocks is dealt into


@pytest.fixture()
def G(dev):
    return gb.Device.Gpu(dev)


def step64(q, kq, ks, vq, vs, lens, scale):
    """out, and a tolerance for logits whose sums f32 holds exactly (in a unit that the test chooses).

    Counted in half steps of f32 (h = 2^-24), relative to sum_j p_j |v_j| unless said otherwise:
    * a base-2 logit x = (hi + lo 2^-12) f: the sum, the constant scale log2(e), f and the product are rounded once each, 4 h |x|; so
      is its distance to the maximum, to the block's and the piece's (3 h of it): at most 7 h R, R = max |x| + (max x - min x), twice (the sum of
      the probabilities has it too), times ln 2: 10 h R
    * exponentials: three of them (in the block, of the block, of the piece), 2^-22 = 4 h each, twice: 24 h
    * two F16 of 11 bits hold 22 bits: 2^-22 = 4 h of a query number or a probability; of a query number it is in the logits' (none here)
    * 32 rows are summed on the tensor cores, in two steps of 16 terms and the sum before, each cut off at 2 h of the largest: 68 h
    * a block is added to a piece's sums by at most 12 roundings, a piece to the result by at most 64 in all; 10 for the products with
      scales, means and shares
    A probability that lies below 2^-30 of the largest of its 32 rows has fewer bits: 2^-52 of that, times |v_j|."""
    seqs, heads, hd = q.shape
    kv = kq.shape[1]
    group = heads // kv
    tiles = (group + 7) // 8
    blocks = sum((int(n) + 31) // 32 for n in lens) * kv * tiles
    per_piece = (blocks + WARPS - 1) // WARPS
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for s in range(seqs):
        n = int(lens[s])
        if n == 0:
            continue
        by = np.arange(n) // 32
        for h in range(heads):
            c = h // group
            k = kq[s, c, :n].astype(np.float64) * ks[s, c][by].astype(np.float64)[:, None]
            v = vq[s, c, :n].astype(np.float64) * vs[s, c][by].astype(np.float64)[:, None]
            x = k @ q[s, h].astype(np.float64) * scale
            e = np.exp(x - x.max())
            p = e / e.sum()
            out[s, h] = p @ v
            span = (np.abs(x).max() + x.max() - x.min()) * np.log2(np.e)
            eps = (24 + 4 + 68 + 12 * per_piece + 64 + 10 + 10 * span) * 2.0**-24
            tol[s, h] = eps * (p @ np.abs(v))
            for b in range(0, n, 32):
                tol[s, h] += 2.0**-52 * p[b:b + 32].max() * np.abs(v[b:b + 32]).sum(0)
    return out, tol


def attend(dev, G, q, parts, lens, scale):
    cache, dst = upload(G, parts), put(G, np.full_like(q, 3))
    ws = gb.Tensor.zeros((gb.galois_cache_attention_workspace(cache, q.shape[1]) // 4,), F32, G)
    gb.galois_cache_attention(put(G, q), cache, put(G, np.array(lens, np.int32)), dst, scale, ws)
    dev.synchronize()
    return dst.to_numpy().astype(np.float64)


def close(got, out, tol):
    assert np.all(np.isfinite(got))
    worst = np.max(np.abs(got - out) / np.where(tol == 0, 1, tol))
    assert np.all(np.abs(got - out) <= tol), f"{worst:.3g} of the tolerance"


EXACT = [(128, 1, 1, [33]), (128, 4, 1, [700, 32, 5]), (64, 16, 2, [513, 64]), (128, 10, 1, [96, 200]), (64, 3, 3, [2000])]
SINKS = [(128, 32), (128, 33), (64, 700), (128, 8192)]


def exact_inputs(hd, heads, kv, lens):
    """Query numbers of 14 bits and values without a sign: both halves of the query and of the probabilities have to count."""
    rng = np.random.default_rng(hd + heads)
    ctx, seqs = max(lens), len(lens)
    # |q| < 2^14, |k| <= 7: hi (multiples of 8, 11 bits) and lo sum to less than 2^24 of their units
    q = rng.integers(-(2**14) + 1, 2**14, (seqs, heads, hd)).astype(np.float32)
    kq = rng.integers(-7, 8, (seqs, kv, ctx, hd)).astype(np.int8)
    vq = rng.integers(1, 128, (seqs, kv, ctx, hd)).astype(np.int8)
    ks = np.ones((seqs, kv, (ctx + 31) // 32), np.float32)
    vs = np.exp(rng.normal(-3, 1, ks.shape)).astype(np.float32)
    return q, (kq, ks, vq, vs), 2.0**-18  # logits of some +-6


@pytest.mark.parametrize("hd,heads,kv,lens", EXACT)
def test_exact_logits(dev, G, hd, heads, kv, lens):
    q, parts, scale = exact_inputs(hd, heads, kv, lens)
    out, tol = step64(q, *parts, lens, scale)
    close(attend(dev, G, q, parts, lens, scale), out, tol)


def sink_inputs(gap, hd, n):
    rng = np.random.default_rng(gap + n)
    q = np.zeros((1, 2, hd), np.float32)
    q[0, 0, 0], q[0, 1, 0] = gap, gap - 3
    kq = np.zeros((1, 1, n, hd), np.int8)
    vq = rng.integers(1, 128, (1, 1, n, hd)).astype(np.int8)
    at = n // 3
    kq[0, 0, at, 0], vq[0, 0, at] = 1, 0
    ks = np.ones((1, 1, (n + 31) // 32), np.float32)
    vs = np.exp(rng.normal(-3, 1, ks.shape)).astype(np.float32)
    return q, (kq, ks, vq, vs)


@pytest.mark.parametrize("gap", [8, 10, 14, 17, 20, 25])
@pytest.mark.parametrize("hd,n", SINKS)
def test_a_sink_of_values_near_zero(dev, G, gap, hd, n):
    """One row takes nearly all of the probability and has nothing to give: the result is what the others' small probabilities make."""
    q, parts = sink_inputs(gap, hd, n)
    out, tol = step64(q, *parts, [n], 1.0)
    close(attend(dev, G, q, parts, [n], 1.0), out, tol)


def test_a_loud_block_that_has_no_weight(dev, G):
    """Behind a block of values near 2^-83 lies, in the same warp's part, one of 2^120 that no probability reaches."""
    seqs, kv, hd = 150, 8, 64  # 2400 blocks over 1184 parts
    rng = np.random.default_rng(5)
    kq = np.zeros((seqs, kv, 64, hd), np.int8)
    kq[:, :, 32:, 0] = -100
    vq = rng.integers(1, 128, kq.shape).astype(np.int8)
    ks = np.ones((seqs, kv, 2), np.float32)
    vs = np.empty_like(ks)
    vs[..., 0], vs[..., 1] = 1e-25, 2e36
    q = np.zeros((seqs, kv, hd), np.float32)
    q[..., 0] = 4
    out, tol = step64(q, kq, ks, vq, vs, [64] * seqs, 1.0)
    close(attend(dev, G, q, (kq, ks, vq, vs), [64] * seqs, 1.0), out, tol)


@pytest.mark.parametrize("low,high", [(2.0**-120, 2.0**-110), (1e-3, 1.0), (2.0**100, 2.0**119), (2.0**124, 2.0**127), (-3.0, -0.5)])
def test_scales_of_any_size(dev, G, low, high):
    """Whole numbers of a few units under value scales that only a caller's own cache has, below 2^-100 and up to f32's end."""
    rng = np.random.default_rng(10)
    n, hd = 300, 64
    q = rng.integers(-100, 101, (2, 3, hd)).astype(np.float32)
    kq = rng.integers(-7, 8, (2, 1, n, hd)).astype(np.int8)
    vq = np.ones((2, 1, n, hd), np.int8)
    ks = np.ones((2, 1, 10), np.float32)
    vs = rng.uniform(low, high, ks.shape).astype(np.float32)
    out, tol = step64(q, kq, ks, vq, vs, [n, 40], 2.0**-11)
    close(attend(dev, G, q, (kq, ks, vq, vs), [n, 40], 2.0**-11), out, tol + 2.0**-140)


@pytest.mark.parametrize("what", ["loud first", "loud last", "rising"])
def test_blocks_that_rise_one_after_the_other(dev, G, what):
    """Logits and value scales that rise, or fall, from block to block of one warp's part by less, and by more, than what lets the sums be
    rescaled."""
    rng = np.random.default_rng(11)
    seqs, kv, n, hd = 30, 8, 1600, 64  # 12000 blocks over 1184 parts: ten each
    kq = np.zeros((seqs, kv, n, hd), np.int8)
    kq[..., 0] = np.repeat(rng.integers(-2, 9, (seqs, kv, n // 32)).cumsum(-1) % 100, 32, axis=-1) if what == "rising" else rng.integers(-60, 61, (seqs, kv, n))
    vq = rng.integers(1, 128, kq.shape).astype(np.int8)
    ks = np.ones((seqs, kv, n // 32), np.float32)
    order = np.argsort(rng.random(ks.shape), -1) if what == "rising" else np.broadcast_to(np.arange(n // 32), ks.shape)
    vs = (2.0 ** (order * 4.0 - 78.0) * (1 + rng.random(ks.shape))).astype(np.float32)
    if what == "loud first":
        vs = np.ascontiguousarray(vs[..., ::-1])
    q = np.zeros((seqs, kv, hd), np.float32)
    q[..., 0] = 1
    out, tol = step64(q, kq, ks, vq, vs, [n] * seqs, 1.0)
    close(attend(dev, G, q, (kq, ks, vq, vs), [n] * seqs, 1.0), out, tol)


@pytest.mark.parametrize("hd", [64, 128])
def test_a_loud_channel_of_the_query_that_no_key_has(dev, G, hd):
    rng = np.random.default_rng(6)
    n = 200
    q = (rng.integers(-(2**14) + 1, 2**14, (1, 4, hd)) / 2.0**10).astype(np.float32)
    q[:, :, 7] = 2.0**30
    kq = rng.integers(-7, 8, (1, 1, n, hd)).astype(np.int8)
    kq[..., 7] = 0
    vq = rng.integers(1, 128, (1, 1, n, hd)).astype(np.int8)
    ks, vs = np.ones((1, 1, 7), np.float32), np.full((1, 1, 7), 0.02, np.float32)
    out, tol = step64(q, kq, ks, vq, vs, [n], 2.0**-6)
    close(attend(dev, G, q, (kq, ks, vq, vs), [n], 2.0**-6), out, tol)


def test_a_factor_below_the_range_of_f32(dev, G):
    """Small queries, a small scale, large keys: only their product is an ordinary number."""
    rng = np.random.default_rng(7)
    n, hd = 100, 64
    q = (rng.integers(-(2**14) + 1, 2**14, (1, 3, hd)) * 2.0**-119).astype(np.float32)
    kq = rng.integers(-7, 8, (1, 1, n, hd)).astype(np.int8)
    vq = rng.integers(1, 128, (1, 1, n, hd)).astype(np.int8)
    ks, vs = np.full((1, 1, 4), 2.0**120, np.float32), np.full((1, 1, 4), 0.02, np.float32)
    out, tol = step64(q, kq, ks, vq, vs, [n], 2.0**-17)
    assert tol.max() < 1e-3 * out.min()
    close(attend(dev, G, q, (kq, ks, vq, vs), [n], 2.0**-17), out, tol)


def test_keys_of_zeros_under_a_factor_beyond_the_range_of_f32(dev, G):
    """A logit of 0 stays 0 beside others that f32 does not hold."""
    n, hd = 100, 64
    rng = np.random.default_rng(8)
    q = np.full((1, 2, hd), -(2.0**127), np.float32)
    kq = np.zeros((1, 1, n, hd), np.int8)
    kq[0, 0, ::2] = 5
    vq = rng.integers(1, 128, (1, 1, n, hd)).astype(np.int8)
    ks, vs = np.full((1, 1, 4), 2.0**20, np.float32), np.full((1, 1, 4), 0.02, np.float32)
    got = attend(dev, G, q, (kq, ks, vq, vs), [n], 1.0)
    want = (vq[0, 0, 1::2].astype(np.float64) * np.float64(vs[0, 0, 0])).mean(0)
    assert np.all(np.abs(got - want) <= 2.0**-16 * want)  # as step64 counts, without logits


# ------------------------------------------------------------------------------------------------ prompts


@pytest.mark.parametrize("hd,heads", [(64, 2), (128, 1)])
@pytest.mark.parametrize("gap", [8, 12, 14, 16])
@pytest.mark.parametrize("first", [0, 100, 2999])
def test_prompt_sink_of_values_near_zero(dev, G, hd, heads, gap, first):
    """As above for prompts, whose probabilities are rounded to F16: 11 bits down to 2^-21 of the row's largest, below that to
    multiples of 2^-31 of it."""
    n, nq = 3000, 3
    q = np.zeros((nq, heads, hd), np.float16)
    q[:, :, 0] = gap
    k, v = np.zeros((n, 1, hd), np.float16), np.ones((n, 1, hd), np.float16)
    k[first, 0, 0], v[first] = 1, 0
    dst = put(G, np.zeros(q.shape, np.float32))
    gb.galois_prompt_attention(put(G, q), put(G, k), put(G, v), put(G, np.array([0, nq], np.int32)), put(G, np.array([0, n], np.int32)), dst, 1.0)
    dev.synchronize()
    got = dst.to_numpy().astype(np.float64)
    for i in range(nq):
        seen = n - nq + i + 1
        x = q[i, 0, 0].astype(np.float64) * k[:seen, 0, 0].astype(np.float64)
        e = np.exp(x - x.max())
        mass = (e * v[:seen, 0, 0]).sum()
        out = mass / e.sum()
        # half a step of F16, of its smallest numbers at 2^7 of the largest; logits' constant and product 2 h |x|; sums of n terms
        # in blocks of 64, cut off at 2 h of the largest (4 steps of 17 terms, then one a block), exponentials 8 h
        tol = out * (2.0**-11 + (2 * gap * 1.45 * 2 + 136 + 2 * (n / 64) * 2 + 16) * 2.0**-24) + 2.0**-32 * (v[:seen, 0, 0] != 0).sum() / e.sum()
        assert np.all(np.abs(got[i] - out) <= tol), (i, np.max(np.abs(got[i] - out) / out))


@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_results_at_the_end_of_f16(dev, G, hd):
    """The mean of values that are all the largest F16 is that number, whichever way their probabilities were rounded."""
    n = 101
    q, k = np.full((1, 1, hd), 0, np.float16), np.zeros((n, 1, hd), np.float16)
    q[0, 0, 0] = -1
    k[1:, 0, 0] = 1
    v = np.full((n, 1, hd), 65504, np.float16)
    v[:, 0, 1::2] *= -1
    scale = -float(np.log(0.5 + 2.0**-12 + 2.0**-19))  # probabilities of the others, next to where F16 rounds up
    for kind in (np.float16, np.float32):
        dst = put(G, np.zeros((1, 1, hd), kind))
        gb.galois_prompt_attention(put(G, q), put(G, k), put(G, v), put(G, np.array([0, 1], np.int32)), put(G, np.array([0, n], np.int32)), dst, scale)
        dev.synchronize()
        got = dst.to_numpy().astype(np.float64)
        assert np.all(np.isfinite(got))
        assert np.all(np.abs(got - v[0].astype(np.float64)) <= 65504 * 2.0**-11 * 1.01)


def test_prompt_attention_is_the_same_every_time(dev, G):
    rng = np.random.default_rng(9)
    lens = [700, 3, 260, 1, 129]
    n = sum(lens)
    st = put(G, np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
    q, k, v = (put(G, rng.normal(0, 2, (n, h, 128)).astype(np.float16)) for h in (8, 2, 2))
    seen = set()
    for _ in range(8):
        dst = put(G, np.zeros((n, 8, 128), np.float32))
        gb.galois_prompt_attention(q, k, v, st, st, dst, 0.3)
        dev.synchronize()
        seen.add(dst.to_numpy().tobytes())
    assert len(seen) == 1
