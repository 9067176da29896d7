"""Prompt attention and the 8-bit cache where calls are at their edges: starts that are wrong, numbers at the end of f32, no heads, long
evictions, operands that lie over one another, and the library's own mat-mul, rope and copy in front of them."""
import numpy as np
import pytest

import cache_reference as R
import galois_b200 as gb
from galois_b200 import GError, GGmlType
from test_cache import back, f16_bound, parts_of, prompt_inputs, put, random_cache, spread, upload

pytestmark = pytest.mark.gpu

I32, F16, F32 = GGmlType.I32, GGmlType.F16, GGmlType.F32
F32_MAX = np.finfo(np.float32).max


@pytest.fixture()
def G(dev):
    return gb.Device.Gpu(dev)


def reported(dev, text="out of range"):
    with pytest.raises(GError) as e:
        dev.synchronize()
    assert e.value.code == -1 and text in str(e.value) and "wait" not in str(e.value), str(e.value)


# ------------------------------------------------------------------------------------------------ starts and positions


@pytest.mark.parametrize("what", ["append", "read", "prompt", "step", "evict"])
def test_what_is_out_of_range_is_said_to_be(dev, G, what):
    rng = np.random.default_rng(1)
    cache = upload(G, random_cache(rng, 1, 1, 64, 64))
    x, starts, pos = put(G, np.ones((5, 1, 64), np.float32)), put(G, np.array([0, 9], np.int32)), put(G, np.zeros(1, np.int32))
    if what == "append":
        gb.galois_cache_append(x, x, starts, pos, cache)
    elif what == "read":
        gb.galois_cache_read(cache, starts, pos, x, put(G, np.ones((5, 1, 64), np.float32)))
    elif what == "prompt":
        h = put(G, np.ones((5, 1, 64), np.float16))
        gb.galois_prompt_attention(h, h, h, starts, starts, x, 0.1)
    elif what == "step":
        ws = gb.Tensor.zeros((gb.galois_cache_attention_workspace(cache, 1) // 4,), F32, G)
        q = put(G, np.ones((1, 1, 64), np.float32))
        gb.galois_cache_attention(q, cache, put(G, np.array([65], np.int32)), put(G, np.ones((1, 1, 64), np.float32)), 0.1, ws)
    else:
        cut = gb.CacheQ8.zeros(64, 32, 1, 1, G)
        gb.galois_cache_evict(cache, put(G, np.array([65], np.int32)), put(G, np.ones((1, 1, 64), np.float32)), 4, cut, put(G, np.zeros(1, np.int32)),
                              put(G, np.zeros((1, 1, 32), np.float32)), put(G, np.zeros((1, 1, 32), np.int32)))
    reported(dev)
    dev.synchronize()


@pytest.mark.parametrize("starts,pos,fine", [
    ([0, 5, 9999], [3, 0], [0]),       # no token lies in the second sequence
    ([0, 5, 5, 6], [3, 0, 0], [0]),
    ([0, 2, 5, 4], [3, 7, 0], [0, 1]),  # the last one's end lies in front of its start
    ([0, 5, 5], [3, 999], [0, 1]),     # nothing is wanted of the second: its position does not matter
])
def test_sequences_without_tokens_of_their_own(dev, G, starts, pos, fine):
    rng = np.random.default_rng(2)
    seqs = len(pos)
    parts = random_cache(rng, seqs, 2, 64, 64)
    x = [rng.normal(0, 1, (5, 2, 64)).astype(np.float32) for _ in range(2)]
    cache, want = upload(G, parts), [p.copy() for p in parts]
    s, p = put(G, np.array(starts, np.int32)), put(G, np.array(pos, np.int32))
    gb.galois_cache_append(put(G, x[0]), put(G, x[1]), s, p, cache)
    bad = len(fine) < seqs
    reported(dev) if bad else dev.synchronize()
    for i in fine:
        a, b = starts[i], starts[i + 1]
        for h in range(2):
            R.append(x[h][a:b], [0, b - a], [pos[i]], want[2 * h][i:i + 1], want[2 * h + 1][i:i + 1])
    for got, w in zip(parts_of(cache, want), want):
        assert np.array_equal(got, w)
    outs = [put(G, np.full((5, 2, 64), 9, np.float32)) for _ in range(2)]
    gb.galois_cache_read(cache, s, p, *outs)
    reported(dev) if bad else dev.synchronize()
    for h, out in enumerate(outs):
        rows, expect = R.values(want[2 * h], want[2 * h + 1]).astype(np.float32), np.full((5, 2, 64), 9, np.float32)
        for i in fine:
            a, b = starts[i], starts[i + 1]
            expect[a:b] = rows[i, :, pos[i]:pos[i] + b - a].transpose(1, 0, 2)
        assert np.array_equal(out.to_numpy(), expect)


def descending(seqs, at, rng):
    """Starts of `seqs` sequences of 3 to 70 tokens; those behind sequence `at` begin again from the front."""
    lens = rng.integers(3, 71, seqs)
    starts = R.starts_of(lens)
    tokens = int(starts[-1])
    starts[at + 1:] -= starts[at + 1] - 1
    return starts.astype(np.int32), tokens


@pytest.mark.parametrize("seqs,at", [(3, 1), (40, 20), (70, 33), (70, 31), (70, 32), (70, 64)])
def test_starts_that_descend_leave_out_what_comes_behind(dev, G, seqs, at):
    """Sequences that would share tokens are not served one over the other: from the first descent on all are left out."""
    rng = np.random.default_rng(seqs + at)
    starts, tokens = descending(seqs, at, rng)
    parts = random_cache(rng, seqs, 1, 80, 64)
    x = [rng.normal(0, 1, (tokens, 1, 64)).astype(np.float32) for _ in range(2)]
    pos = rng.integers(0, 10, seqs).astype(np.int32)
    cache, want = upload(G, parts), [p.copy() for p in parts]
    s, p = put(G, starts), put(G, pos)
    gb.galois_cache_append(put(G, x[0]), put(G, x[1]), s, p, cache)
    reported(dev)
    for h in range(2):
        R.append(x[h], starts[:at + 1], pos[:at], want[2 * h][:at], want[2 * h + 1][:at])
    for got, w in zip(parts_of(cache, want), want):
        assert np.array_equal(got, w)
    outs = [put(G, np.full((tokens, 1, 64), 9, np.float32)) for _ in range(2)]
    gb.galois_cache_read(cache, s, p, *outs)
    reported(dev)
    n = int(starts[at])
    for h, out in enumerate(outs):
        rows, got = R.values(want[2 * h], want[2 * h + 1]).astype(np.float32), out.to_numpy()
        assert np.all(got[n:] == 9)
        for i in range(at):
            a, b = starts[i], starts[i + 1]
            assert np.array_equal(got[a:b], rows[i, :, pos[i]:pos[i] + b - a].transpose(1, 0, 2))
    q, k, v = (rng.normal(0, 1, (tokens, 2 if i == 0 else 1, 64)).astype(np.float16) for i in range(3))
    out, bound = R.prompt(q, k, v, starts[:at + 1], starts[:at + 1], 0.125)
    dst = put(G, np.full(q.shape, 3, np.float32))
    gb.galois_prompt_attention(put(G, q), put(G, k), put(G, v), s, s, dst, 0.125)
    reported(dev)
    got = dst.to_numpy()
    assert np.all(got[n:] == 3)
    assert np.all(np.abs(got[:n] - out[:n]) <= bound[:n])


# ------------------------------------------------------------------------------------------------ numbers at the end of f32


def test_infinities_come_back_as_the_largest_number(dev, G):
    """127 times the scale f32(largest / 127) is beyond f32; what was stored as the largest finite number is read as that."""
    x = np.zeros((40, 1, 64), np.float32)
    x[0, 0, :4] = [np.inf, -np.inf, F32_MAX, -F32_MAX]
    x[35, 0, :3] = [3e38, -3e38, 1]
    cache = gb.CacheQ8.zeros(64, 64, 1, 1, G)
    s, p = put(G, np.array([0, 40], np.int32)), put(G, np.zeros(1, np.int32))
    gb.galois_cache_append(put(G, x), put(G, -x), s, p, cache)
    outs = [put(G, np.full(x.shape, 9, np.float32)) for _ in range(2)]
    gb.galois_cache_read(cache, s, p, *outs)
    dev.synchronize()
    want = np.clip(x.astype(np.float64), -F32_MAX, F32_MAX)
    for sign, out in zip((1, -1), outs):
        got = out.to_numpy().astype(np.float64) * sign
        assert np.all(np.isfinite(got))
        assert np.array_equal(got[0], want[0]) and not got[1:32].any()
        assert np.all(np.abs(got[35] - want[35]) <= 3e38 / 127 * 0.5000001)
    half = [put(G, np.full(x.shape, 9, np.float16)) for _ in range(2)]
    gb.galois_cache_read(cache, s, p, *half)
    dev.synchronize()
    assert list(half[0].to_numpy()[0, 0, :4]) == [np.inf, -np.inf, np.inf, -np.inf]  # what F16 makes of them


@pytest.mark.parametrize("hd", [64, 128])
def test_cache_attention_over_infinite_values(dev, G, hd):
    """A row that alone counts gives the largest number; one that does not count gives nothing, not NaN."""
    rng = np.random.default_rng(3)
    ctx = 96
    x = rng.normal(0, 1, (3, ctx, hd)).astype(np.float32)
    x[0, 0, ::2], x[0, 0, 1::2] = np.inf, -np.inf
    x[1, 5], x[2, 40] = np.inf, -np.inf
    k = np.zeros((3, ctx, hd), np.float32)
    k[1, :32, 0], k[2, 32:64, 0] = -127, -127  # the whole block, as its other rows are zeros now
    cache = gb.CacheQ8.zeros(hd, ctx, 1, 3, G)
    starts = put(G, np.arange(4, dtype=np.int32) * ctx)
    gb.galois_cache_append(put(G, k.reshape(-1, 1, hd)), put(G, x.reshape(-1, 1, hd)), starts, put(G, np.zeros(3, np.int32)), cache)
    q = np.zeros((3, 2, hd), np.float32)
    q[..., 0] = 8
    dst = put(G, np.zeros_like(q))
    ws = gb.Tensor.zeros((gb.galois_cache_attention_workspace(cache, 2) // 4,), F32, G)
    gb.galois_cache_attention(put(G, q), cache, put(G, np.array([1, ctx, ctx], np.int32)), dst, 1.0, ws)
    dev.synchronize()
    got = dst.to_numpy().astype(np.float64)
    assert np.all(got[0, :, ::2] == F32_MAX) and np.all(got[0, :, 1::2] == -F32_MAX)
    for s, gone in ((1, slice(0, 32)), (2, slice(32, 64))):
        rows = np.delete(x[s].astype(np.float64), np.r_[gone], axis=0)
        step = np.abs(rows).max() / 127 / 2  # what the 8 bits are off by, at most
        assert np.all(np.abs(got[s] - rows.mean(0)) <= step * 1.001)


# ------------------------------------------------------------------------------------------------ no heads, long rows, large counts


def test_weights_of_no_heads_are_the_weights_there_were(dev, G):
    rng = np.random.default_rng(4)
    cache = upload(G, random_cache(rng, 2, 3, 50, 64))
    w, lens = rng.random((2, 3, 50)).astype(np.float32), np.array([50, 20], np.int32)
    none = gb.Tensor.zeros((64, 0, 2), F32, G)
    wo = put(G, np.full_like(w, 7))
    ws = gb.Tensor.zeros((max(1, gb.galois_cache_attention_workspace(cache, 0, True) // 4),), F32, G)
    gb.galois_cache_attention(none, cache, put(G, lens), none, 0.1, ws, weights=put(G, w), weights_out=wo)
    dev.synchronize()
    got = wo.to_numpy()
    for s, n in enumerate(lens):
        assert np.array_equal(got[s, :, :n], w[s, :, :n]) and np.all(got[s, :, n:] == 7)
    gb.galois_cache_attention(none, cache, put(G, np.array([51, 20], np.int32)), none, 0.1, ws, weights=put(G, w), weights_out=wo)
    reported(dev)


def test_lengths_in_a_cache_without_rows(dev, G):
    cache = gb.CacheQ8.zeros(64, 0, 2, 3, G)
    q, o = put(G, np.ones((3, 2, 64), np.float32)), put(G, np.full((3, 2, 64), 3, np.float32))
    ws = gb.Tensor.zeros((gb.galois_cache_attention_workspace(cache, 2) // 4,), F32, G)
    gb.galois_cache_attention(q, cache, put(G, np.array([0, 1, 0], np.int32)), o, 0.1, ws)
    reported(dev)
    assert not o.to_numpy().any()


@pytest.mark.parametrize("n,budget,recent", [(20000, 4097, 300), (8193, 8192, 1), (16384, 9000, 0), (17000, 16999, 16000)])
@pytest.mark.parametrize("kind", ["steps", "equal", "odd"])
def test_evict_of_more_rows_than_a_chunk(dev, G, n, budget, recent, kind):
    rng = np.random.default_rng(n)
    lens = np.array([n, n - 4000], np.int32)
    parts = random_cache(rng, 2, 1, n, 64)
    w = np.exp(rng.normal(0, 2, (2, 1, n))).astype(np.float32)
    if kind == "steps":
        w = (np.floor(w * 4) / 4).astype(np.float32)
    elif kind == "equal":
        w[:] = 0.25
    else:
        w -= 1
        w.reshape(-1)[rng.integers(0, w.size, w.size // 4)] = rng.choice([np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-45, -1e-45], w.size // 4)
    cut_parts = [np.full((2, 1, budget, 64), 99, np.int8), np.full((2, 1, (budget + 31) // 32), 5, np.float32)] * 2
    cut = upload(G, cut_parts)
    ol, ow, ix = put(G, np.full(2, -7, np.int32)), put(G, np.full((2, 1, budget), 6, np.float32)), put(G, np.full((2, 1, budget), -1, np.int32))
    gb.galois_cache_evict(upload(G, parts), put(G, lens), put(G, w), recent, cut, ol, ow, ix)
    dev.synchronize()
    want = R.evict(*parts, lens, w, budget, recent)
    assert np.array_equal(ix.to_numpy(), want[6]) and np.array_equal(ol.to_numpy(), want[4])
    got, got_w = parts_of(cut, cut_parts), ow.to_numpy()
    for s in range(2):
        m = want[4][s]
        assert np.array_equal(got_w[s, :, :m], want[5][s, :, :m], equal_nan=True) and np.all(got_w[s, :, m:] == 6)
        for i in (0, 2):
            assert np.array_equal(got[i][s, :, :m], want[i][s, :, :m]) and np.all(got[i][s, :, m:] == 99)


@pytest.mark.parametrize("recent,same", [(2**32, 40), (2**32 + 3, 40), (2**31, 40)])
def test_a_count_of_recent_rows_beyond_32_bits(dev, G, recent, same):
    rng = np.random.default_rng(5)
    parts = random_cache(rng, 1, 1, 100, 64)
    w, lens = rng.random((1, 1, 100)).astype(np.float32), np.array([100], np.int32)
    cut = gb.CacheQ8.zeros(64, 40, 1, 1, G)
    ol, ow, ix = put(G, np.zeros(1, np.int32)), put(G, np.zeros((1, 1, 40), np.float32)), put(G, np.zeros((1, 1, 40), np.int32))
    gb.galois_cache_evict(upload(G, parts), put(G, lens), put(G, w), recent, cut, ol, ow, ix)
    dev.synchronize()
    assert np.array_equal(ix.to_numpy(), R.evict(*parts, lens, w, 40, same)[6])
    with pytest.raises(GError):
        gb.galois_cache_evict(upload(G, parts), put(G, lens), put(G, w), -(2**32), cut, ol, ow, ix)
    with pytest.raises(GError):
        gb.galois_cache_attention_workspace(cut, 2**32 + 4)


# ------------------------------------------------------------------------------------------------ operands over one another


@pytest.mark.parametrize("heads,kv", [(4, 4), (3, 3), (4, 2)])
def test_prompt_attention_of_keys_that_all_heads_share(dev, G, heads, kv):
    """Key/value heads, and tokens of the queries, at a stride of 0: operands may lie over one another, they are only read."""
    rng = np.random.default_rng(6)
    q, k, v, qs, ks = prompt_inputs(rng, 64, heads, 1, [(150, 150), (20, 70)], 0)
    one = [put(G, x) for x in (k, v)]
    shared = [t.view((64, kv, k.shape[0]), (1, 0, 64, 64 * k.shape[0])) for t in one]
    out, bound = R.prompt(q, np.repeat(k, kv, 1), np.repeat(v, kv, 1), qs, ks, 0.125)
    dst = put(G, np.zeros(q.shape, np.float32))
    gb.galois_prompt_attention(put(G, q), *shared, put(G, qs), put(G, ks), dst, 0.125)
    dev.synchronize()
    assert np.all(np.abs(dst.to_numpy() - out) <= bound)


def test_append_of_keys_that_all_heads_share(dev, G):
    rng = np.random.default_rng(7)
    x = [rng.normal(0, 1, (50, 1, 128)).astype(np.float32) for _ in range(2)]
    shared = [put(G, a).view((128, 3, 50), (1, 0, 128, 128 * 50)) for a in x]
    parts = random_cache(rng, 1, 3, 64, 128)
    cache, want = upload(G, parts), [p.copy() for p in parts]
    gb.galois_cache_append(*shared, put(G, np.array([0, 50], np.int32)), put(G, np.array([7], np.int32)), cache)
    dev.synchronize()
    for i in range(2):
        R.append(np.repeat(x[i], 3, 1), [0, 50], [7], want[2 * i], want[2 * i + 1])
    for got, w in zip(parts_of(cache, want), want):
        assert np.array_equal(got, w)


# ------------------------------------------------------------------------------------------------ behind the library's own operators


def test_a_layer_s_attention_from_projections_to_tokens(dev, G, oracle):
    """Q4_0 projections, rope, the copy to F16, prompt attention, append; then a token: projections, rope, append, attention over the
    cache, output projection.  Each of the new operators is compared with its plain form on what the library's others gave it."""
    rng = np.random.default_rng(8)
    hd, heads, kv, lens, ctx = 64, 4, 2, [40, 25], 64
    width, n = hd * heads, sum(lens)
    scale = hd**-0.5

    def weight(rows, seed):
        w = oracle.quantize_q4_0(oracle.fill_normal(rows * width, seed, 0, 0.06).reshape(rows, width))
        return gb.Tensor.from_raw(w, (width, rows), GGmlType.Q4_0, G)

    wq, wk, wv, wo = weight(width, 1), weight(hd * kv, 2), weight(hd * kv, 3), weight(width, 4)
    rope = gb.RopeCustomOption(n_dims=hd)

    def project(w, x, count, positions):
        """{head_dim, heads, tokens} of the projection, turned if positions are given."""
        tokens, rows = x.dim().shape[1], count * hd
        y = gb.Tensor.zeros((rows, tokens), F32, G)
        gb.galois_matmul(w, x, y)
        y = y.view((hd, count, tokens), (1, hd, rows, rows * tokens))
        if positions is None:
            return y
        turned = gb.Tensor.zeros((hd, count, tokens), F32, G)
        gb.galois_rope_custom(rope, y, positions, turned)
        return turned

    def half(x):
        y = gb.Tensor.zeros(x.dim().shape[:3], F16, G)
        gb.galois_cpy(x, y)
        return y

    x = put(G, rng.normal(0, 1, (n, width)).astype(np.float32))
    at = put(G, np.concatenate([np.arange(m) for m in lens]).astype(np.int32))
    q, k, v = half(project(wq, x, heads, at)), half(project(wk, x, kv, at)), half(project(wv, x, kv, None))
    starts = R.starts_of(lens)
    st, zero = put(G, starts), put(G, np.zeros(2, np.int32))
    out = gb.Tensor.zeros((hd, heads, n), F32, G)
    cache = gb.CacheQ8.zeros(hd, ctx, kv, 2, G)
    gb.galois_prompt_attention(q, k, v, st, st, out, scale)
    gb.galois_cache_append(k, v, st, zero, cache)
    y = gb.Tensor.zeros((width, n), F32, G)
    gb.galois_matmul(wo, out.view((width, n), (1, width, width * n, width * n)), y)
    ref, bound = R.prompt(q.to_numpy(), k.to_numpy(), v.to_numpy(), starts, starts, scale)
    assert np.abs(ref).max() > 0.1
    assert np.all(np.abs(out.to_numpy() - ref) <= bound)
    want = [np.zeros((2, kv, ctx, hd), np.int8), np.zeros((2, kv, ctx // 32), np.float32)]
    want = want + [a.copy() for a in want]
    R.append(k.to_numpy(), starts, [0, 0], want[0], want[1])
    R.append(v.to_numpy(), starts, [0, 0], want[2], want[3])
    ws = gb.Tensor.zeros((gb.galois_cache_attention_workspace(cache, heads) // 4,), F32, G)
    one = put(G, np.arange(3, dtype=np.int32))
    for t in range(3):
        x1, now = put(G, rng.normal(0, 1, (2, width)).astype(np.float32)), np.array(lens, np.int32) + t
        pos = put(G, now)
        q1, k1, v1 = project(wq, x1, heads, pos), project(wk, x1, kv, pos), project(wv, x1, kv, None)
        o1, y1 = gb.Tensor.zeros((hd, heads, 2), F32, G), gb.Tensor.zeros((width, 2), F32, G)
        gb.galois_cache_append(k1, v1, one, pos, cache)
        gb.galois_cache_attention(q1, cache, put(G, now + 1), o1, scale, ws)
        gb.galois_matmul(wo, o1.view((width, 2), (1, width, 2 * width, 2 * width)), y1)
        R.append(back(k1, (2, kv, hd)), np.arange(3), now, want[0], want[1])
        R.append(back(v1, (2, kv, hd)), np.arange(3), now, want[2], want[3])
        for got, w in zip(parts_of(cache, want), want):
            assert np.array_equal(got, w)
        ref, bound, _, _ = R.step(back(q1, (2, heads, hd)), *want, now + 1, scale)
        assert np.all(np.abs(o1.to_numpy() - ref) <= bound)
        assert np.all(np.isfinite(y1.to_numpy()))


def test_two_threads_with_a_context_each(dev, G):
    """The first calls of two contexts made from two threads at once."""
    import threading

    import torch

    rng = np.random.default_rng(9)
    lens = np.array([200, 90], np.int32)
    parts = random_cache(rng, 2, 2, 200, 64)
    q, k, v, qs, _ = prompt_inputs(rng, 64, 4, 2, [(200, 200), (90, 90)], 0)
    q1 = rng.normal(0, 1, (2, 4, 64)).astype(np.float32)
    places = [gb.CudaDevice(0, torch.cuda.Stream()) for _ in range(2)]
    got, failed = [None, None], []

    def work(i):
        try:
            P = gb.Device.Gpu(places[i])
            cache, o, o1 = upload(P, parts), put(P, np.zeros(q.shape, np.float16)), put(P, np.zeros_like(q1))
            ws = gb.Tensor.zeros((gb.galois_cache_attention_workspace(cache, 4) // 4,), F32, P)
            t = [put(P, a) for a in (q, k, v, qs)]
            q1t, lt = put(P, q1), put(P, lens)
            torch.cuda.synchronize()
            for _ in range(30):
                gb.galois_prompt_attention(*t, t[3], o, 0.125)
                gb.galois_cache_attention(q1t, cache, lt, o1, 0.125, ws)
            places[i].synchronize()
            got[i] = (o.to_numpy(), o1.to_numpy())
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for p in places:
        p.close()
    assert not failed, failed
    out, bound = R.prompt(q, k, v, qs, qs, 0.125)
    step, step_bound, _, _ = R.step(q1, *parts, lens, 0.125)
    for o, o1 in got:
        assert np.all(np.abs(o - out) <= f16_bound(out, bound)) and np.all(np.abs(o1 - step) <= step_bound)


# ------------------------------------------------------------------------------------------------ strides, places, lengths, graphs


@pytest.mark.parametrize("hd,kv,ctx,budget", [(128, 2, 300, 100), (64, 3, 90, 64)])
def test_evict_between_strided_tensors(dev, G, hd, kv, ctx, budget):
    """Heads slowest, rows apart, in everything that is read and written; what lies between the rows stays."""
    rng = np.random.default_rng(10)
    lens = np.array([ctx, ctx - 7, budget - 1], np.int32)
    seqs, blocks = 3, (budget + 31) // 32
    parts = random_cache(rng, seqs, kv, ctx, hd)
    w = rng.random((seqs, kv, ctx)).astype(np.float32)
    w.reshape(-1)[::7] = 0.5

    def apart(x, pad):
        return spread(G, x, (2, 0, 1, 3) if x.ndim == 4 else (1, 0, 2), pad)

    cache = gb.CacheQ8(*(apart(p, 16 if p.ndim == 4 else 3)[0] for p in parts))
    to = [np.full((seqs, kv, budget, hd), 99, np.int8), np.full((seqs, kv, blocks), 5, np.float32)] * 2
    cut = [apart(x, 16 if x.ndim == 4 else 1) for x in to]
    ow, ix, ol = apart(np.full((seqs, kv, budget), 6, np.float32), 5), apart(np.full((seqs, kv, budget), -1, np.int32), 2), put(G, np.zeros(seqs, np.int32))
    gb.galois_cache_evict(cache, put(G, lens), apart(w, 1)[0], 9, gb.CacheQ8(*(t[0] for t in cut)), ol, ow[0], ix[0])
    dev.synchronize()
    want = R.evict(*parts, lens, w, budget, 9)
    assert np.array_equal(back(ix[0], (seqs, kv, budget)), want[6]) and np.array_equal(ol.to_numpy(), want[4])
    got, got_w = [back(t[0], x.shape) for t, x in zip(cut, to)], back(ow[0], (seqs, kv, budget))
    for s in range(seqs):
        m = want[4][s]
        assert np.array_equal(got_w[s, :, :m], want[5][s, :, :m]) and np.all(got_w[s, :, m:] == 6)
        for i in (0, 2):
            assert np.array_equal(got[i][s, :, :m], want[i][s, :, :m]) and np.all(got[i][s, :, m:] == 99)
            assert np.array_equal(got[i + 1][s, :, :(m + 31) // 32], want[i + 1][s, :, :(m + 31) // 32])
    for view, whole, before in cut + [ow, ix]:
        n = view.dim().shape[0]
        assert np.array_equal(whole.to_numpy()[..., n:], before[..., n:], equal_nan=before.dtype.kind == "f")


@pytest.mark.parametrize("heads,kv", [(4, 2), (3, 1)])
def test_prompts_that_do_not_begin_with_the_first_row(dev, G, heads, kv):
    rng = np.random.default_rng(11)
    qs, ks = np.array([70, 200, 201, 260], np.int32), np.array([3, 140, 300, 400], np.int32)
    q, k, v = (rng.normal(0, 1, (n, h, 64)).astype(np.float16) for n, h in ((300, heads), (450, kv), (450, kv)))
    q[:70], q[260:] = np.nan, np.inf
    for x in (k, v):
        x[:3], x[400:] = np.nan, np.inf
    out, bound = R.prompt(q, k, v, qs, ks, 0.125)
    dst = put(G, np.full(q.shape, 3, np.float32))
    gb.galois_prompt_attention(put(G, q), put(G, k), put(G, v), put(G, qs), put(G, ks), dst, 0.125)
    dev.synchronize()
    got = dst.to_numpy()
    assert np.all(got[:70] == 3) and np.all(got[260:] == 3)
    assert np.all(np.abs(got[70:260] - out[70:260]) <= bound[70:260])


@pytest.mark.parametrize("hd,heads,kv,nq,nk", [(64, 2, 1, 3, 70001), (128, 1, 1, 130, 20000), (64, 3, 3, 1, 40000)])
def test_prompts_behind_long_prefixes(dev, G, hd, heads, kv, nq, nk):
    rng = np.random.default_rng(12)
    q, k, v, qs, ks = prompt_inputs(rng, hd, heads, kv, [(nq, nk)], 0)
    out, bound = R.prompt(q, k, v, qs, ks, hd**-0.5)
    dst = put(G, np.full(q.shape, 3, np.float32))
    gb.galois_prompt_attention(put(G, q), put(G, k), put(G, v), put(G, qs), put(G, ks), dst, hd**-0.5)
    dev.synchronize()
    assert np.all(np.abs(dst.to_numpy() - out) <= bound)


@pytest.mark.parametrize("kind", [np.float32, np.float16])
def test_append_of_numbers_that_are_not_finite_into_blocks_that_hold_rows(dev, G, kind):
    rng = np.random.default_rng(13)
    parts = random_cache(rng, 3, 2, 96, 64)
    x = [rng.normal(0, 1, (60, 2, 64)).astype(kind) for _ in range(2)]
    x[0][3, 0, 5], x[0][4, 1, 6], x[1][40, 0, 0], x[1][59, 1, 63] = np.nan, np.inf, -np.inf, np.nan
    x[1][25:30] = np.nan
    starts, pos = np.array([0, 10, 30, 60], np.int32), np.array([20, 31, 50], np.int32)
    cache, want = upload(G, parts), [p.copy() for p in parts]
    gb.galois_cache_append(put(G, x[0]), put(G, x[1]), put(G, starts), put(G, pos), cache)
    dev.synchronize()
    for i in range(2):
        R.append(x[i], starts, pos, want[2 * i], want[2 * i + 1])
    for got, w in zip(parts_of(cache, want), want):
        assert np.array_equal(got, w)


def test_two_graphs_replayed_at_once(dev, G):
    """A graph of each of two contexts, with a workspace each, replayed on two streams."""
    import torch

    rng = np.random.default_rng(14)
    lens = np.array([600, 1000], np.int32)
    work = []
    for _ in range(2):
        stream = torch.cuda.Stream()
        own = gb.CudaDevice(0, stream)
        P = gb.Device.Gpu(own)
        parts = random_cache(rng, 2, 2, 1000, 128)
        q1, w = rng.normal(0, 1, (2, 8, 128)).astype(np.float32), rng.random((2, 2, 1000)).astype(np.float32)
        cache, t, o, wt, wo = upload(P, parts), put(P, q1), put(P, np.zeros_like(q1)), put(P, w), put(P, np.zeros_like(w))
        ws, lt = gb.Tensor.zeros((gb.galois_cache_attention_workspace(cache, 8, True) // 4,), F32, P), put(P, lens)
        torch.cuda.synchronize()
        gb.galois_cache_attention(t, cache, lt, o, 0.09, ws, weights=wt, weights_out=wo)
        own.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            gb.galois_cache_attention(t, cache, lt, o, 0.09, ws, weights=wt, weights_out=wo)
        work.append((own, stream, graph, o, wo, R.step(q1, *parts, lens, 0.09, w), (cache, t, lt, wt, ws)))  # what a graph reads lives as long
    try:
        for _ in range(20):
            for _, stream, graph, *_ in work:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for own, _, _, o, wo, (out, bound, ww, wb), _ in work:
            own.synchronize()
            assert np.all(np.abs(o.to_numpy() - out) <= bound)
            got = wo.to_numpy()
            for s, n in enumerate(lens):
                assert np.all(np.abs(got[s, :, :n] - ww[s, :, :n]) <= wb[s, :, :n]) and not got[s, :, n:].any()
    finally:
        torch.cuda.synchronize()
        for w_ in work:
            w_[2].reset()
            w_[0].close()
