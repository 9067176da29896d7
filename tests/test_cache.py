"""Prompt attention and the 8-bit key/value cache against plain forms in 64 bits, on the GPU."""
import itertools

import numpy as np
import pytest

import cache_reference as R
import galois_b200 as gb
from galois_b200 import GError, GGmlType

pytestmark = pytest.mark.gpu

I8, I32, F16, F32 = GGmlType.I8, GGmlType.I32, GGmlType.F16, GGmlType.F32
KIND = {np.dtype(np.int8): I8, np.dtype(np.int32): I32, np.dtype(np.float16): F16, np.dtype(np.float32): F32}


@pytest.fixture()
def G(dev):
    return gb.Device.Gpu(dev)


def put(G, x):
    return gb.Tensor.from_numpy(x, KIND[x.dtype], G)


def spread(G, x, order=None, pad=0):
    """x as a view with other strides: `order` of the dimensions from slowest to fastest (the last stays), `pad`
    numbers behind every row.  What lies between the rows is 77 (or NaN)."""
    order = order or range(x.ndim)
    y = np.ascontiguousarray(x.transpose(order))
    full = np.full(y.shape[:-1] + (y.shape[-1] + pad,), np.nan if y.dtype.kind == "f" else 77, y.dtype)
    full[..., :y.shape[-1]] = y
    t = put(G, full)
    strides = [int(np.prod(full.shape[i + 1:])) for i in range(full.ndim)]
    by_dim = [0] * x.ndim
    for place, d in enumerate(order):
        by_dim[d] = strides[place]
    nb = by_dim[::-1] + [full.size] * (4 - x.ndim)
    return t.view(x.shape[::-1], nb), t, full


def back(view, shape):
    """The numpy values of a (possibly strided) tensor."""
    flat = view.to_cpu_tensor().storage
    d = view.dim()
    strides = [d.stride[i] * flat.itemsize for i in range(len(shape))][::-1]
    return np.lib.stride_tricks.as_strided(np.asarray(flat)[view.offset:], shape, strides).copy()


def random_cache(rng, seqs, kv, ctx, hd):
    blocks = (ctx + 31) // 32
    q = [rng.integers(-127, 128, (seqs, kv, ctx, hd)).astype(np.int8) for _ in range(2)]
    sc = [np.exp(rng.normal(-3.5, 0.5, (seqs, kv, blocks))).astype(np.float32) for _ in range(2)]
    return q[0], sc[0], q[1], sc[1]


def upload(G, parts):
    return gb.CacheQ8(*(put(G, x) for x in parts))


def parts_of(cache, like):
    return [back(t, x.shape) for t, x in zip((cache.k, cache.k_scale, cache.v, cache.v_scale), like)]


# ------------------------------------------------------------------------------------------------ append and read

APPENDS = [  # head_dim, kv heads, ctx, (new tokens, position) of each sequence
    (128, 1, 1, [(1, 0)]),
    (128, 2, 100, [(1, 0), (1, 31), (1, 32), (1, 99)]),
    (64, 3, 97, [(97, 0), (0, 5), (33, 31), (1, 96), (64, 32), (2, 63)]),
    (128, 8, 300, [(300, 0), (31, 1), (268, 32), (0, 0)]),
    (64, 1, 5000, [(4999, 1), (1, 4000)]),
    (128, 2, 64, [(1, i) for i in range(40)]),
]


@pytest.mark.parametrize("hd,kv,ctx,seqs", APPENDS)
@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("strided", [False, True])
def test_append_and_read(dev, G, hd, kv, ctx, seqs, kind, strided):
    rng = np.random.default_rng(hd + kv + ctx + len(seqs))
    lens, pos = [a for a, _ in seqs], np.array([p for _, p in seqs], np.int32)
    n = sum(lens)
    x = [(rng.normal(0, 1, (n + 3, kv, hd)) * np.exp(rng.normal(0, 1, (n + 3, 1, 1)))).astype(kind) for _ in range(2)]
    parts = random_cache(rng, len(seqs), kv, ctx, hd)
    starts = R.starts_of(lens)
    if strided:  # heads slowest in the new rows; tokens slowest in the cache; rows apart
        new = [spread(G, a, (1, 0, 2), 8)[0] for a in x]
        views = [spread(G, parts[0], (2, 0, 1, 3), 16)[0], spread(G, parts[1], (1, 0, 2), 3)[0], spread(G, parts[2], (2, 0, 1, 3), 16)[0], spread(G, parts[3], (1, 0, 2), 3)[0]]
        cache = gb.CacheQ8(*views)
    else:
        new, cache = [put(G, a) for a in x], upload(G, parts)
    gb.galois_cache_append(new[0], new[1], put(G, starts), put(G, pos), cache)
    want = [p.copy() for p in parts]
    for i in range(2):
        R.append(x[i], starts, pos, want[2 * i], want[2 * i + 1])
    for got, w in zip(parts_of(cache, want), want):
        assert np.array_equal(got, w)  # rows and scales that were not written among them
    # the written rows and a few before them, into destinations whose other rows stay
    first = np.maximum(pos - 3, 0).astype(np.int32)
    rows = np.array([p + a - f for a, p, f in zip(lens, pos, first)])
    to = np.full((rows.sum() + 2, kv, hd), 5, kind)
    outs = [spread(G, to, (1, 0, 2), 8) if strided else (put(G, to), None, None) for _ in range(2)]
    gb.galois_cache_read(cache, put(G, R.starts_of(rows)), put(G, first), outs[0][0], outs[1][0])
    dev.synchronize()
    for (t, _, _), q, sc in zip(outs, want[::2], want[1::2]):
        v = R.values(q, sc).astype(np.float32)  # the product of two f32, rounded once
        expect = to.copy()
        expect[:rows.sum()] = np.concatenate([v[s, :, f:f + r].transpose(1, 0, 2) for s, (f, r) in enumerate(zip(first, rows))]).astype(kind)
        assert np.array_equal(back(t, to.shape), expect)


def test_append_token_by_token_grows_the_scale(dev, G):
    """A block filled one token at a time, each louder than the one before: every step rescales what it holds."""
    rng = np.random.default_rng(5)
    parts = random_cache(rng, 2, 2, 70, 64)
    cache, want = upload(G, parts), [p.copy() for p in parts]
    for t in range(70):
        x = [(rng.normal(0, 1, (2, 2, 64)) * 1.07**t).astype(np.float32) for _ in range(2)]
        pos = np.array([t, max(0, t - 3)], np.int32)
        gb.galois_cache_append(put(G, x[0]), put(G, x[1]), put(G, R.starts_of([1, 1])), put(G, pos), cache)
        for i in range(2):
            R.append(x[i], R.starts_of([1, 1]), pos, want[2 * i], want[2 * i + 1])
    dev.synchronize()
    for got, w in zip(parts_of(cache, want), want):
        assert np.array_equal(got, w)


def test_append_borders_and_odd_numbers(dev, G):
    """Quotients on and next to k + 1/2, NaN, infinities, the smallest and the largest numbers, rows of zeros."""
    d = np.float32(0.37)
    k = np.arange(-127, 128, dtype=np.float64)
    ties = np.concatenate([(k + 0.5) * np.float64(d), k * np.float64(d)]).astype(np.float32)
    near = np.concatenate([np.nextafter(ties, np.float32(9e9)), np.nextafter(ties, np.float32(-9e9))])
    row = np.concatenate([ties, near]).astype(np.float32)
    row = row[np.abs(row) <= 127 * d]
    x = np.zeros((8 * 32, 1, 128), np.float32)
    x[:32].reshape(-1)[:row.size] = row
    x[0, 0, 0] = 127 * d
    half = np.arange(-127, 128, dtype=np.float32)  # a scale of exactly 1: exact ties
    x[32:64].reshape(-1)[:255], x[32:64].reshape(-1)[255:509], x[32, 0, 100] = half, half[:-1] + 0.5, 127
    x[64:96] = np.nan
    x[96, 0, :4] = [np.inf, -np.inf, 1e38, -1e30]
    x[128:160] = 1e-38
    x[160, 0, :3] = [2.0**-93, 2.0**-94, -(2.0**-95)]
    x[192] = 3e38
    x[224, 0, 5], x[225, 0, 6] = np.nan, 2.0
    zero = [np.zeros((1, 1, 256, 128), np.int8), np.zeros((1, 1, 8), np.float32)]
    cache = upload(G, zero + zero)
    s, p = put(G, np.array([0, 256], np.int32)), put(G, np.array([0], np.int32))
    gb.galois_cache_append(put(G, x), put(G, -x), s, p, cache)
    want = [z.copy() for z in zero + zero]
    R.append(x, [0, 256], [0], want[0], want[1])
    R.append(-x, [0, 256], [0], want[2], want[3])
    dev.synchronize()
    for got, w in zip(parts_of(cache, want), want):
        assert np.array_equal(got, w)


@pytest.mark.parametrize("starts,pos,fine", [
    ([0, 2, 5], [0, 61], [0]), ([0, 2, 5], [-1, 3], [1]), ([0, 2, 99], [0, 3], [0]), ([-3, 2, 5], [0, 3], [1]), ([0, 2, 5], [2**31 - 1, 4], [1]),
    ([0, 2, 5], [64, 64], []),
])
def test_append_and_read_out_of_range(dev, G, starts, pos, fine):
    """Sequences whose starts or positions are out of range are left out and reported; the others are served."""
    rng = np.random.default_rng(9)
    parts = random_cache(rng, 2, 1, 63, 128)
    x = [rng.normal(0, 1, (5, 1, 128)).astype(np.float32) for _ in range(2)]
    cache, want = upload(G, parts), [p.copy() for p in parts]
    s, p = put(G, np.array(starts, np.int32)), put(G, np.array(pos, np.int32))
    gb.galois_cache_append(put(G, x[0]), put(G, x[1]), s, p, cache)
    with pytest.raises(GError) as e:
        dev.synchronize()
    assert e.value.code == -1
    for i in fine:
        one = np.array([starts[i], starts[i + 1]])
        for h in range(2):
            R.append(x[h][one[0]:one[1]], one - one[0], [pos[i]], want[2 * h][i:i + 1], want[2 * h + 1][i:i + 1])
    for got, w in zip(parts_of(cache, want), want):
        assert np.array_equal(got, w)
    outs = [put(G, np.full((5, 1, 128), 9, np.float32)) for _ in range(2)]
    gb.galois_cache_read(cache, s, p, outs[0], outs[1])
    with pytest.raises(GError):
        dev.synchronize()
    dev.synchronize()  # reported once


# ------------------------------------------------------------------------------------------------ attention over the cache

STEPS = [  # head_dim, heads, kv heads, ctx, lengths
    (128, 1, 1, 1, [1]),
    (128, 4, 4, 40, [0, 1, 2, 31, 32, 33, 40]),
    (64, 6, 2, 130, [130, 129, 127, 64, 65, 96]),
    (128, 8, 1, 1000, [1000, 17]),
    (64, 12, 1, 333, [333, 0, 5]),
    (128, 32, 2, 777, [777, 500]),
    (128, 7, 1, 5000, [4999]),
    (64, 5, 5, 2049, [2049, 2048, 1]),
    (128, 20, 4, 600, list(range(0, 600, 19))),
]


@pytest.mark.parametrize("hd,heads,kv,ctx,lens", STEPS)
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("strided", [False, True])
def test_cache_attention(dev, G, hd, heads, kv, ctx, lens, weighted, strided):
    rng = np.random.default_rng(hd * heads + ctx)
    seqs = len(lens)
    parts = random_cache(rng, seqs, kv, ctx, hd)
    q = rng.normal(0, 1, (seqs, heads, hd)).astype(np.float32)
    lens = np.array(lens, np.int32)
    w = rng.random((seqs, kv, ctx)).astype(np.float32)
    # what lies behind a length is not used: whole blocks behind it have no scale, its last rows hold other numbers
    for s, n in enumerate(lens):
        for p in parts[1::2]:
            p[s, :, (n + 31) // 32:] = np.nan
        w[s, :, n:] = np.nan
    out, bound, ww, wb = R.step(q, *parts, lens, hd**-0.5, w if weighted else None)
    order3, order4 = ((1, 0, 2), (2, 0, 1, 3)) if strided else (None, None)
    if strided:
        cache = gb.CacheQ8(*(spread(G, p, order4 if p.ndim == 4 else order3, 16)[0] for p in parts))
        qt, dst, wt = spread(G, q, order3, 4)[0], spread(G, np.full_like(q, 3), order3, 4)[0], spread(G, w, order3, 1)[0]
    else:
        cache, qt, dst, wt = upload(G, parts), put(G, q), put(G, np.full_like(q, 3)), put(G, w)
    ws = gb.Tensor.zeros((max(1, gb.galois_cache_attention_workspace(cache, heads, weighted) // 4),), F32, G)
    ws.storage.fill_(float("nan"))
    wo = put(G, np.full_like(w, 7)) if not strided else wt  # in place
    extra = dict(weights=wt, weights_out=wo) if weighted else {}
    gb.galois_cache_attention(qt, cache, put(G, lens), dst, hd**-0.5, ws, **extra)
    dev.synchronize()
    got = back(dst, q.shape).astype(np.float64)
    assert np.all(np.abs(got - out) <= bound), np.max(np.abs(got - out) - bound)
    if weighted:
        got_w = back(wo, w.shape)
        for s, n in enumerate(lens):
            assert np.all(np.abs(got_w[s, :, :n] - ww[s, :, :n]) <= wb[s, :, :n])
            assert np.all(got_w[s, :, n:] == 7) if not strided else np.all(np.isnan(got_w[s, :, n:]))


@pytest.mark.parametrize("what", ["loud query", "far scales", "equal", "zero scale"])
def test_cache_attention_values(dev, G, what):
    """A query far outside F16's range, value scales of 30 orders of magnitude, equal logits, blocks of zeros."""
    rng = np.random.default_rng(3)
    parts = random_cache(rng, 2, 2, 700, 128)
    q = rng.normal(0, 1, (2, 6, 128)).astype(np.float32)
    scale, lens = 128**-0.5, np.array([700, 345], np.int32)
    if what == "loud query":
        q, scale = (q * 3e20).astype(np.float32), 128**-0.5 * 1e-20
    elif what == "far scales":
        parts[3][:] = (10.0 ** rng.uniform(-30, 0, parts[3].shape)).astype(np.float32)
    elif what == "equal":
        q[:] = 0
    else:
        for p in parts[1::2]:
            p[:, :, ::3] = 0
        parts[3][1] = 0
    out, bound, _, _ = R.step(q, *parts, lens, scale)
    cache, dst = upload(G, parts), put(G, np.zeros_like(q))
    ws = gb.Tensor.zeros((gb.galois_cache_attention_workspace(cache, 6) // 4,), F32, G)
    gb.galois_cache_attention(put(G, q), cache, put(G, lens), dst, scale, ws)
    dev.synchronize()
    got = dst.to_numpy().astype(np.float64)
    assert np.all(np.abs(got - out) <= bound), np.max(np.abs(got - out) - bound)


def test_cache_attention_lengths_out_of_range(dev, G):
    rng = np.random.default_rng(4)
    parts = random_cache(rng, 3, 1, 50, 64)
    q = rng.normal(0, 1, (3, 2, 64)).astype(np.float32)
    cache, dst = upload(G, parts), put(G, np.full_like(q, 3))
    ws = gb.Tensor.zeros((gb.galois_cache_attention_workspace(cache, 2) // 4,), F32, G)
    gb.galois_cache_attention(put(G, q), cache, put(G, np.array([-1, 51, 50], np.int32)), dst, 0.1, ws)
    with pytest.raises(GError) as e:
        dev.synchronize()
    assert e.value.code == -1
    out, bound, _, _ = R.step(q, *parts, [0, 0, 50], 0.1)
    assert np.all(np.abs(dst.to_numpy() - out) <= bound)


def test_cache_attention_is_the_same_every_time(dev, G):
    rng = np.random.default_rng(6)
    lens = np.array([900, 3, 0, 512], np.int32)
    parts = random_cache(rng, 4, 2, 900, 128)
    q, w = rng.normal(0, 1, (4, 8, 128)).astype(np.float32), rng.random((4, 2, 900)).astype(np.float32)
    cache, qt, lt, wt = upload(G, parts), put(G, q), put(G, lens), put(G, w)
    ws = gb.Tensor.zeros((gb.galois_cache_attention_workspace(cache, 8, True) // 4,), F32, G)
    seen = set()
    for _ in range(5):
        dst, wo = put(G, np.zeros_like(q)), put(G, np.zeros_like(w))
        gb.galois_cache_attention(qt, cache, lt, dst, 0.09, ws, weights=wt, weights_out=wo)
        dev.synchronize()
        seen.add(dst.to_numpy().tobytes() + wo.to_numpy().tobytes())
    assert len(seen) == 1


# ------------------------------------------------------------------------------------------------ eviction

EVICTS = [  # head_dim, kv heads, ctx, budget, recent, lengths
    (128, 2, 200, 64, 10, [200, 65, 64, 63, 1, 0]),
    (64, 1, 5000, 777, 100, [5000, 1234]),
    (128, 3, 100, 33, 0, [100, 34]),
    (128, 1, 100, 33, 500, [100, 20]),
    (64, 2, 40, 64, 4, [40, 39]),
    (128, 1, 3000, 1, 0, [3000]),
    (64, 4, 1025, 1024, 1, [1025, 1024]),
]


@pytest.mark.parametrize("hd,kv,ctx,budget,recent,lens", EVICTS)
@pytest.mark.parametrize("kind", ["steps", "equal", "odd"])
def test_evict(dev, G, hd, kv, ctx, budget, recent, lens, kind):
    rng = np.random.default_rng(ctx + budget)
    seqs, lens = len(lens), np.array(lens, np.int32)
    parts = random_cache(rng, seqs, kv, ctx, hd)
    w = np.exp(rng.normal(0, 2, (seqs, kv, ctx))).astype(np.float32)
    if kind == "steps":
        w = (np.floor(w * 16) / 16).astype(np.float32)
    elif kind == "equal":
        w[:] = 0.25
    else:
        w -= 1
        w.reshape(-1)[rng.integers(0, w.size, w.size // 4)] = rng.choice([np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-45, -1e-45], w.size // 4)
    cache = upload(G, parts)
    blocks = (budget + 31) // 32
    cut_parts = [np.full((seqs, kv, budget, hd), 99, np.int8), np.full((seqs, kv, blocks), 5, np.float32)] * 2
    cut = upload(G, cut_parts)
    ol, ow, ix = put(G, np.full(seqs, -7, np.int32)), put(G, np.full((seqs, kv, budget), 6, np.float32)), put(G, np.full((seqs, kv, budget), -1, np.int32))
    gb.galois_cache_evict(cache, put(G, lens), put(G, w), recent, cut, ol, ow, ix)
    dev.synchronize()
    want = R.evict(*parts, lens, w, budget, recent)
    assert np.array_equal(ix.to_numpy(), want[6])
    assert np.array_equal(ol.to_numpy(), want[4])
    got = parts_of(cut, cut_parts)
    got_w = ow.to_numpy()
    for s in range(seqs):
        m = want[4][s]
        assert np.array_equal(got_w[s, :, :m], want[5][s, :, :m], equal_nan=True) and np.all(got_w[s, :, m:] == 6)
        for i in (0, 2):
            assert np.array_equal(got[i][s, :, :m], want[i][s, :, :m]) and np.all(got[i][s, :, m:] == 99)
            b = (m + 31) // 32
            assert np.array_equal(got[i + 1][s, :, :b], want[i + 1][s, :, :b]) and np.all(got[i + 1][s, :, b:] == 5)
    for a, b in zip(parts_of(cache, parts), parts):
        assert np.array_equal(a, b)


def test_evict_lengths_out_of_range(dev, G):
    rng = np.random.default_rng(8)
    parts = random_cache(rng, 3, 1, 64, 64)
    cut = gb.CacheQ8.zeros(64, 32, 1, 3, G)
    ol, ow, ix = put(G, np.full(3, 9, np.int32)), put(G, np.zeros((3, 1, 32), np.float32)), put(G, np.full((3, 1, 32), -1, np.int32))
    w = rng.random((3, 1, 64)).astype(np.float32)
    gb.galois_cache_evict(upload(G, parts), put(G, np.array([65, 64, -1], np.int32)), put(G, w), 4, cut, ol, ow, ix)
    with pytest.raises(GError):
        dev.synchronize()
    assert list(ol.to_numpy()) == [0, 32, 0]
    want = R.evict(*parts, np.array([0, 64, 0]), w, 32, 4)
    assert np.array_equal(ix.to_numpy(), want[6])


# ------------------------------------------------------------------------------------------------ prompts

PROMPTS = [  # head_dim, heads, kv heads, (queries, keys) of each sequence
    (128, 1, 1, [(1, 1)]),
    (64, 2, 1, [(5, 5), (1, 1), (3, 9)]),
    (128, 4, 4, [(127, 127), (128, 128), (129, 129), (1, 130)]),
    (64, 6, 2, [(64, 64), (65, 100), (257, 257)]),
    (128, 8, 2, [(300, 300), (2, 513), (0, 7), (130, 258)]),
    (128, 5, 1, [(255, 255), (256, 512)]),
    (64, 7, 7, [(400, 401)]),
    (128, 2, 2, [(9, 4), (3, 0), (140, 130), (2, 2)]),
    (128, 3, 1, [(513, 513)]),
]


def prompt_inputs(rng, hd, heads, kv, seqs, extra=3):
    nq, nk = [a for a, _ in seqs], [b for _, b in seqs]
    q = rng.normal(0, 1, (sum(nq) + extra, heads, hd)).astype(np.float16)
    k = rng.normal(0, 1, (sum(nk) + extra, kv, hd)).astype(np.float16)
    v = rng.normal(0, 1, (sum(nk) + extra, kv, hd)).astype(np.float16)
    return q, k, v, R.starts_of(nq), R.starts_of(nk)


def f16_bound(out, bound):
    """An f32 result rounded to F16: half a step of the value (2^-11), or of the smallest numbers."""
    return bound + 2.0**-11 * (np.abs(out) + bound) + 2.0**-25


@pytest.mark.parametrize("hd,heads,kv,seqs", PROMPTS)
@pytest.mark.parametrize("kind", [np.float16, np.float32])
@pytest.mark.parametrize("strided", [False, True])
def test_prompt_attention(dev, G, hd, heads, kv, seqs, kind, strided):
    rng = np.random.default_rng(hd + heads + len(seqs))
    q, k, v, qs, ks = prompt_inputs(rng, hd, heads, kv, seqs)
    for x, n in ((q, qs[-1]), (k, ks[-1]), (v, ks[-1])):
        x[n:] = np.nan  # rows behind the last sequence
    out, bound = R.prompt(q, k, v, qs, ks, hd**-0.5)
    if kind == np.float16:
        bound = f16_bound(out, bound)
    ops = [spread(G, x, (1, 0, 2), 8)[0] if strided else put(G, x) for x in (q, k, v)]
    to = np.full(q.shape, 3, kind)
    dst = spread(G, to, (1, 0, 2), 8)[0] if strided else put(G, to)
    gb.galois_prompt_attention(*ops, put(G, qs), put(G, ks), dst, hd**-0.5)
    dev.synchronize()
    got = back(dst, q.shape).astype(np.float64)
    assert np.all(got[qs[-1]:] == 3)
    n = qs[-1]
    assert np.all(np.abs(got[:n] - out[:n]) <= bound[:n]), np.max(np.abs(got[:n] - out[:n]) - bound[:n])
    for s, (a, b) in enumerate(seqs):  # queries that see no key
        assert np.all(got[qs[s]:qs[s] + max(0, a - b)] == 0)


@pytest.mark.parametrize("where", ["k", "v", "both"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_attention_masked_places_do_not_matter(dev, G, where, bad, hd):
    """A key or value that is not finite reaches the queries that see it and no other, wherever it lies."""
    rng = np.random.default_rng(11)
    seqs = [(300, 300), (140, 200), (7, 7)]
    q, k, v, qs, ks = prompt_inputs(rng, hd, 4, 2, seqs)
    clean, bound = R.prompt(q, k, v, qs, ks, 0.1)
    places = [(0, 130), (0, 299), (1, 199), (2, 3)]
    for s, j in places:
        for x in (k,) if where == "k" else (v,) if where == "v" else (k, v):
            x[ks[s] + j, 1, 5] = bad
    dst = put(G, np.zeros(q.shape, np.float32))
    gb.galois_prompt_attention(put(G, q), put(G, k), put(G, v), put(G, qs), put(G, ks), dst, 0.1)
    dev.synchronize()
    got = dst.to_numpy().astype(np.float64)
    for s, (a, b) in enumerate(seqs):
        first = min(j for t, j in places if t == s) - (b - a)  # the first query that sees a bad place
        part = slice(qs[s], qs[s] + first)
        assert np.all(np.abs(got[part] - clean[part]) <= bound[part])
        rows = slice(qs[s] + first, qs[s + 1])
        assert np.all(np.abs(got[rows, :2] - clean[rows, :2]) <= bound[rows, :2])  # heads of the other key/value head
        if where == "v":
            hit = got[rows, 2:, 5]
            assert np.all(np.isnan(hit) if np.isnan(bad) else ~np.isfinite(hit))
            others = np.delete(np.arange(hd), 5)
            assert np.all(np.abs(got[rows, 2:][..., others] - clean[rows, 2:][..., others]) <= bound[rows, 2:][..., others])


@pytest.mark.parametrize("what", ["large", "rising", "equal"])
def test_prompt_attention_values(dev, G, what):
    """Logits of hundreds, a maximum that grows from key to key, all logits equal."""
    rng = np.random.default_rng(12)
    q, k, v, qs, ks = prompt_inputs(rng, 128, 2, 2, [(600, 600)], 0)
    scale = 128**-0.5
    if what == "large":
        q = (q * 20).astype(np.float16)
    elif what == "rising":
        q[:], k[:] = 1, np.linspace(-4, 4, 600)[:, None, None].astype(np.float16)
        scale = 0.5
    else:
        k[:] = 0
    out, bound = R.prompt(q, k, v, qs, ks, scale)
    dst = put(G, np.zeros(q.shape, np.float32))
    gb.galois_prompt_attention(put(G, q), put(G, k), put(G, v), put(G, qs), put(G, ks), dst, scale)
    dev.synchronize()
    assert np.all(np.abs(dst.to_numpy() - out) <= bound), np.max(np.abs(dst.to_numpy() - out) - bound)


@pytest.mark.parametrize("qs,ks", [([0, 5, 9], [0, 5, 11]), ([0, 5, 4], [0, 5, 9]), ([-1, 5, 9], [0, 5, 9]), ([0, 5, 9], [0, 12, 9])])
def test_prompt_attention_starts_out_of_range(dev, G, qs, ks):
    rng = np.random.default_rng(13)
    x = [rng.normal(0, 1, (9, 1, 64)).astype(np.float16) for _ in range(3)]
    dst = put(G, np.full((9, 1, 64), 3, np.float32))
    gb.galois_prompt_attention(*(put(G, a) for a in x), put(G, np.array(qs, np.int32)), put(G, np.array(ks, np.int32)), dst, 0.1)
    with pytest.raises(GError) as e:
        dev.synchronize()
    assert e.value.code == -1
    dev.synchronize()


# ------------------------------------------------------------------------------------------------ together


def test_a_conversation(dev, G):
    """Prompts of different lengths, their cache, generated tokens with weights, an eviction, more tokens, and a prompt that
    continues the cached ones: every result against the plain forms fed the operators' own inputs."""
    rng = np.random.default_rng(21)
    hd, heads, kv, ctx, budget = 64, 4, 2, 200, 96
    lens = [150, 33, 90]
    scale = hd**-0.5
    q, k, v, qs, _ = prompt_inputs(rng, hd, heads, kv, [(n, n) for n in lens], 0)
    starts = put(G, qs)
    qt, kt, vt = put(G, q), put(G, k), put(G, v)
    dst = put(G, np.zeros(q.shape, np.float16))
    cache = gb.CacheQ8.zeros(hd, ctx, kv, 3, G)
    like = [np.zeros((3, kv, ctx, hd), np.int8), np.zeros((3, kv, 7), np.float32)] * 2
    want = [x.copy() for x in like]
    gb.galois_prompt_attention(qt, kt, vt, starts, starts, dst, scale)
    gb.galois_cache_append(kt, vt, starts, put(G, np.zeros(3, np.int32)), cache)
    out, bound = R.prompt(q, k, v, qs, qs, scale)
    assert np.all(np.abs(dst.to_numpy() - out) <= f16_bound(out, bound))
    R.append(k, qs, [0, 0, 0], want[0], want[1])
    R.append(v, qs, [0, 0, 0], want[2], want[3])
    ws = gb.Tensor.zeros((gb.galois_cache_attention_workspace(cache, heads, True) // 4,), F32, G)
    one = put(G, np.arange(4, dtype=np.int32))
    w = put(G, np.zeros((3, kv, ctx), np.float32))

    def tokens(cache, want, lens, w, steps):
        for _ in range(steps):
            k1, v1 = (rng.normal(0, 1, (3, kv, hd)).astype(np.float32) for _ in range(2))
            q1 = rng.normal(0, 1, (3, heads, hd)).astype(np.float32)
            at = np.array(lens, np.int32)
            o = put(G, np.zeros_like(q1))
            gb.galois_cache_append(put(G, k1), put(G, v1), one, put(G, at), cache)
            before = w.to_numpy()
            gb.galois_cache_attention(put(G, q1), cache, put(G, at + 1), o, scale, ws, weights=w, weights_out=w)
            R.append(k1, np.arange(4), at, want[0], want[1])
            R.append(v1, np.arange(4), at, want[2], want[3])
            ref, b, ww, wb = R.step(q1, *want, at + 1, scale, before)
            assert np.all(np.abs(o.to_numpy() - ref) <= b)
            assert np.all(np.abs(w.to_numpy() - ww) <= wb + 1e-30)
            lens = [n + 1 for n in lens]
        for got, x in zip(parts_of(cache, want), want):
            assert np.array_equal(got, x)
        return lens

    lens = tokens(cache, want, lens, w, 3)
    cut = gb.CacheQ8.zeros(hd, budget, kv, 3, G)
    ol, ow, ix = gb.Tensor.zeros((3,), I32, G), gb.Tensor.zeros((budget, kv, 3), F32, G), gb.Tensor.zeros((budget, kv, 3), I32, G)
    gb.galois_cache_evict(cache, put(G, np.array(lens, np.int32)), w, 16, cut, ol, ow, ix)
    ref = R.evict(*want, lens, w.to_numpy(), budget, 16)
    assert np.array_equal(ol.to_numpy(), ref[4])
    assert np.array_equal(parts_of(cut, ref[:4])[0], ref[0])
    # the cut cache is full: put it into a larger one by its values, then go on
    lens = [int(n) for n in ref[4]]
    back_starts = R.starts_of(lens)
    kk, vv = (gb.Tensor.zeros((hd, kv, sum(lens)), F32, G) for _ in range(2))
    zero = put(G, np.zeros(3, np.int32))
    gb.galois_cache_read(cut, put(G, back_starts), zero, kk, vv)
    cache = gb.CacheQ8.zeros(hd, ctx, kv, 3, G)
    gb.galois_cache_append(kk, vv, put(G, back_starts), zero, cache)
    want = [x.copy() for x in like]
    R.append(kk.to_numpy(), back_starts, [0, 0, 0], want[0], want[1])
    R.append(vv.to_numpy(), back_starts, [0, 0, 0], want[2], want[3])
    w = put(G, np.zeros((3, kv, ctx), np.float32))
    lens = tokens(cache, want, lens, w, 3)
    # a second prompt behind what the cache holds: earlier rows read back in F16, the new ones behind them
    new = [20, 5, 1]
    total = [a + b for a, b in zip(lens, new)]
    ks = R.starts_of(total)
    allk, allv = (gb.Tensor.zeros((hd, kv, sum(total)), F16, G) for _ in range(2))
    q2, k2, v2, qs2, _ = prompt_inputs(rng, hd, heads, kv, [(n, n) for n in new], 0)
    gb.galois_cache_append(put(G, k2), put(G, v2), put(G, qs2), put(G, np.array(lens, np.int32)), cache)
    gb.galois_cache_read(cache, put(G, ks), zero, allk, allv)
    dst = put(G, np.zeros(q2.shape, np.float32))
    gb.galois_prompt_attention(put(G, q2), allk, allv, put(G, qs2), put(G, ks), dst, scale)
    out, bound = R.prompt(q2, allk.to_numpy(), allv.to_numpy(), qs2, ks, scale)
    dev.synchronize()
    assert np.all(np.abs(dst.to_numpy() - out) <= bound)


def test_captured_and_replayed_and_on_another_stream(dev, G):
    """All five operators in one graph, replayed on new inputs, on a stream of the caller's."""
    import torch

    rng = np.random.default_rng(31)
    hd, heads, kv, ctx = 128, 4, 2, 128
    q, k, v, qs, _ = prompt_inputs(rng, hd, heads, kv, [(70, 70), (20, 20)], 0)
    qt, kt, vt, st = put(G, q), put(G, k), put(G, v), put(G, qs)
    lens = np.array([70, 20], np.int32)
    zero, lt = put(G, np.zeros(2, np.int32)), put(G, lens)
    cache, cut = gb.CacheQ8.zeros(hd, ctx, kv, 2, G), gb.CacheQ8.zeros(hd, 48, kv, 2, G)
    q1 = put(G, rng.normal(0, 1, (2, heads, hd)).astype(np.float32))
    outs = {"p": put(G, np.zeros(q.shape, np.float16)), "o": put(G, np.zeros((2, heads, hd), np.float32)), "w": put(G, np.zeros((2, kv, ctx), np.float32)),
            "ol": gb.Tensor.zeros((2,), I32, G), "ow": gb.Tensor.zeros((48, kv, 2), F32, G), "ix": gb.Tensor.zeros((48, kv, 2), I32, G),
            "k": gb.Tensor.zeros((hd, kv, 90), F16, G), "v": gb.Tensor.zeros((hd, kv, 90), F16, G)}
    w0 = put(G, np.zeros((2, kv, ctx), np.float32))
    ws = gb.Tensor.zeros((gb.galois_cache_attention_workspace(cache, heads, True) // 4,), F32, G)

    def go():
        gb.galois_prompt_attention(qt, kt, vt, st, st, outs["p"], 0.1)
        gb.galois_cache_append(kt, vt, st, zero, cache)
        gb.galois_cache_attention(q1, cache, lt, outs["o"], 0.1, ws, weights=w0, weights_out=outs["w"])
        gb.galois_cache_evict(cache, lt, outs["w"], 8, cut, outs["ol"], outs["ow"], outs["ix"])
        gb.galois_cache_read(cache, st, zero, outs["k"], outs["v"])

    before, stream = dev.stream, torch.cuda.Stream()
    try:
        torch.cuda.synchronize()
        dev.set_stream(stream)
        go()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            go()
        for seed in (41, 42):
            r = np.random.default_rng(seed)
            for t in (qt, kt, vt, q1):
                t.storage.copy_(torch.from_numpy(r.normal(0, 1, t.storage.numel())))
            for t in outs.values():
                t.storage.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = {n: t.storage.clone() for n, t in outs.items()}
            for t in outs.values():
                t.storage.zero_()
            torch.cuda.synchronize()
            go()
            stream.synchronize()
            for n, t in outs.items():
                assert torch.equal(got[n], t.storage), n
            kq = kt.to_numpy()
            out, bound = R.prompt(qt.to_numpy(), kq, vt.to_numpy(), qs, qs, 0.1)
            assert np.all(np.abs(outs["p"].to_numpy() - out) <= f16_bound(out, bound))
        del graph
    finally:
        torch.cuda.synchronize()
        dev.set_stream(before)


def test_offsets_beyond_32_bits(dev, G):
    """The last slot of a cache of more than 4 GB."""
    rng = np.random.default_rng(51)
    hd, ctx, kv, seqs = 128, 65536, 8, 36  # 36 x 64 MB for the keys, as much for the values, slots 2^26 apart
    cache = gb.CacheQ8.zeros(hd, ctx, kv, seqs, G)
    assert (seqs - 1) * kv * ctx * hd > 2**31
    n = 100
    x = [rng.normal(0, 1, (n, kv, hd)).astype(np.float32) for _ in range(2)]
    starts = np.zeros(seqs + 1, np.int32)
    starts[-1] = n
    pos = np.zeros(seqs, np.int32)
    pos[-1] = ctx - n
    gb.galois_cache_append(put(G, x[0]), put(G, x[1]), put(G, starts), put(G, pos), cache)
    outs = [gb.Tensor.zeros((hd, kv, n), F32, G) for _ in range(2)]
    gb.galois_cache_read(cache, put(G, starts), put(G, pos), *outs)
    q = rng.normal(0, 1, (seqs, kv, hd)).astype(np.float32)
    lens = np.zeros(seqs, np.int32)
    lens[-1] = ctx
    dst = put(G, np.zeros_like(q))
    ws = gb.Tensor.zeros((gb.galois_cache_attention_workspace(cache, kv) // 4,), F32, G)
    gb.galois_cache_attention(put(G, q), cache, put(G, lens), dst, hd**-0.5, ws)
    dev.synchronize()
    want = [np.zeros((1, kv, 128, hd), np.int8), np.zeros((1, kv, 4), np.float32)] * 2
    want = [w.copy() for w in want]
    for i in range(2):
        R.append(x[i], [0, n], [128 - n], want[2 * i], want[2 * i + 1])
        assert np.array_equal(outs[i].to_numpy(), R.values(*want[2 * i:2 * i + 2])[0, :, 128 - n:].transpose(1, 0, 2).astype(np.float32))
    # the other rows are zeros: their logits are 0 and their values nothing
    for h in range(kv):
        kk, vv = (R.values(*want[2 * i:2 * i + 2])[0, h, 128 - n:] for i in range(2))
        x_ = kk @ q[-1, h].astype(np.float64) * hd**-0.5
        top = max(0.0, x_.max())
        e = np.exp(x_ - top)
        ref = e @ vv / (e.sum() + (ctx - n) * np.exp(-top))
        assert np.allclose(dst.to_numpy()[-1, h], ref, rtol=1e-4, atol=1e-6)
    assert not dst.to_numpy()[:-1].any()


@pytest.mark.parametrize("hd,heads,kv", list(itertools.product([64, 128], [8], [1, 2, 8])))
def test_a_slot_alone_gives_what_it_gives_in_a_batch(dev, G, hd, heads, kv):
    """A sequence's results do not depend on which others are served with it, up to the order of sums."""
    rng = np.random.default_rng(61)
    lens = np.array([200, 64, 1, 130], np.int32)
    parts = random_cache(rng, 4, kv, 200, hd)
    q = rng.normal(0, 1, (4, heads, hd)).astype(np.float32)

    def attend(parts, q, lens):
        cache, dst = upload(G, parts), put(G, np.zeros_like(q))
        ws = gb.Tensor.zeros((gb.galois_cache_attention_workspace(cache, heads) // 4,), F32, G)
        gb.galois_cache_attention(put(G, q), cache, put(G, lens), dst, 0.1, ws)
        dev.synchronize()
        return dst.to_numpy()

    whole = attend(parts, q, lens)
    for s in range(4):
        one = attend([p[s:s + 1] for p in parts], q[s:s + 1], lens[s:s + 1])
        _, bound, _, _ = R.step(q[s:s + 1], *[p[s:s + 1] for p in parts], lens[s:s + 1], 0.1)
        assert np.all(np.abs(one - whole[s:s + 1]) <= 2 * bound)


# ------------------------------------------------------------------------------------------------ many, none, two at once


@pytest.mark.parametrize("heads,kv", [(4, 2), (3, 1)])
def test_prompt_attention_of_many_sequences(dev, G, heads, kv):
    """More sequences than a warp has lanes, some without queries, some without keys."""
    rng = np.random.default_rng(71)
    seqs = [(int(a), int(max(0, a + b))) for a, b in zip(rng.integers(0, 40, 100), rng.integers(-20, 60, 100))]
    seqs[40], seqs[77] = (700, 900), (130, 64)
    q, k, v, qs, ks = prompt_inputs(rng, 64, heads, kv, seqs, 0)
    out, bound = R.prompt(q, k, v, qs, ks, 0.125)
    dst = put(G, np.full(q.shape, 3, np.float32))
    gb.galois_prompt_attention(put(G, q), put(G, k), put(G, v), put(G, qs), put(G, ks), dst, 0.125)
    dev.synchronize()
    assert np.all(np.abs(dst.to_numpy() - out) <= bound)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-30])
def test_prompt_attention_scales(dev, G, scale):
    rng = np.random.default_rng(72)
    q, k, v, qs, ks = prompt_inputs(rng, 128, 2, 1, [(150, 150), (3, 70)], 0)
    out, _ = R.prompt(q, k, v, qs, ks, scale)
    _, bound = R.prompt(q, k, v, qs, ks, abs(scale))
    if scale < 0:  # the bound's probabilities belong to the other sign: all of them at once
        bound = np.maximum(bound, 2.0**-10 * np.abs(v.astype(np.float64)).max())
    dst = put(G, np.zeros(q.shape, np.float32))
    gb.galois_prompt_attention(put(G, q), put(G, k), put(G, v), put(G, qs), put(G, ks), dst, scale)
    dev.synchronize()
    assert np.all(np.abs(dst.to_numpy() - out) <= bound)


def test_nothing_to_see(dev, G):
    """No keys at all, a cache without rows, no sequences, no tokens."""
    q = put(G, np.ones((5, 2, 64), np.float16))
    none = gb.Tensor.zeros((64, 2, 0), F16, G)
    dst = put(G, np.full((5, 2, 64), 3, np.float32))
    gb.galois_prompt_attention(q, none, none, put(G, np.array([0, 5], np.int32)), put(G, np.array([0, 0], np.int32)), dst, 0.1)
    dev.synchronize()
    assert not dst.to_numpy().any()
    cache = gb.CacheQ8.zeros(64, 0, 2, 3, G)
    q1, o1 = put(G, np.ones((3, 2, 64), np.float32)), put(G, np.full((3, 2, 64), 3, np.float32))
    ws = gb.Tensor.zeros((gb.galois_cache_attention_workspace(cache, 2) // 4,), F32, G)
    gb.galois_cache_attention(q1, cache, put(G, np.zeros(3, np.int32)), o1, 0.1, ws)
    dev.synchronize()
    assert not o1.to_numpy().any()
    cache = gb.CacheQ8.zeros(64, 40, 2, 3, G)
    kv = gb.Tensor.zeros((64, 2, 0), F32, G)
    gb.galois_cache_append(kv, kv, put(G, np.zeros(4, np.int32)), put(G, np.zeros(3, np.int32)), cache)
    cut = gb.CacheQ8.zeros(64, 0, 2, 3, G)
    lens, ol = put(G, np.array([40, 1, 0], np.int32)), put(G, np.full(3, 9, np.int32))
    empty_f, empty_i = gb.Tensor.zeros((0, 2, 3), F32, G), gb.Tensor.zeros((0, 2, 3), I32, G)
    gb.galois_cache_evict(cache, lens, put(G, np.ones((3, 2, 40), np.float32)), 4, cut, ol, empty_f, empty_i)
    dev.synchronize()
    assert not ol.to_numpy().any()


def test_cache_attention_of_many_slots(dev, G):
    """More slots than a warp has lanes, most of them empty or short."""
    rng = np.random.default_rng(73)
    seqs, ctx = 150, 100
    lens = rng.integers(0, 3, seqs) * rng.integers(0, 51, seqs)
    lens[[0, 149]] = 0, 100
    parts = random_cache(rng, seqs, 2, ctx, 64)
    q, w = rng.normal(0, 1, (seqs, 18, 64)).astype(np.float32), rng.random((seqs, 2, ctx)).astype(np.float32)
    out, bound, ww, wb = R.step(q, *parts, lens, 0.125, w)
    cache, dst, wt = upload(G, parts), put(G, np.full_like(q, 3)), put(G, w)
    ws = gb.Tensor.zeros((gb.galois_cache_attention_workspace(cache, 18, True) // 4,), F32, G)
    gb.galois_cache_attention(put(G, q), cache, put(G, lens.astype(np.int32)), dst, 0.125, ws, weights=wt, weights_out=wt)
    dev.synchronize()
    assert np.all(np.abs(dst.to_numpy() - out) <= bound)
    got = wt.to_numpy()
    for s, n in enumerate(lens):
        assert np.all(np.abs(got[s, :, :n] - ww[s, :, :n]) <= wb[s, :, :n]) and np.array_equal(got[s, :, n:], w[s, :, n:])


def test_two_contexts_at_once(dev, G):
    """Two contexts on streams of their own, their launches interleaved: each gives what it gives alone."""
    import torch

    rng = np.random.default_rng(74)
    other = gb.CudaDevice(0, torch.cuda.Stream())
    try:
        places = [G, gb.Device.Gpu(other)]
        lens = np.array([700, 300], np.int32)
        work = []
        for P in places:
            parts = random_cache(rng, 2, 2, 700, 128)
            q, k, v, qs, _ = prompt_inputs(rng, 128, 4, 2, [(260, 260), (90, 90)], 0)
            q1 = rng.normal(0, 1, (2, 4, 128)).astype(np.float32)
            t = {"cache": upload(P, parts), "q": put(P, q), "k": put(P, k), "v": put(P, v), "s": put(P, qs), "q1": put(P, q1), "l": put(P, lens),
                 "o": put(P, np.zeros(q.shape, np.float16)), "o1": put(P, np.zeros_like(q1))}
            t["ws"] = gb.Tensor.zeros((gb.galois_cache_attention_workspace(t["cache"], 4) // 4,), F32, P)
            work.append((t, R.prompt(q, k, v, qs, qs, 0.09), R.step(q1, *parts, lens, 0.09)))
        torch.cuda.synchronize()
        for _ in range(20):
            for t, _, _ in work:
                gb.galois_prompt_attention(t["q"], t["k"], t["v"], t["s"], t["s"], t["o"], 0.09)
                gb.galois_cache_attention(t["q1"], t["cache"], t["l"], t["o1"], 0.09, t["ws"])
        dev.synchronize()
        other.synchronize()
        for t, (out, bound), (step, step_bound, _, _) in work:
            assert np.all(np.abs(t["o"].to_numpy() - out) <= f16_bound(out, bound))
            assert np.all(np.abs(t["o1"].to_numpy() - step) <= step_bound)
    finally:
        other.close()


def test_beside_the_library_s_other_kernels(dev, G, oracle):
    """Prompt attention between mat-muls that hold tensor memory themselves, all launched to overlap."""
    rng = np.random.default_rng(75)
    n = k = 256
    w = oracle.quantize_q4_0(oracle.fill_normal(n * k, 170, 0, 0.02).reshape(n, k))
    wt = gb.Tensor.from_raw(w, (k, n), GGmlType.Q4_0, G)
    x = oracle.fill_normal(256 * k, 171).reshape(256, k)
    xt, y1, y2 = put(G, x), gb.Tensor.zeros((n, 256), F32, G), gb.Tensor.zeros((n, 256), F32, G)
    q, kk, v, qs, _ = prompt_inputs(rng, 64, 4, 4, [(256, 256)], 0)
    qt, kt, vt, st, o = put(G, q), put(G, kk), put(G, v), put(G, qs), put(G, np.zeros(q.shape, np.float16))
    for _ in range(5):
        gb.galois_matmul(wt, xt, y1)
        gb.galois_prompt_attention(qt, kt, vt, st, st, o, 0.125)
        gb.galois_matmul(wt, xt, y2)
    dev.synchronize()
    assert np.array_equal(y1.to_numpy(), y2.to_numpy())
    from conftest import assert_close

    assert_close(y1.to_numpy(), oracle.mul_mat_q4_0(w, x))
    out, bound = R.prompt(q, kk, v, qs, qs, 0.125)
    assert np.all(np.abs(o.to_numpy() - out) <= f16_bound(out, bound))


@pytest.mark.parametrize("hd,heads,kv", [(64, 4, 2), (128, 2, 2)])
def test_prompt_attention_of_short_ragged_prompts_one_after_the_other(dev, G, hd, heads, kv):
    """Every unit is one ragged tile of keys, and each SM goes through several of them: the next unit's values may be under way
    before this one's have arrived.  Each replay finds its operands in HBM."""
    rng = np.random.default_rng(74)
    seqs = [(int(n), int(n)) for n in rng.integers(1, 61, 700)]
    q, k, v, qs, ks = prompt_inputs(rng, hd, heads, kv, seqs, 0)
    args = [put(G, a) for a in (q, k, v, qs, ks)]
    dst = put(G, np.full(q.shape, 3, np.float32))
    out, bound = R.prompt(q, k, v, qs, ks, 0.125)
    for _ in range(3):
        gb.Tensor.zeros((1 << 26,), F32, G)  # 256 MB pass through L2
        gb.galois_prompt_attention(*args, dst, 0.125)
        dev.synchronize()
        assert np.all(np.abs(dst.to_numpy() - out) <= bound)


@pytest.mark.parametrize("first,lens,pos", [(3, [5, 40], [30, 0]), (64, [1, 1], [0, 63]), (45, [64], [0])])
def test_rows_in_front_of_the_first_sequence(dev, G, first, lens, pos):
    """starts need not begin at 0: what lies in front belongs to nobody, and is no error."""
    rng = np.random.default_rng(75)
    starts = R.starts_of(lens) + first
    tokens = int(starts[-1]) + 2
    parts = random_cache(rng, len(lens), 2, 64, 64)
    x = [rng.normal(0, 1, (tokens, 2, 64)).astype(np.float32) for _ in range(2)]
    cache, want = upload(G, parts), [p.copy() for p in parts]
    s, p = put(G, starts.astype(np.int32)), put(G, np.array(pos, np.int32))
    gb.galois_cache_append(put(G, x[0]), put(G, x[1]), s, p, cache)
    outs = [put(G, np.full((tokens, 2, 64), 9, np.float32)) for _ in range(2)]
    gb.galois_cache_read(cache, s, p, outs[0], outs[1])
    dev.synchronize()
    for h in range(2):
        R.append(x[h][first:], starts - first, pos, want[2 * h], want[2 * h + 1])
    for got, w in zip(parts_of(cache, want), want):
        assert np.array_equal(got, w)
    for h, out in enumerate(outs):
        rows, got = R.values(want[2 * h], want[2 * h + 1]), out.to_numpy()
        assert np.all(got[:first] == 9) and np.all(got[starts[-1]:] == 9)
        for i, n in enumerate(lens):
            assert np.array_equal(got[starts[i]:starts[i + 1]], rows[i, :, pos[i]:pos[i] + n].transpose(1, 0, 2).astype(np.float32))


@pytest.mark.parametrize("starts", [[4, 2, 5], [5, 7, 7], [9, 9, 9]])
def test_starts_that_do_not_ascend_or_pass_the_end_are_reported(dev, G, starts):
    cache = upload(G, random_cache(np.random.default_rng(76), 2, 1, 64, 64))
    x = put(G, np.ones((5, 1, 64), np.float32))
    s, p = put(G, np.array(starts, np.int32)), put(G, np.zeros(2, np.int32))
    gb.galois_cache_append(x, x, s, p, cache)
    with pytest.raises(GError) as e:
        dev.synchronize()
    assert e.value.code == -1


@pytest.mark.parametrize("n", [3, 70])
def test_read_leaves_a_sequence_out_as_a_whole(dev, G, n):
    """One row too many for the slot: none of the sequence's rows is written."""
    cache = upload(G, random_cache(np.random.default_rng(77), 2, 1, 100, 64))
    outs = [put(G, np.full((n + 2, 1, 64), 9, np.float32)) for _ in range(2)]
    gb.galois_cache_read(cache, put(G, np.array([0, n, n + 2], np.int32)), put(G, np.array([101 - n, 5], np.int32)), outs[0], outs[1])
    with pytest.raises(GError):
        dev.synchronize()
    for out in outs:
        got = out.to_numpy()
        assert np.all(got[:n] == 9) and not np.any(got[n:] == 9)


@pytest.mark.parametrize("hd", [64, 128])
def test_cache_attention_of_the_largest_values(dev, G, hd):
    """The sum of many large values leaves f32's range, their mean does not."""
    rng = np.random.default_rng(78)
    lens = [3000, 33, 7]
    kq, ks, vq, vs = random_cache(rng, 3, 1, 3000, hd)
    vq[..., : hd // 2] = 120
    vs[:] = np.float32(2.5e36)
    q = rng.normal(0, 0.01, (3, 4, hd)).astype(np.float32)
    out, bound, _, _ = R.step(q, kq, ks, vq, vs, lens, 0.125)
    cache, dst = upload(G, (kq, ks, vq, vs)), put(G, np.zeros_like(q))
    ws = gb.Tensor.zeros((gb.galois_cache_attention_workspace(cache, 4) // 4,), F32, G)
    gb.galois_cache_attention(put(G, q), cache, put(G, np.array(lens, np.int32)), dst, 0.125, ws)
    dev.synchronize()
    assert np.all(np.abs(dst.to_numpy() - out) <= bound)


def test_cache_attention_of_logits_below_the_range(dev, G):
    """Every logit is -inf in f32: nothing counts, the result and the added weights are 0."""
    kq, vq = np.full((1, 1, 40, 64), 127, np.int8), np.full((1, 1, 40, 64), 3, np.int8)
    sc = np.full((1, 1, 2), 1e30, np.float32)
    q, w = np.full((1, 2, 64), -1e30, np.float32), np.arange(40, dtype=np.float32).reshape(1, 1, 40)
    cache, dst, wt = upload(G, (kq, sc, vq, np.ones_like(sc))), put(G, np.full_like(q, 5)), put(G, w)
    ws = gb.Tensor.zeros((gb.galois_cache_attention_workspace(cache, 2, True) // 4,), F32, G)
    gb.galois_cache_attention(put(G, q), cache, put(G, np.array([40], np.int32)), dst, 1.0, ws, weights=wt, weights_out=wt)
    dev.synchronize()
    assert not dst.to_numpy().any() and np.array_equal(wt.to_numpy(), w)


@pytest.mark.parametrize("kind,pad", [(np.float32, 4), (np.float16, 8), (np.float32, 8), (np.float16, 16)])
def test_prompt_attention_into_rows_of_any_alignment(dev, G, kind, pad):
    """Rows of the destination begin at every 16 bytes, or every 32."""
    rng = np.random.default_rng(79)
    q, k, v, qs, ks = prompt_inputs(rng, 64, 3, 1, [(140, 150), (9, 9)], 1)
    out, bound = R.prompt(q, k, v, qs, ks, 0.125)
    bound = f16_bound(out, bound) if kind == np.float16 else bound
    dst, _, _ = spread(G, np.full(q.shape, 3, kind), None, pad)
    gb.galois_prompt_attention(put(G, q), put(G, k), put(G, v), put(G, qs), put(G, ks), dst, 0.125)
    dev.synchronize()
    got, n = back(dst, q.shape).astype(np.float64), qs[-1]
    assert np.all(got[n:] == 3) and np.all(np.abs(got[:n] - out[:n]) <= bound[:n])
