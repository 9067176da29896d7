"""That the tolerances of test_cache_accuracy.py see the mistakes they are there for, planted in the plain form (no GPU)."""
import numpy as np
import pytest

from test_cache_accuracy import EXACT, SINKS, exact_inputs, sink_inputs, step64


def half_of(x, axis):
    """x as one F16 whose largest along `axis` lies in 2^14 .. 2^15: what is left when the lower half is lost."""
    top = np.abs(x).max(axis, keepdims=True)
    up = 2.0 ** (14 - np.floor(np.log2(np.where(top == 0, 1, top))))
    return (x * up).astype(np.float16).astype(np.float64) / up


def step_with(q, kq, ks, vq, vs, lens, scale, change):
    out = np.zeros(q.shape)
    heads, kv = q.shape[1], kq.shape[1]
    for s, n in enumerate(lens):
        by = np.arange(n) // 32
        for h in range(heads):
            c = h // (heads // kv)
            x = (kq[s, c, :n] * ks[s, c][by][:, None].astype(np.float64)) @ q[s, h].astype(np.float64) * scale
            e = np.exp(x - x.max())
            out[s, h] = change(e) @ (vq[s, c, :n] * vs[s, c][by][:, None].astype(np.float64)) / e.sum()
    return out


@pytest.mark.parametrize("hd,heads,kv,lens", EXACT)
def test_a_lost_half_is_seen(hd, heads, kv, lens):
    q, parts, scale = exact_inputs(hd, heads, kv, lens)
    out, tol = step64(q, *parts, lens, scale)
    assert np.all(np.abs(step_with(q, *parts, lens, scale, lambda e: e) - out) <= tol / 100)
    assert np.any(np.abs(step_with(half_of(q.astype(np.float64), -1), *parts, lens, scale, lambda e: e) - out) > tol)
    assert np.any(np.abs(step_with(q, *parts, lens, scale, lambda e: half_of(e, 0)) - out) > tol)


@pytest.mark.parametrize("gap", [14, 17, 20, 25])
@pytest.mark.parametrize("hd,n", SINKS)
def test_probabilities_that_are_cut_off_are_seen(gap, hd, n):
    """Multiples of 2^-25 of the largest, as two F16 halves of numbers up to 1 end."""
    q, parts = sink_inputs(gap, hd, n)
    out, tol = step64(q, *parts, [n], 1.0)
    assert np.any(np.abs(step_with(q, *parts, [n], 1.0, lambda e: np.rint(e * 2.0**24) / 2.0**24) - out) > tol)
