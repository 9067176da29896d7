"""Plain 64-bit forms of the prompt-attention and 8-bit-cache operators, for the tests."""
import numpy as np

BLOCK = 32
TINY = 2.0**-100
F32_MAX = np.finfo(np.float32).max


def starts_of(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def append(x, starts, pos, q, scale):
    """x [tokens][kv][hd] into q [seqs][kv][ctx][hd] (i8) and scale [seqs][kv][blocks], in place."""
    with np.errstate(all="ignore"):
        x = np.nan_to_num(x.astype(np.float64), nan=0.0, posinf=F32_MAX, neginf=-F32_MAX)
        for s in range(len(starts) - 1):
            n, p = int(starts[s + 1] - starts[s]), int(pos[s])
            rows = x[starts[s]:starts[s + 1]].transpose(1, 0, 2)  # [kv][n][hd]
            for b in range(p // BLOCK, (p + n - 1) // BLOCK + 1 if n else p // BLOCK):
                lo, hi = max(p, b * BLOCK), min(p + n, (b + 1) * BLOCK)
                part = rows[:, lo - p:hi - p]
                d = (np.abs(part).max((1, 2)) / 127).astype(np.float32)
                held = scale[s, :, b].copy() if lo > b * BLOCK else np.zeros_like(d)
                d = np.maximum(d, held)
                d[d < TINY] = 0
                by = np.where(d == 0, 1, d).astype(np.float64)[:, None, None]
                old = np.rint(q[s, :, b * BLOCK:lo].astype(np.float64) * held.astype(np.float64)[:, None, None] / by)
                new = np.rint(part / by)
                q[s, :, b * BLOCK:lo] = np.where(d[:, None, None] == 0, 0, np.clip(old, -127, 127))
                q[s, :, lo:hi] = np.where(d[:, None, None] == 0, 0, np.clip(new, -127, 127))
                scale[s, :, b] = d


def values(q, scale):
    return q.astype(np.float64) * np.repeat(scale.astype(np.float64), BLOCK, axis=2)[:, :, :q.shape[2], None]


def step(q, kq, ks, vq, vs, lens, scale, weights=None):
    """(out [seqs][heads][hd], weights + probabilities, bound on |out| of an f32 evaluation)."""
    seqs, heads, hd = q.shape
    kv, ctx = kq.shape[1:3]
    group = heads // kv
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    w = None if weights is None else weights.astype(np.float64).copy()
    wb = None if weights is None else np.zeros(w.shape)
    for s in range(seqs):
        n = int(lens[s])
        if n == 0:
            continue
        by = np.arange(n) // BLOCK
        for h in range(heads):
            c = h // group
            k = kq[s, c, :n].astype(np.float64) * ks[s, c][by].astype(np.float64)[:, None]
            v = vq[s, c, :n].astype(np.float64) * vs[s, c][by].astype(np.float64)[:, None]
            qd = q[s, h].astype(np.float64)
            x = k @ qd * scale
            p = np.exp(x - x.max())
            p /= p.sum()
            out[s, h] = p @ v
            # logits: hd products summed in f32 in any order, q split into two halves of 11 bits (2^-22 left over), two
            # more products (scales); exp of an argument that is off by |x| 2^-23; sums of n terms; each counted twice
            delta = scale * (np.abs(k) @ np.abs(qd)).max() * (hd * 2.0**-24 + 2.0**-21)
            eps = 2 * delta + np.abs(x - x.max()).max() * 2.0**-22 + 2.0**-20 + n * 2.0**-24
            bound[s, h] = 2 * eps * np.abs(v).max(0) + 2.0**-22 * np.abs(v).max()
            if w is not None:
                w[s, c, :n] += p
                wb[s, c, :n] += 2 * eps * p + 2.0**-23 * w[s, c, :n]
    return out, bound, w, wb


def prompt(q, k, v, q_starts, k_starts, scale):
    """(out [tokens][heads][hd], bound on the error of an evaluation with F16 probabilities and an f32 result)."""
    heads, hd = q.shape[1:]
    group = heads // k.shape[1]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for s in range(len(q_starts) - 1):
        q0, q1, k0, k1 = int(q_starts[s]), int(q_starts[s + 1]), int(k_starts[s]), int(k_starts[s + 1])
        nq, nk = q1 - q0, k1 - k0
        for h in range(heads):
            kk, vv = k[k0:k1, h // group].astype(np.float64), v[k0:k1, h // group].astype(np.float64)
            for i in range(nq):
                n = i + nk - nq + 1
                if n <= 0:
                    continue
                qi = q[q0 + i, h].astype(np.float64)
                with np.errstate(all="ignore"):
                    x = kk[:n] @ qi * scale
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    out[q0 + i, h] = p @ vv[:n]
                    delta = scale * (np.abs(kk[:n]) @ np.abs(qi)).max() * (hd * 2.0**-24 + 2.0**-22)
                    eps = 2 * delta + np.abs(x - x.max()).max() * 2.0**-22 + 2.0**-20 + n * 2.0**-24
                    # probabilities are rounded to F16 relative to the largest (half a step, 2^-11, and 2^-25 where they
                    # are below F16's normal range)
                    bound[q0 + i, h] = (2.0**-11 + 2 * eps) * (p @ np.abs(vv[:n])) + 2.0**-25 * np.abs(vv[:n]).sum(0) / np.exp(x - x.max()).sum()
    return out, bound


def evict(kq, ks, vq, vs, lens, weights, budget, recent):
    """(k, k_scale, v, v_scale, out_lens, out_weights, index) of the cut cache; rows behind a length are zero / -1."""
    seqs, kv, ctx, hd = kq.shape
    blocks = (budget + BLOCK - 1) // BLOCK
    index = np.full((seqs, kv, budget), -1, np.int32)
    ow = np.zeros((seqs, kv, budget), np.float32)
    out = [(np.zeros((seqs, kv, budget, hd), np.int8), np.zeros((seqs, kv, blocks), np.float32)) for _ in range(2)]
    for s in range(seqs):
        n = int(lens[s])
        m = min(n, budget)
        r = min(recent, m)
        for c in range(kv):
            w = np.where(np.isnan(weights[s, c]), -np.inf, weights[s, c].astype(np.float64))
            nan = np.isnan(weights[s, c])
            order = sorted(range(n - r), key=lambda j: (bool(nan[j]), -w[j], j))[:m - r]
            kept = np.array(sorted(order) + list(range(n - r, n)), np.int64)
            index[s, c, :m] = kept
            ow[s, c, :m] = weights[s, c, kept]
            for (q, sc), (oq, osc) in zip(((kq, ks), (vq, vs)), out):
                d_old = sc[s, c, kept // BLOCK]
                for b in range(0, m, BLOCK):
                    part = slice(b, min(m, b + BLOCK))
                    d = d_old[part].max()
                    if d < TINY:
                        d = np.float32(0)
                    osc[s, c, b // BLOCK] = d
                    x = q[s, c, kept[part]].astype(np.float64) * d_old[part].astype(np.float64)[:, None]
                    oq[s, c, part] = np.rint(x / np.float64(d)) if d > 0 else 0
    return out[0][0], out[0][1], out[1][0], out[1][1], np.minimum(lens, budget).astype(np.int32), ow, index
