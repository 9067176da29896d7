"""What the prompt-attention and 8-bit key/value-cache operators are measured on.

Each case is one pass through one operator at sizes that a decoder with this library's layers meets: 32 heads of
128 (or grouped over 8 key/value heads), contexts of 2048 and up to 8192 tokens, one sequence or a batch of them
with different lengths.  ``run`` computes the plain form (elementary torch operations, 32 bits, 64 bits for the
quotients that are rounded to whole numbers) or, with ``own``, calls the library.

  prompt  attention of packed prompts: causal within each sequence, grouped heads, optionally behind a prefix
  append  keys and values of new tokens into an 8-bit cache, one scale for each 32 tokens of a head; the rows of
          the blocks that were written are read back as the values they stand for
  read    rows of the 8-bit cache as F16 / F32 values
  step    attention of one new token per sequence over the cache, optionally adding up each token's weight
  evict   the cache cut down to a budget: the newest tokens and those with the largest added-up weight
"""
import functools
import random

import torch

own = False

BLOCK = 32        # tokens that share a scale
TINY = 2.0**-100  # a scale below this stands for a block of zeros


def listed():
    return [
        # a handful of short questions packed into one call, grouped heads of 64: latency
        {"name": "prompt short", "op": "prompt", "head_dim": 64, "heads": 8, "kv_heads": 2, "seqs": 7, "tokens": 300, "prefix": 0},
        # the decode layer's shape (32 heads x 128) filling its context of 2048 from one prompt
        {"name": "prompt layer", "op": "prompt", "head_dim": 128, "heads": 32, "kv_heads": 32, "seqs": 1, "tokens": 2048, "prefix": 0},
        # a prefill batch of a grouped-head model: ragged prompts, part of them continuing a cached prefix
        {"name": "prompt packed", "op": "prompt", "head_dim": 128, "heads": 32, "kv_heads": 8, "seqs": 3, "tokens": 8192, "prefix": 500},
        # one generated token for each of 48 conversations, in the type the projections write
        {"name": "append tokens", "op": "append", "head_dim": 128, "kv_heads": 8, "seqs": 48, "tokens": 48, "ctx": 4096, "half": False},
        # the prompts of a prefill batch put into the cache
        {"name": "append prompts", "op": "append", "head_dim": 128, "kv_heads": 8, "seqs": 5, "tokens": 8000, "ctx": 8192, "half": True},
        # a short conversation read back for the continuation of its prompt
        {"name": "read one", "op": "read", "head_dim": 128, "kv_heads": 32, "seqs": 1, "ctx": 2048, "rows": 333, "half": True},
        # a batch of long ones
        {"name": "read batch", "op": "read", "head_dim": 128, "kv_heads": 8, "seqs": 8, "ctx": 8192, "rows": 50000, "half": True},
        # one conversation, the decode layer's shape with its cache full
        {"name": "step one", "op": "step", "head_dim": 128, "heads": 32, "kv_heads": 32, "seqs": 1, "ctx": 2048, "full": True, "weights": False},
        # a serving batch of conversations of different lengths, grouped heads
        {"name": "step batch", "op": "step", "head_dim": 128, "heads": 32, "kv_heads": 8, "seqs": 64, "ctx": 8192, "full": False, "weights": False},
        # a batch whose cache is going to be cut: the weights are added up
        {"name": "step weights", "op": "step", "head_dim": 128, "heads": 32, "kv_heads": 8, "seqs": 16, "ctx": 4096, "full": False, "weights": True},
        # one conversation that has filled its context, cut to half of it
        {"name": "evict one", "op": "evict", "head_dim": 128, "kv_heads": 32, "seqs": 1, "ctx": 2048, "budget": 1024, "recent": 128},
        # a batch of grouped-head conversations cut to 2048 tokens each
        {"name": "evict batch", "op": "evict", "head_dim": 128, "kv_heads": 8, "seqs": 16, "ctx": 8192, "budget": 2048, "recent": 256},
    ]


def draw(rng):
    log = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))  # noqa: E731
    op = rng.choice(["prompt", "prompt", "append", "read", "step", "step", "evict"])
    c = {"op": op, "head_dim": rng.choice([64, 128, 128])}
    kv = rng.choice([1, 2, 3, 4, 5, 8, 8, 10, 16, 32])
    if op == "prompt":
        group = rng.choice([1, 1, 2, 3, 4, 4, 5, 7, 8])
        kv = max(1, min(kv, 32 // group))
        c |= {"heads": kv * group, "kv_heads": kv, "seqs": log(1, 16)}
        c |= {"tokens": log(max(4, c["seqs"]), 6500), "prefix": rng.choice([0, 0, 0, log(1, 700)])}
    elif op == "append":
        c |= {"kv_heads": kv, "seqs": log(1, 64)}
        c |= {"tokens": c["seqs"] if rng.random() < 0.5 else max(c["seqs"], log(40, 8000 * 8 // max(8, kv))), "half": rng.random() < 0.5}
        c["ctx"] = min(8192, c["tokens"] + log(32, 2000))
    elif op == "read":
        c |= {"kv_heads": kv, "seqs": log(1, 16), "ctx": log(64, 8192), "half": rng.random() < 0.7}
        c["rows"] = min(c["seqs"] * c["ctx"], log(max(16, c["seqs"]), 50000 * 8 // max(8, kv)))
    elif op == "step":
        group = rng.choice([1, 1, 2, 3, 4, 4, 5, 7, 8, 12, 16])
        kv = max(1, min(kv, 64 // group))
        c |= {"heads": kv * group, "kv_heads": kv, "ctx": log(64, 8192), "full": rng.random() < 0.3, "weights": rng.random() < 0.3}
        c["seqs"] = log(1, max(1, min(64, 64 * 8 * 8192 // (kv * c["ctx"] * 4 if c["weights"] else kv * c["ctx"] * 2))))
    else:
        c |= {"kv_heads": kv, "ctx": log(100, 8192)}
        c["seqs"] = log(1, max(1, min(32, 8 * 8 * 8192 // (kv * c["ctx"]))))
        c["budget"] = max(1, min(c["ctx"], log(max(1, c["ctx"] // 8), max(2, c["ctx"]))))
        c["recent"] = rng.randint(0, c["budget"] // 2)
    return c


# ---------------------------------------------------------------------------------------------- lengths


def _parts(total, parts, key, least=1):
    """`total` dealt into `parts` lengths of at least `least`, unevenly, the same way for the same sizes."""
    r = random.Random(key)
    cuts = sorted(r.random() for _ in range(parts - 1))
    spare = total - parts * least
    edges = [0] + [int(spare * c) for c in cuts] + [spare]
    return [least + b - a for a, b in zip(edges, edges[1:])]


def _lengths(case):
    """What the case's sizes say of its sequences, as lists of whole numbers."""
    n = case["seqs"]
    key = ":".join("%s" % case[k] for k in sorted(case) if k != "name")
    r = random.Random(key)
    if case["op"] == "prompt":
        q = _parts(case["tokens"], n, key)
        before = [case["prefix"] if i % 2 == 0 else 0 for i in range(n)]
        return {"q": q, "k": [a + b for a, b in zip(q, before)]}
    if case["op"] == "append":
        new = _parts(case["tokens"], n, key)
        return {"new": new, "pos": [r.randint(0, case["ctx"] - a) for a in new]}
    if case["op"] == "read":
        least = min(1, case["rows"] // n)
        rows = _parts(case["rows"], n, key, least)
        over = 0
        for i in range(n):  # what does not fit a sequence's context goes to the others
            over += max(0, rows[i] - case["ctx"])
            rows[i] = min(rows[i], case["ctx"])
        for i in range(n):
            more = min(over, case["ctx"] - rows[i])
            rows[i] += more
            over -= more
        return {"rows": rows, "pos": [r.randint(0, case["ctx"] - a) for a in rows]}
    if case["op"] == "step":
        if case["full"]:
            return {"len": [case["ctx"]] * n}
        lens = [max(1, int(case["ctx"] * (0.1 + 0.9 * r.random()))) for _ in range(n)]
        if n > 8:
            lens[3] = 0  # a slot of the batch that holds no conversation
            lens[5] = case["ctx"]
        return {"len": lens}
    return {"len": [case["ctx"]] + [max(1, int(case["ctx"] * (0.2 + 0.8 * r.random()))) for _ in range(n - 1)]}


def _starts(lens):
    out = [0]
    for x in lens:
        out.append(out[-1] + x)
    return out


# ---------------------------------------------------------------------------------------------- inputs


def _cache(g, case, ctx):
    """An 8-bit cache as a run of the model leaves it: whole numbers that fill -127..127, scales that differ by
    head and block (a few channels and heads of the keys are far larger than the rest)."""
    shape = (case["seqs"], case["kv_heads"], ctx, case["head_dim"])
    blocks = (ctx + BLOCK - 1) // BLOCK
    out = {}
    for name, size in (("k", 0.03), ("v", 0.02)):
        x = torch.randn(shape, device="cuda", generator=g).mul_(40).round_().clamp_(-127, 127)
        out[name] = x.to(torch.int8)
        del x
        spread = torch.randn(shape[:2] + (blocks,), device="cuda", generator=g).mul_(0.3).exp_()
        out[name + "_scale"] = spread * size * (1 + torch.rand(shape[:2] + (1,), device="cuda", generator=g))
    return out


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, device="cuda", generator=g)  # noqa: E731
    lens, hd, kv = _lengths(case), case["head_dim"], case["kv_heads"]
    s = {"case": dict(case)}
    if case["op"] == "prompt":
        loud = randn(kv, hd).mul(0.4).exp()  # channels of the keys that are larger than others
        s["q"] = randn(case["tokens"], case["heads"], hd).half()
        s["k"] = (randn(sum(lens["k"]), kv, hd) * loud).half()
        s["v"] = randn(sum(lens["k"]), kv, hd).half()
        s["q_starts"], s["k_starts"] = _ints(_starts(lens["q"])), _ints(_starts(lens["k"]))
    elif case["op"] == "append":
        s |= _cache(g, case, case["ctx"])
        kind = torch.float16 if case["half"] else torch.float32
        loud = randn(kv, hd).mul(0.4).exp()
        s["new_k"] = (randn(case["tokens"], kv, hd) * loud * 1.5).to(kind)
        s["new_v"] = randn(case["tokens"], kv, hd).to(kind)
        s["starts"], s["pos"] = _ints(_starts(lens["new"])), _ints(lens["pos"])
        # the rows of the blocks that the new tokens lie in, up to the last new token
        first = [p // BLOCK * BLOCK for p in lens["pos"]]
        back = [p + n - f for p, n, f in zip(lens["pos"], lens["new"], first)]
        s["back_starts"], s["back_pos"], s["back_rows"] = _ints(_starts(back)), _ints(first), sum(back)
        s["most"] = max(lens["new"])
    elif case["op"] == "read":
        s |= _cache(g, case, case["ctx"])
        s["starts"], s["pos"], s["rows"] = _ints(_starts(lens["rows"])), _ints(lens["pos"]), sum(lens["rows"])
    elif case["op"] == "step":
        s |= _cache(g, case, case["ctx"])
        s["q"] = randn(case["seqs"], case["heads"], hd)
        s["len"] = _ints(lens["len"])
        if case["weights"]:
            s["weights"] = torch.rand((case["seqs"], kv, case["ctx"]), device="cuda", generator=g)
    else:
        s |= _cache(g, case, case["ctx"])
        s["len"] = _ints(lens["len"])
        # long-tailed and, for rarely used tokens, equal: steps of 1/64
        s["weights"] = randn(case["seqs"], kv, case["ctx"]).mul(2).exp().mul(16).floor().div(64)
        kept = [min(n, case["budget"]) for n in lens["len"]]
        s["kept_starts"], s["kept_pos"], s["kept_rows"] = _ints(_starts(kept)), _ints([0] * len(kept)), sum(kept)
    return s


# ---------------------------------------------------------------------------------------------- plain forms


def _segments(starts, n):
    """For each of n packed tokens: its sequence and its place in it."""
    at = torch.arange(n, device="cuda")
    seq = torch.bucketize(at, starts[1:].long(), right=True)
    return seq, at - starts.long()[seq]


def _prompt(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    (tq, heads, hd), (tk, kv, _) = q.shape, k.shape
    qs, ks = s["q_starts"].long(), s["k_starts"].long()
    q_seq, q_at = _segments(s["q_starts"], tq)
    k_seq, k_at = _segments(s["k_starts"], tk)
    q_at = q_at + ((ks[1:] - ks[:-1]) - (qs[1:] - qs[:-1]))[q_seq]  # the last query stands at the last key
    seen = (q_seq[:, None] == k_seq[None]) & (k_at[None] <= q_at[:, None])
    grouped = q.view(tq, kv, heads // kv, hd).permute(1, 2, 0, 3).reshape(kv, -1, hd)
    x = torch.bmm(grouped, k.permute(1, 2, 0)).mul_(hd**-0.5).view(heads, tq, tk)
    x.masked_fill_(~seen, float("-inf"))
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    out = torch.bmm(x.view(kv, -1, tk), v.permute(1, 0, 2)).view(heads, tq, hd)
    return {"out": (out / torch.where(total == 0, 1.0, total)).permute(1, 0, 2).half()}


def _values(q, scale):
    """[seqs][heads][tokens][head_dim] whole numbers and a scale for each 32 tokens -> the values they stand for."""
    return q.float() * scale.repeat_interleave(BLOCK, dim=2)[:, :, : q.shape[2], None]


def _rows(q, scale, starts, pos, n):
    """The values of packed rows: row i of sequence s is position pos[s] + i."""
    seq, at = _segments(starts, n)
    at = at + pos.long()[seq]
    return q[seq, :, at].float() * scale[seq, :, at // BLOCK][..., None]


def _put(x, starts, pos, most, q, scale):
    """New tokens x into one of the two halves of a cache, in place."""
    seqs, kv, ctx, hd = q.shape
    starts, pos = starts.long(), pos.long()
    count = starts[1:] - starts[:-1]
    first = pos // BLOCK
    blocks = (most + BLOCK - 1) // BLOCK + 1
    at = first[:, None] * BLOCK + torch.arange(blocks * BLOCK, device="cuda")  # [seqs][window]
    i = at - pos[:, None]
    new = (i >= 0) & (i < count[:, None])
    touched = new.view(seqs, blocks, BLOCK).any(-1)
    x = torch.where(new[..., None, None], x[(starts[:-1, None] + i).clamp(0, len(x) - 1)].float(), 0.0)  # [seqs][window][kv][hd]
    x = x.view(seqs, blocks, BLOCK, kv, hd)
    fresh = (x.abs().amax((2, 4)).double() / 127).float()  # [seqs][blocks][kv]
    block = (first[:, None] + torch.arange(blocks, device="cuda")).clamp_max(scale.shape[2] - 1)
    seq = torch.arange(seqs, device="cuda")
    held = scale[seq[:, None], :, block] * ((at[:, ::BLOCK] < pos[:, None]) & touched)[..., None]
    d = torch.maximum(fresh, held)
    d = torch.where(d < TINY, 0.0, d)
    by = torch.where(d == 0, 1.0, d).double()[:, :, None, :, None]
    put = torch.round(x.double() / by)
    old = q[seq[:, None], :, at.clamp_max(ctx - 1)].view(seqs, blocks, BLOCK, kv, hd).double()
    old = torch.round(old * held.double()[:, :, None, :, None] / by)
    keep = (at < pos[:, None]) & touched.repeat_interleave(BLOCK, 1)
    put = torch.where(new.view(seqs, blocks, BLOCK, 1, 1), put, old) * (d != 0)[:, :, None, :, None]
    put = put.clamp(-127, 127).to(torch.int8).view(seqs, blocks * BLOCK, kv, hd)
    s_at, w_at = torch.nonzero(new | keep, as_tuple=True)
    q[s_at, :, at[s_at, w_at]] = put[s_at, w_at]
    s_at, b_at = torch.nonzero(touched, as_tuple=True)
    scale[s_at, :, block[s_at, b_at]] = d[s_at, b_at]


def _append(s):
    out = {}
    for name in ("k", "v"):
        _put(s["new_" + name], s["starts"], s["pos"], s["most"], s[name], s[name + "_scale"])
        out[name] = _rows(s[name], s[name + "_scale"], s["back_starts"], s["back_pos"], s["back_rows"])
    return out


def _read(s):
    kind = torch.float16 if s["case"]["half"] else torch.float32
    return {n: _rows(s[n], s[n + "_scale"], s["starts"], s["pos"], s["rows"]).to(kind) for n in ("k", "v")}


def _step(s):
    q, lens = s["q"], s["len"]
    k = _values(s["k"], s["k_scale"])
    seqs, kv, ctx, hd = k.shape
    x = torch.matmul(q.view(seqs, kv, -1, hd), k.transpose(2, 3)).mul_(hd**-0.5)  # [seqs][kv][group][ctx]
    del k
    seen = (torch.arange(ctx, device="cuda") < lens[:, None])[:, None, None]
    x.masked_fill_(~seen, float("-inf"))
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    x.div_(torch.where(total == 0, 1.0, total))
    out = {"out": torch.matmul(x, _values(s["v"], s["v_scale"])).reshape(seqs, -1, hd)}
    if s["case"]["weights"]:
        out["weights"] = torch.where(seen[:, :, 0], s["weights"] + x.sum(2), 0.0)
    return out


def _evict(s):
    c, lens, w = s["case"], s["len"].long(), s["weights"]
    seqs, kv, ctx = w.shape
    budget, recent = c["budget"], c["recent"]
    at = torch.arange(ctx, device="cuda")
    # 0: kept for being new, 1: kept by weight, 2: no token
    rank = torch.where(at >= lens[:, None], 2, torch.where(at >= lens[:, None] - recent, 0, 1))[:, None].expand(seqs, kv, ctx)
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices
    order = order.gather(-1, torch.sort(rank.gather(-1, order), dim=-1, stable=True).indices)[..., :budget]
    count = lens.clamp_max(budget)
    row = torch.arange(budget, device="cuda")
    held = (row < count[:, None])[:, None].expand(seqs, kv, budget)
    index = torch.sort(torch.where(held, order, ctx), dim=-1).values
    src = index.clamp_max(ctx - 1)
    out = {"index": torch.where(held, index, -1).int(), "len": count.int(), "weights": torch.where(held, w.gather(-1, src), 0.0)}
    blocks = (budget + BLOCK - 1) // BLOCK
    pad = blocks * BLOCK - budget
    for name in ("k", "v"):
        d_old = torch.where(held, s[name + "_scale"].gather(-1, src // BLOCK), 0.0)
        d = torch.nn.functional.pad(d_old, (0, pad)).view(seqs, kv, blocks, BLOCK).amax(-1)
        d = torch.where(d < TINY, 0.0, d).repeat_interleave(BLOCK, -1)[..., :budget]
        q = s[name].gather(2, src[..., None].expand(-1, -1, -1, c["head_dim"])).double()
        q = torch.round(q * d_old.double()[..., None] / torch.where(d == 0, 1.0, d).double()[..., None])
        value = (q * (d != 0)[..., None]).float() * d[..., None]
        seq, place = _segments(s["kept_starts"], s["kept_rows"])
        out[name] = value[seq, :, place]
    return out


# ---------------------------------------------------------------------------------------------- the library's calls


@functools.lru_cache(None)
def _library():
    import galois_b200 as gb

    return gb, gb.Device.Gpu(gb.CudaDevice(0))


def _tensor(x):
    """A torch tensor as one of the library's, its dimensions in ggml order."""
    gb, place = _library()
    kind = {torch.float32: gb.GGmlType.F32, torch.float16: gb.GGmlType.F16, torch.int32: gb.GGmlType.I32, torch.int8: gb.GGmlType.I8}[x.dtype]
    return gb.Tensor(kind, gb.Dim.ggml(tuple(x.shape)[::-1], kind), x.view(-1), place)


def _handle(s):
    """The library's tensors of this state, made on its first pass and kept with it, as a program keeps them."""
    h = s.get("handle")
    if h is None:
        gb, _ = _library()
        c = s["case"]
        h = s["handle"] = {n: _tensor(x) for n, x in s.items() if isinstance(x, torch.Tensor)}
        new = lambda *shape, dtype=torch.float32: torch.zeros(shape, dtype=dtype, device="cuda")  # noqa: E731
        if c["op"] != "prompt":
            h["cache"] = gb.CacheQ8(h["k"], h["k_scale"], h["v"], h["v_scale"])
        if c["op"] == "prompt":
            out = {"out": torch.empty_like(s["q"])}
        elif c["op"] == "append":
            out = {n: new(s["back_rows"], c["kv_heads"], c["head_dim"]) for n in ("k", "v")}
        elif c["op"] == "read":
            out = {n: new(s["rows"], c["kv_heads"], c["head_dim"], dtype=torch.float16 if c["half"] else torch.float32) for n in ("k", "v")}
        elif c["op"] == "step":
            out = {"out": torch.empty_like(s["q"])}
            if c["weights"]:
                out["weights"] = torch.zeros_like(s["weights"])
            size = gb.galois_cache_attention_workspace(h["cache"], c["heads"], c["weights"])
            h["workspace"] = _tensor(torch.empty(size // 4, device="cuda"))
        else:
            rows = (c["seqs"], c["kv_heads"], c["budget"])
            out = {"index": new(*rows, dtype=torch.int32).fill_(-1), "len": new(c["seqs"], dtype=torch.int32), "weights": new(*rows)}
            out |= {n: new(s["kept_rows"], c["kv_heads"], c["head_dim"]) for n in ("k", "v")}
            blocks = (c["budget"] + BLOCK - 1) // BLOCK
            cut = [x for n in ("k", "v") for x in (new(*rows, c["head_dim"], dtype=torch.int8), new(*rows[:2], blocks))]
            h["cut"] = gb.CacheQ8(*(_tensor(x) for x in cut))
        h["out"], h["to"] = out, {n: _tensor(x) for n, x in out.items()}
    return h


def _call(s):
    gb, _ = _library()
    h, c = _handle(s), s["case"]
    to = h["to"]
    if c["op"] == "prompt":
        gb.galois_prompt_attention(h["q"], h["k"], h["v"], h["q_starts"], h["k_starts"], to["out"], c["head_dim"] ** -0.5)
    elif c["op"] == "append":
        gb.galois_cache_append(h["new_k"], h["new_v"], h["starts"], h["pos"], h["cache"])
        gb.galois_cache_read(h["cache"], h["back_starts"], h["back_pos"], to["k"], to["v"])
    elif c["op"] == "read":
        gb.galois_cache_read(h["cache"], h["starts"], h["pos"], to["k"], to["v"])
    elif c["op"] == "step":
        gb.galois_cache_attention(h["q"], h["cache"], h["len"], to["out"], c["head_dim"] ** -0.5, h["workspace"],
                                  weights=h.get("weights"), weights_out=to.get("weights"))
    else:
        gb.galois_cache_evict(h["cache"], h["len"], h["weights"], c["recent"], h["cut"], to["len"], to["weights"], to["index"])
        gb.galois_cache_read(h["cut"], h["kept_starts"], h["kept_pos"], to["k"], to["v"])
    return h["out"]


def run(state):
    if own:
        return _call(state)
    return {"prompt": _prompt, "append": _append, "read": _read, "step": _step, "evict": _evict}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    lens, hd, kv = _lengths(case), case["head_dim"], case["kv_heads"]
    if case["op"] == "prompt":
        pairs = sum(q * (k - q) + q * (q + 1) // 2 for q, k in zip(lens["q"], lens["k"]))
        return {"bytes": 2 * hd * (2 * case["heads"] * sum(lens["q"]) + 2 * kv * sum(lens["k"])), "flops": 4 * hd * case["heads"] * pairs}
    row = 2 * kv * hd  # values of a token's keys and values
    scales = lambda n: 2 * kv * 4 * ((n + BLOCK - 1) // BLOCK)  # noqa: E731
    if case["op"] == "append":
        size = 0
        for n, p in zip(lens["new"], lens["pos"]):
            old = p % BLOCK  # the tokens that share the first block are read and may be written
            size += row * n * ((2 if case["half"] else 4) + 1) + 2 * row * old + 2 * scales(n + old)
            size += row * (n + old) * 4 + row * (n + old)  # read back
        return {"bytes": size, "flops": 4 * row * sum(lens["new"])}
    if case["op"] == "read":
        n = sum(lens["rows"])
        return {"bytes": row * n * (1 + (2 if case["half"] else 4)) + sum(scales(r) for r in lens["rows"]), "flops": row * n}
    if case["op"] == "step":
        n = sum(lens["len"])
        size = row * n + sum(scales(r) for r in lens["len"]) + 8 * hd * case["heads"] * case["seqs"]
        return {"bytes": size + (8 * kv * n if case["weights"] else 0), "flops": 4 * hd * case["heads"] * n}
    n = sum(lens["len"])
    kept = sum(min(x, case["budget"]) for x in lens["len"])
    # weights once; kept rows and their scales in and out, then read back; indices and weights out
    return {"bytes": 4 * kv * n + row * kept * 2 + row * kept * 5 + sum(scales(x) for x in lens["len"]) + 2 * scales(kept) + 8 * kv * kept, "flops": kv * n + row * kept}


# ---------------------------------------------------------------------------------------------- in 64 bits


def _exact_put(x, new, pos, q, scale):
    """One half of a cache with the new tokens in it, sequence by sequence and block by block."""
    q, scale = q.double(), scale.clone()
    done = 0
    for s, (n, p) in enumerate(zip(new, pos)):
        rows = x[done : done + n].double()  # [n][kv][hd]
        done += n
        for b in range(p // BLOCK, (p + n - 1) // BLOCK + 1):
            lo, hi = max(p, b * BLOCK), min(p + n, (b + 1) * BLOCK)
            part = rows[lo - p : hi - p].transpose(0, 1)  # [kv][m][hd]
            d = (part.abs().amax((1, 2)) / 127).float()
            if lo > b * BLOCK:
                d = torch.maximum(d, scale[s, :, b])
                old = q[s, :, b * BLOCK : lo] * scale[s, :, b].double()[:, None, None]
                q[s, :, b * BLOCK : lo] = torch.nan_to_num((old / d.double()[:, None, None]).round())
            q[s, :, lo:hi] = torch.nan_to_num((part / d.double()[:, None, None]).round())
            scale[s, :, b] = d
    return q, scale


def _exact_rows(q, scale, rows, pos):
    out = []
    for s, (n, p) in enumerate(zip(rows, pos)):
        at = torch.arange(p, p + n, device="cuda")
        out.append((q[s][:, at].double() * scale[s][:, at // BLOCK].double()[..., None]).transpose(0, 1))
    return torch.cat(out)


def exact(case, seed):
    s, lens = prepare(case, seed), _lengths(case)
    scaling = case["head_dim"] ** -0.5
    if case["op"] == "prompt":
        group = case["heads"] // case["kv_heads"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        q0 = k0 = 0
        for n, m in zip(lens["q"], lens["k"]):
            past = torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1)
            for h in range(case["heads"]):
                x = s["q"][q0 : q0 + n, h].double() @ s["k"][k0 : k0 + m, h // group].double().T * scaling
                p = torch.softmax(x.masked_fill(past, float("-inf")), -1)
                out[q0 : q0 + n, h] = p @ s["v"][k0 : k0 + m, h // group].double()
            q0, k0 = q0 + n, k0 + m
        return {"out": out}
    if case["op"] == "append":
        out = {}
        for name in ("k", "v"):
            q, scale = _exact_put(s["new_" + name], lens["new"], lens["pos"], s[name], s[name + "_scale"])
            first = [p // BLOCK * BLOCK for p in lens["pos"]]
            out[name] = _exact_rows(q, scale, [p + n - f for p, n, f in zip(lens["pos"], lens["new"], first)], first)
        return out
    if case["op"] == "read":
        return {n: _exact_rows(s[n], s[n + "_scale"], lens["rows"], lens["pos"]) for n in ("k", "v")}
    if case["op"] == "step":
        kv, hd = case["kv_heads"], case["head_dim"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        weights = torch.zeros(case["seqs"], kv, case["ctx"], dtype=torch.float64, device="cuda")
        for i, n in enumerate(lens["len"]):
            if n == 0:
                continue
            by = torch.arange(n, device="cuda") // BLOCK
            k = s["k"][i, :, :n].double() * s["k_scale"][i][:, by].double()[..., None]
            v = s["v"][i, :, :n].double() * s["v_scale"][i][:, by].double()[..., None]
            p = torch.softmax(s["q"][i].double().view(kv, -1, hd) @ k.transpose(1, 2) * scaling, -1)
            out[i] = (p @ v).reshape(-1, hd)
            if case["weights"]:
                weights[i, :, :n] = s["weights"][i, :, :n].double() + p.sum(1)
        return {"out": out, "weights": weights} if case["weights"] else {"out": out}
    kv, budget, recent = case["kv_heads"], case["budget"], case["recent"]
    index = torch.full((case["seqs"], kv, budget), -1, dtype=torch.int32)
    weights = torch.zeros(case["seqs"], kv, budget, dtype=torch.float64)
    rows = {"k": [], "v": []}
    host = s["weights"].cpu()
    for i, n in enumerate(lens["len"]):
        m = min(n, budget)
        new = min(recent, m)
        kept = []
        for h in range(kv):
            w = host[i, h, : n - new].tolist()
            best = sorted(range(n - new), key=lambda j: (-w[j], j))[: m - new]
            kept.append(sorted(best) + list(range(n - new, n)))
        at = torch.tensor(kept)  # [kv][m]
        index[i, :, :m] = at.int()
        weights[i, :, :m] = host[i].gather(1, at).double()
        at = at.cuda()
        for name in ("k", "v"):
            d_old = s[name + "_scale"][i].gather(1, at // BLOCK).double()
            q = s[name][i].gather(1, at[..., None].expand(-1, -1, case["head_dim"])).double()
            for b in range(0, m, BLOCK):
                d = d_old[:, b : b + BLOCK].amax(1)[:, None, None]
                part = q[:, b : b + BLOCK]
                part.mul_(d_old[:, b : b + BLOCK, None]).div_(d).round_().mul_(d)
            rows[name].append(q.transpose(0, 1))
    return {"index": index, "len": torch.tensor([min(n, budget) for n in lens["len"]], dtype=torch.int32), "weights": weights,
            "k": torch.cat(rows["k"]), "v": torch.cat(rows["v"])}
