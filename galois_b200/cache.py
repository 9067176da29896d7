"""Attention of prompts, and the 8-bit key/value cache with its operators.

The reference composes attention from mat-muls and soft_max over an F16 cache (src/op.rs:3093-3111, 3216-3230) and
has none of these; they take and check their tensors like the ``galois_*`` functions in ``op.py`` and forward to one
``galois_b200_*`` entry point each.  A serving loop uses them together:

    galois_prompt_attention(q, k, v, starts, starts, out, scale)         # F16 q, k, v of the packed prompts
    galois_cache_append(k, v, starts, pos, cache)                        # their keys and values into the cache
    galois_cache_append(k1, v1, one_each, lens, cache)                   # then, per generated token:
    galois_cache_attention(q1, cache, lens_plus_1, out1, scale, ws)

with ``galois_cache_evict`` when a cache is full and ``galois_cache_read`` to continue a prompt behind cached tokens.
"""
from __future__ import annotations

import ctypes as C

from ._lib import GaloisCacheQ8, lib
from .tensor import Device, GError, GGmlType, Tensor, _check
from .op import _gpu_ctx, _p, _want

BLOCK = 32  # rows of a head that share a scale


class CacheQ8:
    """Keys and values of ``seqs`` sequences in 8 bits: row j of a head stands for ``k[j] * k_scale[j // 32]``.

    ``k``, ``v``: I8 {head_dim, ctx, kv_heads, seqs}; ``k_scale``, ``v_scale``: F32 {ceil(ctx / 32), kv_heads, seqs}.
    The two halves are laid out alike.  The tensors may be views; their storage must not move while the cache is used."""

    def __init__(self, k: Tensor, k_scale: Tensor, v: Tensor, v_scale: Tensor):
        _gpu_ctx(k, k_scale, v, v_scale)
        for t in (k, v):
            _want(t, GGmlType.I8, "CacheQ8")
        for t in (k_scale, v_scale):
            _want(t, GGmlType.F32, "CacheQ8 scale")
        for a, b in ((k, v), (k_scale, v_scale)):
            if tuple(a.dim().shape) != tuple(b.dim().shape) or tuple(a.dim().stride) != tuple(b.dim().stride):
                raise GError("CacheQ8: the keys and the values must be laid out alike")
        self.head_dim, self.ctx, self.kv_heads, self.seqs = k.dim().shape
        if tuple(k_scale.dim().shape) != ((self.ctx + BLOCK - 1) // BLOCK, self.kv_heads, self.seqs, 1):
            raise GError("CacheQ8: scales must be {ceil(ctx / 32), kv_heads, seqs}")
        self.k, self.k_scale, self.v, self.v_scale = k, k_scale, v, v_scale
        self.device = k.device
        self._c = GaloisCacheQ8(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), k.dim().c_struct(), k_scale.dim().c_struct())

    @staticmethod
    def zeros(head_dim: int, ctx: int, kv_heads: int, seqs: int, device: Device) -> "CacheQ8":
        rows = lambda: Tensor.zeros((head_dim, ctx, kv_heads, seqs), GGmlType.I8, device)  # noqa: E731
        scales = lambda: Tensor.zeros(((ctx + BLOCK - 1) // BLOCK, kv_heads, seqs), GGmlType.F32, device)  # noqa: E731
        return CacheQ8(rows(), scales(), rows(), scales())

    def _ref(self):
        return C.byref(self._c)


def _ctx_of(cache: CacheQ8, *tensors: Tensor):
    return _gpu_ctx(cache.k, *tensors)


def _ints(t: Tensor, n: int | None, what: str) -> int:
    """`t` as a row of at least n whole numbers (n None: how many it has)."""
    _want(t, GGmlType.I32, what)
    d = t.dim()
    if d.stride[0] != 1 or any(x != 1 for x in d.shape[1:]):
        raise GError(f"{what}: a contiguous row of i32 is wanted")
    if n is not None and d.shape[0] < n:
        raise GError(f"{what}: {d.shape[0]} numbers, {n} are wanted")
    return d.shape[0]


def galois_prompt_attention(q: Tensor, k: Tensor, v: Tensor, q_starts: Tensor, k_starts: Tensor, dst: Tensor, scale: float) -> None:
    """Causal attention of packed prompts: queries ``q_starts[s] .. q_starts[s + 1]`` of ``q`` see the keys
    ``k_starts[s] .. k_starts[s + 1]`` up to their own, the last query standing at the last key (so a sequence with more
    keys than queries continues earlier tokens).  q, dst {head_dim, heads, tokens}, k, v {head_dim, kv_heads, tokens}: F16, dst
    F16 or F32; head_dim 64 or 128; heads a multiple of kv_heads.  Queries without a key give zeros."""
    ctx = _gpu_ctx(q, k, v, q_starts, k_starts, dst)
    for t in (q, k, v):
        _want(t, GGmlType.F16, "galois_prompt_attention")
    nseq = _ints(q_starts, None, "galois_prompt_attention q_starts") - 1
    _ints(k_starts, nseq + 1, "galois_prompt_attention k_starts")
    if nseq < 0:
        raise GError("galois_prompt_attention: starts hold one number more than there are sequences")
    if dst.dtype == GGmlType.F16:
        fn = lib.galois_b200_prompt_attention_f16
    elif dst.dtype == GGmlType.F32:
        fn = lib.galois_b200_prompt_attention_f16_f32
    else:
        raise GError(f"galois_prompt_attention: dst is {dst.dtype.name}, F16 and F32 are built")
    rc = fn(ctx, _p(q), q.c_dim(), _p(k), k.c_dim(), _p(v), v.c_dim(), _p(q_starts), _p(k_starts), nseq, _p(dst), dst.c_dim(), scale)
    _check(ctx, rc, "galois_prompt_attention")


def _rows(ctx, name: str, cache: CacheQ8, k: Tensor, v: Tensor, starts: Tensor, pos: Tensor) -> tuple:
    if k.dtype not in (GGmlType.F16, GGmlType.F32) or v.dtype != k.dtype:
        raise GError(f"{name}: k and v must both be F16 or both F32, got {k.dtype.name} and {v.dtype.name}")
    nseq = _ints(starts, None, f"{name} starts") - 1
    if nseq < 0:
        raise GError(f"{name}: starts hold one number more than there are sequences")
    _ints(pos, nseq, f"{name} pos")
    return nseq, "f16" if k.dtype == GGmlType.F16 else "f32"


def galois_cache_append(k: Tensor, v: Tensor, starts: Tensor, pos: Tensor, cache: CacheQ8) -> None:
    """Rows ``starts[s] + i`` of k and v ({head_dim, kv_heads, tokens}, F32 or F16) become rows ``pos[s] + i`` of slot s of the
    cache.  A block of 32 rows takes the scale f32(max|x| / 127); rows it held before ``pos[s]`` are brought to it."""
    ctx = _ctx_of(cache, k, v, starts, pos)
    nseq, kind = _rows(ctx, "galois_cache_append", cache, k, v, starts, pos)
    fn = lib.galois_b200_cache_append_f16 if kind == "f16" else lib.galois_b200_cache_append_f32
    _check(ctx, fn(ctx, cache._ref(), _p(k), k.c_dim(), _p(v), v.c_dim(), _p(starts), _p(pos), nseq), "galois_cache_append")


def galois_cache_read(cache: CacheQ8, starts: Tensor, pos: Tensor, k: Tensor, v: Tensor) -> None:
    """The values of rows ``pos[s] + i`` of slot s into rows ``starts[s] + i`` of k and v ({head_dim, kv_heads, tokens}, F32 or
    F16): what galois_get_rows is for a Q4_0 table."""
    ctx = _ctx_of(cache, k, v, starts, pos)
    nseq, kind = _rows(ctx, "galois_cache_read", cache, k, v, starts, pos)
    fn = lib.galois_b200_cache_read_f16 if kind == "f16" else lib.galois_b200_cache_read_f32
    _check(ctx, fn(ctx, cache._ref(), _p(starts), _p(pos), nseq, _p(k), k.c_dim(), _p(v), v.c_dim()), "galois_cache_read")


def galois_cache_attention_workspace(cache: CacheQ8, heads: int, weights: bool = False) -> int:
    """Bytes of workspace that galois_cache_attention wants for `heads` query heads."""
    ctx = _ctx_of(cache)
    need = C.c_size_t()
    rc = lib.galois_b200_cache_attention_workspace_bytes(ctx, cache._ref(), heads, 1 if weights else 0, C.byref(need))
    _check(ctx, rc, "galois_cache_attention_workspace")
    return need.value


def galois_cache_attention(q: Tensor, cache: CacheQ8, lens: Tensor, dst: Tensor, scale: float, workspace: Tensor, *, weights: Tensor | None = None,
                           weights_out: Tensor | None = None) -> None:
    """One query per slot over the first ``lens[s]`` rows of its cache.  q, dst F32 {head_dim, heads, seqs}; ``workspace``:
    galois_cache_attention_workspace bytes (any dtype, contents irrelevant; one for each call that may run at the
    same time).  With ``weights`` and ``weights_out`` (F32 {ctx, kv_heads, seqs}; they may be the same tensor) each row's
    probabilities, summed over the heads of its group, are added to its weight."""
    given = [t for t in (weights, weights_out) if t is not None]
    ctx = _ctx_of(cache, q, lens, dst, workspace, *given)
    for t in (q, dst, *given):
        _want(t, GGmlType.F32, "galois_cache_attention")
    _ints(lens, cache.seqs, "galois_cache_attention lens")
    if not workspace.dim().ggml_is_contiguous():
        raise GError("galois_cache_attention: the workspace must be contiguous")
    size = workspace.dim().elem_count() * workspace.storage.element_size()
    w = (None, None) if weights is None else (_p(weights), weights.c_dim())
    wo = (None, None) if weights_out is None else (_p(weights_out), weights_out.c_dim())
    rc = lib.galois_b200_cache_attention_f32(ctx, _p(q), q.c_dim(), cache._ref(), _p(lens), _p(dst), dst.c_dim(), scale, *w, *wo, _p(workspace), size)
    _check(ctx, rc, "galois_cache_attention")


def galois_cache_evict(cache: CacheQ8, lens: Tensor, weights: Tensor, recent: int, out: CacheQ8, out_lens: Tensor, out_weights: Tensor,
                       index: Tensor) -> None:
    """Cuts every slot and head to the ``out.ctx`` rows of `out`: the last `recent` rows and, of the others, those of largest
    weight (equal: the lowest row), in their order.  ``index`` (I32 {out.ctx, kv_heads, seqs}) receives their old
    rows, ``out_weights`` their weights, ``out_lens`` the new lengths; what lies behind a new length is left as it was."""
    ctx = _ctx_of(cache, lens, weights, out.k, out_lens, out_weights, index)
    for t in (weights, out_weights):
        _want(t, GGmlType.F32, "galois_cache_evict")
    _want(index, GGmlType.I32, "galois_cache_evict index")
    _ints(lens, cache.seqs, "galois_cache_evict lens")
    _ints(out_lens, cache.seqs, "galois_cache_evict out_lens")
    rc = lib.galois_b200_cache_evict(ctx, cache._ref(), _p(lens), _p(weights), weights.c_dim(), recent, out._ref(), _p(out_lens), _p(out_weights),
                                     out_weights.c_dim(), _p(index), index.c_dim())
    _check(ctx, rc, "galois_cache_evict")
