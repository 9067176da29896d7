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
from .op import _gpu_ctx, _want
from .tensor import Device, GError, GGmlType, Tensor, _check

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
        self._ref = C.byref(self._c)

    @staticmethod
    def zeros(head_dim: int, ctx: int, kv_heads: int, seqs: int, device: Device) -> "CacheQ8":
        rows = lambda: Tensor.zeros((head_dim, ctx, kv_heads, seqs), GGmlType.I8, device)  # noqa: E731
        scales = lambda: Tensor.zeros(((ctx + BLOCK - 1) // BLOCK, kv_heads, seqs), GGmlType.F32, device)  # noqa: E731
        return CacheQ8(rows(), scales(), rows(), scales())


# A serving loop makes these calls for a few microseconds of GPU work each, so their checks are written for the case that
# passes; whatever fails goes through the ones in op.py, which say why.
_F16, _F32, _I32 = GGmlType.F16, GGmlType.F32, GGmlType.I32


def _ctx_of(first: Tensor, *rest: Tensor):
    gpu = first.device.gpu
    if gpu is None:
        return _gpu_ctx(first, *rest)
    for t in rest:
        if t.device.gpu is not gpu:
            return _gpu_ctx(first, *rest)
    return gpu.ctx


def _ints(t: Tensor, n: int | None, what: str) -> int:
    """`t` as a row of at least n whole numbers (n None: how many it has)."""
    if t.dtype is not _I32:
        _want(t, _I32, what)
    d = t._dim
    have, *others = d.shape
    if d.stride[0] != 1 or others != [1, 1, 1]:
        raise GError(f"{what}: a contiguous row of i32 is wanted")
    if n is not None and have < n:
        raise GError(f"{what}: {have} numbers, {n} are wanted")
    return have


def galois_prompt_attention(q: Tensor, k: Tensor, v: Tensor, q_starts: Tensor, k_starts: Tensor, dst: Tensor, scale: float) -> None:
    """Causal attention of packed prompts: queries ``q_starts[s] .. q_starts[s + 1]`` of ``q`` see the keys
    ``k_starts[s] .. k_starts[s + 1]`` up to their own, the last query standing at the last key (so a sequence with more
    keys than queries continues earlier tokens).  q, dst {head_dim, heads, tokens}, k, v {head_dim, kv_heads, tokens}: F16, dst
    F16 or F32; head_dim 64 or 128; heads a multiple of kv_heads.  Queries without a key give zeros."""
    ctx = _ctx_of(q, k, v, q_starts, k_starts, dst)
    for t in (q, k, v):
        if t.dtype is not _F16:
            _want(t, _F16, "galois_prompt_attention")
    nseq = _ints(q_starts, None, "galois_prompt_attention q_starts") - 1
    _ints(k_starts, nseq + 1, "galois_prompt_attention k_starts")
    if nseq < 0:
        raise GError("galois_prompt_attention: starts hold one number more than there are sequences")
    if dst.dtype is _F16:
        fn = lib.galois_b200_prompt_attention_f16
    elif dst.dtype is _F32:
        fn = lib.galois_b200_prompt_attention_f16_f32
    else:
        raise GError(f"galois_prompt_attention: dst is {dst.dtype.name}, F16 and F32 are built")
    rc = fn(ctx, q.data_ptr(), q.c_dim(), k.data_ptr(), k.c_dim(), v.data_ptr(), v.c_dim(), q_starts.data_ptr(), k_starts.data_ptr(), nseq, dst.data_ptr(), dst.c_dim(), scale)
    _check(ctx, rc, "galois_prompt_attention")


def _rows(name: str, k: Tensor, v: Tensor, starts: Tensor, pos: Tensor) -> int:
    """Checks packed rows; how many sequences there are."""
    kind = k.dtype
    if v.dtype is not kind or (kind is not _F16 and kind is not _F32):
        raise GError(f"{name}: k and v must both be F16 or both F32, got {k.dtype.name} and {v.dtype.name}")
    nseq = _ints(starts, None, name + " starts") - 1
    if nseq < 0:
        raise GError(f"{name}: starts hold one number more than there are sequences")
    _ints(pos, nseq, name + " pos")
    return nseq


def galois_cache_append(k: Tensor, v: Tensor, starts: Tensor, pos: Tensor, cache: CacheQ8) -> None:
    """Rows ``starts[s] + i`` of k and v ({head_dim, kv_heads, tokens}, F32 or F16) become rows ``pos[s] + i`` of slot s of the
    cache.  A block of 32 rows takes the scale f32(max|x| / 127); rows it held before ``pos[s]`` are brought to it."""
    ctx = _ctx_of(cache.k, k, v, starts, pos)
    nseq = _rows("galois_cache_append", k, v, starts, pos)
    fn = lib.galois_b200_cache_append_f16 if k.dtype is _F16 else lib.galois_b200_cache_append_f32
    _check(ctx, fn(ctx, cache._ref, k.data_ptr(), k.c_dim(), v.data_ptr(), v.c_dim(), starts.data_ptr(), pos.data_ptr(), nseq), "galois_cache_append")


def galois_cache_read(cache: CacheQ8, starts: Tensor, pos: Tensor, k: Tensor, v: Tensor) -> None:
    """The values of rows ``pos[s] + i`` of slot s into rows ``starts[s] + i`` of k and v ({head_dim, kv_heads, tokens}, F32 or
    F16): what galois_get_rows is for a Q4_0 table."""
    ctx = _ctx_of(cache.k, k, v, starts, pos)
    nseq = _rows("galois_cache_read", k, v, starts, pos)
    fn = lib.galois_b200_cache_read_f16 if k.dtype is _F16 else lib.galois_b200_cache_read_f32
    _check(ctx, fn(ctx, cache._ref, starts.data_ptr(), pos.data_ptr(), nseq, k.data_ptr(), k.c_dim(), v.data_ptr(), v.c_dim()), "galois_cache_read")


def galois_cache_attention_workspace(cache: CacheQ8, heads: int, weights: bool = False) -> int:
    """Bytes of workspace that galois_cache_attention wants for `heads` query heads."""
    ctx = _ctx_of(cache.k)
    if not 0 <= heads <= 65535:  # the C argument has 32 bits
        raise GError(f"galois_cache_attention_workspace: {heads} heads")
    need = C.c_size_t()
    rc = lib.galois_b200_cache_attention_workspace_bytes(ctx, cache._ref, heads, 1 if weights else 0, C.byref(need))
    _check(ctx, rc, "galois_cache_attention_workspace")
    return need.value


def galois_cache_attention(q: Tensor, cache: CacheQ8, lens: Tensor, dst: Tensor, scale: float, workspace: Tensor, *, weights: Tensor | None = None,
                           weights_out: Tensor | None = None) -> None:
    """One query per slot over the first ``lens[s]`` rows of its cache.  q, dst F32 {head_dim, heads, seqs}; ``workspace``:
    galois_cache_attention_workspace bytes (any dtype, contents irrelevant; one for each call that may run at the
    same time).  With ``weights`` and ``weights_out`` (F32 {ctx, kv_heads, seqs}; they may be the same tensor) each row's
    probabilities, summed over the heads of its group, are added to its weight."""
    if weights is None and weights_out is None:
        f32 = (q, dst)
    else:
        f32 = tuple(t for t in (q, dst, weights, weights_out) if t is not None)
    ctx = _ctx_of(cache.k, lens, workspace, *f32)
    for t in f32:
        if t.dtype is not _F32:
            _want(t, _F32, "galois_cache_attention")
    _ints(lens, cache.seqs, "galois_cache_attention lens")
    size = workspace.room()
    if size < 0:
        raise GError("galois_cache_attention: the workspace must be contiguous")
    w = (None, None) if weights is None else (weights.data_ptr(), weights.c_dim())
    wo = (None, None) if weights_out is None else (weights_out.data_ptr(), weights_out.c_dim())
    rc = lib.galois_b200_cache_attention_f32(ctx, q.data_ptr(), q.c_dim(), cache._ref, lens.data_ptr(), dst.data_ptr(), dst.c_dim(), scale, *w, *wo, workspace.data_ptr(), size)
    _check(ctx, rc, "galois_cache_attention")


def galois_cache_evict(cache: CacheQ8, lens: Tensor, weights: Tensor, recent: int, out: CacheQ8, out_lens: Tensor, out_weights: Tensor,
                       index: Tensor) -> None:
    """Cuts every slot and head to the ``out.ctx`` rows of `out`: the last `recent` rows and, of the others, those of largest
    weight (equal: the lowest row), in their order.  ``index`` (I32 {out.ctx, kv_heads, seqs}) receives their old
    rows, ``out_weights`` their weights, ``out_lens`` the new lengths; what lies behind a new length is left as it was."""
    ctx = _ctx_of(cache.k, lens, weights, out.k, out_lens, out_weights, index)
    for t in (weights, out_weights):
        if t.dtype is not _F32:
            _want(t, _F32, "galois_cache_evict")
    if index.dtype is not _I32:
        _want(index, _I32, "galois_cache_evict index")
    _ints(lens, cache.seqs, "galois_cache_evict lens")
    _ints(out_lens, cache.seqs, "galois_cache_evict out_lens")
    if recent < 0:
        raise GError(f"galois_cache_evict: {recent} recent rows")
    recent = min(recent, out.ctx)  # no more are kept; the C argument has 32 bits
    rc = lib.galois_b200_cache_evict(ctx, cache._ref, lens.data_ptr(), weights.data_ptr(), weights.c_dim(), recent, out._ref, out_lens.data_ptr(), out_weights.data_ptr(),
                                     out_weights.c_dim(), index.data_ptr(), index.c_dim())
    _check(ctx, rc, "galois_cache_evict")
