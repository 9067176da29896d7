"""What the prompt-attention and 8-bit-cache entry points refuse, checked without a GPU: every check comes before the
first CUDA call, so a zeroed stand-in for the context and made-up addresses are enough."""
import ctypes as C

import numpy as np
import pytest

from galois_b200 import GError, GGmlType
from galois_b200._lib import GaloisCacheQ8, GaloisDim, lib

BADARG, SHAPE, LAYOUT, DST, BROADCAST, UNSUPPORTED, NOMEM, STATE = -1, -2, -3, -4, -5, -6, -8, -10


@pytest.fixture()
def ctx():
    return C.create_string_buffer(1 << 20)


def dim(shape, stride=None):
    d = GaloisDim()
    ne = list(shape) + [1] * (4 - len(shape))
    nb = [1]
    for n in ne[:3]:
        nb.append(nb[-1] * n)
    d.n_dims = len(shape)
    for i in range(4):
        d.ne[i], d.nb[i] = ne[i], (stride or nb)[i]
    return d


def addr(n):
    return C.c_void_p(n << 30)


def cache(hd=128, ctx=100, kv=2, seqs=3, **over):
    h = GaloisCacheQ8(1 << 40, 2 << 40, 3 << 40, 4 << 40, dim((hd, ctx, kv, seqs)), dim(((ctx + 31) // 32, kv, seqs)))
    for k, v in over.items():
        setattr(h, k, v)
    return h


def rows(hd=128, kv=2, tokens=5):
    return dim((hd, kv, tokens))


def append(ctx, h, kd=None, vd=None, k=addr(1), v=addr(2), starts=addr(3), pos=addr(4), nseq=3, fn="append_f32"):
    kd, vd = kd or rows(), vd or kd or rows()
    return getattr(lib, "galois_b200_cache_" + fn)(ctx, C.byref(h), k, C.byref(kd), v, C.byref(vd), starts, pos, nseq)


@pytest.mark.parametrize("h,code", [
    (cache(hd=96), UNSUPPORTED), (cache(hd=256), UNSUPPORTED), (cache(k=None), BADARG), (cache(v_scale=None), BADARG), (cache(k=(1 << 40) + 8), LAYOUT),
    (cache(v=(1 << 40) + 1024), LAYOUT), (cache(k_scale=(2 << 40) + 64), LAYOUT), (cache(sd=dim((3, 2, 3))), SHAPE), (cache(sd=dim((4, 2, 2))), SHAPE),
    (cache(qd=dim((128, 100, 2, 3), (1, 136, 13600, 27200))), LAYOUT), (cache(qd=dim((128, 100, 2, 3), (1, 128, 128, 25600))), LAYOUT),
    (cache(qd=dim((128, 100, 2, 3), (2, 256, 25600, 51200))), LAYOUT), (cache(qd=dim((128, -1, 2, 3))), BADARG),
    (cache(sd=dim((4, 2, 3), (1, 2, 8, 24))), LAYOUT),
])
def test_a_bad_cache_is_refused_by_every_entry_point(ctx, h, code):
    assert append(ctx, h) == code
    assert append(ctx, h, fn="append_f16") == code
    kd = rows()
    assert lib.galois_b200_cache_read_f32(ctx, C.byref(h), addr(3), addr(4), 3, addr(1), C.byref(kd), addr(2), C.byref(kd)) == code
    need = C.c_size_t()
    assert lib.galois_b200_cache_attention_workspace_bytes(ctx, C.byref(h), 4, 1, C.byref(need)) == code
    assert attend(ctx, h) == code
    assert evict(ctx, h) == code
    assert evict(ctx, cache(), out=h) == code


@pytest.mark.parametrize("change,code", [
    (dict(kd=rows(64)), SHAPE), (dict(kd=rows(kv=3)), SHAPE), (dict(vd=rows(tokens=4)), SHAPE), (dict(k=None), BADARG), (dict(starts=None), BADARG),
    (dict(pos=None), BADARG), (dict(nseq=4), SHAPE), (dict(nseq=-1), SHAPE), (dict(k=C.c_void_p((1 << 30) + 8)), LAYOUT),
    (dict(kd=dim((128, 2, 5), (1, 130, 260, 1300))), LAYOUT), (dict(kd=dim((128, 2, 5), (2, 256, 512, 2560))), LAYOUT),
    (dict(kd=dim((128, 2, 5), (1, 128, -256, 0))), BADARG), (dict(k=C.c_void_p(1 << 40)), BADARG), (dict(v=C.c_void_p(4 << 40)), BADARG),
    (dict(starts=C.c_void_p((3 << 30) + 2)), LAYOUT),
])
def test_append_refuses(ctx, change, code):
    assert append(ctx, cache(), **change) == code
    assert lib.galois_b200_last_error(ctx)


def test_nothing_to_do_is_no_error(ctx):
    none = rows(tokens=0)
    assert append(ctx, cache(), kd=none, k=None, v=None) == 0
    assert append(ctx, cache(), nseq=0, starts=None, pos=None) == 0
    assert append(ctx, cache(seqs=0), nseq=0) == 0
    d = dim((128, 0, 3))
    assert lib.galois_b200_cache_attention_f32(ctx, None, C.byref(d), C.byref(cache()), None, None, C.byref(d), 1.0, None, None, None, None, None, 0) == 0


@pytest.mark.parametrize("change,code", [
    (dict(k=C.c_void_p((1 << 40) + 256)), DST), (dict(k=addr(2)), DST), (dict(kd=dim((128, 2, 5), (1, 128, 128, 640))), DST), (dict(kd=rows(tokens=6), vd=rows()), SHAPE),
])
def test_read_refuses(ctx, change, code):
    kd = change.get("kd", rows())
    vd = change.get("vd", kd)
    for fn in (lib.galois_b200_cache_read_f32, lib.galois_b200_cache_read_f16):
        assert fn(ctx, C.byref(cache()), addr(3), addr(4), 3, change.get("k", addr(1)), C.byref(kd), addr(2), C.byref(vd)) == code


def attend(ctx, h, heads=4, **o):
    qd = o.get("qd", dim((128, heads, 3)))
    dd = o.get("dd", dim((128, heads, 3)))
    wd, wod = o.get("wd", dim((100, 2, 3))), o.get("wod", dim((100, 2, 3)))
    w, wo = o.get("w", None), o.get("wo", None)
    return lib.galois_b200_cache_attention_f32(ctx, o.get("q", addr(1)), C.byref(qd), C.byref(h), o.get("lens", addr(2)), o.get("dst", addr(3)), C.byref(dd), 1.0,
                                               w, C.byref(wd), wo, C.byref(wod), o.get("ws", addr(5)), o.get("size", 1 << 29))


@pytest.mark.parametrize("change,code", [
    (dict(heads=3), BROADCAST), (dict(qd=dim((64, 4, 3))), SHAPE), (dict(qd=dim((128, 4, 2)), dd=dim((128, 4, 2))), SHAPE), (dict(dd=dim((128, 2, 3))), SHAPE),
    (dict(q=None), BADARG), (dict(lens=None), BADARG), (dict(ws=None), BADARG), (dict(size=0), NOMEM), (dict(ws=C.c_void_p((5 << 30) + 4)), LAYOUT),
    (dict(qd=dim((128, 4, 3), (1, 129, 516, 1548))), LAYOUT), (dict(dd=dim((128, 4, 3), (1, 0, 512, 1536))), DST), (dict(dst=addr(1)), DST),
    (dict(dst=C.c_void_p((1 << 40) + 1024)), DST), (dict(w=addr(6)), BADARG), (dict(wo=addr(6)), BADARG), (dict(w=addr(6), wo=C.c_void_p((6 << 30) + 4)), DST),
    (dict(w=addr(6), wo=addr(7), wd=dim((99, 2, 3))), SHAPE), (dict(w=addr(6), wo=addr(7), wod=dim((100, 2, 3), (1, 0, 200, 600))), DST),
    (dict(w=addr(6), wo=addr(7), wd=dim((100, 2, 3), (2, 200, 400, 1200))), LAYOUT), (dict(w=addr(6), wo=addr(3)), DST), (dict(w=addr(3), wo=addr(7)), DST),
])
def test_cache_attention_refuses(ctx, change, code):
    assert attend(ctx, cache(), **change) == code


def evict(ctx, h, out=None, recent=4, **o):
    out = out or cache(ctx=40, k=5 << 40, v=6 << 40, k_scale=7 << 40, v_scale=8 << 40)
    wd, owd, idd = o.get("wd", dim((100, 2, 3))), o.get("owd", dim((40, 2, 3))), o.get("idd", dim((40, 2, 3)))
    return lib.galois_b200_cache_evict(ctx, C.byref(h), o.get("lens", addr(1)), o.get("w", addr(2)), C.byref(wd), recent, C.byref(out), o.get("ol", addr(3)),
                                       o.get("ow", addr(4)), C.byref(owd), o.get("index", addr(5)), C.byref(idd))


@pytest.mark.parametrize("change,code", [
    (dict(recent=-1), BADARG), (dict(out=cache(ctx=40)), DST), (dict(out=cache(seqs=2, k=5 << 40, v=6 << 40, k_scale=7 << 40, v_scale=8 << 40)), SHAPE),
    (dict(lens=None), BADARG), (dict(w=None), BADARG), (dict(index=None), BADARG), (dict(wd=dim((40, 2, 3))), SHAPE), (dict(idd=dim((41, 2, 3))), SHAPE),
    (dict(owd=dim((40, 2, 3), (1, 40, 40, 0))), DST), (dict(ol=addr(1)), DST), (dict(ow=addr(2)), DST), (dict(index=addr(4)), DST), (dict(ow=C.c_void_p((4 << 30) + 1)), LAYOUT),
    (dict(wd=dim((100, 2, 3), (2, 200, 400, 1200))), LAYOUT),
])
def test_evict_refuses(ctx, change, code):
    assert evict(ctx, cache(), **change) == code


def prompt(ctx, **o):
    qd = o.get("qd", dim((128, 4, 9)))
    kd, vd, dd = o.get("kd", dim((128, 2, 9))), o.get("vd", o.get("kd", dim((128, 2, 9)))), o.get("dd", qd)
    fn = lib.galois_b200_prompt_attention_f16_f32 if o.get("f32") else lib.galois_b200_prompt_attention_f16
    return fn(ctx, o.get("q", addr(1)), C.byref(qd), o.get("k", addr(2)), C.byref(kd), o.get("v", addr(3)), C.byref(vd), o.get("qs", addr(4)), o.get("ks", addr(4)),
              o.get("nseq", 2), o.get("dst", addr(5)), C.byref(dd), 1.0)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("change,code", [
    (dict(qd=dim((96, 4, 9))), UNSUPPORTED), (dict(kd=dim((64, 2, 9))), SHAPE), (dict(kd=dim((128, 3, 9))), BROADCAST), (dict(vd=dim((128, 2, 8))), SHAPE),
    (dict(dd=dim((128, 4, 8))), SHAPE), (dict(q=None), BADARG), (dict(qs=None), BADARG), (dict(nseq=-1), BADARG), (dict(q=C.c_void_p((1 << 30) + 8)), LAYOUT),
    (dict(qd=dim((128, 4, 9), (1, 132, 528, 4752))), LAYOUT), (dict(dst=addr(1)), DST), (dict(dst=addr(3)), DST), (dict(dst=addr(4)), DST),
    (dict(dd=dim((128, 4, 9), (1, 128, 0, 0))), DST), (dict(kd=dim((128, 0, 9))), BROADCAST), (dict(qd=dim((128, 4, 9, 2))), SHAPE),
])
def test_prompt_attention_refuses(ctx, f32, change, code):
    assert prompt(ctx, f32=f32, **change) == code


def test_no_context_is_a_status():
    d, h = rows(), cache()
    assert append(None, h) == STATE and attend(None, h) == STATE and evict(None, h) == STATE and prompt(None) == STATE
    assert lib.galois_b200_cache_read_f32(None, C.byref(h), None, None, 0, None, C.byref(d), None, C.byref(d)) == STATE


def test_cpu_tensors_are_refused():
    import galois_b200 as gb

    z = lambda *ne, t=GGmlType.F32: gb.Tensor.zeros(ne, t, gb.Device.Cpu())  # noqa: E731
    with pytest.raises(GError):
        gb.CacheQ8.zeros(128, 64, 2, 1, gb.Device.Cpu())
    h, i = z(128, 2, 4, t=GGmlType.F16), z(2, t=GGmlType.I32)
    with pytest.raises(GError):
        gb.galois_prompt_attention(h, h, h, i, i, h, 1.0)
    assert np.array_equal(z(4, t=GGmlType.I8).to_numpy(), np.zeros(4, np.int8))


def test_metadata_inside_what_is_written_is_refused(ctx):
    assert append(ctx, cache(), starts=C.c_void_p((1 << 40) + 64)) == BADARG
    assert append(ctx, cache(), pos=C.c_void_p((4 << 40) + 4)) == BADARG
    kd = rows()
    for a, b in ((1, 4), (3, 1), (2, 4), (3, 2)):  # starts, positions: in k, in k, in v, in v
        assert lib.galois_b200_cache_read_f32(ctx, C.byref(cache()), addr(a), addr(b), 3, addr(1), C.byref(kd), addr(2), C.byref(kd)) == DST


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf")])
def test_a_scale_that_is_not_finite_is_refused(ctx, scale):
    qd, kd, sd = dim((128, 4, 9)), dim((128, 2, 9)), dim((128, 4, 3))
    for fn in (lib.galois_b200_prompt_attention_f16, lib.galois_b200_prompt_attention_f16_f32):
        assert fn(ctx, addr(1), C.byref(qd), addr(2), C.byref(kd), addr(3), C.byref(kd), addr(4), addr(4), 2, addr(5), C.byref(qd), scale) == BADARG
    assert lib.galois_b200_cache_attention_f32(ctx, addr(1), C.byref(sd), C.byref(cache()), addr(2), addr(3), C.byref(sd), scale, None, None, None, None, addr(5), 1 << 29) == BADARG
