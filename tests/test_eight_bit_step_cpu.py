"""Host-side checks of the 8-bit decoder-step entry points: they refuse bad arguments with a status
and a message before they touch a device (every pointer here is made up or NULL)."""
import ctypes as C

import pytest

FAKE = 1 << 20  # never dereferenced: each call fails in its checks


def tensor(capi, dtype, shape, data=FAKE):
    return capi.Desc(data, dtype, shape)


def cache_of(capi, dtype=None, k=(4, 2, 16, 64), v=None, ks=(4, 2), table=(3, 2), lengths=(3,),
             table_dtype=None):
    dtype = capi.INT8 if dtype is None else dtype
    ds = [tensor(capi, dtype, k), tensor(capi, dtype, v or k), tensor(capi, capi.FLOAT, ks),
          tensor(capi, capi.FLOAT, ks), tensor(capi, table_dtype or capi.INT32, table),
          tensor(capi, capi.INT32, lengths)]
    return capi.B2QuantizedCache(*[C.pointer(d.t) for d in ds]), ds


def test_norm_arguments(b2):
    from onnx_light_b200 import _capi as c
    f = c.lib().b2_rms_normalization_quantize
    x, w = tensor(c, c.FLOAT16, (4, 64)), tensor(c, c.FLOAT16, (64,))
    y, s = tensor(c, c.INT8, (4, 64)), tensor(c, c.FLOAT, (4, 1))
    assert f(None, None, w.ref, 1e-5, 0, y.ref, s.ref, None, None) == c.B2_ERR_INVALID_ARGUMENT
    cases = [
        (dict(x=tensor(c, c.INT32, (4, 64))), "X must be"),
        (dict(w=tensor(c, c.FLOAT16, (63,))), "scale must have"),
        (dict(y=tensor(c, c.UINT8, (4, 64))), "Y must be"),
        (dict(y=tensor(c, c.INT8, (4, 32))), "Y must be"),
        (dict(s=tensor(c, c.FLOAT, (4, 2))), "Y_scale must be"),
        (dict(s=tensor(c, c.FLOAT16, (4, 1))), "Y_scale must be"),
        (dict(group=24), "group_size"), (dict(group=-1), "group_size"),
        (dict(res=tensor(c, c.FLOAT16, (4, 32))), "residual"),
        (dict(sum=tensor(c, c.FLOAT, (4, 64))), "sum"),
        (dict(x=tensor(c, c.FLOAT16, (4, 64), 0)), "no data"),
    ]
    for change, message in cases:
        a = dict(x=x, w=w, y=y, s=s, group=0, res=None, sum=None) | change
        with pytest.raises(ValueError, match=message):
            c.check(f(a["x"].ref, a["res"].ref if a["res"] else None, a["w"].ref, 1e-5, a["group"],
                      a["y"].ref, a["s"].ref, a["sum"].ref if a["sum"] else None, None))


def test_product_arguments(b2):
    from onnx_light_b200 import _capi as c
    f = c.lib().b2_scaled_matmul
    base = dict(a=(c.INT8, (4, 64)), sa=(c.FLOAT, (4,)), w=(c.INT8, (8, 64)), sw=(c.FLOAT, (8,)),
                y=(c.FLOAT16, (4, 8)))
    cases = [
        (dict(w=(c.FLOAT8E4M3FN, (8, 64))), "one dtype"), (dict(a=(c.UINT8, (4, 64))), "one dtype"),
        (dict(w=(c.INT8, (64, 8))), r"\[N, K\]"), (dict(sa=(c.FLOAT, (5,))), "A_scale"),
        (dict(sw=(c.FLOAT, (7,))), "W_scale"), (dict(sw=(c.FLOAT16, (8,))), "scales must be FLOAT"),
        (dict(y=(c.FLOAT16, (4, 9))), "Y must be"), (dict(y=(c.INT32, (4, 8))), "Y must be"),
    ]
    for change, message in cases:
        d = {k: tensor(c, *v) for k, v in (base | change).items()}
        with pytest.raises(ValueError, match=message):
            c.check(f(d["a"].ref, d["sa"].ref, d["w"].ref, d["sw"].ref, d["y"].ref, None, None, None))
    assert f(None, None, None, None, None, None, None, None) == c.B2_ERR_INVALID_ARGUMENT
    d = {k: tensor(c, *v) for k, v in (base | dict(a=(c.INT8, (4, 1 << 17)), w=(c.INT8, (8, 1 << 17)))).items()}
    with pytest.raises(c.UnsupportedOnGpu, match="K above"):
        c.check(f(d["a"].ref, d["sa"].ref, d["w"].ref, d["sw"].ref, d["y"].ref, None, None, None))


CACHE_FAULTS = [
    (dict(k=(4, 2, 16)), "must be"), (dict(v=(4, 2, 16, 32)), "one shape"), (dict(dtype=2), "INT8 or FLOAT8E4M3FN"),
    (dict(ks=(4, 3)), "cache scales"), (dict(table_dtype=7), "block_table"), (dict(table=(6,)), "block_table"),
    (dict(lengths=(2,)), "lengths"), (dict(k=(4, 0, 16, 64), ks=(4, 0)), "empty dimension"),
]


def test_append_arguments(b2):
    from onnx_light_b200 import _capi as c
    f = c.lib().b2_kv_cache_append
    kv = tensor(c, c.FLOAT16, (3, 2, 1, 64))
    for change, message in CACHE_FAULTS:
        cache, keep = cache_of(c, **change)
        with pytest.raises(ValueError, match=message):
            c.check(f(kv.ref, kv.ref, C.byref(cache), None, None))
    cache, keep = cache_of(c)
    for shape, dtype, message in (((3, 1, 1, 64), c.FLOAT16, "do not fit"), ((3, 1, 127), c.FLOAT16, "do not fit"),
                                  ((3, 64), c.FLOAT16, "must be"), ((3, 2, 1, 64), c.INT8, "K and V must be")):
        bad = tensor(c, dtype, shape)
        with pytest.raises(ValueError, match=message):
            c.check(f(bad.ref, bad.ref, C.byref(cache), None, None))
    counts = tensor(c, c.INT32, (2,))
    with pytest.raises(ValueError, match="new_lengths"):
        c.check(f(kv.ref, kv.ref, C.byref(cache), counts.ref, None))
    assert f(kv.ref, kv.ref, None, None, None) == c.B2_ERR_INVALID_ARGUMENT
    huge, keep = cache_of(c, k=(1 << 30, 2, 16, 64), ks=(1 << 30, 2))
    with pytest.raises(c.UnsupportedOnGpu, match="too large"):
        c.check(f(kv.ref, kv.ref, C.byref(huge), None, None))


def test_attention_arguments(b2):
    from onnx_light_b200 import _capi as c
    f = c.lib().b2_cache_attention
    q = tensor(c, c.FLOAT16, (3, 4, 1, 64))
    ok = c.B2CacheAttentionAttrs(0, 0.0, 1, 0.0, -1, 0)
    for change, message in CACHE_FAULTS:
        cache, keep = cache_of(c, **change)
        with pytest.raises(ValueError, match=message):
            c.check(f(q.ref, C.byref(cache), None, C.byref(ok), q.ref, None, None, None))
    cache, keep = cache_of(c)
    attrs = c.B2CacheAttentionAttrs
    for query, out, at, message in (
            (tensor(c, c.FLOAT, (3, 4, 1, 64)), None, ok, "FLOAT16 or BFLOAT16"),
            (tensor(c, c.FLOAT16, (3, 3, 1, 64)), None, ok, "multiple"),
            (tensor(c, c.FLOAT16, (2, 4, 1, 64)), None, ok, "batch"),
            (tensor(c, c.FLOAT16, (3, 4, 1, 32)), None, ok, "head_size"),
            (tensor(c, c.FLOAT16, (3, 1, 100)), None, ok, "head_size"),
            (q, tensor(c, c.BFLOAT16, (3, 4, 1, 64)), ok, "Y must have"),
            (q, None, attrs(0, 0.0, 1, 0.0, -2, 0), "left_window_size"),
            (q, None, attrs(0, 0.0, 0, 0.0, 5, 0), "needs is_causal"),
            (q, None, attrs(0, 0.0, 1, 0.0, 5, -1), "sink_tokens")):
        y = out or query
        with pytest.raises(ValueError, match=message):
            c.check(f(query.ref, C.byref(cache), None, C.byref(at), y.ref, None, None, None))
    big, keep = cache_of(c, k=(4, 2, 16, 576))
    with pytest.raises(c.UnsupportedOnGpu, match="head sizes"):
        wide = tensor(c, c.FLOAT16, (3, 4, 1, 576))
        c.check(f(wide.ref, C.byref(big), None, C.byref(ok), wide.ref, None, None, None))


def test_operators_are_registered(b2):
    from onnx_light_b200 import dispatch as d
    t = b2.RegisterB200KernelFunctions(b2.KernelDispatchTable(), num_gpus=1)
    for op in ("RMSNormalizationQuantize", "ScaledMatMul", "KVCacheAppend", "QuantizedCacheAttention"):
        assert t.resolve("b200", op, d.DEVICE_GPU0) is getattr(b2, op)
