"""The operators of a decoder step with 8-bit activations and cache at the ends of their ranges:
scales that are not finite, very large or subnormal, mis-declared buffers, large batches.

Tolerances are those of test_gpu_eight_bit_step, or derived at the test.
"""
import math

import pytest
import torch

from test_gpu_eight_bit_step import (QMAX, TYPES, assert_codes, check_attention,  # noqa: F401
                                     clean_status, gen, half_step, kind_of, make_cache, reference,
                                     storage, values)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# Scales that are not finite
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("name", ["k_scale", "v_scale"])
@pytest.mark.parametrize("rows", [1, 3, 160])
@pytest.mark.parametrize("head,page", [(128, 16), (64, 64), (40, 10)])
def test_attention_scales_not_finite_reach_only_what_sees_them(b2, head, page, rows, name, value):
    """A page whose scale is NaN or infinite (its codes are zeros then, as the append leaves them)
    makes the queries that see it NaN and no other."""
    total, window = 400 + rows, 60
    q = torch.randn(1, 2, rows, head, generator=gen(5), device="cuda").half()
    attrs = b2.CacheAttributes(left_window_size=window, sink_tokens=3)
    for block in (300 // page, (total - 1) // page):  # before every window; the last token's
        cache = make_cache(b2, "fp8", [total], [0], 1, head, page, seed=12)
        cache.lengths.fill_(400)
        clean, _ = reference(cache, q, [rows], window=window, sinks=3)
        at = int(cache.block_table[0, block])
        getattr(cache, name)[at] = value
        if math.isinf(value):
            getattr(cache, name[0])[at] = 0
        y = b2.QuantizedCacheAttention()(q, cache, attrs)
        first = rows if block == 300 // page else max(0, block * page - 400)  # that sees the page
        assert bool(torch.isnan(y[:, :, first:]).all())
        assert bool(torch.isfinite(y[:, :, :first]).all())
        if first:
            err, size = (y.double() - clean)[:, :, :first].norm(), clean[:, :, :first].norm()
            assert float(err / size) < 2e-3


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("rows", [12, 300])
def test_prompt_with_a_value_not_finite(b2, rows, value, codes):
    """One value of a prompt's last page is not finite: earlier queries do not notice."""
    x = torch.randn(2, 1, 2, rows, 128, generator=gen(rows), device="cuda").half()
    q = torch.randn(1, 8, rows, 128, generator=gen(1), device="cuda").half()
    ys = []
    for bad in (False, True):
        cache = b2.QuantizedKVCache.allocate(1, 2, rows, 128, page_size=16, dtype=kind_of(b2, codes))
        v = x[1].clone()
        if bad:
            v[0, 1, rows - 1, 7] = value
        b2.KVCacheAppend()(x[0], v, cache)
        ys.append(b2.QuantizedCacheAttention()(q, cache))
    first = (rows - 1) // 16 * 16  # the first query that sees the last page
    assert torch.equal(ys[0][:, :, :first], ys[1][:, :, :first])
    assert torch.equal(ys[0][:, :4], ys[1][:, :4])  # the other KV head's
    assert bool(torch.isnan(ys[1][:, 4:, first:]).all())


# ---------------------------------------------------------------------------
# Buffers declared larger than they are, or off their type's boundary
# ---------------------------------------------------------------------------


def test_declared_types_must_fit_the_storage(b2):
    """A QTensor's storage is measured by its declared type, and must start on that type's boundary."""
    f16, f32 = 10, 1
    raw = torch.zeros(2 * 64, dtype=torch.uint8, device="cuda")
    small16, small32 = b2.QTensor(raw, f16, (2, 64)), b2.QTensor(raw, f32, (2, 64))
    x, w = torch.zeros(2, 64, device="cuda").half(), torch.ones(64, device="cuda").half()
    norm, mm = b2.RMSNormalizationQuantize(), b2.ScaledMatMul()
    for args, kw in (((small16, w), {}), ((x, w), {"residual": small16}), ((x, w), {"out_sum": small16}),
                     ((x, b2.QTensor(raw[:64], f16, (64,))), {}),
                     ((x, w), {"out_scale": b2.QTensor(raw[:7], f32, (2, 1))})):
        with pytest.raises(ValueError, match="storage is smaller"):
            norm(*args, **kw)
    a = torch.zeros(2, 64, dtype=torch.int8, device="cuda")
    one = torch.ones(1, device="cuda")
    with pytest.raises(ValueError, match="storage is smaller"):
        mm(a, b2.QTensor(raw[:2], f32, (2,)), a, one)
    with pytest.raises(ValueError, match="storage is smaller"):
        mm(a, one, a, one, out=b2.QTensor(raw[:4], f16, (2, 2)))
    cache = b2.QuantizedKVCache.allocate(1, 1, 32, 64, page_size=16)
    kv = torch.zeros(1, 1, 2, 64, device="cuda").half()
    small = b2.QTensor(raw, f16, (1, 1, 2, 64))
    for k, v in ((small, kv), (kv, small), (b2.QTensor(raw, f32, (1, 1, 2, 64)), kv)):
        with pytest.raises(ValueError, match="storage is smaller"):
            b2.KVCacheAppend()(k, v, cache)
    with pytest.raises(ValueError, match="storage is smaller"):
        b2.KVCacheAppend()(kv, kv, cache, new_lengths=b2.QTensor(raw[:1], 6, (1,)))
    with pytest.raises(ValueError, match="storage is smaller"):
        b2.QuantizedCacheAttention()(small, cache)
    with pytest.raises(ValueError, match="storage is smaller"):
        b2.QuantizedCacheAttention()(kv, cache, out=small)
    with pytest.raises(ValueError, match="storage is smaller"):
        norm(small32, torch.ones(64, device="cuda"))
    # a shape whose count passes 64 bits
    with pytest.raises(ValueError, match="storage is smaller"):
        norm(b2.QTensor(raw, f16, (1 << 32, 1 << 32)), w)
    # off the boundary of its type
    odd = torch.zeros(4 * 64 + 1, dtype=torch.uint8, device="cuda")[1:]
    with pytest.raises(ValueError, match="boundary"):
        norm(b2.QTensor(odd, f16, (2, 64)), w)
    with pytest.raises(ValueError, match="boundary"):
        b2.KVCacheAppend()(b2.QTensor(odd, f16, (1, 1, 2, 64)), kv, cache)
    # a type that has no size
    with pytest.raises(ValueError, match="dtype"):
        norm(b2.QTensor(raw, 8, (2, 64)), w)
    # what fits and lies right runs
    y = mm(a, b2.QTensor(one.view(torch.uint8), f32, (1,)), b2.QTensor(a.view(torch.uint8), b2.INT8, (2, 64)), one)
    assert y.shape == (2, 2)


# ---------------------------------------------------------------------------
# Subnormal values: the scale is a few units of 2^-149
# ---------------------------------------------------------------------------


def units(g, *shape):
    """Whole multiples of 2^-149 up to 700 of either sign, as FLOAT."""
    n = torch.randint(0, 701, shape, generator=g, device="cuda", dtype=torch.int32)
    sign = torch.randint(0, 2, shape, generator=g, device="cuda", dtype=torch.int32) * -(1 << 31)
    return (n | sign).view(torch.float32)


UNIT_F32 = 2.0 ** -149


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("head", [64, 33])
def test_append_subnormal_values(b2, head, codes):
    """The stored scale is a / 127 or 448 rounded to whole units of 2^-149, so quotients pass 127 by
    up to a half: codes stay at the largest one and keep their sign."""
    cache = b2.QuantizedKVCache.allocate(40, 1, 8, head, page_size=8, dtype=kind_of(b2, codes))
    top = torch.randint(20, 701, (40, 1, 1, 1), generator=gen(head), device="cuda", dtype=torch.int32)
    bits = units(gen(head + 1), 40, 1, 8, head).view(torch.int32)
    x = ((bits & 0x7fffffff) % top + 1 | bits & -(1 << 31)).view(torch.float32)
    b2.KVCacheAppend()(x, x, cache)
    for pool, sc in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        s = sc[:, 0].double()
        assert bool(((s - x.double().abs().amax((1, 2, 3)) / QMAX[codes]).abs() <= 0.5 * UNIT_F32).all())
        want = torch.nan_to_num(x.double() / s[:, None, None, None], nan=0.0, posinf=0.0, neginf=0.0)
        assert_codes(pool, want, codes, slack=1e-6)


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("width,group", [(256, 0), (256, 64), (240, 24), (99, 0), (99, 9)])
def test_norm_subnormal_weights(b2, width, group, codes):
    """n = h / rms * w with w of a few hundred units u = 2^-149.  The kernel rounds n to units twice
    (the second after a factor below 2): within 1.5 u and 2^-20 of it; the scale once more, within
    0.6 u; a code is off by half a step and what 1.5 u make in units of the stored scale."""
    x = torch.randn(64, width, generator=gen(width), device="cuda")
    w = units(gen(width + 1), width)
    r = b2.RMSNormalizationQuantize()(x, w, dtype=kind_of(b2, codes), group_size=group)
    h = x.double()
    n = (h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-5) * w.double()).view(64, -1, group or width)
    s = r.Y_scale.double().view(64, -1)
    assert bool(((s - n.abs().amax(-1) / QMAX[codes]).abs() <= 0.6 * UNIT_F32 + 2e-6 * s).all())
    live = s > 0
    want = (n / s[..., None].clamp(min=UNIT_F32)).clamp(-QMAX[codes], QMAX[codes])
    c = values(storage(r.Y)).view(n.shape)
    bound = half_step(want.abs() + 2, codes) * 1.001 + 1.5 * UNIT_F32 / s[..., None].clamp(min=UNIT_F32) + 1e-3
    assert bool(((c - want).abs() <= bound)[live].all())
    assert float(c[~live].abs().sum()) == 0 and bool(live.any())


# ---------------------------------------------------------------------------
# Value scales near the top of the range
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("rows", [1, 6, 140])
@pytest.mark.parametrize("head,page", [(128, 16), (64, 32), (256, 16), (40, 10)])
def test_attention_large_value_scales(b2, head, page, rows):
    """Values up to 8e37, also beside pages of values 2^90 below: sums of products stay finite."""
    cache = make_cache(b2, "int8", [500 + rows], [0], 1, head, page, seed=8)
    cache.lengths.fill_(500)
    pages = cache.block_table[0].long()
    pages = pages[pages < cache.v_scale.shape[0]]
    q = torch.randn(1, 4, rows, head, generator=gen(3), device="cuda").bfloat16()
    ordinary = cache.v_scale[pages]
    cache.v_scale[pages] = ordinary * 2.0 ** 124  # 2^117 to 2^119
    check_attention(b2, cache, q)
    cache.v_scale[pages[1::3]] = ordinary[1::3] * 2.0 ** 34
    check_attention(b2, cache, q)


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("rows", [1, 6, 140])
@pytest.mark.parametrize("head,page", [(128, 16), (64, 32), (256, 16), (40, 10)])
def test_attention_of_values_near_the_largest(b2, head, page, rows, codes):
    """Values of 1e38 to 3e38, as the append quantizes them: their mean is as large, their sum is not
    a FLOAT any more."""
    total = 300 + rows
    cache = b2.QuantizedKVCache.allocate(1, 1, total, head, page, kind_of(b2, codes))
    k = torch.randn(1, 1, total, head, generator=gen(1), device="cuda").bfloat16()
    v = ((1 + 2 * torch.rand(1, 1, total, head, generator=gen(2), device="cuda")) * 1e38).bfloat16()
    b2.KVCacheAppend()(k, v, cache)
    cache.lengths.fill_(300)
    check_attention(b2, cache, torch.randn(1, 4, rows, head, generator=gen(3), device="cuda").bfloat16())


# ---------------------------------------------------------------------------
# Large batches: the split kernel's ways to share the keys out
# ---------------------------------------------------------------------------


def many_sequences(b2, batch, Hkv, Hq, rows, head, page, longest, codes, seed):
    """Short sequences of different lengths, some without new tokens or with nothing before them."""
    g = gen(seed)
    past = torch.randint(0, longest + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
    past[torch.rand(batch, generator=g, device="cuda") < 0.2] = 0
    past[batch // 2] = longest
    new = torch.randint(0, rows + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
    new[batch - 1] = rows
    per = -(-(longest + rows) // page)
    pages = batch * per
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).view(batch, per)
    cache = b2.QuantizedKVCache.allocate(batch, Hkv, per * page, head, page, kind_of(b2, codes), pages=pages,
                                         block_table=order)
    for pool in (cache.k, cache.v):
        v = torch.randn(pool.shape, generator=g, device="cuda") * (40.0 if codes == "int8" else 120.0)
        pool.copy_(v.round().clamp(-127, 127) if codes == "int8" else
                   v.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8))
    for sc in (cache.k_scale, cache.v_scale):
        sc.copy_(torch.rand(sc.shape, generator=g, device="cuda") * 0.02 + 0.01)
    cache.lengths.copy_(past)
    q = torch.randn(batch, Hq, rows, head, generator=g, device="cuda").half()
    return cache, q, new


def check_many(b2, cache, q, new, window=-1, sinks=0):
    batch, Hq, rows, head = q.shape
    Hkv, page = cache.k.shape[1:3]
    sides = []
    for pool, sc in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        ids = cache.block_table.long()
        v = values(pool[ids]) * sc[ids].double()[..., None, None]
        sides.append(v.transpose(1, 2).reshape(batch, Hkv, -1, head))
    k, v = sides
    at = torch.arange(rows, device="cuda")
    j = torch.arange(k.shape[2], device="cuda")
    p = (cache.lengths[:, None] + at)[:, None, :, None]
    seen = (j <= p) & (at < new[:, None])[:, None, :, None]
    if window >= 0:
        seen = seen & ((p - j <= window) | (j < sinks))
    z = (q.double().view(batch, Hkv, -1, head) @ k.transpose(-1, -2)).view(batch, Hq, rows, -1) / math.sqrt(head)
    prob = torch.nan_to_num(torch.softmax(z.masked_fill(~seen, -math.inf), -1), nan=0.0).view(batch, Hkv, -1, len(j))
    want, size = (prob @ x for x in (v, v.abs()))
    y = b2.QuantizedCacheAttention()(q, cache, b2.CacheAttributes(left_window_size=window, sink_tokens=sinks),
                                     new_lengths=new)
    err = (y.double().view_as(want) - want).abs()
    limit = 2.0 ** -11 * want.abs() * 1.001 + (2.0 ** -11 + 3e-4) * size + 2.0 ** -25
    assert bool((err <= limit).all()), float((err / limit).max())
    assert torch.equal(y, b2.QuantizedCacheAttention()(
        q, cache, b2.CacheAttributes(left_window_size=window, sink_tokens=sinks), new_lengths=new))


MANY = [  # batch, KV heads, query heads, rows, head, page, longest
    (33, 1, 1, 1, 128, 16, 900), (33, 8, 8, 1, 64, 16, 300), (100, 1, 4, 1, 128, 64, 700), (147, 1, 1, 2, 64, 8, 130),
    (192, 8, 8, 1, 128, 16, 90), (192, 1, 1, 12, 128, 16, 200), (256, 1, 1, 12, 64, 16, 100),
    (256, 8, 16, 1, 64, 32, 100), (257, 1, 12, 1, 128, 16, 100), (384, 1, 1, 1, 128, 16, 200),
    (385, 1, 1, 1, 64, 16, 300), (385, 8, 8, 1, 64, 16, 40), (500, 1, 1, 9, 256, 16, 60), (500, 8, 32, 1, 128, 16, 60),
    (2100, 8, 8, 1, 64, 16, 40), (2100, 8, 16, 2, 64, 8, 70), (32, 16, 16, 530, 144, 16, 60)]


@pytest.mark.parametrize("batch,Hkv,Hq,rows,head,page,longest", MANY)
def test_attention_many_sequences(b2, batch, Hkv, Hq, rows, head, page, longest):
    """Ranges worked out per warp (up to 32 sequences), per block, and in runs past a block's
    threads; CTAs of one pair each, ranges that cut pairs, and, with more pairs than counters (about
    16380), ranges of whole pairs."""
    codes = "int8" if batch % 2 else "fp8"
    cache, q, new = many_sequences(b2, batch, Hkv, Hq, rows, head, page, longest, codes, batch + Hkv)
    check_many(b2, cache, q, new)
    check_many(b2, cache, q, new, window=longest // 4, sinks=2)
    check_many(b2, cache, q, torch.zeros_like(new))
