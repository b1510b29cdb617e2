"""The operators of a decoder step with 8-bit activations and an 8-bit paged KV cache, against plain
implementations in 64 bits.

Tolerances, set from the arithmetic:
 * a scale: fp32 statistic over up to a few thousand values in a tree of at most 64 additions, plus
   a handful of roundings: relative 64 * 2^-24 + 2^-21 < 5e-6;
 * a code: within half a step of value / scale, plus what the 5e-6 of the scale and of the
   value make of its magnitude (at most 448 * 1e-5);
 * INT8 products: the integer sum is exact, so one fp32 conversion, two fp32 products and the
   output's rounding remain; FLOAT8 products: fp32 sums of K terms, bounded by K 2^-23 sum |a w|
   (one rounding or truncation per term, in any order);
 * attention: probabilities rounded to 16 bits (2^-11 relative), scores off by at most 1e-4, the
   output's rounding: |error| <= u |y| + (2^-11 + 3e-4) sum p |v| with u = 2^-11 or 2^-8.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
QMAX = {"int8": 127.0, "fp8": 448.0}
NAN_CODE = 0x7F  # FLOAT8E4M3FN NaN


@pytest.fixture(autouse=True)
def clean_status(b2, cuda):
    from onnx_light_b200 import _capi
    _capi.lib().b2_kernel_status(1)
    yield
    assert _capi.lib().b2_kernel_status(1) == 0


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def kind_of(b2, codes):
    return b2.INT8 if codes == "int8" else b2.FLOAT8E4M3FN


def storage(t):
    return t.data if hasattr(t, "dtype") and isinstance(t.dtype, int) else t


def values(codes):
    """8-bit codes (torch.int8, or uint8 storage of FLOAT8E4M3FN) in 64 bits."""
    return (codes.view(torch.float8_e4m3fn) if codes.dtype == torch.uint8 else codes).double()


def half_step(v, codes):
    """Half the distance between neighbouring codes at magnitude v."""
    if codes == "int8":
        return torch.full_like(v, 0.5)
    return torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 4)


def assert_codes(got, want, codes, slack=1e-5):
    """got: codes; want: value / scale in 64 bits."""
    err = (values(got) - want.clamp(-QMAX[codes], QMAX[codes])).abs()
    assert bool((err <= half_step(want, codes) * (1 + 1e-3) + slack * QMAX[codes]).all()), float(err.max())


# ---------------------------------------------------------------------------
# RMSNormalizationQuantize
# ---------------------------------------------------------------------------

NORM_SHAPES = [((1, 8), 0), ((3, 64), 32), ((5, 7), 0), ((2, 3, 1000), 0), ((4, 4096), 0),
               ((2, 4096), 128), ((1, 11008), 0), ((3, 11008), 256), ((2, 96), 24), ((2, 90), 9),
               ((1, 16392), 0), ((2, 20000), 8), ((1, 32768), 64), ((1, 40001), 0), ((300, 272), 16),
               ((2, 1), 0)]


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("tname", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape,group", NORM_SHAPES, ids=lambda s: str(s).replace(" ", ""))
def test_norm(b2, shape, group, tname, codes):
    t = TYPES[tname]
    for residual in (False, True):
        g = gen(len(shape) + shape[-1] + residual)
        x = (torch.randn(shape, generator=g, device="cuda") * 3).to(t)
        w = (1 + 0.3 * torch.randn(shape[-1], generator=g, device="cuda")).to(t)
        more = torch.randn(shape, generator=g, device="cuda").to(t) if residual else None
        r = b2.RMSNormalizationQuantize()(x, w, residual=more, epsilon=1e-5, dtype=kind_of(b2, codes),
                                          group_size=group)
        h = x.double() + (more.double() if residual else 0.0)
        n = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-5) * w.double()
        parts = n.view(*shape[:-1], -1, group or shape[-1])
        scale = parts.abs().amax(-1) / QMAX[codes]
        assert r.Y_scale.shape == scale.shape and tuple(r.Y.shape) == shape
        assert torch.allclose(r.Y_scale.double(), scale, rtol=5e-6, atol=0)
        assert_codes(storage(r.Y).view(parts.shape), parts / scale[..., None], codes)
        if residual:  # one rounding of an fp32 sum: bit for bit
            assert torch.equal(r.sum, (x.float() + more.float()).to(t))
        else:
            assert r.sum is None


@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_norm_zero_and_not_finite_rows(b2, codes):
    x = torch.randn(6, 256, generator=gen(3), device="cuda")
    x[1] = 0
    x[2, 7] = math.nan
    x[3, 9] = math.inf
    x[4] = 1e-30
    x[5, 100] = 3e38  # the square overflows: the row divides by infinity
    r = b2.RMSNormalizationQuantize()(x, torch.ones(256, device="cuda"), dtype=kind_of(b2, codes))
    s, c = r.Y_scale[:, 0], values(storage(r.Y))
    assert bool(torch.isfinite(c).all())
    assert float(s[1]) == 0 and float(c[1].abs().max()) == 0
    assert bool(torch.isnan(s[2])) and bool(torch.isnan(s[3]))
    want = x[4].double() / math.sqrt(1e-5)
    assert abs(float(s[4]) / float(want.max() / QMAX[codes]) - 1) < 1e-5
    assert float(s[5]) == 0 and float(c[5].abs().max()) == 0
    assert bool(torch.isfinite(s[[0]]).all())


def test_norm_sum_in_place(b2):
    """The sum may take the residual's or x's own buffer."""
    for width in (4096, 999):
        x = torch.randn(5, width, generator=gen(1), device="cuda").half()
        res = torch.randn(5, width, generator=gen(2), device="cuda").half()
        w = torch.ones(width, device="cuda").half()
        want = b2.RMSNormalizationQuantize()(x, w, residual=res)
        for alias in (0, 1):
            xs, rs = x.clone(), res.clone()
            got = b2.RMSNormalizationQuantize()(xs, w, residual=rs, out_sum=rs if alias else xs)
            assert torch.equal(got.sum, want.sum) and torch.equal(got.Y.data, want.Y.data)
            assert torch.equal(got.Y_scale, want.Y_scale)


def test_norm_unaligned_rows(b2):
    """A buffer that starts off the 16-byte boundary takes the scalar kernel."""
    base = torch.randn(4 * 128 + 1, generator=gen(5), device="cuda").half()
    x, w = base[1:].view(4, 128), torch.ones(128, device="cuda").half()
    got, want = b2.RMSNormalizationQuantize()(x, w), b2.RMSNormalizationQuantize()(x.clone(), w)
    assert torch.allclose(got.Y_scale, want.Y_scale, rtol=1e-5, atol=0)
    assert_codes(got.Y.data, values(want.Y.data), "fp8", slack=0.08)  # a neighbouring code at most


def test_norm_feeds_dequantize_linear(b2):
    """Y and Y_scale are DequantizeLinear's blocked layout along the last axis."""
    x = torch.randn(3, 512, generator=gen(6), device="cuda")
    r = b2.RMSNormalizationQuantize()(x, torch.ones(512, device="cuda"), dtype=b2.INT8, group_size=64)
    y = b2.DequantizeLinear()(r.Y, r.Y_scale, axis=1)
    want = r.Y.view(3, 8, 64).float() * r.Y_scale[..., None]
    assert torch.equal(y, want.view(3, 512))


# ---------------------------------------------------------------------------
# ScaledMatMul
# ---------------------------------------------------------------------------

PRODUCTS = [(1, 1, 1), (1, 64, 128), (1, 4096, 257), (2, 100, 33), (3, 272, 200), (5, 16, 8),
            (8, 4096, 512), (9, 1040, 130), (16, 2064, 96), (17, 512, 1000), (33, 4112, 77),
            (64, 1024, 300), (65, 768, 129), (100, 130, 50), (128, 4096, 256), (200, 999, 130),
            (257, 528, 511), (300, 4096, 640), (1000, 2048, 1100), (1, 32, 11008), (7, 65536, 40)]


def operand(g, codes, rows, k):
    v = torch.randn(rows, k, generator=g, device="cuda")
    if codes == "int8":
        return (v * 50).round().clamp(-128, 127).to(torch.int8)
    return (v * 120).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def as_arg(b2, t):
    return t if t.dtype == torch.int8 else b2.QTensor(t, b2.FLOAT8E4M3FN, tuple(t.shape))


def check_product(b2, a, as_, w, ws, t, codes):
    y = b2.ScaledMatMul()(as_arg(b2, a), as_, as_arg(b2, w), ws, dtype=t)
    av, wv = values(a), values(w)
    scale = as_.double().reshape(-1, 1) * ws.double().reshape(1, -1)
    want = av @ wv.t() * scale
    size = av.abs() @ wv.abs().t() * scale.abs()
    # exact sums: its conversion and two products (fp32); fp32 sums: one rounding per term
    slack = 4 * 2.0 ** -24 * want.abs() if codes == "int8" else a.shape[1] * 2.0 ** -23 * size
    tiny = 2.0 ** -25 if t == torch.float16 else 0.0  # half a subnormal step
    err = (y.double() - want).abs()
    assert bool((err <= UNIT[t] * want.abs() * (1 + 1e-3) + slack * 1.01 + tiny).all()), \
        float((err / (want.abs() + 1e-30)).max())
    if want.numel() > 500:
        assert float((y.double() - want).norm() / want.norm()) <= UNIT[t] + 3e-5


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("m,k,n", PRODUCTS)
def test_product(b2, m, k, n, codes):
    g = gen(m * 7 + n)
    a, w = operand(g, codes, m, k), operand(g, codes, n, k)
    as_ = torch.rand(m, generator=g, device="cuda") * 0.01 + 0.001
    ws = torch.rand(n, generator=g, device="cuda") * 0.001 + 0.0001
    for t in (torch.float16, torch.bfloat16, torch.float32):
        check_product(b2, a, as_, w, ws, t, codes)


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("m,k,n", [(2500, 400, 4000), (2561, 1040, 4001), (300, 144, 19000), (9000, 4096, 1300),
                                   (38000, 16, 250)])
def test_product_large(b2, m, k, n, codes):
    """Outputs of several hundred tiles: last tiles cut in both directions, several rounds of tiles."""
    g = gen(m + n)
    a, w = operand(g, codes, m, k), operand(g, codes, n, k)
    as_ = torch.rand(m, generator=g, device="cuda") * 0.01 + 0.001
    ws = torch.rand(n, generator=g, device="cuda") * 0.001 + 0.0001
    for t in (torch.float16, torch.bfloat16, torch.float32):
        check_product(b2, a, as_, w, ws, t, codes)


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("m,k,n", [(32, 272, 11008), (128, 272, 11001), (600, 144, 4096), (577, 144, 4090), (200, 400, 11008),
                                   (129, 400, 11000), (512, 144, 11008), (1500, 80, 4097)])
def test_product_between_powers_of_two(b2, m, k, n, codes):
    """Sizes that tiles of 96, 160 and 192 columns fit better, also with a cut last tile."""
    g = gen(m + 3 * n)
    a, w = operand(g, codes, m, k), operand(g, codes, n, k)
    as_ = torch.rand(m, generator=g, device="cuda") * 0.01 + 0.001
    ws = torch.rand(n, generator=g, device="cuda") * 0.001 + 0.0001
    for t in (torch.float16, torch.bfloat16, torch.float32):
        check_product(b2, a, as_, w, ws, t, codes)


@pytest.mark.parametrize("m", [1, 40, 130])
def test_product_one_scale_and_shapes(b2, m):
    g = gen(m)
    a, w = operand(g, "int8", m, 256), operand(g, "int8", 192, 256)
    one = torch.tensor(0.01, device="cuda")
    check_product(b2, a, one, w, torch.rand(192, generator=g, device="cuda"), torch.float32, "int8")
    check_product(b2, a, torch.rand(m, generator=g, device="cuda"), w, one.view(1), torch.float32, "int8")
    if m == 40:  # leading dimensions of A carry over
        y = b2.ScaledMatMul()(a.view(2, 20, 256), one, w, one)
        assert y.shape == (2, 20, 192)
        assert torch.equal(y.view(40, 192), b2.ScaledMatMul()(a, one, w, one))


@pytest.mark.parametrize("m", [1, 8, 33, 129])
def test_product_extreme_codes_are_exact(b2, m):
    """-128 times -128 over a long K: the sum passes 2^24 and stays exact in int32."""
    a = torch.full((m, 65536), -128, dtype=torch.int8, device="cuda")
    w = torch.full((130, 65536), -128, dtype=torch.int8, device="cuda")
    w[:, 0] = 127
    one = torch.ones(1, device="cuda")
    y = b2.ScaledMatMul()(a, one, w, one, dtype=torch.float32)
    want = 65535 * 16384 - 128 * 127
    assert bool((y.double() == float(torch.tensor(want, dtype=torch.float64).float())).all())


@pytest.mark.parametrize("m", [1, 8, 33, 129])
def test_product_nan_and_zero_scales(b2, m):
    """A NaN code or scale reaches its own row or column alone; a zero scale gives zeros."""
    g = gen(9)
    a, w = operand(g, "fp8", m, 512), operand(g, "fp8", 160, 512)
    as_, ws = torch.ones(m, device="cuda"), torch.ones(160, device="cuda")
    w[3, 17] = NAN_CODE
    ws[5], ws[6] = math.nan, 0.0
    y = b2.ScaledMatMul()(as_arg(b2, a), as_, as_arg(b2, w), ws, dtype=torch.float32)
    nan = torch.isnan(y).all(0)
    assert bool(nan[3]) and bool(nan[5]) and int(torch.isnan(y).sum()) == 2 * m
    assert float(y[:, 6].abs().max()) == 0


def test_product_unaligned(b2):
    """Operands off the 16-byte boundary."""
    g = gen(10)
    for m in (1, 30, 200):
        a = operand(g, "int8", 1, m * 64 + 3)[0, 3:].view(m, 64)
        w = operand(g, "int8", 1, 100 * 64 + 1)[0, 1:].view(100, 64)
        one = torch.ones(1, device="cuda")
        y = b2.ScaledMatMul()(a, one, w, one, dtype=torch.float32)
        assert torch.equal(y.double(), a.double() @ w.double().t())


# ---------------------------------------------------------------------------
# The cache
# ---------------------------------------------------------------------------


def make_cache(b2, codes, past, new, heads, head, page, seed=0, spare=3, holes=True):
    """A cache whose sequences hold `past` tokens, with room for `new` more, random pages, and
    everything that belongs to no token set to what must never be used: NaN codes (int8: -128), NaN
    scales, page numbers far outside the pool."""
    g = gen(seed)
    need = [max(1, -(-(p + n) // page)) for p, n in zip(past, new)]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    table = torch.full((len(past), max(need) + (2 if holes else 0)), 1 << 30, dtype=torch.int32)
    if codes == "int8":
        pools = [torch.full((pages, heads, page, head), -128, dtype=torch.int8, device="cuda") for _ in range(2)]
    else:
        pools = [torch.full((pages, heads, page, head), NAN_CODE, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.full((pages, heads), math.nan, device="cuda") for _ in range(2)]
    spread = 40.0 if codes == "int8" else 120.0
    for b, (p, n) in enumerate(zip(past, need)):
        for i in range(n):
            at = order.pop()
            table[b, i] = at
            rows = min(page, max(0, p - i * page))
            if rows:
                for pool, sc in zip(pools, scales):
                    v = torch.randn(heads, rows, head, generator=g, device="cuda") * spread
                    if codes == "int8":
                        pool[at, :, :rows] = v.round().clamp(-127, 127).to(torch.int8)
                    else:
                        pool[at, :, :rows] = v.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
                    sc[at] = torch.rand(heads, generator=g, device="cuda") * 0.02 + 0.01
    return b2.QuantizedKVCache(pools[0], pools[1], scales[0], scales[1], table.cuda(),
                               torch.tensor(past, dtype=torch.int32, device="cuda"), kind_of(b2, codes))


def side(cache, name, b, total):
    """[heads, total, head] of one sequence in 64 bits."""
    pool, sc = getattr(cache, name), getattr(cache, name + "_scale")
    page = pool.shape[2]
    ids = cache.block_table[b, :-(-total // page)].long()
    v = values(pool[ids]) * sc[ids].double()[:, :, None, None]
    return v.permute(1, 0, 2, 3).reshape(pool.shape[1], -1, pool.shape[3])[:, :total]


APPENDS = [  # past, new rows, new lengths, heads, head, page
    ([0], 1, None, 1, 64, 16), ([5, 16, 31], 1, None, 2, 128, 16), ([0, 1, 63, 64], 70, [70, 1, 0, 33], 2, 96, 64),
    ([3, 17], 40, None, 1, 80, 8), ([7], 200, [129], 3, 128, 128), ([2, 9], 5, None, 2, 33, 10),
    ([100, 3], 3, None, 2, 256, 32), ([1, 2, 3], 2, None, 1, 5, 1), ([30], 300, None, 1, 136, 256)]


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("tname", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("past,rows,count,heads,head,page", APPENDS, ids=lambda v: str(v).replace(" ", ""))
def test_append(b2, past, rows, count, heads, head, page, tname, codes):
    t = TYPES[tname]
    new = count or [rows] * len(past)
    cache = make_cache(b2, codes, past, new, heads, head, page, seed=rows)
    before = {n: getattr(cache, n).clone() for n in ("k", "v", "k_scale", "v_scale")}
    g = gen(rows + 1)
    # amplitudes from far below to far above what the pages hold, so that some scales grow
    amp = torch.exp(2 * torch.randn(len(past), heads, 1, 1, generator=g, device="cuda"))
    kv = [(torch.randn(len(past), heads, rows, head, generator=g, device="cuda") * amp).to(t) for _ in range(2)]
    counts = torch.tensor(new, dtype=torch.int32, device="cuda") if count else None
    for rank3 in (False, True):
        for n, old in before.items():
            getattr(cache, n).copy_(old)
        args = [x.transpose(1, 2).reshape(len(past), rows, -1).contiguous() for x in kv] if rank3 else kv
        b2.KVCacheAppend()(args[0], args[1], cache, new_lengths=counts)
        assert torch.equal(cache.lengths.cpu(), torch.tensor(past, dtype=torch.int32))
        for name, x in zip(("k", "v"), kv):
            pool, sc = getattr(cache, name), getattr(cache, name + "_scale")
            want_pool, want_sc = before[name].clone(), before[name + "_scale"].double()
            grown = 0
            for b, (p, n) in enumerate(zip(past, new)):
                for slot in range(p // page, (p + n + page - 1) // page if n else 0):
                    at = int(cache.block_table[b, slot])
                    lo, hi = max(p, slot * page), min(p + n, slot * page + page)
                    older = lo - slot * page
                    z = x[b, :, lo - p:hi - p].double()
                    had = want_sc[at].clone() if older else torch.zeros(heads, dtype=torch.float64, device="cuda")
                    s = torch.maximum(had, z.abs().amax((1, 2)) / QMAX[codes])
                    want_sc[at] = s
                    assert_codes(pool[at, :, older:older + hi - lo], z / s[:, None, None], codes, slack=1e-6)
                    for h in range(heads):
                        if older and s[h] > had[h] * (1 + 1e-6):
                            grown += 1
                            again = values(before[name][at, h, :older]) * (had[h] / s[h])
                            assert_codes(pool[at, h, :older], again, codes, slack=1e-6)
                        elif older:
                            assert torch.equal(pool[at, h, :older], before[name][at, h, :older])
                    want_pool[at, :, :older + hi - lo] = pool[at, :, :older + hi - lo]
            assert torch.equal(pool, want_pool)  # nothing else was touched
            assert torch.equal(torch.isnan(sc), torch.isnan(want_sc))
            assert torch.allclose(sc.double(), want_sc, rtol=2.0 ** -22, atol=0, equal_nan=True)


@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_append_token_by_token_equals_the_definition(b2, codes):
    """A page filled one token at a time: the scale ends as the largest magnitude, and each code is
    within one step (half for its own rounding, half for each of the at most few growths)."""
    cache = b2.QuantizedKVCache.allocate(2, 2, 64, 64, page_size=16, dtype=kind_of(b2, codes))
    g = gen(2)
    x = torch.randn(2, 2, 40, 64, generator=g, device="cuda").half()
    for i in range(40):
        b2.KVCacheAppend()(x[:, :, i:i + 1].contiguous(), x[:, :, i:i + 1].contiguous(), cache)
        cache.advance(1)
    for b in range(2):
        for slot in range(3):
            rows = x[b, :, slot * 16:min(40, slot * 16 + 16)].double()
            at = int(cache.block_table[b, slot])
            s = rows.abs().amax((1, 2)) / QMAX[codes]
            assert torch.allclose(cache.k_scale[at].double(), s, rtol=1e-6, atol=0)
            got = values(cache.k[at, :, :rows.shape[1]]) * s[:, None, None]
            steps = 16 * 2 * half_step(rows / s[:, None, None], codes) * s[:, None, None]
            assert bool(((got - rows).abs() <= steps).all())
            assert float((got - rows).norm() / rows.norm()) < (0.02 if codes == "int8" else 0.06)
    assert torch.equal(cache.k, cache.v)


@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_append_zeros_and_not_finite(b2, codes):
    cache = b2.QuantizedKVCache.allocate(3, 1, 16, 32, page_size=16, dtype=kind_of(b2, codes))
    x = torch.zeros(3, 1, 2, 32, device="cuda")
    x[1, 0, 0, 3], x[2, 0, 1, 5] = math.nan, math.inf
    b2.KVCacheAppend()(x, x, cache)
    s = cache.k_scale[:, 0]
    assert float(s[0]) == 0 and bool(torch.isnan(s[1])) and bool(torch.isinf(s[2]))
    assert float(values(cache.k).abs().max()) == 0
    cache.advance(2)
    one = torch.ones(3, 1, 1, 32, device="cuda")  # after zeros; after a NaN; after an infinity
    b2.KVCacheAppend()(one, one, cache)
    assert abs(float(s[0]) * QMAX[codes] - 1) < 1e-6 and float(values(cache.k[0, 0, 2]).min()) == QMAX[codes]
    assert bool(torch.isnan(s[1])) and bool(torch.isinf(s[2]))


def test_append_out_of_range_is_reported(b2):
    """Lengths past the table and pages outside the pool are skipped and reported."""
    from onnx_light_b200 import _capi
    lib = _capi.lib()
    x = torch.ones(3, 1, 4, 16, device="cuda").half()
    cache = b2.QuantizedKVCache.allocate(3, 1, 16, 16, page_size=8, dtype=b2.INT8)
    cache.lengths.copy_(torch.tensor([14, -3, 0], dtype=torch.int32))
    cache.block_table[2, 0] = 99
    b2.KVCacheAppend()(x, x, cache)
    assert lib.b2_kernel_status(1) == 4
    assert bool((cache.k[1, 0, 6:] == 127).all()) and bool((cache.k[1, 0, :6] == 0).all())  # two fit
    assert float(cache.k_scale[4].abs().max()) == 0
    q = torch.ones(3, 2, 4, 16, device="cuda").half()
    y = b2.QuantizedCacheAttention()(q, cache)
    assert lib.b2_kernel_status(1) == 4 and bool(torch.isfinite(y).all())
    assert float(y[2].abs().max()) == 0  # its only page does not exist


# ---------------------------------------------------------------------------
# QuantizedCacheAttention
# ---------------------------------------------------------------------------


def reference(cache, q, new, causal=True, window=-1, sinks=0, scale=None, softcap=0.0):
    """(y, sum p |v|) in 64 bits."""
    B, Hq, S, D = q.shape
    Hkv = cache.k.shape[1]
    y, size = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), None
    size = torch.zeros_like(y)
    for b in range(B):
        p, n = int(cache.lengths[b]), new[b]
        total = p + n
        if n == 0:
            continue
        k, v = side(cache, "k", b, total), side(cache, "v", b, total)
        z = torch.einsum("kgsd,kjd->kgsj", q[b].double().view(Hkv, -1, S, D)[:, :, :n], k)
        z = z * (scale if scale is not None else 1 / math.sqrt(D))
        if softcap > 0:
            z = softcap * torch.tanh(z / softcap)
        at = p + torch.arange(n, device="cuda")[:, None]
        j = torch.arange(total, device="cuda")
        seen = torch.ones(n, total, dtype=torch.bool, device="cuda")
        if causal:
            seen = j <= at
            if window >= 0:
                seen = seen & ((at - j <= window) | (j < sinks))
        prob = torch.softmax(z.masked_fill(~seen, -math.inf), -1)
        y[b, :, :n] = torch.einsum("kgsj,kjd->kgsd", prob, v).reshape(Hq, n, D)
        size[b, :, :n] = torch.einsum("kgsj,kjd->kgsd", prob, v.abs()).reshape(Hq, n, D)
    return y, size


def check_attention(b2, cache, q, new=None, **kw):
    S = q.shape[2]
    counts = torch.tensor(new, dtype=torch.int32, device="cuda") if new else None
    attrs = b2.CacheAttributes(is_causal=kw.get("causal", True), left_window_size=kw.get("window", -1),
                               sink_tokens=kw.get("sinks", 0), softcap=kw.get("softcap", 0.0),
                               has_scale=kw.get("scale") is not None, scale=kw.get("scale") or 0.0)
    y = b2.QuantizedCacheAttention()(q, cache, attrs, new_lengths=counts)
    want, size = reference(cache, q, new or [S] * q.shape[0], **kw)
    err = (y.double() - want).abs()
    limit = UNIT[q.dtype] * want.abs() * 1.001 + (2.0 ** -11 + 3e-4) * size + 2.0 ** -25
    assert bool((err <= limit).all()), float((err / limit).max())
    q3 = q.transpose(1, 2).reshape(q.shape[0], S, -1).contiguous()
    y3 = b2.QuantizedCacheAttention()(q3, cache, attrs, new_lengths=counts)
    assert torch.equal(y3.view(q.shape[0], S, q.shape[1], -1).transpose(1, 2), y)
    return y


ATTENTIONS = [  # past, rows, new lengths, Hq, Hkv, head, page
    ([0], 1, None, 1, 1, 64, 16), ([0, 3, 15, 16, 17], 1, None, 4, 2, 128, 16),
    ([63, 64, 200, 1000], 1, None, 8, 1, 128, 64), ([31, 2047], 1, None, 32, 8, 128, 64),
    ([5, 900], 1, None, 16, 1, 64, 32), ([700], 1, None, 32, 1, 128, 64), ([129, 40], 1, None, 48, 1, 96, 128),
    ([10, 500], 1, None, 6, 2, 80, 8), ([10, 300], 1, None, 4, 2, 256, 16), ([9, 50], 1, None, 2, 1, 40, 10),
    ([9, 77], 1, None, 3, 3, 33, 7), ([0, 5], 1, [1, 0], 4, 4, 128, 16), ([77], 1, None, 70, 1, 64, 16),
    ([100, 0], 4, None, 8, 2, 128, 16), ([100, 7], 5, [5, 2], 4, 4, 64, 32), ([333], 8, None, 8, 2, 128, 64),
    ([0], 130, None, 4, 1, 128, 64), ([0, 60], 70, [70, 33], 4, 2, 64, 16), ([250], 257, None, 8, 8, 128, 32),
    ([31, 0, 512], 33, [33, 0, 20], 6, 2, 96, 64), ([1000], 300, None, 16, 2, 128, 128),
    ([17], 140, None, 2, 1, 80, 48), ([40], 64, None, 2, 2, 256, 16), ([5], 50, None, 2, 1, 50, 6),
    ([4000], 129, None, 8, 1, 128, 64), ([0], 1024, None, 2, 2, 128, 64)]


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("tname", ["f16", "bf16"])
@pytest.mark.parametrize("past,rows,count,Hq,Hkv,head,page", ATTENTIONS, ids=lambda v: str(v).replace(" ", ""))
def test_attention(b2, past, rows, count, Hq, Hkv, head, page, tname, codes):
    new = count or [rows] * len(past)
    cache = make_cache(b2, codes, [p + n for p, n in zip(past, new)], [0] * len(past), Hkv, head, page, seed=rows)
    cache.lengths.copy_(torch.tensor(past, dtype=torch.int32))
    q = torch.randn(len(past), Hq, rows, head, generator=gen(head + rows), device="cuda").to(TYPES[tname])
    y = check_attention(b2, cache, q, count)
    for b, n in enumerate(new):
        assert float(y[b, :, n:].abs().sum()) == 0
    longest = max(past)
    check_attention(b2, cache, q, count, window=longest // 3, sinks=2)
    check_attention(b2, cache, q, count, window=0, sinks=0)
    check_attention(b2, cache, q, count, window=7, sinks=40)
    check_attention(b2, cache, q, count, causal=False)
    check_attention(b2, cache, q, count, scale=0.3, softcap=2.0)


@pytest.mark.parametrize("rows", [1, 6, 200])
@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_attention_large_scores(b2, codes, rows):
    """Scores of several hundred: the running maximum is replaced many times, one key takes all."""
    cache = make_cache(b2, codes, [700 + rows], [0], 2, 128, 32, seed=4)
    cache.lengths.fill_(700)
    q = (torch.randn(1, 4, rows, 128, generator=gen(1), device="cuda") * 20).half()
    # scores reach 1e3: fp32 leaves 1e3 * 2^-22, within the 3e-4 of the bound
    check_attention(b2, cache, q)
    check_attention(b2, cache, -q, scale=-0.05)


@pytest.mark.parametrize("rows", [1, 5, 150])
@pytest.mark.parametrize("tname", ["f16", "bf16"])
def test_attention_uneven_scales(b2, rows, tname):
    """Pages whose value scales differ by a factor of a million."""
    cache = make_cache(b2, "int8", [500 + rows], [0], 1, 128, 16, seed=8)
    cache.lengths.fill_(500)
    pages = cache.block_table[0].long()
    pages = pages[pages < cache.v_scale.shape[0]]
    cache.v_scale[pages] *= 10.0 ** (torch.arange(len(pages), device="cuda") % 7 - 4.0)[:, None]
    q = torch.randn(1, 4, rows, 128, generator=gen(3), device="cuda").to(TYPES[tname])
    check_attention(b2, cache, q)


@pytest.mark.parametrize("rows", [1, 4, 140])
@pytest.mark.parametrize("amplitude", [1e-7, 1e-3, 300.0])
def test_attention_query_amplitudes(b2, rows, amplitude):
    """Queries from far below to far above 1, bfloat16's range."""
    cache = make_cache(b2, "fp8", [300 + rows], [0], 2, 128, 64, seed=6)
    cache.lengths.fill_(300)
    q = (torch.randn(1, 4, rows, 128, generator=gen(3), device="cuda") * amplitude).bfloat16()
    check_attention(b2, cache, q, scale=0.1 / amplitude)


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("rows", [1, 3, 160])
@pytest.mark.parametrize("head,page", [(128, 16), (64, 64), (40, 10)])
def test_attention_not_finite_values_stay_where_they_are_seen(b2, rows, codes, head, page):
    """A block whose scale is NaN or infinite reaches the queries that see it and no other."""
    total = 400 + rows
    cache = make_cache(b2, codes, [total], [0], 1, head, page, seed=12)
    cache.lengths.fill_(400)
    q = torch.randn(1, 2, rows, head, generator=gen(5), device="cuda").half()
    window = 60
    clean, _ = reference(cache, q, [rows], window=window, sinks=3)
    for name in ("k_scale", "v_scale"):
        sc = getattr(cache, name)
        block = 300 // page  # before the window of query 0: seen by none
        keep = sc.clone()
        sc[int(cache.block_table[0, block])] = math.nan
        y = b2.QuantizedCacheAttention()(q, cache, b2.CacheAttributes(left_window_size=window, sink_tokens=3))
        far = (block + 1) * page <= 400 - window
        assert far and bool(torch.isfinite(y).all())
        assert float((y.double() - clean).norm() / clean.norm()) < 2e-3
        sc.copy_(keep)
        last = (total - 1) // page  # holds the last token: seen by the last query alone, or a few
        sc[int(cache.block_table[0, last])] = math.nan
        y = b2.QuantizedCacheAttention()(q, cache, b2.CacheAttributes(left_window_size=window, sink_tokens=3))
        first = max(0, last * page - 400)  # the first query that sees a token of that block
        assert bool(torch.isnan(y[:, :, first:]).all())
        assert bool(torch.isfinite(y[:, :, :first]).all())
        sc.copy_(keep)


@pytest.mark.parametrize("rows", [1, 40])
def test_cache_past_4_gib(b2, rows):
    """Pages whose codes lie past 2^32 bytes of their pool, for the append and both tensor-core kernels."""
    pages, heads, page, head = 66000, 8, 64, 128  # 4.3e9 bytes each of K and V
    cache = b2.QuantizedKVCache.allocate(1, heads, 128, head, page_size=page, dtype=b2.INT8, pages=pages,
                                         block_table=torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32,
                                                                  device="cuda"))
    assert cache.k.numel() > 1 << 32
    kv = torch.randn(2, 1, heads, 100, head, generator=gen(1), device="cuda").half()
    b2.KVCacheAppend()(kv[0], kv[1], cache)
    cache.advance(100)
    for pool, x in ((cache.k, kv[0]), (cache.v, kv[1])):
        got = values(pool[pages - 1]) * cache.k_scale[pages - 1].double()[:, None, None] if pool is cache.k else \
            values(pool[pages - 1]) * cache.v_scale[pages - 1].double()[:, None, None]
        step = (cache.k_scale if pool is cache.k else cache.v_scale)[pages - 1].double()[:, None, None]
        assert bool(((got - x[0, :, :64].double()).abs() <= 0.501 * step).all())
    cache.lengths.fill_(100 - rows)
    q = torch.randn(1, 16, rows, head, generator=gen(2), device="cuda").half()
    check_attention(b2, cache, q)


def test_attention_identical_runs(b2):
    """The same call twice gives the same bits, whatever order blocks finish in."""
    for past, rows in (([3000, 17, 900], 1), ([2500], 3), ([600], 500)):
        cache = make_cache(b2, "fp8", [p + rows for p in past], [0] * len(past), 2, 128, 64, seed=1)
        cache.lengths.copy_(torch.tensor(past, dtype=torch.int32))
        q = torch.randn(len(past), 8, rows, 128, generator=gen(5), device="cuda").half()
        first = b2.QuantizedCacheAttention()(q, cache)
        for _ in range(5):
            assert torch.equal(b2.QuantizedCacheAttention()(q, cache), first)


def test_attention_on_two_streams(b2):
    """Calls on two streams at once keep to their own workspaces."""
    cache = make_cache(b2, "int8", [4000] * 4, [0] * 4, 2, 128, 64, seed=2)
    cache.lengths.fill_(3999)
    qs = [torch.randn(4, 8, 1, 128, generator=gen(i), device="cuda").half() for i in range(2)]
    want = [b2.QuantizedCacheAttention()(q, cache) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(b2.QuantizedCacheAttention()(qs[i], cache))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_step_in_a_cuda_graph(b2):
    """Append, attention and the count of tokens replayed: nothing waits for the host."""
    cache = b2.QuantizedKVCache.allocate(2, 2, 256, 128, page_size=32, dtype=b2.FLOAT8E4M3FN)
    cache2 = b2.QuantizedKVCache.allocate(2, 2, 256, 128, page_size=32, dtype=b2.FLOAT8E4M3FN)
    x = torch.randn(40, 3, 2, 2, 1, 128, generator=gen(7), device="cuda").half()
    q = torch.randn(40, 2, 8, 1, 128, generator=gen(8), device="cuda").half()
    sk, sv, sq = x[0, 0].clone(), x[0, 1].clone(), q[0].clone()

    def step(c, k, v, qq):
        b2.KVCacheAppend()(k, v, c)
        y = b2.QuantizedCacheAttention()(qq, c)
        c.advance(1)
        return y

    want = [step(cache2, x[i, 0], x[i, 1], q[i]) for i in range(40)]
    side_stream = torch.cuda.Stream()
    with torch.cuda.stream(side_stream):
        step(cache, sk, sv, sq)
    torch.cuda.synchronize()
    cache.lengths.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side_stream):
        y = step(cache, sk, sv, sq)
    cache.lengths.zero_()
    for i in range(40):
        sk.copy_(x[i, 0])
        sv.copy_(x[i, 1])
        sq.copy_(q[i])
        graph.replay()
        assert torch.equal(y, want[i])
    assert torch.equal(cache.k, cache2.k) and torch.equal(cache.v_scale, cache2.v_scale)


def test_empty_calls(b2):
    one = torch.ones(1, device="cuda")
    y = b2.ScaledMatMul()(torch.zeros(0, 32, dtype=torch.int8, device="cuda"), one,
                          torch.zeros(8, 32, dtype=torch.int8, device="cuda"), one)
    assert y.shape == (0, 8)
    y = b2.ScaledMatMul()(torch.zeros(3, 0, dtype=torch.int8, device="cuda"), one,
                          torch.zeros(8, 0, dtype=torch.int8, device="cuda"), one)
    assert y.shape == (3, 8) and float(y.abs().max()) == 0
    r = b2.RMSNormalizationQuantize()(torch.zeros(0, 64, device="cuda"), torch.ones(64, device="cuda"))
    assert r.Y_scale.shape == (0, 1)
    cache = b2.QuantizedKVCache.allocate(0, 2, 16, 64, page_size=16)
    x = torch.zeros(0, 2, 1, 64, device="cuda").half()
    b2.KVCacheAppend()(x, x, cache)
    assert b2.QuantizedCacheAttention()(x, cache).shape == x.shape
    cache = b2.QuantizedKVCache.allocate(2, 2, 16, 64, page_size=16)
    x = torch.zeros(2, 2, 0, 64, device="cuda").half()
    b2.KVCacheAppend()(x, x, cache)
    assert b2.QuantizedCacheAttention()(x, cache).shape == x.shape


def test_refusals(b2):
    x, w = torch.zeros(2, 64, device="cuda"), torch.ones(64, device="cuda")
    norm, mm = b2.RMSNormalizationQuantize(), b2.ScaledMatMul()
    with pytest.raises(ValueError, match="group_size"):
        norm(x, w, group_size=48)
    with pytest.raises(ValueError, match="scale must have"):
        norm(x, w.half())
    with pytest.raises(ValueError, match="residual"):
        norm(x, w, residual=x.half())
    with pytest.raises(ValueError, match="8-bit codes"):
        norm(x, w, dtype=1)
    with pytest.raises(ValueError, match="contiguous"):
        norm(torch.zeros(64, 2, device="cuda").t(), w)
    a = torch.zeros(2, 64, dtype=torch.int8, device="cuda")
    one = torch.ones(1, device="cuda")
    with pytest.raises(ValueError, match="one dtype"):
        mm(a, one, b2.QTensor(a.view(torch.uint8), b2.FLOAT8E4M3FN, (2, 64)), one)
    with pytest.raises(ValueError, match=r"\[N, K\]"):
        mm(a, one, torch.zeros(3, 32, dtype=torch.int8, device="cuda"), one)
    with pytest.raises(ValueError, match="A_scale"):
        mm(a, torch.ones(3, device="cuda"), a, one)
    with pytest.raises(ValueError, match="scales must be FLOAT"):
        mm(a, one.half(), a, one)
    cache = b2.QuantizedKVCache.allocate(2, 2, 32, 64, page_size=16)
    kv = torch.zeros(2, 2, 1, 64, device="cuda").half()
    append, attend = b2.KVCacheAppend(), b2.QuantizedCacheAttention()
    with pytest.raises(ValueError, match="do not fit"):
        append(kv[:1].contiguous(), kv[:1].contiguous(), cache)
    with pytest.raises(ValueError, match="one shape|must be"):
        append(kv, kv[:, :, :, :32].contiguous(), cache)
    with pytest.raises(ValueError, match="new_lengths"):
        append(kv, kv, cache, new_lengths=torch.ones(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="FLOAT16 or BFLOAT16"):
        attend(kv.float(), cache)
    with pytest.raises(ValueError, match="multiple"):
        attend(torch.zeros(2, 3, 1, 64, device="cuda").half(), cache)
    with pytest.raises(ValueError, match="left_window_size"):
        attend(kv, cache, b2.CacheAttributes(left_window_size=-2))
    with pytest.raises(ValueError, match="needs is_causal"):
        attend(kv, cache, b2.CacheAttributes(is_causal=False, left_window_size=4))
    with pytest.raises(ValueError, match="sink_tokens"):
        attend(kv, cache, b2.CacheAttributes(sink_tokens=-1))
    with pytest.raises(ValueError, match="INT8 or FLOAT8E4M3FN"):
        b2.QuantizedKVCache(cache.k, cache.v, cache.k_scale, cache.v_scale, cache.block_table, cache.lengths, 10)
