"""Timing cases for the operators of a decoder step whose activations and KV cache are held in
8 bits: RMS normalization (with the residual's addition) that writes 8-bit codes and scales, the
product of two 8-bit operands with row and column scales, the append of new keys and values to a
paged 8-bit cache, and attention over that cache.

A case is a dict of plain values; prepare() makes its inputs, run() is one pass, either in plain
torch operations (32-bit arithmetic, rounded once) or, with `own`, through the package's operators.
exact() computes the same results in 64 bits.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

_TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_QMAX = {"int8": 127.0, "fp8": 448.0}
_F8 = torch.float8_e4m3fn


# ---------------------------------------------------------------------------
# Cases.  Sizes are the repository's own configurations: hidden size 4096, intermediate size
# 11008, 32 query and 8 key/value heads of 128, decode over 4096 cached tokens, prompts of up to
# 8192 tokens.
# ---------------------------------------------------------------------------


def listed():
    return [
        # one decoding user: the norm before a projection, where latency counts
        {"name": "norm decode", "op": "norm", "rows": 1, "width": 4096, "type": "float16",
         "codes": "fp8", "group": 0, "residual": True},
        # an odd number of rows of the intermediate width, scales for groups of 128, no residual
        {"name": "norm groups", "op": "norm", "rows": 517, "width": 11008, "type": "bfloat16",
         "codes": "int8", "group": 128, "residual": False},
        # the norm over a whole prompt
        {"name": "norm prompt", "op": "norm", "rows": 8192, "width": 4096, "type": "bfloat16",
         "codes": "fp8", "group": 0, "residual": True},
        # one new token for each of 32 sequences of different lengths
        {"name": "append decode", "op": "append", "batch": 32, "new": 1, "ragged": False,
         "past": 4095, "kv_heads": 8, "head": 128, "page": 64, "type": "float16", "codes": "fp8"},
        # prompts of different lengths written behind what the cache holds
        {"name": "append prompts", "op": "append", "batch": 4, "new": 2048, "ragged": True,
         "past": 1000, "kv_heads": 8, "head": 128, "page": 64, "type": "bfloat16", "codes": "fp8"},
        # one decoding user at 4096 cached tokens
        {"name": "attention decode", "op": "attention", "batch": 1, "new": 1, "ragged": False,
         "past": 4096, "heads": 32, "kv_heads": 8, "head": 128, "page": 64, "window": -1,
         "sinks": 0, "type": "float16", "codes": "int8"},
        # a decoding batch of sequences of different lengths: the cache's bytes count
        {"name": "attention batch", "op": "attention", "batch": 32, "new": 1, "ragged": False,
         "past": 8191, "heads": 32, "kv_heads": 8, "head": 128, "page": 64, "window": -1,
         "sinks": 0, "type": "bfloat16", "codes": "fp8"},
        # long sequences through a sliding window with four first tokens kept, small pages
        {"name": "attention window", "op": "attention", "batch": 8, "new": 1, "ragged": False,
         "past": 32767, "heads": 32, "kv_heads": 8, "head": 128, "page": 16, "window": 4095,
         "sinks": 4, "type": "float16", "codes": "int8"},
        # the last part of a long prompt: every cached token seen by 2048 new ones
        {"name": "attention prompt", "op": "attention", "batch": 1, "new": 2048, "ragged": False,
         "past": 6144, "heads": 32, "kv_heads": 8, "head": 128, "page": 64, "window": -1,
         "sinks": 0, "type": "bfloat16", "codes": "fp8"},
        # one decoding user's projection: the weight's bytes count
        {"name": "product decode", "op": "product", "rows": 1, "inner": 4096, "columns": 4096,
         "type": "float16", "codes": "fp8"},
        # a decoding batch's up projection
        {"name": "product batch", "op": "product", "rows": 32, "inner": 4096, "columns": 11008,
         "type": "float16", "codes": "int8"},
        # a prompt's up projection: the tensor cores count
        {"name": "product prompt", "op": "product", "rows": 8192, "inner": 4096, "columns": 11008,
         "type": "bfloat16", "codes": "fp8"},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread evenly over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "append", "attention", "attention", "product"])
    codes = rng.choice(["int8", "fp8"])
    half = rng.choice(["float16", "bfloat16"])
    if op == "norm":
        width = _log(rng, 64, 16384)
        group = rng.choice([0, 0, 32, 64, 128])
        width = max(group, width // group * group) if group else width
        rows = _log(rng, 1, max(1, min(8192, 8192 * 4096 // width)))
        return {"op": op, "rows": rows, "width": width,
                "type": rng.choice(["float32", "float16", "bfloat16"]), "codes": codes,
                "group": group, "residual": rng.random() < 0.7}
    if op == "product":
        inner = 16 * _log(rng, 16, 688)
        columns = _log(rng, 64, 11008)
        return {"op": op, "rows": _log(rng, 1, 8192), "inner": inner, "columns": columns,
                "type": half, "codes": codes}
    kv = rng.choice([1, 2, 4, 8])
    head = rng.choice([64, 96, 128])
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        new = 1 if rng.random() < 0.4 else _log(rng, 2, 2048)
        batch = _log(rng, 1, max(1, min(64, 4 * 2048 * 8 * 128 // (new * kv * head))))
        return {"op": op, "batch": batch, "new": new, "ragged": rng.random() < 0.5,
                "past": _log(rng, 1, 4096) - 1, "kv_heads": kv, "head": head, "page": page,
                "type": half, "codes": codes}
    heads = kv * rng.choice([1, 2, 4, 8])
    new = 1 if rng.random() < 0.5 else _log(rng, 2, 2048)
    past = _log(rng, 1, 16384) - 1
    new = min(new, 2048 * 8192 * 32 // ((past + 2048 + page) * heads))
    length = past + new + page
    batch = _log(rng, 1, max(1, min(64, 2048 * 8192 * 32 // (length * new * heads),
                                    32 * 8192 * 8 * 128 // (length * kv * head))))
    windowed = rng.random() < 0.4
    return {"op": op, "batch": batch, "new": new, "ragged": rng.random() < 0.5, "past": past,
            "heads": heads, "kv_heads": kv, "head": head, "page": page,
            "window": _log(rng, 16, 4096) if windowed else -1,
            "sinks": rng.choice([0, 1, 4, 16]) if windowed else 0, "type": half, "codes": codes}


def _lengths(case):
    """(tokens in the cache, new tokens) of each sequence: the first has the most, the others from
    a quarter of it up; with `ragged` their new tokens differ too."""
    part = [1.0 if b == 0 else 0.25 + 0.75 * math.fmod(b * 0.6180339887, 1.0)
            for b in range(case["batch"])]
    past = [int(case["past"] * f) for f in part]
    new = [max(1, int(case["new"] * f)) if case["ragged"] else case["new"] for f in part[::-1]]
    return past, new


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _codes(g, kind, spread, *shape):
    """Random codes of roughly normal values: int8, or 8-bit floats as their bytes."""
    v = _randn(g, *shape).mul_(spread)
    if kind == "int8":
        return v.round_().clamp_(-127, 127).to(torch.int8)
    return v.clamp_(-448, 448).to(_F8).view(torch.uint8)


def _cache(case, g):
    """A paged cache that holds `past` tokens of each sequence and has room for the new ones, its
    pages in random order; page 0 belongs to nobody and fills the tables' unused places."""
    past, new = _lengths(case)
    page, kv, head = case["page"], case["kv_heads"], case["head"]
    need = [max(1, -(-(p + n) // page)) for p, n in zip(past, new)]
    pages = sum(need) + 1
    order = (torch.randperm(pages - 1, generator=g, device="cuda") + 1).to(torch.int32).cpu().tolist()
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [0] * (max(need) - n))
        at += n
    spread = 40.0 if case["codes"] == "int8" else 120.0
    made = {"table": torch.tensor(table, dtype=torch.int32, device="cuda"),
            "past": torch.tensor(past, dtype=torch.int32, device="cuda"),
            "new": torch.tensor(new, dtype=torch.int32, device="cuda")}
    for name in ("k", "v"):
        made[name] = _codes(g, case["codes"], spread, pages, kv, page, head)
        made[name + "_scale"] = torch.exp(0.3 * _randn(g, pages, kv)) / spread
    return made


def prepare(case, seed):
    g = _gen(seed)
    t = _TYPES[case["type"]]
    s = dict(case)
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        x = _randn(g, rows, width)
        # a few channels of a hidden state are much larger than the others
        x *= 1.0 + 15.0 * (torch.rand(width, generator=g, device="cuda") < 0.01)
        s["x"] = x.to(t)
        s["weight"] = (1.0 + 0.2 * _randn(g, width)).to(t)
        s["more"] = _randn(g, rows, width).mul_(0.5).to(t) if case["residual"] else None
    elif case["op"] == "product":
        spread = 32.0 if case["codes"] == "int8" else 100.0
        s["a"] = _codes(g, case["codes"], spread, case["rows"], case["inner"])
        s["w"] = _codes(g, case["codes"], spread, case["columns"], case["inner"])
        s["a_scale"] = torch.exp(0.3 * _randn(g, case["rows"])) / spread
        s["w_scale"] = torch.exp(0.1 * _randn(g, case["columns"])) / (spread * math.sqrt(case["inner"]))
    else:
        s.update(_cache(case, g))
        shape = (case["batch"], case["kv_heads"], case["new"], case["head"])
        if case["op"] == "append":
            s["new_k"], s["new_v"] = (_randn(g, *shape).to(t) for _ in range(2))
        else:
            s["q"] = _randn(g, case["batch"], case["heads"], case["new"], case["head"]).to(t)
    return s


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------


def _value(codes):
    """The values of 8-bit codes in 32 bits."""
    return (codes.view(_F8) if codes.dtype == torch.uint8 else codes).float()


def _encode(v, kind):
    """Values already divided by their scale -> codes; what is not a number gives 0."""
    v = torch.nan_to_num(v, nan=0.0)
    if kind == "int8":
        return v.round().clamp(-127, 127).to(torch.int8)
    return v.clamp(-448, 448).to(_F8).view(torch.uint8)


def _norm_outputs(total, codes, scale, case):
    """The operator's outputs; 8-bit floats as such, whole codes as the values they stand for."""
    if case["codes"] == "fp8":
        values = codes.view(_F8)
    else:
        values = (codes.float().view(*scale.shape, -1) * scale[..., None]).to(_TYPES[case["type"]]).view(codes.shape)
    out = {"values": values, "scale": scale}
    if total is not None:
        out["sum"] = total
    return out


def _norm(s):
    x = s["x"].float()
    if s["more"] is not None:
        x = x + s["more"].float()
    n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * s["weight"].float()
    groups = n.view(n.shape[0], -1, s["group"] or n.shape[1])
    scale = groups.abs().amax(-1) / _QMAX[s["codes"]]
    codes = _encode(groups / scale[..., None], s["codes"]).view(n.shape)
    return _norm_outputs(x.to(s["x"].dtype) if s["more"] is not None else None, codes, scale, s)


def _product(s):
    y = _value(s["a"]) @ _value(s["w"]).t()
    return (y * (s["a_scale"][:, None] * s["w_scale"])).to(_TYPES[s["type"]])


def _append_side(s, name, ids, position, touched, fresh, index):
    """Writes one side's (keys' or values') new tokens into the pages `ids` [batch, slots]."""
    qmax = _QMAX[s["codes"]]
    pool, scales, x = s[name], s[name + "_scale"], s["new_" + name]
    batch, kv, _, head = x.shape
    x = x.float().gather(2, index.view(batch, 1, -1, 1).expand(-1, kv, -1, head))
    x = x.view(batch, kv, *position.shape[1:], head).transpose(1, 2)  # [batch, slots, kv, page, head]
    x = torch.where(fresh[:, :, None, :, None], x, 0.0)
    old, had = pool[ids], scales[ids]
    held = (position < s["past"].view(-1, 1, 1))
    before = torch.where(held.any(-1)[..., None], had, 0.0)
    scale = torch.maximum(before, x.abs().amax((-1, -2)) / qmax)
    grown = scale > before
    again = _encode(_value(old) * (before / scale)[..., None, None], s["codes"])
    kept = torch.where((grown[..., None] & held[:, :, None, :])[..., None], again, old)
    codes = torch.where(fresh[:, :, None, :, None], _encode(x / scale[..., None, None], s["codes"]), kept)
    live = touched[:, :, None]
    pool[ids] = torch.where(live[..., None, None], codes, old)
    scales[ids] = torch.where(live, scale, had)


def _append(s):
    page, new = s["page"], s["new_k"].shape[2]
    slots = (new + page - 2) // page + 1
    first = s["past"] // page
    slot = first[:, None] + torch.arange(slots, device="cuda")
    # positions of the touched pages' rows, and which new token each one is
    position = slot[:, :, None] * page + torch.arange(page, device="cuda")
    index = position - s["past"].view(-1, 1, 1)
    fresh = (index >= 0) & (index < s["new"].view(-1, 1, 1))
    touched = fresh.any(-1)
    ids = s["table"].gather(1, slot.clamp(max=s["table"].shape[1] - 1))
    ids = torch.where(touched, ids, 0).long()
    index = index.clamp(0, new - 1)
    _append_side(s, "k", ids, position, touched, fresh, index)
    _append_side(s, "v", ids, position, touched, fresh, index)
    return _append_outputs(s)


def _append_outputs(s):
    """The updated cache; 8-bit floats as such, whole codes as the values they stand for."""
    if s["codes"] == "fp8":
        return {"k": s["k"].view(_F8), "v": s["v"].view(_F8), "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    t = _TYPES[s["type"]]
    return {"k": (s["k"].float() * s["k_scale"][:, :, None, None]).to(t),
            "v": (s["v"].float() * s["v_scale"][:, :, None, None]).to(t),
            "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _gathered(s, name, length):
    """One side of the cache, sequence by sequence, in 32 bits: [batch, kv_heads, length, head]."""
    ids = s["table"].long()
    v = _value(s[name][ids]) * s[name + "_scale"][ids][..., None, None]
    return v.transpose(1, 2).reshape(ids.shape[0], v.shape[2], length, v.shape[-1])


def _attention(s):
    batch, heads, new, head = s["q"].shape
    kv, length = s["kv_heads"], s["table"].shape[1] * s["page"]
    k, v = _gathered(s, "k", length), _gathered(s, "v", length)
    q = s["q"].float().view(batch, kv, -1, head)
    scores = (q @ k.transpose(-1, -2)).mul_(1.0 / math.sqrt(head)).view(batch, heads, new, length)
    at = torch.arange(new, device="cuda")
    p = s["past"].view(-1, 1, 1, 1) + at.view(-1, 1)
    j = torch.arange(length, device="cuda")
    seen = (j <= p) & (at < s["new"].view(-1, 1)).view(batch, 1, new, 1)
    if s["window"] >= 0:
        seen &= (p - j <= s["window"]) | (j < s["sinks"])
    scores = scores.masked_fill_(~seen, -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min))
    y = e.view(batch, kv, -1, length) @ v
    y = y.view(batch, heads, new, head) / e.sum(-1, keepdim=True).clamp(min=1e-30)
    return y.to(s["q"].dtype)


# ---------------------------------------------------------------------------
# The package's operators
# ---------------------------------------------------------------------------


def _package():
    if "onnx_light_b200" not in sys.modules:
        folder = os.path.join(os.getcwd(), "onnx-light_b200")
        spec = importlib.util.spec_from_file_location("onnx_light_b200", os.path.join(folder, "__init__.py"),
                                                      submodule_search_locations=[folder])
        sys.modules["onnx_light_b200"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["onnx_light_b200"])
    return sys.modules["onnx_light_b200"]


def _run_own(s):
    b2 = _package()
    kind = b2.FLOAT8E4M3FN if s["codes"] == "fp8" else b2.INT8
    if s["op"] == "norm":
        r = b2.RMSNormalizationQuantize()(s["x"], s["weight"], residual=s["more"], epsilon=1e-5,
                                          dtype=kind, group_size=s["group"])
        codes = r.Y.data if s["codes"] == "fp8" else r.Y
        return _norm_outputs(r.sum, codes, r.Y_scale, s)
    if s["op"] == "product":
        a, w = s["a"], s["w"]
        if s["codes"] == "fp8":
            a, w = b2.QTensor(a, kind, a.shape), b2.QTensor(w, kind, w.shape)
        return b2.ScaledMatMul()(a, s["a_scale"], w, s["w_scale"], dtype=_TYPES[s["type"]])
    cache = b2.QuantizedKVCache(s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], s["past"], kind)
    if s["op"] == "append":
        b2.KVCacheAppend()(s["new_k"], s["new_v"], cache, new_lengths=s["new"])
        return _append_outputs(s)
    attrs = b2.CacheAttributes(is_causal=True, left_window_size=s["window"], sink_tokens=s["sinks"])
    return b2.QuantizedCacheAttention()(s["q"], cache, attrs, new_lengths=s["new"])


def run(state):
    if own:
        return _run_own(state)
    return {"norm": _norm, "product": _product, "append": _append, "attention": _attention}[state["op"]](state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    size = 4 if case["type"] == "float32" else 2
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        scales = case["rows"] * (case["width"] // case["group"] if case["group"] else 1)
        return {"bytes": n * (size * (3 if case["residual"] else 1) + 1) + case["width"] * size + 4 * scales,
                "flops": 8 * n}
    if case["op"] == "product":
        m, n, k = case["rows"], case["columns"], case["inner"]
        return {"bytes": (m + n) * k + 2 * m * n + 4 * (m + n), "flops": 2 * m * n * k}
    past, new = _lengths(case)
    kv, head, page = case["kv_heads"], case["head"], case["page"]
    if case["op"] == "append":
        pages = sum((p + n - 1) // page - p // page + 1 for p, n in zip(past, new))
        return {"bytes": 2 * kv * (sum(new) * head * 3 + 4 * pages), "flops": 4 * kv * head * sum(new)}
    w, sinks, pairs, tokens = case["window"], case["sinks"], 0, 0
    for p, n in zip(past, new):
        if w < 0:
            pairs += n * p + n * (n + 1) // 2
            tokens += p + n
            continue
        start = max(0, p - w)  # the first query's window
        tokens += p + n - start + min(sinks, start)
        for i in range(n):
            edge = max(0, p + i - w)
            pairs += p + i + 1 - edge + min(sinks, edge)
    return {"bytes": 2 * kv * tokens * head + 2 * case["heads"] * head * (sum(new) + case["batch"] * case["new"]),
            "flops": 4 * case["heads"] * head * pairs}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------


def _nearest(v, kind):
    """v on the grid of the 8-bit type, ties to even, in 64 bits."""
    if kind == "int8":
        return torch.round(v).clamp(-127, 127)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def _exact_norm(s):
    qmax, width = _QMAX[s["codes"]], s["x"].shape[1]
    h = s["x"].double()
    if s["more"] is not None:
        h = h + s["more"].double()
    rms = ((h ** 2).sum(1) / width + 1e-5).sqrt()
    n = h / rms[:, None] * s["weight"].double()
    parts = n.reshape(n.shape[0], -1, s["group"] if s["group"] else width)
    scale = parts.abs().max(2).values / qmax
    q = _nearest(parts / scale.unsqueeze(2), s["codes"])
    out = {"values": (q if s["codes"] == "fp8" else q * scale.unsqueeze(2)).reshape(n.shape), "scale": scale}
    if s["more"] is not None:
        out["sum"] = h
    return out


def _exact_append(s):
    qmax = _QMAX[s["codes"]]
    past, new, page = s["past"].tolist(), s["new"].tolist(), s["page"]
    out = {}
    for name in ("k", "v"):
        pool, scales = s[name], s[name + "_scale"].double()
        pool = (pool.view(_F8) if s["codes"] == "fp8" else pool).double()
        for b, (p, n) in enumerate(zip(past, new)):
            rows = s["new_" + name][b].double()
            for slot in range(p // page, (p + n - 1) // page + 1):
                lo, hi = max(p, slot * page), min(p + n, (slot + 1) * page)
                at = int(s["table"][b, slot])
                x = rows[:, lo - p:hi - p]
                before = scales[at].clone() if lo > slot * page else torch.zeros_like(scales[at])
                now = torch.maximum(before, x.abs().amax((1, 2)) / qmax)
                older = lo - slot * page
                if older:
                    again = _nearest(pool[at, :, :older] * (before / now)[:, None, None], s["codes"])
                    pool[at, :, :older] = torch.where((now > before)[:, None, None], again, pool[at, :, :older])
                pool[at, :, older:older + hi - lo] = _nearest(x / now[:, None, None], s["codes"])
                scales[at] = now
        out[name] = pool if s["codes"] == "fp8" else pool * scales[:, :, None, None]
        out[name + "_scale"] = scales
    return out


def _exact_attention(s):
    batch, heads, new, head = s["q"].shape
    kv, page = s["kv_heads"], s["page"]
    y = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, (p, n) in enumerate(zip(s["past"].tolist(), s["new"].tolist())):
        total = p + n
        ids = s["table"][b, :-(-total // page)].long()
        sides = []
        for name in ("k", "v"):
            pool = s[name][ids]
            pool = (pool.view(_F8) if s["codes"] == "fp8" else pool).double()
            pool = pool * s[name + "_scale"][ids].double()[:, :, None, None]
            sides.append(pool.permute(1, 0, 2, 3).reshape(kv, -1, head)[:, :total])
        j = torch.arange(total, device="cuda")
        for lo in range(0, n, 256):
            hi = min(n, lo + 256)
            at = p + torch.arange(lo, hi, device="cuda")[:, None]
            seen = j <= at
            if s["window"] >= 0:
                seen = seen & ((at - j <= s["window"]) | (j < s["sinks"]))
            q = s["q"][b, :, lo:hi].double().reshape(kv, -1, hi - lo, head)
            z = torch.einsum("kgsd,kjd->kgsj", q, sides[0]) / math.sqrt(head)
            z = torch.softmax(z.masked_fill(~seen, -math.inf), -1)
            y[b, :, lo:hi] = torch.einsum("kgsj,kjd->kgsd", z, sides[1]).reshape(heads, hi - lo, head)
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "attention":
        return _exact_attention(s)
    a, w = ((s[n].view(_F8) if s["codes"] == "fp8" else s[n]).double() for n in ("a", "w"))
    return torch.einsum("mk,nk->mn", a, w) * s["a_scale"].double()[:, None] * s["w_scale"].double()
