"""A decoder that holds its activations between operators and its KV cache in 8 bits.

Each layer: RMSNormalizationQuantize -> ScaledMatMul (q, k, v) -> RotaryEmbedding -> KVCacheAppend ->
QuantizedCacheAttention -> DequantizeMatMul (int4 output projection) -> RMSNormalizationQuantize with
the residual's addition -> ScaledMatMul (gate, up) -> SwiGLU -> DequantizeMatMul (int4 down
projection).  Weights are random.  The prompts have different lengths; then each step decodes one
token per sequence, replayed as a CUDA graph.

    python examples/quantized_decoder_step.py [--batch 4] [--prompt 300] [--steps 64] [--codes fp8]
"""
from __future__ import annotations

import argparse
import importlib.util
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def load_package():
    """The package directory onnx-light_b200/ as module onnx_light_b200."""
    if "onnx_light_b200" not in sys.modules:
        folder = os.path.join(ROOT, "onnx-light_b200")
        spec = importlib.util.spec_from_file_location(
            "onnx_light_b200", os.path.join(folder, "__init__.py"), submodule_search_locations=[folder])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["onnx_light_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["onnx_light_b200"]


class Config:
    def __init__(self, hidden=1024, heads=8, kv_heads=2, head=128, inner=2816, layers=2,
                 positions=1024, dtype=torch.float16):
        self.hidden, self.heads, self.kv_heads, self.head = hidden, heads, kv_heads, head
        self.inner, self.layers, self.positions, self.dtype = inner, layers, positions, dtype


def quantize_rows(w: torch.Tensor, kind: int, b2):
    """[N, K] weight -> 8-bit codes and one scale per row."""
    top = 127.0 if kind == b2.INT8 else 448.0
    s = w.abs().amax(1) / top
    q = w / s[:, None]
    if kind == b2.INT8:
        return q.round().to(torch.int8), s
    return b2.QTensor(q.to(torch.float8_e4m3fn).view(torch.uint8), kind, tuple(w.shape)), s


def quantize_int4(w: torch.Tensor, b2, block: int = 128):
    """[K, N] weight -> packed int4 codes with FLOAT16 scales for blocks of `block` rows."""
    k, n = w.shape
    s = (w.view(k // block, block, n).abs().amax(1) / 7.0).half()
    q = (w.view(k // block, block, n) / s.float()[:, None]).round().clamp(-8, 7).to(torch.int32)
    q = q.view(-1) & 15
    packed = (q[0::2] | (q[1::2] << 4)).to(torch.uint8)
    return b2.QTensor(packed, 22, (k, n)), s  # 22: ONNX INT4


class Layer:
    """One decoder layer's weights, drawn at random; `plain` keeps them in fp32 for comparison."""

    def __init__(self, cfg: Config, kind: int, b2, gen: torch.Generator):
        def draw(n, k):
            return torch.randn(n, k, generator=gen, device="cuda") / k ** 0.5

        def norm():
            return (1 + 0.1 * torch.randn(cfg.hidden, generator=gen, device="cuda")).to(cfg.dtype)

        q, kv = cfg.heads * cfg.head, cfg.kv_heads * cfg.head
        self.plain = {"qkv": draw(q + 2 * kv, cfg.hidden), "out": draw(cfg.hidden, q),
                      "gate_up": draw(2 * cfg.inner, cfg.hidden), "down": draw(cfg.hidden, cfg.inner)}
        self.norm1, self.norm2 = norm(), norm()
        self.qkv, self.qkv_scale = quantize_rows(self.plain["qkv"], kind, b2)
        self.gate_up, self.gate_up_scale = quantize_rows(self.plain["gate_up"], kind, b2)
        self.out, self.out_scale = quantize_int4(self.plain["out"].t().contiguous(), b2)
        self.down, self.down_scale = quantize_int4(self.plain["down"].t().contiguous(), b2)


class Decoder:
    def __init__(self, cfg: Config, batch: int, codes: str = "fp8", page_size: int = 32, seed: int = 0):
        b2 = load_package()
        self.b2, self.cfg, self.kind = b2, cfg, b2.INT8 if codes == "int8" else b2.FLOAT8E4M3FN
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        self.layers = [Layer(cfg, self.kind, b2, gen) for _ in range(cfg.layers)]
        self.caches = [b2.QuantizedKVCache.allocate(batch, cfg.kv_heads, cfg.positions, cfg.head,
                                                    page_size, self.kind) for _ in range(cfg.layers)]
        for cache in self.caches[1:]:  # one table and one count of tokens serve every layer
            cache.block_table, cache.lengths = self.caches[0].block_table, self.caches[0].lengths
        angle = torch.arange(cfg.positions, device="cuda")[:, None] / 10000.0 ** (
            torch.arange(0, cfg.head, 2, device="cuda") / cfg.head)
        self.cos, self.sin = angle.cos().to(cfg.dtype), angle.sin().to(cfg.dtype)
        self.norm, self.mm, self.rotary = b2.RMSNormalizationQuantize(), b2.ScaledMatMul(), b2.RotaryEmbedding()
        self.append, self.attend = b2.KVCacheAppend(), b2.QuantizedCacheAttention()
        self.int4, self.swiglu = b2.DequantizeMatMul(), b2.SwiGLU()

    def step(self, x: torch.Tensor, new_lengths: torch.Tensor) -> torch.Tensor:
        """x: [batch, new, hidden], of which new_lengths rows count -> the layers' output."""
        cfg, b2 = self.cfg, self.b2
        batch, new, _ = x.shape
        positions = self.caches[0].lengths.long()[:, None] + torch.arange(new, device="cuda")
        positions = positions.clamp(max=cfg.positions - 1)
        q, kv = cfg.heads * cfg.head, cfg.kv_heads * cfg.head
        total, branch = x, None
        for layer, cache in zip(self.layers, self.caches):
            h = self.norm(total, layer.norm1, residual=branch, dtype=self.kind)
            total = h.sum if branch is not None else total
            y = self.mm(h.Y, h.Y_scale, layer.qkv, layer.qkv_scale, dtype=cfg.dtype)
            query, key, value = (t.contiguous() for t in y.split((q, kv, kv), -1))
            query = self.rotary(query, self.cos, self.sin, positions, num_heads=cfg.heads)
            key = self.rotary(key, self.cos, self.sin, positions, num_heads=cfg.kv_heads)
            self.append(key, value, cache, new_lengths=new_lengths)
            a = self.attend(query, cache, new_lengths=new_lengths)
            branch = self.int4(a, layer.out, layer.out_scale)
            h = self.norm(total, layer.norm2, residual=branch, dtype=self.kind)
            total = h.sum
            y = self.mm(h.Y, h.Y_scale, layer.gate_up, layer.gate_up_scale, dtype=cfg.dtype)
            gate, up = (t.contiguous() for t in y.chunk(2, -1))
            branch = self.int4(self.swiglu(gate, up), layer.down, layer.down_scale)
        self.caches[0].advance(new_lengths)
        return total + branch


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=300)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--codes", choices=("fp8", "int8"), default="fp8")
    args = ap.parse_args()
    cfg = Config(positions=args.prompt + args.steps + 8)
    model = Decoder(cfg, args.batch, args.codes)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    prompt = torch.randn(args.batch, args.prompt, cfg.hidden, generator=gen, device="cuda").to(cfg.dtype)
    counts = torch.tensor([max(1, args.prompt - 37 * b) for b in range(args.batch)], dtype=torch.int32,
                          device="cuda")
    y = model.step(prompt, counts)
    x = y[torch.arange(args.batch, device="cuda"), counts.long() - 1][:, None].contiguous()
    one = torch.ones(args.batch, dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        x.copy_(torch.nn.functional.normalize(model.step(x, one), dim=-1) * cfg.hidden ** 0.5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        x.copy_(torch.nn.functional.normalize(model.step(x, one), dim=-1) * cfg.hidden ** 0.5)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    for _ in range(args.steps - 1):
        graph.replay()
    end.record()
    torch.cuda.synchronize()
    us = start.elapsed_time(end) * 1e3 / max(1, args.steps - 1)
    print(f"{args.codes}: {args.batch} sequences, {cfg.layers} layers, tokens held "
          f"{model.caches[0].lengths.tolist()}, {us:.1f} us a step")
    assert bool(torch.isfinite(x).all())


if __name__ == "__main__":
    main()
