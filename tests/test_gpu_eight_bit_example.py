"""The example decoder with 8-bit activations and cache: against the same layers in plain fp32, and a
prompt in one call against the same prompt token by token."""
import importlib.util
import math
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example(b2):
    spec = importlib.util.spec_from_file_location(
        "quantized_decoder_step", os.path.join(ROOT, "examples", "quantized_decoder_step.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def rotate(x, positions, head):
    angle = positions[..., None].double() / 10000.0 ** (torch.arange(0, head, 2, device="cuda") / head)
    c, s = angle.cos()[:, :, None], angle.sin()[:, :, None]
    a, b = x.chunk(2, -1)
    return torch.cat([c * a - s * b, s * a + c * b], -1)


def plain(model, x):
    """All the tokens of each sequence at once, in 64 bits, with the weights before quantization."""
    cfg = model.cfg
    B, S, _ = x.shape
    x = x.double()
    positions = torch.arange(S, device="cuda")[None].expand(B, S)

    def norm(v, w):
        return v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-5) * w.double()

    for layer in model.layers:
        w = {k: v.double() for k, v in layer.plain.items()}
        y = norm(x, layer.norm1) @ w["qkv"].t()
        q, k, v = y.split((cfg.heads * cfg.head, cfg.kv_heads * cfg.head, cfg.kv_heads * cfg.head), -1)
        q = rotate(q.view(B, S, cfg.heads, cfg.head), positions, cfg.head)
        k = rotate(k.view(B, S, cfg.kv_heads, cfg.head), positions, cfg.head)
        g = cfg.heads // cfg.kv_heads
        k, v = k.repeat_interleave(g, 2), v.view(B, S, cfg.kv_heads, cfg.head).repeat_interleave(g, 2)
        z = torch.einsum("bihd,bjhd->bhij", q, k) / math.sqrt(cfg.head)
        z = z.masked_fill(torch.ones(S, S, dtype=torch.bool, device="cuda").triu(1), -math.inf)
        x = x + torch.einsum("bhij,bjhd->bihd", z.softmax(-1), v).reshape(B, S, -1) @ w["out"].t()
        gate, up = (norm(x, layer.norm2) @ w["gate_up"].t()).chunk(2, -1)
        x = x + (gate * torch.sigmoid(gate) * up) @ w["down"].t()
    return x


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_prompt_and_decode_against_plain_layers(example, codes):
    cfg = example.Config(hidden=512, heads=4, kv_heads=2, head=128, inner=1024, layers=2, positions=256)
    model = example.Decoder(cfg, 2, codes)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    x = torch.randn(2, 90, cfg.hidden, generator=g, device="cuda").half()
    want = plain(model, x)
    # int4 weights (two projections a layer) leave about 0.12 of each branch, 8-bit codes 0.01 to
    # 0.03; a branch is of the residual's size at most, so 0.2 of the output bounds two layers
    first = model.step(x[:, :70].contiguous(), torch.tensor([70, 70], dtype=torch.int32, device="cuda"))
    assert rel(first, want[:, :70]) < 0.2
    one = torch.ones(2, dtype=torch.int32, device="cuda")
    for i in range(70, 90):
        y = model.step(x[:, i:i + 1].contiguous(), one)
        assert rel(y, want[:, i:i + 1]) < 0.2
    assert model.caches[0].lengths.tolist() == [90, 90]


@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_ragged_prompts_equal_separate_ones(example, codes):
    """Sequences of different lengths in one call give what each gives alone: the same kernels on the
    same codes, up to the order of sums (fp16 roundings of the output, 2^-10, over two layers)."""
    cfg = example.Config(hidden=512, heads=4, kv_heads=1, head=64, inner=1024, layers=2, positions=128)
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    x = torch.randn(3, 50, cfg.hidden, generator=g, device="cuda").half()
    lengths = [50, 1, 33]
    together = example.Decoder(cfg, 3, codes).step(x, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    for b, n in enumerate(lengths):
        alone = example.Decoder(cfg, 1, codes).step(x[b:b + 1, :n].contiguous(),
                                                    torch.tensor([n], dtype=torch.int32, device="cuda"))
        assert rel(together[b, :n], alone[0]) < 0.02  # codes next to a tie may fall either way


def test_example_runs(example, monkeypatch, capsys):
    monkeypatch.setattr("sys.argv", ["quantized_decoder_step.py", "--steps", "8", "--prompt", "90"])
    example.main()
    assert "us a step" in capsys.readouterr().out
