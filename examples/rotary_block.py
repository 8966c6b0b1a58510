"""One encoder block with rotary positions on the general operators, next to the engine's own attention.

The arctic-embed-s encoder has learned positions and projections tied to its shapes. This block keeps its sizes (384
hidden, 12 heads of 32, 1,536 inside) and its packed ragged batches, but norms its queries and keys for each head,
turns them by their positions, and ends in scores over a vocabulary:

    qkv    = linear_i8(x, W_qkv)                     quantized per token on the way, float out
    q, k   = qk_norm_rope(q, k, table, cu)           in place, where the projection left them
    ctx    = attention_f32(qkv, cu)                  the engine's segment-masked attention
    x      = x + linear_i8(ctx, W_out, inv_smooth)
    x      = x + linear_i8(gelu(linear_i8(x, W_up)), W_down)
    scores = matmul_i8(quantized x, word table)      int8 rows and scales as an `.ae8` pack holds them

Run it on a B200:  python examples/rotary_block.py
"""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "snowflake-arctic-embed-s-rust_b200"))

from arctic_embed_s_int8 import Engine, rope_table  # noqa: E402

HIDDEN, INTER, HEADS, DIM, VOCAB = 384, 1536, 12, 32, 30522


def int8_weights(n: int, k: int, generator) -> dict:
    """Random weights of a linear layer, quantized for each output channel."""
    w = torch.randn(n, k, generator=generator) / k ** 0.5
    scale = w.abs().amax(1) / 127
    return {"w": (w / scale[:, None]).round().to(torch.int8).cuda(), "scale": scale.cuda(),
            "bias": (0.02 * torch.randn(n, generator=generator)).cuda()}


def random_block(seed: int = 0) -> dict:
    g = torch.Generator().manual_seed(seed)
    return {"qkv": int8_weights(3 * HIDDEN, HIDDEN, g), "out": int8_weights(HIDDEN, HIDDEN, g),
            "up": int8_weights(INTER, HIDDEN, g), "down": int8_weights(HIDDEN, INTER, g),
            "words": int8_weights(VOCAB, HIDDEN, g),
            "q_norm": (1 + 0.1 * torch.randn(DIM, generator=g)).cuda(),
            "k_norm": (1 + 0.1 * torch.randn(DIM, generator=g)).cuda(),
            "inv_smooth": torch.exp(0.3 * torch.randn(HIDDEN, generator=g)).cuda(),
            "table": torch.from_numpy(rope_table(512, DIM)).cuda()}


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """int8 rows and their scales."""
    scale = x.abs().amax(1) / 127
    return (x / scale[:, None]).round().to(torch.int8), scale


def run_block(engine: Engine, block: dict, x: torch.Tensor, cu: torch.Tensor, max_len: int) -> dict:
    """x [T, 384] float32 rows of the sequences of cu [n + 1] int32, the longest of max_len (at most 512) rows."""
    T = x.shape[0]

    def linear(rows, layer, inv_smooth=None):
        out = torch.empty(T, layer["w"].shape[0], device=x.device)
        engine.linear_i8(rows, layer["w"], layer["scale"], out, bias=layer["bias"], inv_smooth=inv_smooth)
        return out

    qkv = linear(x, block["qkv"])
    q = qkv[:, :HIDDEN].view(T, HEADS, DIM)
    k = qkv[:, HIDDEN:2 * HIDDEN].view(T, HEADS, DIM)
    engine.qk_norm_rope(q, k, q, k, block["table"], cu=cu, q_weight=block["q_norm"], k_weight=block["k_norm"])
    ctx = torch.empty_like(x)
    engine.attention_f32(qkv, cu, cu.shape[0] - 1, max_len, ctx)
    x = x + linear(ctx, block["out"], block["inv_smooth"])
    x = x + linear(torch.nn.functional.gelu(linear(x, block["up"])), block["down"])
    rows, scale = quantize(x)
    scores = torch.empty(T, VOCAB, dtype=torch.bfloat16, device=x.device)
    engine.matmul_i8(rows, scale, block["words"]["w"], block["words"]["scale"], scores)
    return {"qkv": qkv, "hidden": x, "scores": scores}


def plain_block(block: dict, x: torch.Tensor, cu: torch.Tensor) -> dict:
    """The same in 64 bits, without the int8 rounding of the activations."""
    x = x.double()

    def linear(rows, layer, inv_smooth=None):
        rows = rows if inv_smooth is None else rows * inv_smooth.double()
        return rows @ (layer["w"].double() * layer["scale"].double()[:, None]).T + layer["bias"].double()

    def turned(h, weight, at):
        h = h * (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * weight.double()
        cos, sin = block["table"].double()[at].chunk(2, -1)
        a, b = h.chunk(2, -1)
        return torch.cat([a * cos[:, None] - b * sin[:, None], b * cos[:, None] + a * sin[:, None]], -1)

    qkv = linear(x, block["qkv"])
    ctx = torch.empty_like(x)
    for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()):
        at = torch.arange(b - a, device=x.device)
        q, k, v = (t.reshape(b - a, HEADS, DIM) for t in qkv[a:b].chunk(3, -1))
        q, k = turned(q, block["q_norm"], at), turned(k, block["k_norm"], at)
        p = torch.softmax(torch.einsum("qhd,khd->hqk", q, k) / DIM ** 0.5, -1)
        ctx[a:b] = torch.einsum("hqk,khd->qhd", p, v).reshape(b - a, HIDDEN)
        qkv[a:b] = torch.cat([t.reshape(b - a, HIDDEN) for t in (q, k, v)], -1)
    x = x + linear(ctx, block["out"], block["inv_smooth"])
    x = x + linear(torch.nn.functional.gelu(linear(x, block["up"])), block["down"])
    words = block["words"]
    return {"qkv": qkv, "hidden": x, "scores": x @ (words["w"].double() * words["scale"].double()[:, None]).T}


def main() -> None:
    engine, block = Engine(0), random_block()
    lengths = np.random.default_rng(0).integers(1, 257, 64)
    cu = torch.from_numpy(np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)).cuda()
    x = torch.randn(int(lengths.sum()), HIDDEN, generator=torch.Generator().manual_seed(1)).cuda()
    got, want = run_block(engine, block, x, cu, int(lengths.max())), plain_block(block, x, cu)
    engine.sync()
    for name, value in got.items():
        off = (value.double() - want[name]).norm() / want[name].norm()
        print(f"{name}: {tuple(value.shape)}, {float(off):.4f} of the 64-bit block's norm away")


if __name__ == "__main__":
    main()
