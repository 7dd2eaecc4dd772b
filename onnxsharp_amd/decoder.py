"""An example: a decoder block from the layers of lm_layers, over prompts, pieces of prompts
and single tokens of many sequences in one call.

    x -> RMS norm, 8 bits -> q, k, v -> window attention over the pages -> RMS norm, 8
    bits -> output product -> add, RMS norm, 8 bits -> up, SiLU -> RMS norm, 8 bits ->
    down, add

Six products' worth of operands move in 8 bits; the residual stream stays in 16.  The
attention's and the feed-forward's inner outputs are normalized before they are rounded
to 8 bits, so one operator makes every 8-bit row.  The block knows positions through the
causal window alone; it is no released model's architecture.

`python -m onnxsharp_amd.decoder` runs a prompt and a few tokens on the GPU.
"""
from __future__ import annotations

from typing import Optional

import torch

from .lm_layers import PagedKvCache, QuantMatMulLayer, RmsNormQuantLayer, WindowAttentionLayer

_TOP = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}


def quantize_weight(w: torch.Tensor, q_type: str = "e4m3"):
    """w [n, k] in 8 bits with a scale per output, as QuantMatMulLayer takes it."""
    dtype, top = _TOP[q_type]
    scale = w.float().abs().amax(1).clamp(min=1e-30) / top
    v = (w.float() / scale[:, None]).clamp(-top, top)
    return (v.round() if q_type == "int8" else v).to(dtype), scale


class DecoderBlock:
    """Weights in float, by name: qkv [(q_heads + 2 kv_heads) head_dim, width], out [width,
    q_heads head_dim], up [hidden, width], down [width, hidden], and the norms' gammas norm1
    [width], norm2 [q_heads head_dim], norm3 [width], norm4 [hidden] (of `dtype`)."""

    def __init__(self, weights: dict, q_heads: int, kv_heads: int, head_dim: int, window: Optional[int] = None,
                 sinks: int = 0, q_type: str = "e4m3", eps: float = 1e-5, dtype: torch.dtype = torch.bfloat16):
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.w = {name: quantize_weight(weights[name], q_type) for name in ("qkv", "out", "up", "down")}
        self.gamma = {name: weights[name].to(dtype) for name in ("norm1", "norm2", "norm3", "norm4")}
        self.norm = RmsNormQuantLayer(eps, q_type)
        self.matmul = QuantMatMulLayer(None, dtype)
        self.matmul_silu = QuantMatMulLayer("Silu", dtype)
        self.attention = WindowAttentionLayer(window, sinks)

    def forward(self, x: torch.Tensor, cache: PagedKvCache, cu_seqlens: torch.Tensor, kv_lens: torch.Tensor, max_q: int,
                max_kv: int) -> torch.Tensor:
        """The residual stream [tokens, width] after the block; the new tokens' keys and
        values go to their pages."""
        hq, hkv, d = self.q_heads, self.kv_heads, self.head_dim
        _, q, s = self.norm.forward(x, self.gamma["norm1"])
        qkv = self.matmul.forward(q, s, *self.w["qkv"]).view(-1, hq + 2 * hkv, d)
        o = self.attention.forward(qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:], cache, cu_seqlens, kv_lens, max_q,
                                   max_kv)
        _, q, s = self.norm.forward(o.view(-1, hq * d), self.gamma["norm2"])
        branch = self.matmul.forward(q, s, *self.w["out"])
        h, q, s = self.norm.forward(branch, self.gamma["norm3"], residual=x, out_h=branch)
        up = self.matmul_silu.forward(q, s, *self.w["up"])
        _, q, s = self.norm.forward(up, self.gamma["norm4"])
        return self.matmul.forward(q, s, *self.w["down"], residual=h, out=h)


def random_weights(width: int, hidden: int, q_heads: int, kv_heads: int, head_dim: int, device, seed: int = 0) -> dict:
    g = torch.Generator(device=device).manual_seed(seed)
    t = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    w = {"qkv": t((q_heads + 2 * kv_heads) * head_dim, width) * width ** -0.5,
         "out": t(width, q_heads * head_dim) * (q_heads * head_dim) ** -0.5, "up": t(hidden, width) * width ** -0.5,
         "down": t(width, hidden) * hidden ** -0.5}
    for name, n in (("norm1", width), ("norm2", q_heads * head_dim), ("norm3", width), ("norm4", hidden)):
        w[name] = 1.0 + 0.1 * t(n)
    return w


def main(tokens: int = 300, steps: int = 8) -> None:
    """A prompt through one block, then single tokens."""
    dev, page = torch.device("cuda"), 16
    width, hidden, hq, hkv, d = 1024, 2048, 16, 4, 64
    block = DecoderBlock(random_weights(width, hidden, hq, hkv, d, dev), hq, hkv, d, window=128, sinks=4)
    n = (tokens + steps + page - 1) // page
    pages = torch.zeros(2, n, page, hkv, d, dtype=torch.bfloat16, device=dev)
    cache = PagedKvCache(pages[0], pages[1], torch.randperm(n, device=dev).to(torch.int32)[None])
    x = torch.randn(tokens, width, device=dev).bfloat16()
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    h = block.forward(x, cache, ints(0, tokens), ints(tokens), tokens, tokens)
    print(f"prompt of {tokens}: rms {h.float().pow(2).mean().sqrt().item():.4f}")
    for i in range(steps):
        total = tokens + i + 1
        h = block.forward(h[-1:], cache, ints(0, 1), ints(total), 1, total)
        print(f"token {total}: rms {h.float().pow(2).mean().sqrt().item():.4f}")


if __name__ == "__main__":
    main()
