"""A decoder-only language model that runs on 4-bit weights and a paged key-value cache: what the
text-generation operators are for, in one place.

    python comfy-kitchen_amd/samples/text_generation.py        # random weights, a few tokens

A prompt goes through `ck.window_attention` and leaves its keys and values in a `ck.PagedKVCache`;
then every step runs `F.linear` on GroupInt4Layout weights (`ck.linear_int4`), `ck.apply_rope`, one
`PagedKVCache.write` and one `PagedKVCache.attend` a layer for all sequences together.  Several
continuations of one prompt fork its sequence instead of copying the cache.
"""
from __future__ import annotations

import sys
from dataclasses import dataclass
from pathlib import Path

import torch
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import comfy_kitchen as ck  # noqa: E402
from comfy_kitchen.tensor import QuantizedTensor  # noqa: E402


@dataclass(frozen=True)
class Config:
    vocab: int = 1000
    layers: int = 2
    hidden: int = 512
    heads: int = 8
    kv_heads: int = 2
    head_dim: int = 64
    ffn: int = 1024
    window: int = 0  # of attention; 0: none
    sinks: int = 0
    group_size: int = 128
    eps: float = 1e-6
    rope_base: float = 10000.0


def rope_matrices(positions: torch.Tensor, dim: int, base: float) -> torch.Tensor:
    """The 2x2 rotations of positions, [..., dim / 2, 2, 2] fp32."""
    rate = base ** (-torch.arange(0, dim, 2, device=positions.device, dtype=torch.float32) / dim)
    angle = positions[..., None].float() * rate
    c, s = angle.cos(), angle.sin()
    return torch.stack((c, -s, s, c), -1).reshape(*angle.shape, 2, 2)


class TextDecoder:
    """weights: a dict of [out, in] matrices and norms by name; the matrices are quantized here."""

    def __init__(self, config: Config, weights: dict[str, torch.Tensor], pages: int = 256, page_size: int = 16,
                 cache_dtype: torch.dtype | None = None, cache_scale: float | None = None):
        self.config = config
        self.embedding = weights["embedding"]
        dtype, device = self.embedding.dtype, self.embedding.device
        self.weights = {name: w if name == "embedding" or w.dim() == 1 else
                        QuantizedTensor.from_float(w, "GroupInt4Layout", group_size=config.group_size)
                        for name, w in weights.items()}
        self.cache = ck.PagedKVCache(config.layers, pages, page_size, config.kv_heads, config.head_dim,
                                     cache_dtype or dtype, device, cache_scale, cache_scale)

    @staticmethod
    def random_weights(config: Config, seed: int = 0, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)

        def matrix(rows, cols):
            return (torch.randn(rows, cols, generator=g, device=device) * cols ** -0.5).to(dtype)

        c = config
        w = {"embedding": torch.randn(c.vocab, c.hidden, generator=g, device=device).to(dtype),
             "norm": torch.ones(c.hidden, dtype=dtype, device=device), "head": matrix(c.vocab, c.hidden)}
        for i in range(c.layers):
            w[f"{i}.norm1"] = torch.ones(c.hidden, dtype=dtype, device=device)
            w[f"{i}.norm2"] = torch.ones(c.hidden, dtype=dtype, device=device)
            w[f"{i}.qkv"] = matrix((c.heads + 2 * c.kv_heads) * c.head_dim, c.hidden)
            w[f"{i}.out"] = matrix(c.hidden, c.heads * c.head_dim)
            w[f"{i}.up"] = matrix(2 * c.ffn, c.hidden)
            w[f"{i}.down"] = matrix(c.hidden, c.ffn)
        return w

    def _norm(self, x: torch.Tensor, name: str) -> torch.Tensor:
        y = x.float()
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + self.config.eps)
        return y.to(x.dtype) * self.weights[name]

    def _layers(self, x: torch.Tensor, positions: torch.Tensor, attend) -> torch.Tensor:
        """x [T, hidden] at `positions` [T] through all layers; attend(layer, q, k, v) of [T, heads,
        head_dim] tensors stores k and v and gives [T, heads, head_dim]."""
        c, w = self.config, self.weights
        freqs = rope_matrices(positions, c.head_dim, c.rope_base)[None, :, None]  # [1, T, 1, dim / 2, 2, 2]
        for i in range(c.layers):
            qkv = F.linear(self._norm(x, f"{i}.norm1"), w[f"{i}.qkv"]).unflatten(-1, (-1, c.head_dim))
            q, k, v = qkv.split((c.heads, c.kv_heads, c.kv_heads), 1)
            q, k = (t[0] for t in ck.apply_rope(q[None], k[None], freqs))
            x = x + F.linear(attend(i, q, k, v).flatten(1), w[f"{i}.out"])
            gate, up = F.linear(self._norm(x, f"{i}.norm2"), w[f"{i}.up"]).chunk(2, -1)
            x = x + F.linear(F.silu(gate) * up, w[f"{i}.down"])
        return self._norm(x, "norm")

    def prompt(self, tokens: torch.Tensor) -> tuple[int, torch.Tensor]:
        """A new sequence that holds `tokens` [T]: (its number, the logits behind its last token)."""
        c, n = self.config, tokens.shape[0]
        sequence = self.cache.add()
        slots = self.cache.append([sequence], n)

        def attend(layer, q, k, v):
            self.cache.write(layer, k, v, slots)
            return ck.window_attention(q[None], k[None], v[None], c.window, c.sinks)[0]

        x = self._layers(self.embedding[tokens], torch.arange(n, device=tokens.device), attend)
        return sequence, F.linear(x[-1:], self.weights["head"])[0]

    def step(self, sequences: list[int], tokens: torch.Tensor) -> torch.Tensor:
        """Append one token to each sequence: the logits behind them, [B, vocab]."""
        c = self.config
        slots = self.cache.append(sequences)
        table, lengths = self.cache.tables(sequences)

        def attend(layer, q, k, v):
            self.cache.write(layer, k, v, slots)
            return self.cache.attend(layer, q, table, lengths, window=c.window, sinks=c.sinks)

        x = self._layers(self.embedding[tokens], lengths - 1, attend)
        if c.window:
            for s in sequences:  # pages that left the window
                self.cache.trim(s, c.window, c.sinks)
        return F.linear(x, self.weights["head"])

    def generate(self, tokens: torch.Tensor, steps: int, samples: int = 1, temperature: float = 1.0,
                 generator: torch.Generator | None = None) -> torch.Tensor:
        """`samples` continuations of a prompt, [samples, steps]."""
        first, logits = self.prompt(tokens)
        sequences = [first] + [self.cache.fork(first) for _ in range(samples - 1)]
        logits, out = logits.expand(samples, -1), []
        for i in range(steps):
            p = torch.softmax(logits.float() / temperature, -1)
            out.append(torch.multinomial(p, 1, generator=generator)[:, 0])
            if i + 1 < steps:
                logits = self.step(sequences, out[-1])
        for s in sequences:
            self.cache.free(s)
        return torch.stack(out, 1)


def main() -> None:
    config = Config(window=64, sinks=4)
    model = TextDecoder(config, TextDecoder.random_weights(config))
    prompt = torch.randint(0, config.vocab, (100,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    out = model.generate(prompt, steps=20, samples=4, generator=torch.Generator(device="cuda").manual_seed(2))
    for row in out.tolist():
        print(*row)


if __name__ == "__main__":
    main()
