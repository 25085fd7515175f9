"""A decoder-only language model that runs on 4-bit weights and a paged key-value cache: what the
text-generation operators are for, in one place.

    python comfy-kitchen_amd/samples/text_generation.py        # random weights, a few tokens

A prompt goes through `ck.window_attention` and leaves its keys and values in a `ck.PagedKVCache`;
then every step runs, a layer and for all sequences together, `ck.rms_norm` with the residual's addition,
`F.linear` on GroupInt4Layout weights (`ck.linear_int4`), one `PagedKVCache.write_rope` and one
`PagedKVCache.attend`, and at its end `ck.sample_tokens`.  Several continuations of one prompt fork its
sequence instead of copying the cache, and read what they share of it once (`PagedKVCache.groups`).
With linears="mxfp8" the weights are TensorCoreMXFP8Layout, and the norms in front of linears write MXFP8.
"""
from __future__ import annotations

import sys
from dataclasses import dataclass
from pathlib import Path

import torch
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import comfy_kitchen as ck  # noqa: E402
from comfy_kitchen.tensor import QuantizedTensor, TensorCoreMXFP8Layout  # noqa: E402


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
    linears: str = "int4"  # or "mxfp8"
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
    """weights: a dict of [out, in] matrices and norms by name; the matrices are quantized here.
    share_from: bytes of K and V a layer from which on what sequences share is read once (PagedKVCache.groups; None: its default)."""

    def __init__(self, config: Config, weights: dict[str, torch.Tensor], pages: int = 256, page_size: int = 16,
                 cache_dtype: torch.dtype | None = None, cache_scale: float | None = None, share_from: int | None = None):
        self.config, self.share_from = config, share_from
        self.embedding = weights["embedding"]
        dtype, device = self.embedding.dtype, self.embedding.device
        layout, how = {"int4": ("GroupInt4Layout", {"group_size": config.group_size}), "mxfp8": ("TensorCoreMXFP8Layout", {})}[config.linears]
        self.weights = {name: w if name == "embedding" or w.dim() == 1 else QuantizedTensor.from_float(w, layout, **how)
                        for name, w in weights.items()}
        self.rates = ck.rope_rates(config.head_dim, config.rope_base, device=device)
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

    def _norm(self, x: torch.Tensor, name: str, residual: torch.Tensor | None = None):
        """What the linears behind the norm take, and the sum x + residual."""
        w, eps = self.weights[name], self.config.eps
        if self.config.linears == "mxfp8":
            codes, scales, *h = ck.rms_norm_mxfp8(x, w, residual, eps, pad_32x=True)
            params = TensorCoreMXFP8Layout.Params(scale=scales, orig_dtype=x.dtype, orig_shape=tuple(x.shape))
            return QuantizedTensor(codes, "TensorCoreMXFP8Layout", params), h[0] if h else x
        y = ck.rms_norm(x, w, residual, eps)
        return (y, x) if residual is None else y

    def _linear(self, x: torch.Tensor, name: str) -> torch.Tensor:
        if self.config.linears == "mxfp8" and not isinstance(x, QuantizedTensor):
            x = QuantizedTensor.from_float(x, "TensorCoreMXFP8Layout")
        return F.linear(x, self.weights[name])

    def _layers(self, x: torch.Tensor, attend, rows: slice = slice(None)) -> torch.Tensor:
        """x [T, hidden] through all layers: the logits behind its `rows`.  attend(layer, q, k, v) of [T, heads,
        head_dim] tensors turns them to their positions, stores k and v and gives [T, heads, head_dim]."""
        c = self.config
        more = None  # what is still to be added to x
        for i in range(c.layers):
            y, x = self._norm(x, f"{i}.norm1") if more is None else self._norm(more, f"{i}.norm1", x)
            qkv = self._linear(y, f"{i}.qkv").unflatten(-1, (-1, c.head_dim))
            q, k, v = qkv.split((c.heads, c.kv_heads, c.kv_heads), 1)
            y, x = self._norm(self._linear(attend(i, q, k, v).flatten(1), f"{i}.out"), f"{i}.norm2", x)
            gate, up = self._linear(y, f"{i}.up").chunk(2, -1)
            more = self._linear(F.silu(gate) * up, f"{i}.down")
        y, _ = self._norm(x[rows], "norm") if more is None else self._norm(more[rows], "norm", x[rows])
        return self._linear(y, "head")

    def prompt(self, tokens: torch.Tensor) -> tuple[int, torch.Tensor]:
        """A new sequence that holds `tokens` [T]: (its number, the logits behind its last token)."""
        c, n = self.config, tokens.shape[0]
        sequence = self.cache.add()
        slots = self.cache.append([sequence], n)
        positions = torch.arange(n, device=tokens.device)

        def attend(layer, q, k, v):
            q, k = self.cache.write_rope(layer, q, k, v, positions, self.rates, slots, keep_key=True)
            return ck.window_attention(q[None], k[None], v[None], c.window, c.sinks)[0]

        return sequence, self._layers(self.embedding[tokens], attend, slice(-1, None))[0]

    def step(self, sequences: list[int], tokens: torch.Tensor) -> torch.Tensor:
        """Append one token to each sequence: the logits behind them, [B, vocab]."""
        c = self.config
        slots = self.cache.append(sequences)
        table, lengths = self.cache.tables(sequences)
        positions = lengths - 1
        groups = None if c.window else self.cache.groups(sequences, self.share_from)

        def attend(layer, q, k, v):
            q = self.cache.write_rope(layer, q, k, v, positions, self.rates, slots)
            return self.cache.attend(layer, q, table, lengths, window=c.window, sinks=c.sinks, groups=groups)

        logits = self._layers(self.embedding[tokens], attend)
        if c.window:
            for s in sequences:  # pages that left the window
                self.cache.trim(s, c.window, c.sinks)
        return logits

    def generate(self, tokens: torch.Tensor, steps: int, samples: int = 1, temperature: float = 1.0,
                 generator: torch.Generator | None = None, top_k: int = 0, top_p: float = 1.0,
                 min_p: float = 0.0) -> torch.Tensor:
        """`samples` continuations of a prompt, [samples, steps]."""
        first, logits = self.prompt(tokens)
        sequences = [first] + [self.cache.fork(first) for _ in range(samples - 1)]
        logits, out = logits.expand(samples, -1), []
        u = torch.rand(steps, samples, device=tokens.device, generator=generator)
        for i in range(steps):
            out.append(ck.sample_tokens(logits, u[i], temperature, top_k, top_p, min_p))
            if i + 1 < steps:
                logits = self.step(sequences, out[-1])
        for s in sequences:
            self.cache.free(s)
        return torch.stack(out, 1)


def main() -> None:
    config = Config(window=64, sinks=4)
    model = TextDecoder(config, TextDecoder.random_weights(config))
    prompt = torch.randint(0, config.vocab, (100,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    out = model.generate(prompt, steps=20, samples=4, generator=torch.Generator(device="cuda").manual_seed(2), temperature=0.8,
                         top_p=0.95)
    for row in out.tolist():
        print(*row)


if __name__ == "__main__":
    main()
