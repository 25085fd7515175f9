"""What a step of text generation runs between its linears and around its attention, timed as a program
that serves a language model (a text encoder that also writes, a prompt expander) calls it:

  norm    the residual's addition and the root-mean-square norm in front of a linear, its result in
          16 bits, as E4M3 codes with one scale, or as MXFP8 codes with a scale for each 32
  rope    queries and keys turned to their positions, keys and values stored in a paged cache
  sample  the next token from the logits and a given random number: temperature, top-k, top-p, min-p
  shared  attention of one new token per sequence over a paged cache, for sequences that begin with
          the same tokens (several answers to one prompt)

A case is a dict of plain values with a "kind".  With `own` false, `run` computes the plain form
from elementary torch operations; with `own` true it makes the framework's calls.
"""
from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "comfy-kitchen_amd"))

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}
DEV = "cuda"


# ------------------------------------------------------------------ cases
def _norm(rows, cols, residual, dtype, out):
    return {"kind": "norm", "rows": rows, "cols": cols, "residual": residual, "dtype": dtype, "out": out}


def _rope(tokens, pages, page, heads, kv_heads, dim, rotary, interleaved, context, keep, dtype, cache):
    return {"kind": "rope", "tokens": tokens, "pages": pages, "page": page, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "rotary": rotary, "interleaved": interleaved, "context": context, "keep": keep,
            "dtype": dtype, "cache": cache}


def _sample(rows, vocab, temperature, top_k, top_p, min_p, dtype):
    return {"kind": "sample", "rows": rows, "vocab": vocab, "temperature": temperature, "top_k": top_k,
            "top_p": top_p, "min_p": min_p, "dtype": dtype}


def _shared(groups, members, prefix, suffix, heads, kv_heads, dim, page, dtype, cache):
    return {"kind": "shared", "groups": groups, "members": members, "prefix": prefix, "suffix": suffix,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "cache": cache}


def listed():
    return [
        # one generated token
        {"name": "norm_step", **_norm(1, 5120, True, "bf16", "same")},
        # a short prompt in front of a linear on E4M3 weights, an odd number of rows
        {"name": "norm_fp8_text", **_norm(777, 4608, True, "f16", "e4m3")},
        # a batch of prompts in front of a linear on MXFP8 weights
        {"name": "norm_mxfp8_prompt", **_norm(16384, 5120, True, "bf16", "mxfp8")},
        # a decode step of a batch, one token each, deep in their contexts
        {"name": "rope_step", **_rope(48, 2048, 16, 40, 8, 128, 128, False, 60000, False, "bf16", "bf16")},
        # a long prompt of odd length, half of each head turned, cache in 8 bits, keys kept for the prompt's attention
        {"name": "rope_prompt", **_rope(16001, 300, 64, 40, 8, 128, 64, True, 16001, True, "bf16", "e4m3")},
        # one sequence, a filtered choice
        {"name": "sample_one", **_sample(1, 32000, 0.8, 50, 0.9, 0.0, "f32")},
        # a batch over a large odd vocabulary, 16-bit logits (many equal ones)
        {"name": "sample_batch", **_sample(64, 150001, 1.0, 0, 0.95, 0.02, "bf16")},
        # many sequences without a filter, flattened: nearly every token can be drawn
        {"name": "sample_flat", **_sample(256, 128000, 1.6, 0, 1.0, 0.0, "f32")},
        # four answers to a short prompt
        {"name": "shared_few", **_shared(1, 4, 777, 100, 40, 8, 128, 16, "bf16", "bf16")},
        # many answers to one long document, cache in 8 bits
        {"name": "shared_batch", **_shared(1, 64, 16384, 512, 40, 8, 128, 64, "bf16", "e4m3")},
        # several documents with a dozen answers each, a key-value head per query head
        {"name": "shared_groups", **_shared(6, 12, 9001, 700, 24, 24, 64, 32, "f16", "f16")},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(["norm", "rope", "sample", "shared"])
    dtype = rng.choice(["bf16", "f16"])
    if kind == "norm":
        out = rng.choice(["same", "e4m3", "mxfp8"])
        cols = 32 * _spread(rng, 8, 400) if out == "mxfp8" else _spread(rng, 256, 12800)
        rows = _spread(rng, 1, max(1, min(20000, 80_000_000 // cols)))
        return _norm(rows, cols, rng.random() < 0.7, dtype, out)
    if kind == "sample":
        vocab = _spread(rng, 1000, 250000)
        return _sample(_spread(rng, 1, max(1, min(256, 30_000_000 // vocab))), vocab, rng.choice([0.0, 0.6, 1.0, 1.3]),
                       rng.choice([0, 0, 1, _spread(rng, 2, 1000)]), rng.choice([1.0, 0.5, 0.9, 0.99]),
                       rng.choice([0.0, 0.0, 0.05]), rng.choice(["f32", dtype]))
    kv_heads = rng.choice([1, 2, 4, 8, 10])
    dim = rng.choice([64, 96, 128, 128, 256])
    page = rng.choice([8, 16, 20, 64, 128])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8])
    cache = rng.choice([dtype, dtype, "e4m3"])
    if kind == "rope":
        tokens = _spread(rng, 1, min(16000, 80_000_000 // (heads * dim)))
        return _rope(tokens, -(-tokens // page) + _spread(rng, 8, 512), page, heads, kv_heads, dim,
                     rng.choice([dim, dim, dim // 2]), rng.random() < 0.5, _spread(rng, max(tokens, 100), 1000000),
                     rng.random() < 0.5, dtype, cache)
    members = _spread(rng, 1, 64)
    groups = _spread(rng, 1, max(1, 64 // members))
    total = groups * members
    prefix = _spread(rng, 1, max(1, min(16000, 1_200_000_000 // (total * heads * dim))))
    suffix = _spread(rng, 1, max(1, min(2000, 60_000_000 // (total * kv_heads * dim))))
    return _shared(groups, members, prefix, suffix, heads, kv_heads, dim, page, dtype, cache)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def _cache_like(g, shape, dtype):
    """A cache long in use: keys and values of unit size, in 8 bits as codes in units of 1/64."""
    if dtype != torch.float8_e4m3fn:
        return torch.empty(shape, dtype=dtype, device=DEV).normal_(generator=g)
    x = torch.empty(shape, dtype=dtype, device=DEV)
    for i in range(0, shape[0], 4096):
        x[i:i + 4096] = (_randn(g, *x[i:i + 4096].shape) * 64).clamp(-448, 448).to(dtype)  # the largest stay under 448
    return x


def _shared_lengths(case):
    """Every sequence's number of tokens: the common ones, then 1 .. suffix of its own, none alike."""
    n, total = case["suffix"], case["groups"] * case["members"]
    return [_prefix(case, i // case["members"]) + 1 + (n - 1) * ((5 * i) % total + 1) // total for i in range(total)]


def _prefix(case, group):
    """The documents are of unlike lengths."""
    return max(1, case["prefix"] * (case["groups"] - group) // case["groups"])


def _inputs(case, seed):
    g = _gen(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    if kind == "norm":
        shape = (case["rows"], case["cols"])
        t = {"x": _randn(g, *shape).to(dtype), "residual": (_randn(g, *shape) * 3).to(dtype) if case["residual"] else None,
             "weight": (1 + 0.2 * _randn(g, case["cols"])).to(dtype)}
        t["scale"] = torch.tensor(5.5 / 448, device=DEV) if case["out"] == "e4m3" else None
        return t
    if kind == "sample":
        # logits of a language model: a few tokens well above a bell of the others
        logits = _randn(g, case["rows"], case["vocab"]) * 2.5
        logits += 6.0 * (torch.rand(logits.shape, device=DEV, generator=g) < 20 / case["vocab"])
        return {"logits": logits.to(dtype), "u": torch.rand(case["rows"], device=DEV, generator=g)}
    page, heads, hk, d = case["page"], case["heads"], case["kv_heads"], case["dim"]
    cache = DTYPES[case["cache"]]
    scale = torch.tensor(1 / 64, device=DEV) if case["cache"] == "e4m3" else None
    if kind == "rope":
        n, pages = case["tokens"], case["pages"]
        slots = torch.randperm(pages, device=DEV, generator=g)[:, None] * page + torch.arange(page, device=DEV)
        qkv = _randn(g, n, heads + 2 * hk, d).to(dtype)  # as the projection leaves them
        first = case["context"] - n
        at = torch.arange(n, device=DEV) + first if case["keep"] else torch.randint(
            0, case["context"], (n,), device=DEV, generator=g)
        rates = 10000.0 ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64) / case["rotary"])
        return {"q": qkv[:, :heads], "k": qkv[:, heads:heads + hk], "v": qkv[:, heads + hk:],
                "positions": at.to(torch.int32), "rates": rates.float().to(DEV),
                "slots": slots.flatten()[:n].to(torch.int32).contiguous(), "scale": scale,
                "k_cache": torch.zeros(pages, page, hk, d, device=DEV).to(cache),
                "v_cache": torch.zeros(pages, page, hk, d, device=DEV).to(cache)}
    # the whole pages of a group's document are common, what lies behind is each sequence's own
    lengths, members = _shared_lengths(case), case["members"]
    need = [-(-n // page) for n in lengths]
    common = [_prefix(case, i) // page for i in range(case["groups"])]
    total = sum(common) + sum(c - common[i // members] for i, c in enumerate(need))
    order = torch.randperm(total, device=DEV, generator=g).to(torch.int32)  # a pool long in use
    table = torch.zeros(len(need), max(need), dtype=torch.int32, device=DEV)
    at = 0
    for i, c in enumerate(common):
        table[i * members:(i + 1) * members, :c] = order[at:at + c]
        at += c
    for i, n in enumerate(need):
        c = common[i // members]
        table[i, c:n] = order[at:at + n - c]
        at += n - c
    return {"q": _randn(g, len(need), heads, d).to(dtype), "table": table,
            "lengths": torch.tensor(lengths, dtype=torch.int32, device=DEV),
            "groups": torch.arange(case["groups"] + 1, dtype=torch.int32, device=DEV) * members,
            "shared": torch.tensor([c * page for c in common], dtype=torch.int32, device=DEV),
            "k": _cache_like(g, (total, page, hk, d), cache), "v": _cache_like(g, (total, page, hk, d), cache),
            "scale": scale}


def prepare(case, seed):
    return {"case": case, **_inputs(case, seed)}


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    return (_own if own else _plain)[case["kind"]](case, state)


def _own_norm(case, s):
    import comfy_kitchen as ck

    if case["out"] == "same":
        return ck.rms_norm(s["x"], s["weight"], s["residual"])
    if case["out"] == "e4m3":
        return ck.rms_norm_fp8(s["x"], s["scale"], s["weight"], s["residual"])
    return ck.rms_norm_mxfp8(s["x"], s["weight"], s["residual"])


def _own_rope(case, s):
    import comfy_kitchen as ck

    turned = ck.paged_write_rope(s["q"], s["k"], s["v"], s["positions"], s["rates"], s["k_cache"], s["v_cache"],
                                 s["slots"], interleaved=case["interleaved"], k_scale=s["scale"], v_scale=s["scale"],
                                 keep_key=case["keep"])
    return [turned, s["k_cache"], s["v_cache"]]


def _own_sample(case, s):
    import comfy_kitchen as ck

    return ck.sample_tokens(s["logits"], s["u"], case["temperature"], case["top_k"], case["top_p"], case["min_p"])


def _own_shared(case, s):
    import comfy_kitchen as ck

    return ck.shared_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], s["groups"], s["shared"],
                               k_scale=s["scale"], v_scale=s["scale"])


_own = {"norm": _own_norm, "rope": _own_rope, "sample": _own_sample, "shared": _own_shared}


def _plain_norm(case, s):
    h = s["x"]
    if s["residual"] is not None:
        h = (h.float() + s["residual"].float()).to(h.dtype)
    y = h.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * s["weight"].float()
    y = y.to(h.dtype)
    if case["out"] == "same":
        out = [y]
    elif case["out"] == "e4m3":
        out = [(y.float() * (1.0 / s["scale"])).clamp(-448, 448).to(torch.float8_e4m3fn)]
    else:
        rows, cols = y.shape
        blocks = y.float().reshape(rows, cols // 32, 32)
        top = blocks.abs().amax(-1)
        # the least power of two that brings the block under 448
        e = torch.ceil(torch.log2((top / 448).clamp(min=2.0 ** -127))).clamp(-127, 127)
        codes = (blocks * torch.exp2(-e)[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).reshape(rows, cols)
        bytes_ = torch.where(top > 0, e + 127, torch.zeros_like(e)).to(torch.uint8)
        pad = torch.nn.functional.pad(bytes_, (0, -(cols // 32) % 4, 0, -rows % 128))
        tiles = pad.reshape(pad.shape[0] // 128, 4, 32, pad.shape[1] // 4, 4).permute(0, 3, 2, 1, 4)
        out = [codes, tiles.reshape(pad.shape).contiguous().view(torch.float8_e8m0fnu)]
    if s["residual"] is not None:
        out.append(h)
    return out if len(out) > 1 else out[0]


def _plain_rope(case, s):
    angle = s["positions"].double()[:, None] * s["rates"].double()
    c, n = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    r = case["rotary"]

    def turn(x):
        x = x.float()
        y = x.clone()
        a, b = (slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
        y[..., a] = x[..., a] * c - x[..., b] * n
        y[..., b] = x[..., a] * n + x[..., b] * c
        return y

    q, k = turn(s["q"]), turn(s["k"])
    slots = s["slots"].long()
    for x, cache in ((k, s["k_cache"]), (s["v"].float(), s["v_cache"])):
        if s["scale"] is not None:
            x = (x / s["scale"]).clamp(-448, 448)
        cache.view(-1, *cache.shape[2:])[slots] = x.to(cache.dtype)
    q = q.to(s["q"].dtype)
    return [(q, k.to(q.dtype)) if case["keep"] else q, s["k_cache"], s["v_cache"]]


def _plain_sample(case, s):
    logits = s["logits"]
    if case["temperature"] == 0:
        # the first of the largest
        at = torch.arange(logits.shape[1], device=DEV)
        return torch.where(logits == logits.amax(-1, keepdim=True), at, logits.shape[1]).amin(-1)
    values, index = torch.sort(logits.float(), dim=-1, descending=True, stable=True)
    # weights next to a border decide: 64 bits
    w = torch.exp((values.double() - values[:, :1].double()) / case["temperature"])
    if case["top_k"]:
        w[:, case["top_k"]:] = 0
    if case["top_p"] < 1:
        before = torch.cumsum(w, -1) - w
        w = w * (before < case["top_p"] * w.sum(-1, keepdim=True))
    w = w * (w >= case["min_p"])
    running = torch.cumsum(w, -1)
    past = (running > s["u"].double()[:, None] * running[:, -1:]) & (w > 0)
    first = torch.where(past, torch.arange(w.shape[1], device=DEV), w.shape[1] - 1).amin(-1, keepdim=True)
    return torch.gather(index, 1, first)[:, 0]


def _plain_shared(case, s):
    b, hk, d = s["q"].shape[0], case["kv_heads"], case["dim"]
    rep = case["heads"] // hk
    table = s["table"].long()
    q = s["q"].float().reshape(b, hk, rep, d)
    out = torch.empty(b, hk, rep, d, device=DEV)
    capacity = table.shape[1] * case["page"]
    seen = torch.arange(capacity, device=DEV) < s["lengths"].long()[:, None]
    step = max(1, 400_000_000 // (capacity * hk * d))  # sequences whose cache is widened at once
    for i in range(0, b, step):
        k = s["k"][table[i:i + step]].float().reshape(-1, capacity, hk, d).permute(0, 2, 3, 1)
        if s["scale"] is not None:
            k = k * s["scale"]
        p = (q[i:i + step] @ k) * d ** -0.5
        p = p.masked_fill(~seen[i:i + step, None, None, :], float("-inf"))
        p = torch.exp(p - p.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        del k
        v = s["v"][table[i:i + step]].float().reshape(-1, capacity, hk, d).permute(0, 2, 1, 3)
        if s["scale"] is not None:
            v = v * s["scale"]
        out[i:i + step] = p @ v
    return out.reshape(b, case["heads"], d).to(s["q"].dtype)


_plain = {"norm": _plain_norm, "rope": _plain_rope, "sample": _plain_sample, "shared": _plain_shared}


# ------------------------------------------------------------------ bounds
def work(case):
    kind, size = case["kind"], 4 if case["dtype"] == "f32" else 2
    if kind == "norm":
        n = case["rows"] * case["cols"]
        out = {"same": 2 * n, "e4m3": n, "mxfp8": n + n // 32}[case["out"]]
        return {"bytes": 2 * n + (4 * n if case["residual"] else 0) + 2 * case["cols"] + out, "flops": 6 * n}
    if kind == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": size * n + 12 * case["rows"], "flops": 4 * n}
    row, es = case["kv_heads"] * case["dim"], 1 if case["cache"] == "e4m3" else 2
    if kind == "rope":
        q, t = case["heads"] * case["dim"], case["tokens"]
        moved = 4 * q + 4 * row + 2 * row * es + (2 * row if case["keep"] else 0) + 8
        return {"bytes": t * moved, "flops": 3 * t * (case["heads"] + case["kv_heads"]) * case["rotary"]}
    lengths, page = _shared_lengths(case), case["page"]
    common = [_prefix(case, i) // page * page for i in range(case["groups"])]
    read = sum(common) + sum(n - common[i // case["members"]] for i, n in enumerate(lengths))
    return {"bytes": 2 * read * row * es + 4 * len(lengths) * case["heads"] * case["dim"],
            "flops": 4 * sum(lengths) * case["heads"] * case["dim"]}


# ------------------------------------------------- the same results in 64 bits
def exact(case, seed):
    t = _inputs(case, seed)
    kind = case["kind"]
    if kind == "sample":
        return None  # a token's number is chosen, not computed
    if kind == "norm":
        h = t["x"].double()
        if t["residual"] is not None:
            h = h + t["residual"].double()
        # the norm is of the sum as it is stored
        kept = h.to(t["x"].dtype).double()
        y = kept / torch.sqrt(kept.pow(2).sum(-1, keepdim=True) / case["cols"] + 1e-6) * t["weight"].double()
        if case["out"] == "e4m3":
            y = (y / t["scale"].double()).clamp(-448, 448)
        out = [y]
        if case["out"] == "mxfp8":
            top = y.to(t["x"].dtype).double().unflatten(-1, (-1, 32)).abs().amax(-1)  # of the rounded results
            out = [y / torch.pow(2.0, torch.ceil(torch.log2(top / 448))).repeat_interleave(32, -1), None]
        if t["residual"] is not None:
            out.append(h)
        return out if len(out) > 1 else out[0]
    if kind == "rope":
        r, half = case["rotary"], case["rotary"] // 2
        turns = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                            torch.outer(t["positions"].double(), t["rates"].double()))[:, None]

        def turned(x):
            head, rest = x.double().split((r, case["dim"] - r), -1)
            if case["interleaved"]:
                z = torch.view_as_complex(head.unflatten(-1, (half, 2)).contiguous()) * turns
                head = torch.view_as_real(z).flatten(-2)
            else:
                z = torch.complex(*head.split(half, -1)) * turns
                head = torch.cat((z.real, z.imag), -1)
            return torch.cat((head, rest), -1)

        q, k = turned(t["q"]), turned(t["k"])
        caches = []
        for x in (k, t["v"].double()):
            if t["scale"] is not None:
                x = torch.clip(x / t["scale"].double(), -448, 448)
            cache = torch.zeros(t["k_cache"].shape, dtype=torch.float64, device=DEV)
            cache.flatten(0, 1).index_copy_(0, t["slots"].long(), x)
            caches.append(cache)
        return [(q, k) if case["keep"] else q, *caches]
    rep, d, page = case["heads"] // case["kv_heads"], case["dim"], case["page"]
    out = torch.empty(t["q"].shape, dtype=torch.float64, device=DEV)
    factor = 1.0 if t["scale"] is None else t["scale"].double()
    for i, n in enumerate(_shared_lengths(case)):
        at = torch.arange(n, device=DEV)
        pages = t["table"][i].long()[at // page]
        for h in range(case["kv_heads"]):
            k, v = t["k"][pages, at % page, h].double(), t["v"][pages, at % page, h].double()
            scores = torch.matmul(t["q"][i, h * rep:(h + 1) * rep].double(), (k * factor).T) / d ** 0.5
            weight = (scores - scores.max(-1, keepdim=True).values).exp()
            out[i, h * rep:(h + 1) * rep] = torch.matmul(weight, v * factor) / weight.sum(-1, keepdim=True)
    return out
