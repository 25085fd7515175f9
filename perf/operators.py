"""The operators of text generation that are timed here, as a program that serves a language
model (a text encoder that also writes, a prompt expander) calls them between its linears:

  linear   y = x W^T + bias with a weight of 4-bit codes, one scale (and zero point) for each row
           and group of inputs, for one to some dozens of activation rows
  decode   attention of one new token per sequence over a key-value cache held in pages
  prompt   causal attention of a prompt with a sliding window and a few first tokens (sinks) that
           stay visible
  write    keys and values of new tokens scattered to their slots of the paged cache
  copy     token rows copied from slots to slots of the paged caches of all layers: the partly
           filled pages of forked sequences, and the kept tokens of compacted ones

A case is a dict of plain values with a "kind".  With `own` false, `run` computes the plain form
from elementary torch operations in 32 bits; with `own` true it makes the framework's calls.
"""
from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "comfy-kitchen_amd"))

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
DEV = "cuda"


# ------------------------------------------------------------------ cases
def _linear(m, n, k, group, zeros, bias, dtype):
    return {"kind": "linear", "m": m, "n": n, "k": k, "group": group, "zeros": zeros, "bias": bias, "dtype": dtype}


def _decode(batch, length, ragged, heads, kv_heads, dim, page, window, sinks, dtype, cache):
    return {"kind": "decode", "batch": batch, "length": length, "ragged": ragged, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "window": window, "sinks": sinks, "dtype": dtype,
            "cache": cache}


def _prompt(batch, queries, keys, heads, kv_heads, dim, window, sinks, dtype):
    return {"kind": "prompt", "batch": batch, "queries": queries, "keys": keys, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "window": window, "sinks": sinks, "dtype": dtype}


def _write(tokens, pages, page, kv_heads, dim, dtype):
    return {"kind": "write", "tokens": tokens, "pages": pages, "page": page, "kv_heads": kv_heads, "dim": dim,
            "dtype": dtype}


def _copy(layers, tokens, run, pages, page, kv_heads, dim, dtype):
    return {"kind": "copy", "layers": layers, "tokens": tokens, "run": run, "pages": pages, "page": page,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype}


def listed():
    return [
        # one generated token: the key projection of a layer with 8 key-value heads
        {"name": "linear_key_1", **_linear(1, 1024, 5120, 128, False, False, "bf16")},
        # one generated token: the feed-forward's up-projection, small groups with zero points
        {"name": "linear_up_1", **_linear(1, 13824, 5120, 64, True, False, "f16")},
        # two dozen sequences generated together: the feed-forward's down-projection
        {"name": "linear_down_24", **_linear(24, 5120, 13824, 128, False, True, "bf16")},
        # one sequence soon after its prompt: a short cache that ends inside a page
        {"name": "decode_short", **_decode(1, 333, False, 40, 8, 128, 16, 0, 0, "bf16", "bf16")},
        # a batch of sequences of unlike lengths, cache in 8 bits
        {"name": "decode_batch", **_decode(48, 8192, True, 40, 8, 128, 64, 0, 0, "bf16", "e4m3")},
        # one very long document, a key-value head per query head, an odd length
        {"name": "decode_long", **_decode(1, 80003, False, 30, 30, 128, 128, 0, 0, "f16", "f16")},
        # a short prompt of a small model: an odd length, a window that covers a third of it
        {"name": "prompt_short", **_prompt(1, 777, 777, 24, 8, 64, 256, 4, "f16")},
        # a long document read in one go
        {"name": "prompt_long", **_prompt(1, 16384, 16384, 40, 8, 128, 4096, 16, "bf16")},
        # a decode step of a batch: one token each
        {"name": "write_step", **_write(48, 2048, 16, 8, 128, "bf16")},
        # a batch of prompts
        {"name": "write_prompt", **_write(32000, 1024, 64, 8, 128, "bf16")},
        # eight sequences forked: the filled parts of their last pages, for every layer
        {"name": "copy_fork", **_copy(40, 8 * 37, 37, 100, 64, 8, 128, "bf16")},
        # a long sequence compacted to the tokens worth keeping, single tokens and short runs
        {"name": "copy_compact", **_copy(20, 6001, 3, 384, 64, 8, 128, "bf16")},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(["linear", "decode", "prompt", "write", "copy"])
    dtype = rng.choice(["bf16", "f16"])
    if kind == "linear":
        group = rng.choice([32, 64, 128])
        return _linear(_spread(rng, 1, 64), _spread(rng, 256, 16000), 32 * _spread(rng, 32, 448), group,
                       rng.random() < 0.5, rng.random() < 0.5, dtype)
    kv_heads = rng.choice([1, 2, 4, 8, 10])
    dim = rng.choice([64, 96, 128, 128, 256])
    if kind == "decode":
        heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8, 16])
        length = _spread(rng, 1, 60000)
        batch = _spread(rng, 1, max(1, min(128, 200_000_000 // (length * kv_heads * dim))))
        window = rng.choice([0, 0, _spread(rng, 16, 8192)])
        return _decode(batch, length, rng.random() < 0.6, heads, kv_heads, dim, rng.choice([8, 16, 20, 32, 64, 128, 256]),
                       window, rng.choice([0, 1, 4, 33]) if window else 0, dtype, rng.choice([dtype, dtype, "e4m3"]))
    if kind == "prompt":
        heads = kv_heads * rng.choice([1, 2, 3, 5])
        keys = _spread(rng, 1, min(10000, 6_000_000 // (heads * dim) * 4))
        queries = keys if rng.random() < 0.7 else _spread(rng, 1, keys)
        batch = _spread(rng, 1, max(1, min(16, 20000 // keys, 20_000_000_000 // (keys * queries * heads * dim))))
        return _prompt(batch, queries, keys, heads, kv_heads, dim, _spread(rng, 16, 6000), rng.choice([0, 1, 4, 33]), dtype)
    page = rng.choice([8, 16, 20, 64, 128])
    if kind == "write":
        tokens = _spread(rng, 1, 32000)
        return _write(tokens, -(-tokens // page) + _spread(rng, 8, 512), page, kv_heads, dim, dtype)
    layers = rng.choice([1, 4, 20])
    tokens = _spread(rng, 1, min(6000, 100_000_000 // (layers * kv_heads * dim)))
    run = _spread(rng, 1, 64)
    return _copy(layers, tokens, run, 2 * -(-4 * tokens // page) + 8, page, kv_heads, dim, dtype)


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """Every sequence's number of cached tokens, the new one among them."""
    b, n = case["batch"], case["length"]
    if not case["ragged"]:
        return [n] * b
    return [max(1, n * ((7 * i) % b + 1) // b) for i in range(b)] if b % 7 else [max(1, n * (i + 1) // b) for i in range(b)]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def _inputs(case, seed):
    g = _gen(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    if kind == "linear":
        m, n, k, group = case["m"], case["n"], case["k"], case["group"]
        w = _randn(g, n, k) * 0.02
        groups = -(-k // group)
        pad = torch.nn.functional.pad(w, (0, groups * group - k)).reshape(n, groups, group)
        if case["zeros"]:
            lo, hi = pad.amin(-1).clamp(max=0), pad.amax(-1).clamp(min=0)
            scales = ((hi - lo) / 15).clamp(min=1e-6).to(dtype)
            zeros = torch.round(-lo / scales.float()).clamp(0, 15)
        else:
            scales = (pad.abs().amax(-1) / 7).clamp(min=1e-6).to(dtype)
            zeros = torch.full((n, groups), 8.0, device=DEV)
        q = (torch.round(pad / scales.float().unsqueeze(-1)) + zeros.unsqueeze(-1)).clamp(0, 15)
        q = q.reshape(n, -1)[:, :k].to(torch.uint8)
        codes = q[:, 0::2] | (q[:, 1::2] << 4)  # two codes a byte, the even one in the low nibble
        x = _randn(g, m, k).to(dtype)
        bias = _randn(g, n).to(dtype) if case["bias"] else None
        return {"x": x, "codes": codes.contiguous(), "scales": scales,
                "zeros": zeros.to(torch.uint8) if case["zeros"] else None, "bias": bias}
    if kind == "decode":
        lengths = _lengths(case)
        page, hk, d = case["page"], case["kv_heads"], case["dim"]
        need = [-(-n // page) for n in lengths]
        total = sum(need)
        order = torch.randperm(total, device=DEV, generator=g).to(torch.int32)  # a pool long in use
        table = torch.zeros(len(need), max(need), dtype=torch.int32, device=DEV)
        at = 0
        for i, c in enumerate(need):
            table[i, :c] = order[at:at + c]
            at += c
        t = {"q": _randn(g, case["batch"], case["heads"], d).to(dtype), "table": table,
             "lengths": torch.tensor(lengths, dtype=torch.int32, device=DEV)}
        cache = DTYPES[case["cache"]]
        for name in ("k", "v"):
            x = torch.empty(total, page, hk, d, dtype=cache, device=DEV)
            if case["cache"] == "e4m3":
                # keys and values of unit size in units of 1/64: the largest stay under 448
                for i in range(0, total, 4096):
                    x[i:i + 4096] = (_randn(g, *x[i:i + 4096].shape) * 64).clamp(-448, 448).to(cache)
                t[name + "_scale"] = torch.tensor(1 / 64, device=DEV)
            else:
                x.normal_(generator=g)
                t[name + "_scale"] = None
            t[name] = x
        return t
    if kind == "prompt":
        b, d = case["batch"], case["dim"]
        return {"q": _randn(g, b, case["queries"], case["heads"], d).to(dtype),
                "k": _randn(g, b, case["keys"], case["kv_heads"], d).to(dtype),
                "v": _randn(g, b, case["keys"], case["kv_heads"], d).to(dtype)}
    page, hk, d, pages = case["page"], case["kv_heads"], case["dim"], case["pages"]
    if kind == "write":
        slots = torch.randperm(pages, device=DEV, generator=g)[:, None] * page + torch.arange(page, device=DEV)
        return {"k": _randn(g, case["tokens"], hk, d).to(dtype), "v": _randn(g, case["tokens"], hk, d).to(dtype),
                "k_cache": torch.zeros(pages, page, hk, d, dtype=dtype, device=DEV),
                "v_cache": torch.zeros(pages, page, hk, d, dtype=dtype, device=DEV),
                "slots": slots.flatten()[:case["tokens"]].to(torch.int32).contiguous()}
    caches = [torch.empty(case["layers"], pages, page, hk, d, dtype=dtype, device=DEV).normal_(generator=g)
              for _ in range(2)]
    # runs of tokens from one half of the pool to fresh pages of the other, whose order is mixed
    tokens, run = case["tokens"], case["run"]
    order = torch.randperm(pages, device=DEV, generator=g)
    old, new = order[:pages // 2], order[pages // 2:]
    runs = -(-tokens // run)
    place = (old.numel() * page) // run
    start = torch.randperm(max(place, runs), device=DEV, generator=g)[:runs].sort().values * run
    at = (start[:, None] + torch.arange(run, device=DEV)).flatten()[:tokens] % (old.numel() * page)
    to = torch.arange(tokens, device=DEV)
    return {"k_cache": caches[0], "v_cache": caches[1],
            "src": (old[at // page] * page + at % page).to(torch.int32),
            "dst": (new[to // page] * page + to % page).to(torch.int32)}


def prepare(case, seed):
    return {"case": case, **_inputs(case, seed)}


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    return (_own if own else _plain)[case["kind"]](case, state)


def _own_linear(case, s):
    import comfy_kitchen as ck

    return ck.linear_int4(s["x"], s["codes"], s["scales"], s["zeros"], s["bias"], group_size=case["group"])


def _own_decode(case, s):
    import comfy_kitchen as ck

    return ck.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], window=case["window"],
                              sinks=case["sinks"], k_scale=s["k_scale"], v_scale=s["v_scale"])


def _own_prompt(case, s):
    import comfy_kitchen as ck

    return ck.window_attention(s["q"], s["k"], s["v"], window=case["window"], sinks=case["sinks"])


def _own_write(case, s):
    import comfy_kitchen as ck

    ck.paged_write(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"])
    return [s["k_cache"], s["v_cache"]]


def _own_copy(case, s):
    import comfy_kitchen as ck

    ck.paged_copy(s["k_cache"], s["v_cache"], s["src"], s["dst"])
    return [s["k_cache"], s["v_cache"]]


_own = {"linear": _own_linear, "decode": _own_decode, "prompt": _own_prompt, "write": _own_write, "copy": _own_copy}


def _plain_linear(case, s):
    codes, group = s["codes"], case["group"]
    q = torch.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1).float()
    k = q.shape[1]
    if s["zeros"] is None:
        q = q - 8.0
    else:
        q = q - s["zeros"].float().repeat_interleave(group, 1)[:, :k]
    w = q * s["scales"].float().repeat_interleave(group, 1)[:, :k]
    y = s["x"].float() @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


def _plain_decode(case, s):
    b, hk, d = case["batch"], case["kv_heads"], case["dim"]
    rep = case["heads"] // hk
    table = s["table"].long()
    q = s["q"].float().reshape(b, hk, rep, d)
    out = torch.empty(b, hk, rep, d, device=DEV)
    capacity = table.shape[1] * case["page"]
    pos = torch.arange(capacity, device=DEV)
    n = s["lengths"].long()[:, None]
    seen = pos < n
    if case["window"]:
        seen = seen & ((pos >= n - case["window"]) | (pos < case["sinks"]))
    step = max(1, 400_000_000 // (capacity * hk * d))  # sequences whose cache is widened at once
    for i in range(0, b, step):
        k = s["k"][table[i:i + step]].float().reshape(-1, capacity, hk, d).permute(0, 2, 3, 1)
        if s["k_scale"] is not None:
            k = k * s["k_scale"]
        p = (q[i:i + step] @ k) * d ** -0.5
        p = p.masked_fill(~seen[i:i + step, None, None, :], float("-inf"))
        p = torch.exp(p - p.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        del k
        v = s["v"][table[i:i + step]].float().reshape(-1, capacity, hk, d).permute(0, 2, 1, 3)
        if s["v_scale"] is not None:
            v = v * s["v_scale"]
        out[i:i + step] = p @ v
    return out.reshape(b, case["heads"], d).to(s["q"].dtype)


def _plain_prompt(case, s):
    b, sq, sk, hq, hk = case["batch"], case["queries"], case["keys"], case["heads"], case["kv_heads"]
    out = torch.empty_like(s["q"])
    key = torch.arange(sk, device=DEV)
    rows = max(1, min(sq, 200_000_000 // (sk * (hq // hk))))  # query rows whose scores are held at once
    for i in range(b):
        for h in range(hk):
            heads = slice(h * (hq // hk), (h + 1) * (hq // hk))
            k = s["k"][i, :, h].float().t()
            v = s["v"][i, :, h].float()
            for r in range(0, sq, rows):
                q = s["q"][i, r:r + rows, heads].float().transpose(0, 1)  # heads, rows, dim
                at = torch.arange(r, r + q.shape[1], device=DEV)[:, None] + (sk - sq)
                seen = (key <= at) & ((at - key < case["window"]) | (key < case["sinks"]))
                p = (q @ k) * case["dim"] ** -0.5
                p = p.masked_fill(~seen, float("-inf"))
                p = torch.exp(p - p.amax(-1, keepdim=True))
                p = p / p.sum(-1, keepdim=True)
                out[i, r:r + rows, heads] = (p @ v).transpose(0, 1).to(out.dtype)
    return out


def _plain_write(case, s):
    slots = s["slots"].long()
    for x, cache in ((s["k"], s["k_cache"]), (s["v"], s["v_cache"])):
        cache.view(-1, *cache.shape[2:])[slots] = x
    return [s["k_cache"], s["v_cache"]]


def _plain_copy(case, s):
    src, dst = s["src"].long(), s["dst"].long()
    for cache in (s["k_cache"], s["v_cache"]):
        rows = cache.view(cache.shape[0], -1, *cache.shape[3:])
        rows[:, dst] = rows[:, src]
    return [s["k_cache"], s["v_cache"]]


_plain = {"linear": _plain_linear, "decode": _plain_decode, "prompt": _plain_prompt, "write": _plain_write,
          "copy": _plain_copy}


# ------------------------------------------------------------------ bounds
def _pairs(case):
    """(query, key) pairs that the window leaves, of one head of one batch entry."""
    total, sq, sk, w, s = 0, case["queries"], case["keys"], case["window"], case["sinks"]
    for p in range(sk - sq, sk):
        first = max(0, p - w + 1)
        total += p + 1 - first + min(s, first)
    return total


def work(case):
    kind = case["kind"]
    if kind == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        groups = -(-k // case["group"])
        weight = n * k // 2 + n * groups * (3 if case["zeros"] else 2)
        return {"bytes": weight + 2 * m * k + 2 * m * n + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    row = case["kv_heads"] * case["dim"]
    if kind == "decode":
        w, size = case["window"], 1 if case["cache"] == "e4m3" else 2
        seen = 0
        for n in _lengths(case):
            first = max(0, n - w) if w else 0
            seen += n - first + min(case["sinks"], first)
        qo = 2 * case["batch"] * case["heads"] * case["dim"] * 2
        return {"bytes": 2 * seen * row * size + qo, "flops": 4 * seen * case["heads"] * case["dim"]}
    if kind == "prompt":
        b, d = case["batch"], case["dim"]
        seen_keys = case["keys"]
        return {"bytes": 4 * b * case["queries"] * case["heads"] * d + 4 * b * seen_keys * row,
                "flops": 4 * b * _pairs(case) * case["heads"] * d}
    if kind == "write":
        return {"bytes": 8 * case["tokens"] * row + 4 * case["tokens"], "flops": 0}
    return {"bytes": 8 * case["layers"] * case["tokens"] * row + 8 * case["tokens"], "flops": 0}


# ------------------------------------------------- the same results in 64 bits
def _softmax_rows(scores, values):
    """softmax(scores) values, in the scores' type, from the definition."""
    top = scores.max(-1, keepdim=True).values
    weight = (scores - top).exp()
    return torch.matmul(weight, values) / weight.sum(-1, keepdim=True)


def exact(case, seed):
    t = _inputs(case, seed)
    kind = case["kind"]
    if kind == "linear":
        n, half = t["codes"].shape
        w = torch.empty(n, 2 * half, dtype=torch.float64, device=DEV)
        w[:, 0::2] = (t["codes"] % 16).double()
        w[:, 1::2] = (t["codes"] // 16).double()
        for i in range(t["scales"].shape[1]):
            cols = slice(i * case["group"], min((i + 1) * case["group"], case["k"]))
            zero = 8.0 if t["zeros"] is None else t["zeros"][:, i:i + 1].double()
            w[:, cols] = (w[:, cols] - zero) * t["scales"][:, i:i + 1].double()
        y = torch.matmul(t["x"].double(), w.T)
        return y if t["bias"] is None else y + t["bias"].double()
    if kind == "decode":
        page, rep, d = case["page"], case["heads"] // case["kv_heads"], case["dim"]
        out = torch.empty(case["batch"], case["heads"], d, dtype=torch.float64, device=DEV)
        for i, n in enumerate(_lengths(case)):
            first = max(0, n - case["window"]) if case["window"] else 0
            at = torch.cat((torch.arange(min(case["sinks"], first), device=DEV), torch.arange(first, n, device=DEV)))
            pages = t["table"][i].long()[at // page]
            for h in range(case["kv_heads"]):
                k, v = t["k"][pages, at % page, h].double(), t["v"][pages, at % page, h].double()
                if t["k_scale"] is not None:
                    k, v = k * t["k_scale"].double(), v * t["v_scale"].double()
                q = t["q"][i, h * rep:(h + 1) * rep].double()
                out[i, h * rep:(h + 1) * rep] = _softmax_rows(torch.matmul(q, k.T) / d ** 0.5, v)
        return out
    if kind == "prompt":
        sq, sk, rep = case["queries"], case["keys"], case["heads"] // case["kv_heads"]
        out = torch.empty(t["q"].shape, dtype=torch.float64, device=DEV)
        for i in range(case["batch"]):
            for h in range(case["heads"]):
                k, v = t["k"][i, :, h // rep].double(), t["v"][i, :, h // rep].double()
                for r in range(0, sq, 2048):
                    end = min(r + 2048, sq)
                    p0, p1 = r + sk - sq, end + sk - sq  # positions of these rows
                    first = max(0, p0 - case["window"] + 1)
                    at = torch.cat((torch.arange(min(case["sinks"], first), device=DEV),
                                    torch.arange(first, p1, device=DEV)))
                    row = torch.arange(p0, p1, device=DEV)[:, None]
                    hidden = (at > row) | ((row - at >= case["window"]) & (at >= case["sinks"]))
                    scores = torch.matmul(t["q"][i, r:end, h].double(), k[at].T) / case["dim"] ** 0.5
                    out[i, r:end, h] = _softmax_rows(scores.masked_fill(hidden, -float("inf")), v[at])
        return out
    return None  # rows are moved, not computed
