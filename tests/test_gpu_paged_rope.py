"""Queries and keys turned to their positions, keys and values stored: against the definition in 64 bits.

The bound: one rounding of the result (unit |y|; f16 has steps of 2^-24 under 2^-14), two products and a sum in
fp32 of cosine and sine that are 2^-22 off together: 2^-21 (|x| + |y|) magnitude.  Codes are compared where the exact
quotient is not within 2^-18 of the middle between two codes."""
import numpy as np
import pytest
import torch

import comfy_kitchen as ck

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def turned(x, positions, rates, interleaved, magnitude):
    """(the result, |x| + |y| of its pair) in 64 bits."""
    x, n = x.double(), len(rates)
    angle = np.outer(positions.numpy().astype(np.longdouble), rates.numpy().astype(np.longdouble))  # 64 bits of mantissa
    c, s = (torch.from_numpy(f(angle).astype(np.float64))[:, None] * magnitude for f in (np.cos, np.sin))
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    y, size = x.clone(), torch.zeros_like(x)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    size[..., a] = size[..., b] = (x[..., a].abs() + x[..., b].abs()) * abs(magnitude)
    return y, size


def near(got, ref, size, dtype):
    err = (got.cpu().double() - ref).abs()
    bound = (UNIT[dtype] + 2.0 ** -21) * ref.abs() + 2.0 ** -21 * size + (2.0 ** -25 if dtype == "f16" else 0)
    assert bool((err <= bound).all()), float((err / bound.clamp_min(1e-300)).max())


def near_codes(got, quotient, size):
    """E4M3 codes of quotients known up to 2^-20 of their size."""
    q, slack = quotient.clamp(-448, 448), 2.0 ** -20 * (size + quotient.abs())
    lo, hi = ((q + d).clamp(-448, 448).float().to(DT["e4m3"]).double() for d in (-slack, slack))
    got = got.cpu().double()
    assert bool(((got == lo) | (got == hi)).all())


def run(tokens, heads, hk, dim, rotary, page, interleaved, dtype, cache, first=0, magnitude=1.0, keep=True, layout="plain", kinds=(torch.int32, torch.int64),
        seed=0):
    g = torch.Generator().manual_seed(seed + tokens)
    pages = -(-tokens // page) + 2
    shape = (pages, page, hk, dim)
    k, v = ((torch.randn(shape, generator=g) * 9).to(DT[cache]).cuda() for _ in range(2))
    if layout == "PHTD":
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    before = [t.cpu().clone() for t in (k, v)]
    fused = torch.randn(tokens, heads + 2 * hk, dim, generator=g).to(DT[dtype])
    positions = torch.randint(first, first + 5 * tokens + 1, (tokens,), generator=g)
    rates = ck.rope_rates(rotary, device="cpu")
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    slots[2::7] = -1
    if tokens > 4:
        slots[4] = pages * page
    scales = (0.01, 0.02) if cache == "e4m3" else (None, None)
    dev = fused.cuda()
    if layout == "unaligned":
        dev = torch.zeros(tokens, heads + 2 * hk, dim + 1, dtype=DT[dtype], device="cuda")[..., 1:].copy_(fused)
    out = ck.paged_write_rope(dev[:, :heads], dev[:, heads:heads + hk], dev[:, heads + hk:], positions.to(kinds[0]).cuda(), rates.cuda(), k, v,
                              slots.to(kinds[1]).cuda(), interleaved=interleaved, magnitude=magnitude,
                              k_scale=None if scales[0] is None else torch.tensor(scales[0]), v_scale=None if scales[1] is None else torch.tensor(scales[1]),
                              keep_key=keep)
    q_out, k_out = out if keep else (out, None)
    q, size = turned(fused[:, :heads], positions, rates, interleaved, magnitude)
    assert q_out.is_contiguous() and q_out.dtype == DT[dtype]
    near(q_out, q, size, dtype)
    assert torch.equal(q_out.cpu()[..., rotary:], fused[:, :heads, rotary:])
    ref, size = turned(fused[:, heads:heads + hk], positions, rates, interleaved, magnitude)
    if keep:
        near(k_out, ref, size, dtype)
    live = (slots >= 0) & (slots < pages * page)
    rows_k, rows_v = (t.contiguous().flatten(0, 1).cpu()[slots[live]] for t in (k, v))
    if cache == "e4m3":
        near_codes(rows_k, ref[live] / torch.tensor(scales[0]).double(), size[live] / scales[0])
        near_codes(rows_v, fused[live, heads + hk:].double() / torch.tensor(scales[1]).double(), 0.0)
    else:
        near(rows_k, ref[live], size[live], dtype)
        assert torch.equal(rows_v, fused[live, heads + hk:])
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[slots[live]] = False
    for t, old in zip((k, v), before):
        assert torch.equal(t.contiguous().flatten(0, 1).cpu()[rest].view(torch.uint8), old.contiguous().flatten(0, 1)[rest].view(torch.uint8))


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"), ("f16", "e4m3")])
@pytest.mark.parametrize("dim,rotary", [(16, 16), (64, 64), (96, 96), (128, 64), (128, 16), (128, 0), (256, 256), (128, 20), (96, 24), (64, 2), (112, 108)])
def test_heads(dim, rotary, dtype, cache, interleaved, hip):
    run(37, 5, 2, dim, rotary, 20, interleaved, dtype, cache)


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("tokens,heads,hk", [(0, 4, 2), (1, 1, 1), (1, 40, 8), (3, 7, 7), (300, 40, 8), (2111, 12, 3), (1000, 2, 1)])
def test_tokens(tokens, heads, hk, interleaved, hip):
    run(tokens, heads, hk, 128, 128, 16, interleaved, "bf16", "bf16", keep=False)


@pytest.mark.parametrize("layout", ["PHTD", "unaligned"])
@pytest.mark.parametrize("cache", ["f16", "e4m3"])
def test_layouts(cache, layout, hip):
    run(50, 6, 2, 64, 64, 8, False, "f16", cache, layout=layout, kinds=(torch.int64, torch.int32))


def test_magnitude_and_negative_positions(hip):
    run(40, 4, 2, 64, 64, 8, True, "bf16", "bf16", first=-100, magnitude=1.25)
    run(40, 4, 2, 64, 32, 8, False, "f16", "f16", first=-100, magnitude=-0.5)


def test_far_positions(hip):
    run(64, 4, 2, 128, 128, 16, True, "f16", "f16", first=2_000_000)
    run(64, 4, 2, 128, 128, 16, False, "f16", "f16", first=2 ** 31 - 1000)
    run(8, 4, 2, 128, 128, 16, False, "f16", "f16", first=2 ** 40, kinds=(torch.int64, torch.int32))


def test_values_that_are_not_finite(hip):
    """They reach their own pair, and nothing else; the part that is not turned stays as it is."""
    x = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(1)).bfloat16()
    x[0, 0, 3], x[0, 1, 50], x[1, 2, 40], x[1, 3, 63] = float("nan"), float("inf"), float("nan"), float("-inf")
    k, v = (torch.zeros(2, 8, 1, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    rates = ck.rope_rates(32)
    at = torch.arange(2, device="cuda", dtype=torch.int32)
    for interleaved, partner in ((True, 2), (False, 19)):
        q = ck.paged_write_rope(x[:, :2].cuda(), x[:, 2:3].cuda(), x[:, 3:].cuda(), at + 1, rates, k, v, at, interleaved=interleaved).cpu()
        bad = ~q.isfinite()
        assert bad.nonzero().tolist() == sorted([[0, 0, 3], [0, 0, partner], [0, 1, 50]]) and q[0, 1, 50] == float("inf")
        rows = k.flatten(0, 1)[:2].cpu()
        assert (~rows.isfinite()).nonzero().tolist() == [[1, 0, 40]] and torch.equal(v.flatten(0, 1)[:2].cpu(), x[:, 3:])


def test_as_apply_rope_and_paged_write(hip):
    """The same as the two calls it takes the place of, up to the matrices' 32 bits."""
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k = (torch.randn(30, h, 64, device="cuda", generator=g).bfloat16() for h in (4, 4))
    rates = ck.rope_rates(64)
    angle = torch.arange(30, device="cuda")[:, None] * rates
    f = torch.stack((angle.cos(), -angle.sin(), angle.sin(), angle.cos()), -1).reshape(1, 30, 1, 32, 2, 2)
    want = ck.apply_rope(q[None], k[None], f)
    cache = [torch.zeros(4, 8, 4, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    at = torch.arange(30, device="cuda", dtype=torch.int32)
    version = cache[0]._version
    got = ck.paged_write_rope(q, k, k, at, rates, *cache, at, keep_key=True)
    assert cache[0]._version > version
    for a, b in zip(got, want):
        assert float((a.float() - b[0].float()).abs().max()) <= 2.0 ** -7 * float(b.abs().max())
    assert torch.equal(cache[0].flatten(0, 1)[:30], got[1]) and torch.equal(cache[1].flatten(0, 1)[:30], k)


def test_past_4_gib(hip):
    """A slot whose byte offset does not fit 32 bits."""
    pages = 2 ** 17 + 3
    k, v = (torch.empty(pages, 16, 8, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(2, 24, 128, device="cuda", generator=g).half()
    slots = torch.tensor([pages * 16 - 1, 2 ** 21 + 5], dtype=torch.int32, device="cuda")
    at = torch.tensor([7, 9], dtype=torch.int32, device="cuda")
    _, kept = ck.paged_write_rope(x[:, :8], x[:, 8:16], x[:, 16:], at, ck.rope_rates(128), k, v, slots, keep_key=True)
    assert torch.equal(k.flatten(0, 1)[slots.long()], kept) and torch.equal(v.flatten(0, 1)[slots.long()], x[:, 16:])


def test_captured(hip):
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(9, 12, 128, device="cuda", generator=g).bfloat16()
    at = torch.arange(9, dtype=torch.int32, device="cuda")
    rates = ck.rope_rates(128)
    k, v, k2, v2 = (torch.zeros(8, 16, 2, 128, dtype=torch.bfloat16, device="cuda") for _ in range(4))

    def step(k, v):
        return ck.paged_write_rope(x[:, :8], x[:, 8:10], x[:, 10:], at, rates, k, v, at, interleaved=False)

    step(k, v)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        q = step(k, v)
    for i in range(3):
        at.add_(9)
        x.mul_(-1.25)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q, step(k2, v2))
        n = 9 * (i + 2)
        assert torch.equal(k.flatten(0, 1)[9:n], k2.flatten(0, 1)[9:n]) and torch.equal(v.flatten(0, 1)[9:n], v2.flatten(0, 1)[9:n])


def test_refusals(hip):
    q = torch.zeros(4, 6, 64, dtype=torch.bfloat16, device="cuda")
    cache = torch.zeros(3, 8, 2, 64, dtype=torch.bfloat16, device="cuda")
    i = torch.zeros(4, dtype=torch.int32, device="cuda")
    rates = ck.rope_rates(64)

    def call(q=q, key=q[:, :2], value=q[:, :2], at=i, rates=rates, k=cache, v=cache.clone(), slots=i, **more):
        return ck.paged_write_rope(q, key, value, at, rates, k, v, slots, **more)

    for kwargs, text in ((dict(key=q[:3, :2]), "do not fit"), (dict(value=q[:, :2].half()), "do not fit"), (dict(key=q[:, :3]), "do not fit"),
                         (dict(rates=ck.rope_rates(66)), "head_dim"), (dict(at=i[:3]), "positions"), (dict(slots=i[:3]), "slots"),
                         (dict(k=cache.half(), v=cache.half()), "into a cache"), (dict(k=cache[:2]), "differ"),
                         (dict(k_scale=torch.tensor(1.0)), "float8_e4m3fn"),
                         (dict(q=q[..., :40], key=q[:, :2, :40], value=q[:, :2, :40], k=cache[..., :40], v=cache[..., :40], rates=rates[:4]), "multiple of 16")):
        with pytest.raises(ValueError, match=text):
            call(**kwargs)
    for kwargs in (dict(q=q.float()), dict(at=i.float()), dict(rates=rates.double()), dict(q=q.cpu()), dict(at=i[None])):
        with pytest.raises(ck.NoCapableBackendError):
            call(**kwargs)
