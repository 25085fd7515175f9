"""Attention in 64 bits from its definition, and how far a result computed in 32 bits with 16-bit
weights may be from it (test infrastructure).

The bound: one rounding of the result and one of each weight, unit * (|o| + A) with A = sum p |v| /
sum p and unit 2^-8 (bf16) or 2^-11 (f16); the scores' fp32 sums of at most 256 products err by
2^-16 S, S the largest scale * sum |q k|, which the weights take on as a relative error, with
2^-16 for the exponential; weights under f16's normal range, against a largest of at least 1,
err by 2^-25 each."""
import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def attend(q, k, v, scale, dtype, largest=1.0):
    """q [..., d], k and v [n, d] in 64 bits -> (o, bound); no keys give zeros.  largest: what the
    largest weight is held at, at least."""
    if k.shape[0] == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    s = q @ k.t() * scale
    p = torch.exp(s - s.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    o = p @ v / total
    mass = p @ v.abs() / total
    size = (q.abs() @ k.abs().t()).amax(-1, keepdim=True) * abs(scale)
    bound = 1.01 * UNIT[dtype] * (o.abs() + mass) + 2.0 ** -16 * (1 + size) * mass + 1e-7
    if dtype == torch.float16:
        bound = bound + k.shape[0] * 2.0 ** -25 / largest * v.abs().amax() / total
    return o, bound


def check(got, want, bound):
    err = (got.detach().cpu().double() - want).abs()
    assert got.shape == want.shape
    assert bool((err <= bound).all()), (float((err / bound.clamp_min(1e-30)).max()), int((~(err <= bound)).sum()))


def visible(length, window, sinks):
    """Positions that a query at position length - 1 sees."""
    first = max(0, length - window) if window > 0 else 0
    return list(range(min(sinks, first))) + list(range(first, length))
