"""Attention inputs in which every key counts (test infrastructure).

Head h of a key-value head sees (score 0) the keys of its own segment and next to nothing (score -60)
of the others'; value dimension d of a key is 1 where the key is of class d, else 0.  So result (h, d)
is the share of class d among the visible keys of segment h: weights of 1 and 2^-86, whole-number
sums that are exact, one rounding.  Runs of 32 keys are of one class, and a result counts few keys:
where some are left out or read twice it is off by far more than its rounding."""
import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
FAR = 60.0  # exact in all of the cache's types


def segment(t, reps, run):
    """The head that sees key t: runs of `run` keys in turn."""
    return t // run % reps


def kind(t, dim, reps, run):
    """The class of key t: of runs of 32 keys in turn, counted within the segment's runs."""
    return (t // 32 + t // (run * reps) * 7) % dim


def keys_values(n, reps, dim, run, value, device="cpu"):
    """k, v [n, dim] of one key-value head; value: what v holds in place of 1 (a power of two)."""
    t = torch.arange(n, device=device)
    k = torch.zeros(n, dim, device=device)
    k[:, :reps] = -FAR
    k[t, segment(t, reps, run)] = 0.0
    v = torch.zeros(n, dim, device=device)
    v[t, kind(t, dim, reps, run)] = value
    return k, v


def queries(reps, dim):
    """q [reps, dim] for a scale of 1."""
    return torch.eye(reps, dim)


def counts(see, reps, dim, run):
    """see [..., n] (truth values) -> keys of each segment and class [..., reps, dim] in 64 bits."""
    t = torch.arange(see.shape[-1], device=see.device)
    cell = segment(t, reps, run) * dim + kind(t, dim, reps, run)
    out = torch.zeros(*see.shape[:-1], reps * dim, dtype=torch.float64, device=see.device)
    return out.scatter_add_(-1, cell.expand(see.shape), see.double()).unflatten(-1, (reps, dim))


def shares(count, value=1.0):
    """What attention gives.  A head none of whose own keys are visible weighs all alike."""
    own = count.sum(-1, keepdim=True)
    every = count.sum(-2, keepdim=True).expand_as(count)
    return value * torch.where(own > 0, count / own.clamp(min=1), every / every.sum(-1, keepdim=True).clamp(min=1))


def check(got, want, dtype):
    """One rounding of a value that an fp32 division left 2^-23 off (f16: to 2^-24 where that is more); the
    others' keys are at most a million times e^-60 of it."""
    err = (got.detach().double() - want.to(got.device)).abs()
    bound = 1.01 * UNIT[dtype] * want.to(got.device) + (1.01 * 2.0 ** -25 if dtype == torch.float16 else 1e-16)
    assert got.shape == want.shape and bool((err <= bound).all()), float((err / bound).max())
