"""The next token against its definition in 64 bits: equal, for every row.

A result could differ where a running weight lies within 2^-33 of the border that it is compared with: under 2^-10
in all of this file's draws together, of which none does."""
import numpy as np
import pytest
import torch

import comfy_kitchen as ck
from sample_ref import pick

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
INF, NAN = float("inf"), float("nan")


def same(logits, u, **how):
    """logits [rows, vocab] on the CPU; each of how a number, or a list of one a row."""
    given = {k: torch.tensor(v, dtype=torch.int32 if k == "top_k" else torch.float32).cuda() if isinstance(v, list) else v
             for k, v in how.items()}
    got = ck.sample_tokens(logits.cuda(), u.cuda(), **given)
    assert got.dtype == torch.int64 and got.shape == (logits.shape[0],)
    rows, us = logits.double().numpy(), u.double().numpy()
    want = []
    for i in range(len(rows)):
        one = {k: given[k][i].item() if isinstance(v, list) else v for k, v in how.items()}
        want.append(pick(rows[i], us[i], **one))
    assert got.cpu().tolist() == want


def make(rows, vocab, dtype, seed=0, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * spread
    x += 6.0 * (torch.rand(rows, vocab, generator=g) < 12 / vocab)
    return x.to(DT[dtype]), torch.rand(rows, generator=g)


HOW = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=2), dict(top_k=50), dict(top_p=0.9), dict(top_p=0.3, temperature=1.3),
       dict(min_p=0.05), dict(min_p=1.0), dict(top_k=40, top_p=0.8, min_p=0.02, temperature=0.8), dict(top_k=700, top_p=0.99), dict(temperature=0.0),
       dict(top_p=0.0), dict(temperature=2.0, top_p=0.95), dict(top_k=10 ** 6, top_p=1.0), dict(temperature=1e-3), dict(temperature=50.0, top_p=0.7)]


@pytest.mark.parametrize("how", HOW, ids=lambda h: "-".join(f"{k}{v}" for k, v in h.items()) or "plain")
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_filters(dtype, how, hip):
    same(*make(24, 9001, dtype, 1), **how)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 7), (5, 8), (300, 100), (2, 8191), (2, 8192), (2, 8193), (3, 16385), (2, 40001), (2, 131072),
                                        (1, 250007)])
def test_sizes(rows, vocab, dtype, hip):
    logits, u = make(rows, vocab, dtype, vocab)
    for how in (dict(), dict(top_k=30, top_p=0.9), dict(top_p=0.95, min_p=0.001), dict(temperature=0.0)):
        same(logits, u, **how)


@pytest.mark.parametrize("vocab", [1, 64, 4096, 5000, 32768, 100000])
def test_equal_logits(vocab, hip):
    """All tokens weigh the same: which one a share of the weight falls on is exact."""
    rows = 64
    at = torch.linspace(0, vocab - 1, rows).floor()
    for value in (0.0, -0.0, 3.7, -1e4, 60000.0):
        logits = torch.full((rows, vocab), value)
        if value == 0.0:
            logits[:, ::2] = -0.0  # equal all the same
        if vocab & (vocab - 1) == 0:  # the shares are numbers of 32 bits
            u = at / vocab
            assert ck.sample_tokens(logits.cuda(), u.cuda()).cpu().tolist() == at.long().tolist()
        u = (at + 0.5) / vocab
        assert ck.sample_tokens(logits.cuda(), u.cuda(), temperature=1.7).cpu().tolist() == at.long().tolist()
        same(logits, u, top_k=max(1, vocab // 3))
        same(logits, u, top_p=0.5)
        same(logits.bfloat16(), u, top_p=0.25, min_p=1.0)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("spread", [1e-4, 0.01, 0.2])
def test_crowded_bins(dtype, spread, hip):
    """More logits in a bin than the list in LDS holds."""
    logits, u = make(6, 30000, "f32", 3, spread)
    logits = (logits.clamp(max=1.0) + 2).to(DT[dtype])
    for how in (dict(), dict(top_k=9000), dict(top_p=0.6, top_k=20000), dict(min_p=0.9), dict(temperature=300.0, top_p=0.9, min_p=0.5)):
        same(logits, u, **how)


def test_masked_rows(hip):
    logits, u = make(12, 20000, "f32", 4)
    logits[0] = -INF  # nothing to draw
    logits[1] = NAN
    logits[2] = -INF
    logits[2, 12345] = -3.0
    logits[3, ::2] = -INF
    logits[4, ::3] = NAN
    logits[5, [7, 15000]] = INF
    logits[6] = torch.finfo(torch.float32).min
    logits[7] = torch.finfo(torch.float32).min
    logits[7, 100] = 1.0
    logits[8, 5] = torch.finfo(torch.float32).max
    logits[9] = INF
    logits[10, 19999] = 1e30
    logits[11] *= 1e30
    for how in (dict(), dict(top_k=5), dict(top_p=0.9), dict(min_p=0.1, temperature=0.5), dict(temperature=0.0), dict(temperature=1e-30), dict(temperature=1e30)):
        same(logits, u, **how)


def test_u_at_its_ends(hip):
    logits, _ = make(2, 5000, "f32", 5)
    for u in (0.0, 1.0 - 2.0 ** -24):
        for how in (dict(), dict(top_k=3), dict(top_p=0.5), dict(min_p=0.3)):
            same(logits, torch.full((2,), u), **how)
    out = ck.sample_tokens(logits.cuda(), torch.tensor([1.0, 7.0], device="cuda"), top_k=3).cpu()  # taken as just under 1
    assert out.tolist() == [logits[i].topk(3).indices[2] for i in range(2)]


def test_weights_at_min_p(hip):
    """w = exp(-j) for whole j, and min_p one of these: equal is kept."""
    logits = -torch.arange(20.0).repeat(5, 1)
    u = torch.tensor([0.0, 0.7, 0.95, 0.999, 1 - 2.0 ** -24])
    for j in range(6):
        same(logits, u, min_p=float(np.exp(-float(j))))


def test_values_of_each_row(hip):
    logits, u = make(9, 12000, "bf16", 6)
    how = dict(temperature=[1.0, 0.0, 0.5, -1.0, 2.0, 1.0, 1.0, 0.9, NAN], top_k=[0, 5, 1, 0, 50, -3, 3, 10 ** 9, 0],
               top_p=[1.0, 0.5, 0.9, 0.1, 0.95, 0.0, 2.0, 0.7, 0.5], min_p=[0.0, 0.1, 0.0, 0.5, 0.01, 0.2, 3.0, 0.0, 0.0])
    got = ck.sample_tokens(logits.cuda(), u.cuda(), **{k: torch.tensor(v, dtype=torch.int32 if k == "top_k" else torch.float32).cuda() for k, v in how.items()})
    f = {k: torch.tensor(v, dtype=torch.float32).tolist() if k != "top_k" else v for k, v in how.items()}
    want = [pick(logits[i].double().numpy(), float(u[i]), f["temperature"][i], f["top_k"][i], f["top_p"][i], min(f["min_p"][i], 1.0)) for i in range(9)]
    assert got.cpu().tolist() == want
    for name in how:  # one of them a tensor, the others numbers
        same(logits, u, **{"top_k": 20, "top_p": 0.9, name: how[name][:1] * 5 + [how[name][2]] * 4})


def test_shares(hip):
    """4096 evenly spread numbers hit every token as often as its weight says, within one."""
    n = 4096
    logits = torch.randn(200, generator=torch.Generator().manual_seed(7))
    u = (torch.arange(n) + 0.5) / n
    got = ck.sample_tokens(logits.cuda().expand(n, -1), u.cuda(), temperature=0.8)
    count = torch.bincount(got.cpu(), minlength=200).double()
    p = torch.softmax(logits.double() / 0.8, -1)
    assert bool(((count - n * p).abs() <= 1.0001).all())


def test_strides_streams_and_repeats(hip):
    logits, u = make(6, 9001, "bf16", 8)
    wide = torch.zeros(6, 9100, dtype=torch.bfloat16, device="cuda")
    wide[:, 33:9034] = logits.cuda()
    first = ck.sample_tokens(logits.cuda(), u.cuda(), top_p=0.97)
    for x in (wide[:, 33:9034], logits.cuda().t().contiguous().t()):
        assert torch.equal(ck.sample_tokens(x, u.cuda(), top_p=0.97), first)
    assert torch.equal(torch.ops.comfy_kitchen.sample_tokens(logits.cuda(), u.cuda(), 1.0, 0, 0.97, 0.0, None, None, None, None), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [ck.sample_tokens(wide[:, 33:9034], u.cuda(), top_p=0.97) for _ in range(5)]
    side.synchronize()
    assert all(torch.equal(a, first) for a in again)
    assert ck.sample_tokens(logits[:0].cuda(), u[:0].cuda()).shape == (0,)


def test_captured(hip):
    logits, u = (t.cuda() for t in make(5, 20000, "f32", 9))
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    ck.sample_tokens(logits, u, top_p=0.9)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        a = ck.sample_tokens(logits, u, top_p=0.9)
        b = ck.sample_tokens(logits, u, top_k=40)
    for i in range(4):
        u.copy_(torch.rand(5, generator=torch.Generator().manual_seed(i)))
        logits.mul_(0.9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, ck.sample_tokens(logits, u, top_p=0.9)) and torch.equal(b, ck.sample_tokens(logits, u, top_k=40))


def test_refusals(hip):
    x, u = torch.zeros(3, 50, device="cuda"), torch.zeros(3, device="cuda")
    for kwargs in (dict(temperature=-0.5), dict(temperature=NAN), dict(top_k=-1), dict(top_p=-0.1), dict(min_p=1.5), dict(min_p=-0.1)):
        with pytest.raises(RuntimeError, match="sample"):
            ck.sample_tokens(x, u, **kwargs)
    with pytest.raises(ValueError, match="random numbers"):
        ck.sample_tokens(x, u[:2])
    with pytest.raises(ValueError, match="no logits"):
        ck.sample_tokens(x[:, :0], u)
    for kwargs in (dict(temperature=u[:2]), dict(top_k=u), dict(top_p=u.double()), dict(min_p=u[:, None])):
        with pytest.raises(ValueError, match="for each of 3 rows"):
            ck.sample_tokens(x, u, **kwargs)
    with pytest.raises(ValueError, match="devices"):
        ck.sample_tokens(x, u, top_p=u.cpu())
    for args in ((x.double(), u), (x, u.double()), (x[0], u), (x.cpu(), u)):
        with pytest.raises(ck.NoCapableBackendError):
            ck.sample_tokens(*args)
