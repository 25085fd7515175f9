"""Prompt attention with a sliding window and sinks against its definition in 64 bits (bounds:
attention_ref.py)."""
import pytest
import torch

import comfy_kitchen as ck
from attention_ref import UNIT, attend, check

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def inputs(b, sq, sk, hq, hk, d, dtype, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed + sq * 31 + sk)
    return ((torch.randn(b, sq, hq, d, generator=g) * spread).to(DT[dtype]), torch.randn(b, sk, hk, d, generator=g).to(DT[dtype]),
            torch.randn(b, sk, hk, d, generator=g).to(DT[dtype]))


def seen(sq, sk, window, sinks, length):
    p = torch.arange(sq)[:, None] + sk - sq
    j = torch.arange(sk)[None]
    near = (p - j < window) if window > 0 else torch.ones(1, 1, dtype=torch.bool)
    return (j <= p) & (j < length) & (near | (j < sinks))


def want(q, k, v, window=0, sinks=0, lengths=None, scale=None):
    b, sq, hq, d = q.shape
    sk, hk = k.shape[1:3]
    scale = d ** -0.5 if scale is None else scale
    unit = UNIT[q.dtype]
    q, k, v = ((x.cuda().double()) for x in (q, k, v))
    o, bound = torch.zeros_like(q), torch.zeros_like(q)
    for i in range(b):
        see = seen(sq, sk, window, sinks, sk if lengths is None else lengths[i]).cuda()
        some = see.any(1)
        for h in range(hq):
            kk, vv = k[i, :, h // (hq // hk)], v[i, :, h // (hq // hk)]
            s = (q[i, :, h] @ kk.t() * scale).masked_fill(~see, -float("inf"))
            p = torch.exp(s - s.amax(1, keepdim=True)).masked_fill(~see, 0.0)
            total = p.sum(1, keepdim=True)
            x, mass = p @ vv / total, p @ vv.abs() / total
            size = (q[i, :, h].abs() @ kk.abs().t()).amax(1, keepdim=True) * abs(scale)
            limit = 1.01 * unit * (x.abs() + mass) + 2.0 ** -16 * (1 + size) * mass + 1e-7
            if unit == 2.0 ** -11:
                limit = limit + see.sum(1, keepdim=True) * 2.0 ** -25 * vv.abs().amax() / total
            o[i, :, h] = torch.where(some[:, None], x, 0.0)
            bound[i, :, h] = torch.where(some[:, None], limit, 0.0)
    return o.cpu(), bound.cpu()


def same(q, k, v, window=0, sinks=0, lengths=None, scale=None):
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32).cuda()
    got = ck.window_attention(q.cuda(), k.cuda(), v.cuda(), window, sinks, n, scale)
    assert got.dtype == q.dtype and got.is_contiguous()
    check(got, *want(q, k, v, window, sinks, lengths, scale))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("sq,sk", [(1, 1), (31, 31), (64, 64), (65, 65), (130, 130), (300, 300), (1, 200), (5, 133), (70, 260), (129, 64)])
def test_lengths(sq, sk, d, dtype, hip):
    same(*inputs(2, sq, sk, 3, 1, d, dtype))
    same(*inputs(1, sq, sk, 2, 2, d, dtype), window=50, sinks=3)


@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 4), (8, 2), (5, 1), (17, 1), (40, 8), (33, 3)])
def test_head_layouts(hq, hk, hip):
    same(*inputs(1, 150, 150, hq, hk, 64, "bf16"), window=70, sinks=2)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (63, 4), (64, 64), (65, 100), (200, 33), (5000, 4), (0, 7)])
@pytest.mark.parametrize("sq,sk", [(400, 400), (100, 431), (3, 700)])
def test_window_and_sinks(sq, sk, window, sinks, hip):
    same(*inputs(1, sq, sk, 4, 2, 64, "bf16"), window=window, sinks=sinks)
    same(*inputs(2, sq, sk, 2, 2, 128, "f16"), window=window, sinks=sinks)


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 5)])
def test_padded_batch(window, sinks, hip):
    """Lengths of none, one, inside and past the padded length; rows past them that see nothing."""
    same(*inputs(6, 150, 150, 4, 2, 64, "bf16"), window=window, sinks=sinks, lengths=[0, 1, 64, 100, 150, 999])
    same(*inputs(3, 20, 150, 4, 2, 128, "f16"), window=window, sinks=sinks, lengths=[0, 131, -3])


def test_no_keys_and_no_queries(hip):
    q, k, v = (x.cuda() for x in inputs(2, 5, 9, 4, 2, 64, "bf16"))
    assert bool((ck.window_attention(q, k[:, :0], v[:, :0]) == 0).all())
    assert ck.window_attention(q[:, :0], k, v).shape == (2, 0, 4, 64)
    assert ck.window_attention(q[:0], k[:0], v[:0]).shape == (0, 5, 4, 64)


def test_long(hip):
    same(*inputs(1, 3001, 3001, 5, 1, 128, "bf16"), window=1000, sinks=70)
    same(*inputs(1, 2500, 4100, 2, 2, 64, "f16"))


@pytest.mark.parametrize("d", [64, 96, 128, 256])
def test_few_rows_over_many_keys(d, hip):
    """Keys split over workgroups: ranges without a visible pair, sinks in the first, rows that see
    nothing, values that are not finite where they are not seen."""
    same(*inputs(1, 1, 5000, 4, 2, d, "bf16"))
    same(*inputs(2, 3, 3333, 5, 1, d, "f16"), window=2000, sinks=40)
    same(*inputs(3, 7, 2100, 4, 4, d, "bf16"), window=0, sinks=0, lengths=[0, 900, 2098])
    q, k, v = inputs(1, 40, 4000, 2, 1, d, "bf16")
    w, bound = want(q, k, v, 1500, 0)
    v[0, 3980] = float("inf")
    got = ck.window_attention(q.cuda(), k.cuda(), v.cuda(), 1500).cpu()
    check(got[:, :20], w[:, :20], bound[:, :20])
    assert bool((got[:, 20:] == float("inf")).all())


def test_large_scores_and_scales(hip):
    same(*inputs(1, 200, 200, 4, 2, 64, "bf16", spread=20.0))
    same(*inputs(1, 200, 200, 4, 2, 64, "f16", spread=8.0), window=100)
    q, k, v = inputs(1, 100, 130, 2, 1, 128, "bf16")
    same(q, k, v, scale=-0.3)
    same(q, k, v, scale=0.0)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_many_small_weights(dtype, hip):
    """One near key among far ones whose weights e^-far add up; f16 has 2^-24 for e^-16.25 = 1.47 2^-24,
    so its weights are held 2^7 larger."""
    g = torch.Generator().manual_seed(2)
    n, d, heads, rows = 400000, 64, 64, 512
    k = torch.zeros(n, d)
    k[100, 0] = 16.25
    v = torch.randn(n, d, generator=g) + 1
    v[100] = -3.0
    q = torch.zeros(1, rows, heads, d)
    q[..., 0] = 8.0  # scale 1/8
    k, v, q = (x.to(DT[dtype]) for x in (k, v, q))
    got = ck.window_attention(q.cuda(), k.cuda()[None, :, None], v.cuda()[None, :, None])[0, -1]
    check(got, *attend(q[0, -1].double(), k.double(), v.double(), 0.125, DT[dtype], 2.0 ** 7))


def test_strides(hip):
    g = torch.Generator().manual_seed(3)
    fused = torch.randn(2, 90, 8, 64, generator=g).bfloat16()  # q, k, v heads of one projection
    q, k, v = fused[:, :, :4], fused[:, :, 4:6], fused[:, :, 6:]
    w = want(q, k, v, 33, 2)
    d = fused.cuda()
    check(ck.window_attention(d[:, :, :4], d[:, :, 4:6], d[:, :, 6:], 33, 2), *w)
    heads_first = [x.transpose(1, 2).contiguous().cuda().transpose(1, 2) for x in (q, k, v)]
    check(ck.window_attention(*heads_first, 33, 2), *w)
    odd = torch.zeros(2, 90, 8, 67).bfloat16().cuda()
    odd[..., 1:65] = d
    check(ck.window_attention(odd[:, :, :4, 1:65], odd[:, :, 4:6, 1:65], odd[:, :, 6:, 1:65], 33, 2), *w)
    one = k[:, :1].expand(2, 90, 2, 64)  # every key the same row
    check(ck.window_attention(q.cuda(), one.cuda()[:, :1].expand(2, 90, 2, 64), v.cuda()), *want(q, one, v))


@pytest.mark.parametrize("bad", [float("inf"), float("nan"), -float("inf")])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_not_finite_where_it_is_not_seen(d, dtype, bad, hip):
    """Keys and values that are not finite reach the queries that see them, and no others."""
    q, k, v = inputs(1, 300, 300, 2, 1, d, dtype, seed=5)
    w, bound = want(q, k, v, 100, 3)
    for tensor, at in ((v, 150), (v, 299), (k, 130), (v, 10)):
        x = tensor.clone()
        x[0, at, 0, 7] = bad
        kk, vv = (x, v) if tensor is k else (k, x)
        got = ck.window_attention(q.cuda(), kk.cuda(), vv.cuda(), 100, 3).cpu()
        see = seen(300, 300, 100, 3, 300)[:, at]
        check(got[:, ~see], w[:, ~see], bound[:, ~see])
        if tensor is v:  # other elements of the rows that see it are as they were
            others = [i for i in range(d) if i != 7]
            check(got[:, see][..., others], w[:, see][..., others], bound[:, see][..., others])
            hit = got[:, see][..., 7]
            assert bool(hit.isnan().all()) if bad != bad else bool((hit == bad).all())
        elif bad != -float("inf"):
            assert not bool(got[:, see].isfinite().all(-1).any()) or bad == float("inf")
    lengths = torch.tensor([200], dtype=torch.int32).cuda()  # padding that holds anything
    k2, v2 = k.clone(), v.clone()
    k2[:, 200:], v2[:, 200:] = bad, bad
    check(ck.window_attention(q.cuda(), k2.cuda(), v2.cuda(), 0, 0, lengths), *want(q, k, v, 0, 0, [200]))


def test_stream_and_graph(hip):
    q, k, v = (x.cuda() for x in inputs(1, 200, 200, 4, 2, 64, "bf16"))
    first = ck.window_attention(q, k, v, 64, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ck.window_attention(q, k, v, 64, 4)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ck.window_attention(q, k, v, 64, 4)
    for i in range(3):
        q.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ck.window_attention(q, k, v, 64, 4))


def test_offsets_past_4_gib(hip):
    """Batch and head offsets that need more than 32 bits."""
    k = torch.empty(3, 2, 6_000_000, 128, dtype=torch.bfloat16, device="cuda").transpose(1, 2)  # 9.2 GB
    v = k  # keys and values from one tensor
    k[:, :300].normal_()
    q = torch.randn(3, 40, 2, 128, device="cuda").bfloat16()
    got = ck.window_attention(q, k[:, :300], v[:, :300], 128, 4)
    check(got, *want(q.cpu(), k[:, :300].cpu(), v[:, :300].cpu(), 128, 4))


def test_refusals(hip):
    q, k, v = (x.cuda() for x in inputs(1, 8, 8, 4, 2, 64, "bf16"))
    with pytest.raises(ck.NoCapableBackendError):
        ck.window_attention(q.float(), k, v)
    with pytest.raises(ck.NoCapableBackendError):
        ck.window_attention(q[0], k, v)
    with pytest.raises(ck.NoCapableBackendError):
        ck.window_attention(q, k, v, lengths=torch.tensor([8]).cuda())
    for args, match in (((q, k.half(), v), "dtypes"), ((q, k, v[:, :4]), "fit"), ((q[:, :, :3], k, v), "fit"),
                        ((q[..., :32], k[..., :32], v[..., :32]), "head_dim"), ((q, k, v, -1), "negative"), ((q, k, v, 4, -1), "negative"),
                        ((q, k, v, 0, 0, torch.zeros(2, dtype=torch.int32).cuda()), "lengths")):
        with pytest.raises(ValueError, match=match):
            ck.window_attention(*args)
