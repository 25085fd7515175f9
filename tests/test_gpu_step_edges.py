"""Calls at the ends of what the operators of a generation step allow: numbers outside their range, the largest rows, two
streams at once, gradients being recorded, the same sequence twice."""
import pytest
import torch

import comfy_kitchen as ck

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("how", [dict(), dict(top_p=0.8), dict(top_k=40, min_p=0.01)], ids=["plain", "top_p", "top_k"])
def test_random_numbers_outside_their_range(how, hip):
    logits = torch.randn(5, 9000, generator=torch.Generator().manual_seed(0)).cuda() * 3
    got = ck.sample_tokens(logits, torch.tensor([NAN, -3.0, -INF, 1.0, INF], device="cuda"), **how)
    # as at the ends of the range
    assert torch.equal(got, ck.sample_tokens(logits, torch.tensor([0.0, 0.0, 0.0, 1 - 2.0 ** -24, 1 - 2.0 ** -24], device="cuda"), **how))


def test_an_infinite_temperature_weighs_all_alike(hip):
    logits = torch.randn(64, 1000, generator=torch.Generator().manual_seed(1)).cuda()
    logits[:, ::4] = -INF
    logits[:, 1] = NAN
    u = (torch.arange(64, device="cuda") + 0.5) / 64
    for temperature in (torch.full((64,), INF, device="cuda"), INF):
        got = ck.sample_tokens(logits, u, temperature=temperature)
        order = logits.nan_to_num(nan=-INF, neginf=-INF).sort(dim=-1, descending=True, stable=True).indices
        # the first whose number of tokens up to itself exceeds u times 749
        assert torch.equal(got, order.gather(1, (u.double() * 749).floor().long()[:, None])[:, 0])


def test_the_largest_vocabulary(hip):
    n = 1 << 24
    logits = torch.full((2, n), -5.0, dtype=torch.bfloat16, device="cuda")
    logits[0, n - 1] = 30.0
    logits[1, 5], logits[1, n - 2] = 20.0, 20.0
    got = ck.sample_tokens(logits, torch.tensor([0.99, 0.75], device="cuda"), top_p=0.5)
    # 2^24 exp(-25) = 2.3e-4 stands behind the two of weight 1: the first falls short of half of it all
    assert got.tolist() == [n - 1, n - 2]
    assert ck.sample_tokens(logits, torch.tensor([0.99, 0.75], device="cuda"), top_k=2).tolist() == [n - 1, n - 2]
    flat = ck.sample_tokens(torch.zeros(1, n, device="cuda"), torch.tensor([0.5], device="cuda"))
    assert flat.item() == n // 2  # counts and weights of 2^24 equal logits
    with pytest.raises(RuntimeError, match="logits"):
        ck.sample_tokens(torch.zeros(1, 1, device="cuda").expand(1, n + 1).half(), torch.zeros(1, device="cuda"))
    many = ck.sample_tokens(logits[:1, :9].expand(65535, -1), torch.zeros(65535, device="cuda"))
    assert bool((many == 0).all())
    with pytest.raises(RuntimeError, match="rows"):
        ck.sample_tokens(logits[:1, :9].expand(65536, -1), torch.zeros(65536, device="cuda"))


def make_cache(pages, page, kv, dim, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(pages, page, kv, dim, device="cuda", generator=g).bfloat16() for _ in range(2)]


def test_on_two_streams_at_once(hip):
    g = torch.Generator(device="cuda").manual_seed(2)
    x, r = (torch.randn(300, 5120, device="cuda", generator=g).bfloat16() for _ in range(2))
    logits = torch.randn(40, 50001, device="cuda", generator=g) * 2
    u = torch.rand(40, device="cuda", generator=g)
    k, v = make_cache(200, 16, 2, 128)
    q = torch.randn(20, 16, 128, device="cuda", generator=g).bfloat16()
    table = torch.arange(200, device="cuda", dtype=torch.int32)[None].repeat(20, 1)
    lengths = i32([1500 + 70 * i for i in range(20)])

    def run():
        return (*ck.rms_norm(x, None, r), *ck.rms_norm_mxfp8(x), ck.sample_tokens(logits, u, top_p=0.9),
                ck.shared_attention(q, k, v, table, lengths, i32([0, 8, 20]), i32([1400, 1600])))

    want = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    for one in got:
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(one, want))


def test_where_gradients_are_recorded(hip):
    """The custom ops around the calls give the same; nothing here has a gradient."""
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = make_cache(40, 16, 2, 64)
    q = torch.randn(6, 8, 64, device="cuda", generator=g).bfloat16()
    table = torch.arange(40, device="cuda", dtype=torch.int32).view(1, -1).repeat(6, 1)
    lengths, groups, shared = i32([300, 320, 500, 640, 10, 0]), i32([0, 3, 6]), i32([290, 400])
    want = ck.shared_attention(q, k, v, table, lengths, groups, shared)
    x = torch.randn(6, 8, 64, device="cuda", generator=g).bfloat16()
    key, value = (torch.randn(6, 2, 64, device="cuda", generator=g).bfloat16() for _ in range(2))
    rates, positions, slots = ck.rope_rates(64), torch.arange(6, device="cuda") * 1000, i32([5, 80, -1, 639, 640, 7])
    rates = rates.cuda()
    a, b = [t.clone() for t in (k, v)], [t.clone() for t in (k, v)]
    y, yk = ck.paged_write_rope(x, key, value, positions, rates, *a, slots, keep_key=True)
    before = b[0]._version
    x.requires_grad_()
    q.requires_grad_()
    assert torch.equal(ck.shared_attention(q, k, v, table, lengths, groups, shared).detach(), want)
    y2, yk2 = ck.paged_write_rope(x, key, value, positions, rates, *b, slots, keep_key=True)
    assert torch.equal(y, y2.detach()) and torch.equal(yk, yk2.detach()) and b[0]._version > before
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.equal(ck.rms_norm(x).detach(), ck.rms_norm(x.detach()))
    with torch.no_grad():
        assert not ck.rms_norm(x).requires_grad


def test_one_sequence_several_times(hip):
    """The same pages in every row of the table, all of a sequence's tokens shared."""
    k, v = make_cache(30, 64, 2, 128, 4)
    q = torch.randn(17, 16, 128, device="cuda").bfloat16()
    table = torch.arange(30, device="cuda", dtype=torch.int32)[None].expand(17, -1)
    for n in (1, 64, 1919, 1920):
        got = ck.shared_attention(q, k, v, table, i32([n] * 17), i32([0, 17]), i32([n]))
        one = [ck.shared_attention(q[i:i + 1], k, v, table[:1], i32([n]), i32([0]), i32([])) for i in range(17)]
        # both within their bounds of the exact value: a rounding of the result each, and of the weights
        top = v.float().abs().amax()
        assert bool(((got.float() - torch.cat(one).float()).abs() <= 2 * 2.0 ** -8 * got.float().abs() + 4 * 2.0 ** -8 * top).all())


@pytest.mark.parametrize("page", [16, 24])
def test_one_key_value_head_for_many(page, hip):
    """64 query heads on one key-value head, in no group: a sequence's own tokens have many rows too."""
    k, v = make_cache(600, page, 1, 128, 5)
    q = torch.randn(9, 64, 128, device="cuda").bfloat16()
    table = torch.randperm(600, device="cuda")[:9 * 64].view(9, 64).int()
    lengths = i32([1, 64 * page, 63, 65, 0, 1000, 129, 128, 900])
    got = ck.shared_attention(q, k, v, table, lengths, i32([3]), i32([]))
    want = ck.paged_attention(q, k, v, table, lengths)
    top = v.float().abs().amax()
    assert bool(((got.float() - want.float()).abs() <= 2 * 2.0 ** -8 * want.float().abs() + 4 * 2.0 ** -8 * top).all()) and bool((got[4] == 0).all())
