"""Arguments of the text-generation calls: one sequence, token or head cut from something wider gives what
a copy of it gives, and scales are taken where they mean something."""
import pytest
import torch

import comfy_kitchen as ck

pytestmark = pytest.mark.gpu


def cut(batch, heads, width, off, dtype=torch.bfloat16, seed=0):
    """`batch` rows of heads of 64 from rows of any width, `off` elements behind their begin."""
    g = torch.Generator().manual_seed(seed)
    wide = torch.randn(batch + 1, width, generator=g).to(dtype).cuda()
    return wide[:, off:off + heads * 64].unflatten(1, (heads, 64))[:batch]


@pytest.mark.parametrize("batch", [1, 2])
@pytest.mark.parametrize("width,off", [(772, 0), (771, 0), (772, 4), (771, 3), (768, 0), (768, 1)])
def test_attention_and_writes(batch, width, off, hip):
    q, k, v = cut(batch, 4, width, off), cut(batch, 2, width, off, seed=1), cut(batch, 2, width, off, seed=2)
    plain = [t.clone(memory_format=torch.contiguous_format).reshape(-1).clone().view(t.shape) for t in (q, k, v)]
    caches = []
    for key, value in ((k, v), plain[1:]):
        pair = [torch.zeros(3, 16, 2, 64, dtype=q.dtype, device="cuda") for _ in range(2)]
        ck.paged_write(key, value, *pair, torch.arange(batch, device="cuda") * 16)
        caches.append(pair)
    assert all(torch.equal(a, b) for a, b in zip(*caches)) and torch.equal(caches[0][0][0, 0], k[0])
    table = torch.arange(batch, dtype=torch.int32, device="cuda")[:, None]
    lengths = torch.ones(batch, dtype=torch.int32, device="cuda")
    want = ck.paged_attention(plain[0], *caches[1], table, lengths)
    assert torch.equal(ck.paged_attention(q, *caches[0], table, lengths), want)
    assert torch.equal(want, v.repeat_interleave(2, 1))  # one visible token each
    # queries as a prompt of one sequence, and as one token of each sequence
    for shape in ((lambda t: t[None]), (lambda t: t[:, None])):
        got = ck.window_attention(*(shape(t) for t in (q, k, v)), 1)
        assert torch.equal(got, shape(want))


@pytest.mark.parametrize("pages,page,heads", [(1, 16, 2), (3, 1, 2), (3, 16, 1)])
def test_caches_with_a_dimension_of_one(pages, page, heads, hip):
    """Their odd strides there address nothing: used in place."""
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(pages, page, heads, 64, generator=g).bfloat16().cuda() for _ in range(2))
    odd = [t.as_strided(t.shape, [s if n > 1 else 2 * s + 3 for n, s in zip(t.shape[:-1], t.stride())] + [1]) for t in (k, v)]
    q = torch.randn(1, 4, 64, generator=g).bfloat16().cuda()
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    lengths = torch.tensor([pages * page - 1], dtype=torch.int32, device="cuda")
    assert torch.equal(ck.paged_attention(q, *odd, table, lengths), ck.paged_attention(q, k, v, table, lengths))
    row = torch.randn(1, heads, 64, generator=g).bfloat16().cuda()
    last = torch.tensor([pages * page - 1], device="cuda")
    ck.paged_write(row, -row, *odd, last)
    assert torch.equal(k[-1, -1], row[0]) and torch.equal(v[-1, -1], -row[0])
    ck.paged_copy(*odd, last, torch.zeros_like(last))
    assert torch.equal(k[0, 0], row[0]) and torch.equal(v[0, 0], -row[0])


def test_nothing_to_do(hip):
    codes = torch.zeros(8, 64, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(8, 1, dtype=torch.bfloat16, device="cuda")
    x = torch.zeros(128, 9, dtype=torch.bfloat16, device="cuda").t()
    assert ck.linear_int4(x[:0], codes, scales).shape == (0, 8)
    assert ck.linear_int4(x[:0].unflatten(0, (0, 3)), codes, scales).shape == (0, 3, 8)
    k = torch.zeros(2, 9, 2, 64, dtype=torch.bfloat16, device="cuda")
    assert ck.window_attention(x[:0, :64].reshape(0, 64)[None, :, None].expand(2, 0, 4, 64), k, k).shape == (2, 0, 4, 64)


def test_scales_of_16_bit_caches(hip):
    """Rows are written as they are there: a scale is refused; attention multiplies by it."""
    k, v = (torch.randn(2, 16, 2, 64, device="cuda").bfloat16() for _ in range(2))
    row, slot, two = k[0, :1], torch.zeros(1, dtype=torch.int32, device="cuda"), torch.tensor(2.0, device="cuda")
    for scales in (dict(k_scale=two), dict(v_scale=two)):
        with pytest.raises(ValueError, match="float8_e4m3fn"):
            ck.paged_write(row, row, k, v, slot, **scales)
    q = torch.randn(1, 2, 64, device="cuda").bfloat16()
    args = (torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), torch.tensor([20], dtype=torch.int32, device="cuda"))
    assert torch.equal(ck.paged_attention(q, k, v, *args, k_scale=two, v_scale=two), ck.paged_attention(q, k * 2, v * 2, *args))
