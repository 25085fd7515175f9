"""Writing and copying token rows of a paged cache, and the sequences of PagedKVCache: exact to the
bit against plain indexing."""
import pytest
import torch

import comfy_kitchen as ck
from attention_ref import attend, check

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}


def caches(pages, page, hk, d, dtype, layout, layers=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    shape = (pages, page, hk, d) if layers is None else (layers, pages, page, hk, d)
    out = []
    for _ in range(2):
        x = torch.randn(shape, generator=g).to(DT[dtype])
        if layout == "PHTD":
            x = x.cuda().transpose(-3, -2).contiguous().transpose(-3, -2)
        elif layout == "wide":  # a view of wider pages and heads
            big = torch.zeros(*shape[:-3], page + 3, hk + 1, d).to(DT[dtype]).cuda()
            big[..., :page, :hk, :] = x.cuda()
            x = big[..., :page, :hk, :]
        out.append(x.cuda())
    return out


def bits(t):
    return t.contiguous().view(torch.uint8).cpu()


@pytest.mark.parametrize("layout", ["plain", "PHTD", "wide"])
@pytest.mark.parametrize("cache", ["same", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,hk,d,page", [(0, 2, 64, 16), (1, 1, 16, 1), (37, 3, 96, 20), (300, 8, 128, 64)])
def test_write(tokens, hk, d, page, dtype, cache, layout, hip):
    g = torch.Generator().manual_seed(tokens + d)
    pages = -(-tokens // page) + 2
    k, v = caches(pages, page, hk, d, dtype if cache == "same" else cache, layout)
    fused = (torch.randn(tokens, 3 * hk, d, generator=g) * 200).to(DT[dtype])  # q, k and v of one projection
    if tokens:
        fused[0, :, :2] = torch.tensor([float("inf"), -0.0]).to(DT[dtype])
    key, value = fused[:, hk:2 * hk], fused[:, 2 * hk:]
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    slots[::5] = torch.where(torch.arange(len(slots[::5])) % 2 == 0, -1, pages * page)
    scales = (0.5, 1.75) if cache == "e4m3" else (None, None)
    want = []
    for x, c, s in ((key, k, scales[0]), (value, v, scales[1])):
        w = c.cpu().clone(memory_format=torch.contiguous_format)
        live = (slots >= 0) & (slots < pages * page)
        row = x[live]
        if s is not None:
            row = (row.float() / s).clamp(-448, 448).to(DT["e4m3"])
        w.view(torch.uint8 if w.element_size() == 1 else torch.int16).view(-1, hk, d)[slots[live]] = row.view(
            torch.uint8 if w.element_size() == 1 else torch.int16)
        want.append(w)
    args = [None if s is None else torch.tensor(s).cuda() for s in scales]
    for kind in (torch.int64, torch.int32):
        ck.paged_write(fused.cuda()[:, hk:2 * hk], fused.cuda()[:, 2 * hk:], k, v, slots.to(kind).cuda(), *args)
        assert torch.equal(bits(k), bits(want[0])) and torch.equal(bits(v), bits(want[1]))


@pytest.mark.parametrize("layers", [None, 1, 3])
@pytest.mark.parametrize("layout", ["plain", "PHTD", "wide"])
@pytest.mark.parametrize("dtype,hk,d,page,rows", [("bf16", 2, 64, 16, 40), ("f16", 3, 8, 5, 11), ("e4m3", 1, 96, 20, 1),
                                                  ("e4m3", 8, 128, 64, 333), ("bf16", 8, 128, 64, 0), ("bf16", 5, 256, 7, 200)])
def test_copy(dtype, hk, d, page, rows, layout, layers, hip):
    g = torch.Generator().manual_seed(rows)
    pages = 2 * -(-rows // page) + 3
    k, v = caches(pages, page, hk, d, dtype, layout, layers)
    order = torch.randperm(pages * page, generator=g)
    src, dst = order[:rows].clone(), order[rows:2 * rows].clone()
    if rows > 10:
        src[3], dst[7], src[5] = -1, pages * page, src[4]  # skipped twice; one row to two places
    live = (src >= 0) & (dst < pages * page)
    want = []
    for c in (k, v):
        w = c.cpu().clone(memory_format=torch.contiguous_format)
        flat = w.view(torch.uint8 if w.element_size() == 1 else torch.int16).view(layers or 1, -1, hk, d)
        flat[:, dst[live]] = flat[:, src[live]]
        want.append(w)
    for kind in (torch.int32, torch.int64):
        ck.paged_copy(k, v, src.to(kind).cuda(), dst.to(kind).cuda())
        assert torch.equal(bits(k), bits(want[0])) and torch.equal(bits(v), bits(want[1]))


def test_copy_past_4_gib(hip):
    k = torch.empty(2, 20000, 64, 8, 128, dtype=torch.bfloat16, device="cuda")  # 5.2 GB a tensor
    v = torch.empty_like(k)
    src = torch.arange(64, dtype=torch.int32, device="cuda") + 19999 * 64
    dst = torch.arange(64, dtype=torch.int32, device="cuda") + 7 * 64
    k[:, 19999].normal_()
    v[:, 19999].normal_()
    ck.paged_copy(k, v, src, dst)
    assert torch.equal(k[:, 7], k[:, 19999]) and torch.equal(v[:, 7], v[:, 19999])
    x = torch.randn(64, 8, 128, device="cuda").bfloat16()
    ck.paged_write(x, -x, k[1], v[1], src)
    assert torch.equal(k[1, 19999], x) and torch.equal(v[1, 19999], -x)


def test_refusals(hip):
    k, v = caches(4, 16, 2, 64, "bf16", "plain")
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    s = torch.arange(3, dtype=torch.int32, device="cuda")
    with pytest.raises(ck.NoCapableBackendError):
        ck.paged_write(x.float(), x.float(), k, v, s)
    with pytest.raises(ck.NoCapableBackendError):
        ck.paged_write(x, x, k, v, s.float())
    with pytest.raises(ck.NoCapableBackendError):
        ck.paged_copy(k.float(), v.float(), s, s + 8)
    for bad, match in ((dict(value=x[:2]), "fit"), (dict(key=x.half(), value=x.half()), "into a cache"), (dict(slots=s[:2]), "slots for"),
                       (dict(v_cache=v[:, :8]), "differ"), (dict(key=x[..., :32], value=x[..., :32]), "fit"),
                       (dict(k_cache=k.half()), "differ")):
        args = dict(key=x, value=x, k_cache=k, v_cache=v, slots=s)
        args.update(bad)
        with pytest.raises(ValueError, match=match):
            ck.paged_write(**args)
    with pytest.raises(ValueError, match="differ"):
        ck.paged_copy(k, v, s, s[:2] + 8)
    with pytest.raises(ValueError, match="contiguous"):
        ck.paged_copy(k[..., 1:], v[..., 1:], s, s + 8)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("page", [16, 10])
def test_sequences_end_to_end(dtype, page, hip):
    """Appends, forks, trims and compactions against lists of rows, attention after every step."""
    g = torch.Generator().manual_seed(page)
    layers, hk, heads, d = 2, 2, 4, 64
    cache = ck.PagedKVCache(layers, 60, page, hk, d, DT[dtype], k_scale=1 / 64 if dtype == "e4m3" else None,
                            v_scale=1 / 64 if dtype == "e4m3" else None)
    rows = {}  # sequence -> per layer (k, v) in 64 bits

    def append(sequences, counts):
        slots = cache.append(sequences, counts)
        for layer in range(layers):
            k, v = (torch.randn(sum(counts), hk, d, generator=g).bfloat16() for _ in range(2))
            cache.write(layer, k.cuda(), v.cuda(), slots)
            if dtype == "e4m3":
                k, v = ((x.float() * 64).clamp(-448, 448).to(DT["e4m3"]).double() / 64 for x in (k, v))
            at = 0
            for s, n in zip(sequences, counts):
                old = rows[s][layer]
                rows[s][layer] = tuple(torch.cat((o, x[at:at + n].double())) for o, x in zip(old, (k, v)))
                at += n

    def start():
        s = cache.add()
        rows[s] = [(torch.zeros(0, hk, d).double(),) * 2 for _ in range(layers)]
        return s

    def fork(s):
        c = cache.fork(s)
        rows[c] = list(rows[s])
        return c

    def look(sequences, window=0, sinks=0):
        table, lengths = cache.tables(sequences)
        for layer in range(layers):
            q = torch.randn(len(sequences), heads, d, generator=g).bfloat16()
            got = cache.attend(layer, q.cuda(), table, lengths, window=window, sinks=sinks)
            for b, s in enumerate(sequences):
                k, v = rows[s][layer]
                first = max(0, len(k) - window) if window else 0
                at = list(range(min(sinks, first))) + list(range(first, len(k)))
                for h in range(hk):
                    check(got[b, 2 * h:2 * h + 2], *attend(q[b, 2 * h:2 * h + 2].double(), k[at, h], v[at, h], d ** -0.5, torch.bfloat16))

    a, b = start(), start()
    append([a, b], [37, 5])
    look([a, b])
    c, e = fork(a), fork(a)
    append([c, a, e], [1, 3, 2])  # three owners of one partly filled page
    look([a, b, c, e])
    append([b], [page - 5])
    f = fork(b)  # a full last page is shared without a copy
    append([b, f], [1, 1])
    look([b, f])
    keep = [0, 1, 5, 6, 7, 20, 30, 33, 39]
    cache.compact(a, keep)
    rows[a] = [tuple(x[keep] for x in kv) for kv in rows[a]]
    append([a], [9])
    look([a, c, e])
    append([e], [80])
    assert cache.trim(e, 30, 4) > 0
    look([e], 30, 4)
    append([e], [3])
    look([e, c], 30, 4)
    for s in (a, b, c, e, f):
        cache.free(s)
    assert cache.free_pages == 60


def test_sequences_of_no_tokens(hip):
    cache = ck.PagedKVCache(1, 4, 16, 2, 64)
    a, b = cache.add(), cache.add()
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    assert cache.append([a, b], [0, 0]).shape == (0,)
    out = cache.attend(0, q, *cache.tables([a, b]))  # a table without a column
    assert out.shape == q.shape and bool((out == 0).all())
    slots = cache.append([b], [1])
    row = torch.randn(1, 2, 64, device="cuda").bfloat16()
    cache.write(0, row, row, slots)
    out = cache.attend(0, q, *cache.tables([a, b]))
    assert bool((out[0] == 0).all()) and torch.equal(out[1], row[0].repeat_interleave(2, 0))
    assert cache.attend(0, q[:0], *cache.tables([])).shape == (0, 4, 64)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    ck.paged_write(row[:0], row[:0], cache.k[0], cache.v[0], none)
    ck.paged_copy(cache.k, cache.v, none, none)
