"""Attention over a cache held in pages against its definition in 64 bits (bounds: attention_ref.py)."""
import pytest
import torch

import comfy_kitchen as ck
from attention_ref import attend, check, visible

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
NAN = float("nan")


class Pool:
    """A cache whose every element that no visible token owns is NaN, and whose page table holds
    nonsense where it is not needed."""

    def __init__(self, lengths, heads, kv_heads, dim, page, dtype="bf16", cache=None, window=0, sinks=0, seed=0,
                 layout="PTHD", spread=1.0):
        g = torch.Generator().manual_seed(seed)
        cache = cache or dtype
        self.window, self.sinks, self.lengths = window, sinks, lengths
        need = [-(-n // page) for n in lengths]
        total = sum(need) + 3
        order = torch.randperm(total, generator=g).tolist()
        k = torch.full((total, page, kv_heads, dim), NAN)
        v = torch.full((total, page, kv_heads, dim), NAN)
        self.table = torch.full((len(lengths), max(need, default=0) + 1), -7, dtype=torch.int32)
        self.rows = []
        for b, n in enumerate(lengths):
            pages = [order.pop() for _ in range(need[b])]
            seen = visible(n, window, sinks)
            kb = torch.randn(len(seen), kv_heads, dim, generator=g) * spread
            vb = torch.randn(len(seen), kv_heads, dim, generator=g)
            if cache == "e4m3":
                kb, vb = (x.mul(64).clamp(-448, 448).to(DT["e4m3"]).float() for x in (kb, vb))
            else:
                kb, vb = (x.to(DT[cache]).float() for x in (kb, vb))
            for i in {t // page for t in seen}:
                self.table[b, i] = pages[i]
            at = torch.tensor([pages[t // page] * page + t % page for t in seen], dtype=torch.long)
            k.view(-1, kv_heads, dim)[at] = kb
            v.view(-1, kv_heads, dim)[at] = vb
            self.rows.append((kb.double(), vb.double()))
        self.k, self.v = k.to(DT[cache]).cuda(), v.to(DT[cache]).cuda()
        if layout == "PHTD":  # heads before tokens in memory
            self.k, self.v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (self.k, self.v))
        elif layout == "layers":  # one layer of a cache whose pages hold all layers
            self.k, self.v = (torch.stack((torch.full_like(x.float(), NAN).to(x.dtype), x), 1)[:, 1] for x in (self.k, self.v))
        self.scales = (0.015625, 0.03125) if cache == "e4m3" else (None, None)
        self.q = torch.randn(len(lengths), heads, dim, generator=g).to(DT[dtype])
        self.kv_heads, self.dim = kv_heads, dim

    def run(self, q=None, scale=None):
        ks, vs = (None if s is None else torch.tensor(s).cuda() for s in self.scales)
        return ck.paged_attention(self.q.cuda() if q is None else q, self.k, self.v, self.table.cuda(),
                                  torch.tensor(self.lengths, dtype=torch.int32).cuda(), scale=scale, window=self.window,
                                  sinks=self.sinks, k_scale=ks, v_scale=vs)

    def want(self, scale=None):
        scale = self.dim ** -0.5 if scale is None else scale
        ks, vs = (1.0 if s is None else s for s in self.scales)
        rep = self.q.shape[1] // self.kv_heads
        o, bound = torch.zeros(self.q.shape, dtype=torch.float64), torch.zeros(self.q.shape, dtype=torch.float64)
        for b, (k, v) in enumerate(self.rows):
            for h in range(self.kv_heads):
                hs = slice(h * rep, (h + 1) * rep)
                o[b, hs], bound[b, hs] = attend(self.q[b, hs].double(), k[:, h] * ks, v[:, h] * vs, scale, self.q.dtype)
        return o, bound


def same(pool, scale=None):
    check(pool.run(scale=scale), *pool.want(scale))


# lengths of nothing, one token, inside and at the ends of tiles of 32 and of pages; several chunks
LENGTHS = [0, 1, 15, 16, 17, 31, 32, 33, 64, 100, 511, 513, 1030, 2500]


@pytest.mark.parametrize("page", [1, 8, 16, 20, 24, 32, 48, 128])
@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"), ("f16", "e4m3")])
def test_lengths_and_pages(dtype, cache, page, hip):
    same(Pool(LENGTHS, 8, 2, 64, page, dtype, cache, seed=page))


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"), ("f16", "e4m3")])
@pytest.mark.parametrize("page", [16, 20])
def test_head_dims(dim, dtype, cache, page, hip):
    same(Pool([1, 47, 333, 1200], 6, 2, dim, page, dtype, cache, seed=dim))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (7, 7), (5, 1), (16, 1), (17, 1), (40, 1), (24, 2), (40, 8)])
@pytest.mark.parametrize("page", [12, 16])
def test_head_layouts(heads, kv_heads, page, hip):
    same(Pool([700, 33, 5], heads, kv_heads, 128, page, seed=heads))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (100, 0), (100, 33), (333, 64), (5000, 4), (0, 9)])
@pytest.mark.parametrize("page", [1, 16, 20, 64])
def test_window_and_sinks(window, sinks, page, hip):
    same(Pool([0, 1, 40, 101, 130, 500, 1777], 4, 2, 64, page, "bf16", window=window, sinks=sinks, seed=window))
    same(Pool([900, 31], 4, 4, 128, page, "f16", "e4m3", window=window, sinks=sinks, seed=sinks))


@pytest.mark.parametrize("layout", ["PHTD", "layers"])
@pytest.mark.parametrize("page", [16, 20])
@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_cache_layouts(layout, page, cache, hip):
    same(Pool([77, 600], 8, 4, 128, page, "bf16", cache, layout=layout, seed=1))


def test_many_sequences(hip):
    """More than a wave of sequences, of unlike lengths."""
    lengths = [(i * 37) % 300 for i in range(150)] + [4000]
    same(Pool(lengths, 4, 2, 64, 16, seed=3))
    same(Pool(lengths, 4, 2, 64, 10, seed=4))


def test_long_sequences_in_many_chunks(hip):
    same(Pool([70001], 2, 1, 64, 16, seed=5))
    same(Pool([30000, 3, 45001], 10, 2, 128, 256, "f16", seed=6))


def test_large_scores_and_scale(hip):
    """Scores whose maximum keeps rising and far ones that vanish; a negative scale; a scale of zero."""
    same(Pool([600, 70], 4, 2, 64, 16, spread=20.0, seed=7))
    same(Pool([600, 70], 4, 2, 64, 24, "f16", spread=8.0, seed=8))
    pool = Pool([300], 4, 2, 64, 16, seed=9)
    same(pool, scale=-0.3)
    same(pool, scale=0.0)


def test_not_a_number_where_it_is_seen(hip):
    """A NaN or infinity in a visible row reaches its heads and no others."""
    for page in (16, 20):
        pool = Pool([200, 100], 4, 2, 64, page, seed=10)
        want, bound = pool.want()
        row = int(pool.table[0, 3]) * page + 2
        pool.k.view(-1, 2, 64)[row, 1, 5] = NAN
        got = pool.run()
        assert bool(got[0, 2:].isnan().all())
        check(got[0, :2], want[0, :2], bound[0, :2])
        check(got[1], want[1], bound[1])


def test_query_strides_and_stream(hip):
    pool = Pool([90, 300], 4, 2, 128, 16, seed=11)
    q = pool.q.cuda()
    want = pool.run()
    fused = torch.randn(2, 12, 128, device="cuda").bfloat16()
    fused[:, 3:7] = q
    assert torch.equal(pool.run(fused[:, 3:7]), want)
    odd = torch.zeros(2, 4, 131, device="cuda").bfloat16()
    odd[..., 1:129] = q
    assert torch.equal(pool.run(odd[..., 1:129]), want)
    assert torch.equal(pool.run(q.transpose(0, 1).contiguous().transpose(0, 1)), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pool.run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_captured_with_changing_lengths(hip):
    """A captured call reads the lengths that the device holds at replay."""
    pool = Pool([2000, 1500, 40], 4, 2, 64, 16, seed=12)
    q, table = pool.q.cuda(), pool.table.cuda()
    lengths = torch.tensor(pool.lengths, dtype=torch.int32).cuda()
    ck.paged_attention(q, pool.k, pool.v, table, lengths)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ck.paged_attention(q, pool.k, pool.v, table, lengths)
    for now in ([2000, 1500, 40], [1, 0, 39], [777, 1500, 8], [2000, 20, 1]):
        lengths.copy_(torch.tensor(now, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ck.paged_attention(q, pool.k, pool.v, table, lengths))
        rows = [(k[:n], v[:n]) for (k, v), n in zip(pool.rows, now)]
        for b, (k, v) in enumerate(rows):
            for h in range(2):
                check(out[b, 2 * h:2 * h + 2], *attend(pool.q[b, 2 * h:2 * h + 2].double(), k[:, h], v[:, h], 0.125, torch.bfloat16))


def test_rows_past_4_gib(hip):
    """Pages whose offsets need more than 32 bits, as elements and as bytes."""
    pages, page, hk, d = 40000, 64, 8, 128  # 2.6e9 elements
    g = torch.Generator(device="cuda").manual_seed(1)
    for page_view in (64, 40):
        k = torch.empty(pages, page, hk, d, dtype=torch.bfloat16, device="cuda")
        v = torch.empty(pages, page, hk, d, dtype=torch.bfloat16, device="cuda")
        k, v = k[:, :page_view], v[:, :page_view]
        use = [39999, 3, 20000, 39998]
        for i in use:
            k[i].normal_(generator=g)
            v[i].normal_(generator=g)
        q = torch.randn(1, hk, d, device="cuda", generator=g).bfloat16()
        n = 4 * page_view - 7
        got = ck.paged_attention(q, k, v, torch.tensor([use], dtype=torch.int32, device="cuda"),
                                 torch.tensor([n], dtype=torch.int32, device="cuda"))
        rk, rv = (x[torch.tensor(use, device="cuda")].reshape(-1, hk, d)[:n].double().cpu() for x in (k, v))
        for h in range(hk):
            check(got[0, h:h + 1], *attend(q[0, h:h + 1].double().cpu(), rk[:, h], rv[:, h], d ** -0.5, torch.bfloat16))
        del k, v


def test_entries_outside_the_cache_are_safe(hip):
    """Page numbers and lengths outside the cache give some finite result, and no fault."""
    k = torch.randn(6, 16, 2, 64, device="cuda").bfloat16()
    table = torch.tensor([[99, -5, 2 ** 31 - 1], [1, 2, -2 ** 31]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([10 ** 9, -4], dtype=torch.int32, device="cuda")
    for cache in (k, k[:, :10]):
        out = ck.paged_attention(torch.randn(2, 4, 64, device="cuda").bfloat16(), cache, cache, table, lengths)
        assert bool(out.isfinite().all()) and bool((out[1] == 0).all())


def test_refusals(hip):
    pool = Pool([20], 4, 2, 64, 16)
    q, k, v, t = pool.q.cuda(), pool.k, pool.v, pool.table.cuda()
    n = torch.tensor([20], dtype=torch.int32).cuda()
    with pytest.raises(ck.NoCapableBackendError):
        ck.paged_attention(q.float(), k, v, t, n)
    with pytest.raises(ck.NoCapableBackendError):
        ck.paged_attention(q, k, v, t.long(), n)
    with pytest.raises(ck.NoCapableBackendError):
        ck.paged_attention(q, k, v, t, n.cpu())
    for bad, match in ((dict(q=q.half()), "a cache of"), (dict(q=q[:, :3]), "does not fit"), (dict(q=q[..., :32]), "does not fit"),
                       (dict(v_cache=v[:2]), "differ"), (dict(window=-1), "negative"), (dict(sinks=-1), "negative"),
                       (dict(page_table=t.repeat(2, 1)), "sequences"), (dict(k_cache=k[..., :32], v_cache=v[..., :32], q=q[..., :32]), "head_dim"),
                       (dict(k_cache=k.transpose(1, 3), v_cache=v.transpose(1, 3)), "contiguous|fit"),
                       (dict(k_scale=torch.zeros(2, device="cuda")), "one element")):
        args = dict(q=q, k_cache=k, v_cache=v, page_table=t, lengths=n)
        args.update(bad)
        with pytest.raises(ValueError, match=match):
            ck.paged_attention(**args)
