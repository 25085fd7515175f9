"""Attention of sequences that begin with the same tokens against its definition in 64 bits (bounds: attention_ref.py)."""
import pytest
import torch

import comfy_kitchen as ck
from attention_ref import attend, check

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
NAN = float("nan")


class Pool:
    """groups: [(common tokens, [own tokens of each sequence])], None in place of a number of common tokens at
    either end: sequences in no group.  Every element of the cache that no token owns is NaN, and the page
    tables hold nonsense where they are not needed, the common tokens' of all but a group's first among that."""

    def __init__(self, groups, heads, kv_heads, dim, page, dtype="bf16", cache=None, seed=0, layout="PTHD", spread=1.0):
        g = torch.Generator().manual_seed(seed)
        cache = cache or dtype
        self.lengths, self.starts, self.shared, self.rows = [], [], [], []
        plan = []  # of each sequence: tokens of the group that its table places, its own
        for common, own in groups:
            for i, n in enumerate(own):
                plan.append((common or 0, n, i == 0))
                self.lengths.append((common or 0) + n)
            if common is not None:
                self.starts = (self.starts or [len(plan) - len(own)]) + [len(plan)]
                self.shared.append(common)
        need = [-(-n // page) for n in self.lengths]
        total = sum(need) + 3
        order = torch.randperm(total, generator=g).tolist()
        k = torch.full((total, page, kv_heads, dim), NAN)
        v = torch.full((total, page, kv_heads, dim), NAN)
        self.table = torch.full((len(plan), max(need, default=0) + 1), -7, dtype=torch.int32)
        head = None
        for b, (common, own, first) in enumerate(plan):
            kb, vb = (torch.randn(common + own, kv_heads, dim, generator=g) * s for s in (spread, 1.0))
            if cache == "e4m3":
                kb, vb = (x.mul(64).clamp(-448, 448).to(DT["e4m3"]).float() for x in (kb, vb))
            else:
                kb, vb = (x.to(DT[cache]).float() for x in (kb, vb))
            if first:
                head = kb[:common], vb[:common]
            kb[:common], vb[:common] = head
            seen = list(range(0 if first else common, common + own))
            pages = [order.pop() for _ in range(need[b])]
            for i in {t // page for t in seen}:
                self.table[b, i] = pages[i]
            at = torch.tensor([pages[t // page] * page + t % page for t in seen], dtype=torch.long)
            k.view(-1, kv_heads, dim)[at] = kb[seen]
            v.view(-1, kv_heads, dim)[at] = vb[seen]
            self.rows.append((kb.double(), vb.double()))
        self.k, self.v = k.to(DT[cache]).cuda(), v.to(DT[cache]).cuda()
        if layout == "PHTD":
            self.k, self.v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (self.k, self.v))
        elif layout == "layers":
            self.k, self.v = (torch.stack((torch.full_like(x.float(), NAN).to(x.dtype), x), 1)[:, 1] for x in (self.k, self.v))
        self.scales = (0.015625, 0.03125) if cache == "e4m3" else (None, None)
        self.q = torch.randn(len(plan), heads, dim, generator=g).to(DT[dtype])
        self.kv_heads, self.dim = kv_heads, dim

    def run(self, q=None, scale=None, starts=None, shared=None, lengths=None):
        def i32(x):
            return torch.tensor(x, dtype=torch.int32).cuda()

        ks, vs = (None if s is None else torch.tensor(s).cuda() for s in self.scales)
        return ck.shared_attention(self.q.cuda() if q is None else q, self.k, self.v, self.table.cuda(), i32(lengths or self.lengths),
                                   i32(self.starts if starts is None else starts), i32(self.shared if shared is None else shared), scale=scale,
                                   k_scale=ks, v_scale=vs)

    def want(self, scale=None, lengths=None):
        scale = self.dim ** -0.5 if scale is None else scale
        ks, vs = (1.0 if s is None else s for s in self.scales)
        rep = self.q.shape[1] // self.kv_heads
        o, bound = torch.zeros(self.q.shape, dtype=torch.float64), torch.zeros(self.q.shape, dtype=torch.float64)
        for b, (k, v) in enumerate(self.rows):
            n = (lengths or self.lengths)[b]
            for h in range(self.kv_heads):
                hs = slice(h * rep, (h + 1) * rep)
                o[b, hs], bound[b, hs] = attend(self.q[b, hs].double(), k[:n, h] * ks, v[:n, h] * vs, scale, self.q.dtype)
        return o, bound


def same(pool, **how):
    want = pool.want(**{k: v for k, v in how.items() if k in ("scale", "lengths")})
    check(pool.run(**how), *want)


MIXED = [(None, [40, 0, 200]), (100, [1, 30, 5]), (333, [0, 0, 7, 64, 65]), (64, [9]), (0, [3, 4]), (500, []), (1000, [1] * 40), (None, [77, 3])]


@pytest.mark.parametrize("page", [1, 8, 16, 20, 64, 256])
@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"), ("f16", "e4m3")])
def test_groups_and_pages(dtype, cache, page, hip):
    same(Pool(MIXED, 4, 2, 64, page, dtype, cache, seed=page))


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"), ("f16", "e4m3")])
@pytest.mark.parametrize("page", [12, 16])
def test_head_dims(dim, dtype, cache, page, hip):
    same(Pool([(300, [5, 70, 1]), (None, [33])], 6, 2, dim, page, dtype, cache, seed=dim))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (7, 7), (5, 1), (16, 1), (40, 1), (24, 2), (40, 8), (130, 1), (300, 2)])
def test_head_layouts(heads, kv_heads, hip):
    same(Pool([(200, [33, 5, 1, 2]), (65, [10] * 9)], heads, kv_heads, 64, 16, seed=heads))


@pytest.mark.parametrize("tokens", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257])
def test_lengths(tokens, hip):
    same(Pool([(tokens, [1, 0, 2]), (3, [tokens, 1]), (None, [tokens])], 4, 2, 64, 16, seed=tokens))


def test_rows_in_several_blocks(hip):
    """32 to some hundred rows: waves and workgroups that are partly and wholly used."""
    for members in (8, 9, 31, 32, 33, 64, 100):
        same(Pool([(150, [1 + i % 3 for i in range(members)])], 4, 1, 64, 16, seed=members))


@pytest.mark.parametrize("layout", ["PHTD", "layers"])
@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_cache_layouts(layout, cache, hip):
    same(Pool(MIXED, 8, 4, 128, 16, "bf16", cache, layout=layout, seed=1))


def test_long_prefix_in_many_chunks(hip):
    same(Pool([(30001, [400, 1, 77])], 4, 1, 64, 16, seed=2))
    same(Pool([(9000, [3000, 2]), (5000, [1, 1]), (None, [7001])], 4, 2, 128, 64, "f16", "e4m3", seed=3))


def test_many_sequences(hip):
    same(Pool([(70 + i, [(7 * j + i) % 50 for j in range(1 + i % 5)]) for i in range(250)], 2, 1, 64, 16, seed=4))
    same(Pool([(40, [1 + j % 3 for j in range(1500)])], 2, 1, 64, 8, seed=5))


def test_large_scores_and_scale(hip):
    same(Pool(MIXED, 4, 2, 64, 16, spread=20.0, seed=7))
    same(Pool(MIXED, 4, 2, 64, 24, "f16", spread=8.0, seed=8))
    pool = Pool(MIXED, 4, 2, 64, 16, seed=9)
    same(pool, scale=-0.3)
    same(pool, scale=0.0)


def test_more_shared_than_a_sequence_holds(hip):
    """Then as many as the shortest of the group holds."""
    pool = Pool([(300, [50, 1, 20])], 4, 2, 64, 16, seed=10)
    for b in range(1, 3):  # the tables place all tokens of all sequences
        pool.table[b, :300 // 16] = pool.table[0, :300 // 16]
    own = pool.k, pool.v
    full = [(k.clone(), v.clone()) for k, v in pool.rows]
    for b in range(3):  # a row of the page that is common only in part: its copies
        for t in range(288, 300):
            at = int(pool.table[b, 18]) * 16 + t % 16
            own[0].view(-1, 2, 64)[at] = full[b][0][t].bfloat16().cuda()
            own[1].view(-1, 2, 64)[at] = full[b][1][t].bfloat16().cuda()
    for lengths in ([350, 301, 320], [350, 100, 7], [0, 301, 320], [64, 64, 64]):
        same(pool, lengths=lengths)
        if min(lengths) <= 300:  # or more were said to be common than are
            same(pool, lengths=lengths, shared=[10 ** 9])
        same(pool, lengths=lengths, shared=[-5])
        same(pool, lengths=lengths, shared=[], starts=[2])


def test_a_value_that_is_not_finite(hip):
    """It reaches the heads that see it, all the group's where it is common, and no others."""
    for cache in ("bf16", "e4m3"):
        pool = Pool([(100, [30, 40]), (100, [20])], 4, 2, 64, 16, "bf16", cache, seed=11)
        want, bound = pool.want()
        at = int(pool.table[0, 3]) * 16 + 2
        pool.k.view(-1, 2, 64)[at, 1, 5] = NAN
        at = int(pool.table[1, 7]) * 16 + 2
        pool.v.view(-1, 2, 64)[at, 0, 5] = NAN
        got = pool.run()
        assert bool(got[:2, 2:].isnan().all()) and bool(got[1, :2, 5].isnan().all())
        got[1, :2, 5] = want[1, :2, 5].to(got)
        check(got[:2, :2], want[:2, :2], bound[:2, :2] + 1)
        check(got[0, :2], want[0, :2], bound[0, :2])
        check(got[2], want[2], bound[2])


def test_as_paged_attention(hip):
    """What it takes the place of, on tables that place every token."""
    pool = Pool([(320, [50, 1, 20]), (None, [100])], 8, 2, 128, 16, seed=12)
    pool.table[1:3, :20] = pool.table[0, :20]
    n = torch.tensor(pool.lengths, dtype=torch.int32).cuda()
    other = ck.paged_attention(pool.q.cuda(), pool.k, pool.v, pool.table.cuda(), n)
    check(pool.run(), other.cpu().double(), 2 * pool.want()[1])


def test_query_strides_and_stream(hip):
    pool = Pool(MIXED, 4, 2, 128, 16, seed=13)
    q = pool.q.cuda()
    want = pool.run()
    fused = torch.randn(len(q), 12, 128, device="cuda").bfloat16()
    fused[:, 3:7] = q
    assert torch.equal(pool.run(fused[:, 3:7]), want)
    odd = torch.zeros(len(q), 4, 131, device="cuda").bfloat16()
    odd[..., 1:129] = q
    assert torch.equal(pool.run(odd[..., 1:129]), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pool.run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_captured_with_changing_lengths(hip):
    pool = Pool([(700, [300, 40, 1]), (64, [5, 6])], 4, 2, 64, 16, seed=14)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    args = [pool.q.cuda(), pool.k, pool.v, pool.table.cuda(), i32(pool.lengths), i32(pool.starts), i32(pool.shared)]
    ck.shared_attention(*args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ck.shared_attention(*args)
        second = ck.shared_attention(args[0] * 2, *args[1:])
    for now in (pool.lengths, [701, 740, 700, 64, 70], [1000, 700, 701, 69, 65]):
        args[4].copy_(i32(now))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ck.shared_attention(*args)) and torch.equal(second, ck.shared_attention(args[0] * 2, *args[1:]))
        check(out, *pool.want(lengths=now))


def test_rows_past_4_gib(hip):
    pages, page, hk, d = 40000, 64, 8, 128
    g = torch.Generator(device="cuda").manual_seed(1)
    for cache in (torch.bfloat16, torch.float8_e4m3fn):
        k, v = (torch.empty(2 * pages if cache.itemsize == 1 else pages, page, hk, d, dtype=cache, device="cuda") for _ in range(2))
        use = [len(k) - 1, 3, len(k) // 2, len(k) - 2]
        for i in use:
            for x in (k, v):
                x[i] = torch.randn(page, hk, d, device="cuda", generator=g).to(cache)
        q = torch.randn(2, hk, d, device="cuda", generator=g).bfloat16()
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        got = ck.shared_attention(q, k, v, i32([use[:3], [0, 0, use[3]]]), i32([150, 170]), i32([0, 2]), i32([128]))
        for b, (last, n) in enumerate(((use[2], 150), (use[3], 170))):
            at = torch.tensor([*use[:2], last], device="cuda")
            rk, rv = (x[at].reshape(-1, hk, d)[:n].double().cpu() for x in (k, v))
            for h in range(hk):
                check(got[b, h:h + 1], *attend(q[b, h:h + 1].double().cpu(), rk[:, h], rv[:, h], d ** -0.5, torch.bfloat16))
        del k, v


def test_bounds_that_make_no_sense_are_safe(hip):
    """Group bounds, lengths and pages outside what they count give some finite result, and no fault."""
    k = torch.randn(6, 16, 2, 64, device="cuda").bfloat16()
    q = torch.randn(5, 4, 64, device="cuda").bfloat16()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    table = i32([[99, -5, 2 ** 31 - 1]] * 5)
    for starts in ([0, 5, 3, 8], [-4, 99, -1, 2], [5, 0, 0, 0], [2 ** 31 - 1, -2 ** 31, 7, 3], [3, 1, 4, 1]):
        out = ck.shared_attention(q, k, k, table, i32([10 ** 9, -4, 3, 40, 17]), i32(starts), i32([2 ** 31 - 1, -7, 20]))
        assert bool(out.isfinite().all()) and bool((out[1] == 0).all())


def test_nothing_to_do(hip):
    k = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    none = i32([])
    assert ck.shared_attention(q[:0], k, k, i32([]).reshape(0, 2), none, i32([0]), none).shape == (0, 4, 64)
    out = ck.shared_attention(q + 1, k + 1, k + 1, i32([]).reshape(3, 0), i32([0, 5, 0]), i32([0, 3]), i32([4]))
    assert bool((out == 0).all())  # tables without a column hold no tokens


def test_refusals(hip):
    pool = Pool([(20, [1, 2])], 4, 2, 64, 16)
    q, k, v, t = pool.q.cuda(), pool.k, pool.v, pool.table.cuda()
    n = torch.tensor(pool.lengths, dtype=torch.int32).cuda()
    args = dict(q=q, k_cache=k, v_cache=v, page_table=t, lengths=n, groups=n, shared=n[:1])
    for bad, match in ((dict(q=q.half()), "a cache of"), (dict(q=q[:, :3]), "does not fit"), (dict(v_cache=v[:2]), "differ"),
                       (dict(page_table=t.repeat(2, 1)), "sequences"), (dict(shared=n), "groups"), (dict(groups=n[:0], shared=n[:0]), "groups"),
                       (dict(k_cache=k[..., :32], v_cache=v[..., :32], q=q[..., :32]), "head_dim"),
                       (dict(k_scale=torch.zeros(2, device="cuda")), "one element")):
        with pytest.raises(ValueError, match=match):
            ck.shared_attention(**{**args, **bad})
    for bad in (dict(q=q.float()), dict(page_table=t.long()), dict(lengths=n.cpu()), dict(groups=n.long()), dict(shared=n.float())):
        with pytest.raises(ck.NoCapableBackendError):
            ck.shared_attention(**{**args, **bad})
    many = torch.zeros(4097, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="4096"):
        ck.shared_attention(q[:1].expand(4097, -1, -1), k, v, many[:, None], many, many[:1], many[:0])
