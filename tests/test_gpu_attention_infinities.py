"""Infinities in keys that are seen: a query whose score there is -inf gives that key no weight, one whose
score is +inf has no defined result and gives NaN; nothing else changes."""
import pytest
import torch

import comfy_kitchen as ck
from attention_ref import attend, check

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
INF = float("inf")


def judge(got, q, k, v, see, at, bad, dtype):
    """got, q [rows, d] of one head, see [rows, n]; key `at` of k (finite here) held bad at element 7."""
    for i in range(len(q)):
        if not see[i, at] or q[i, 7] * bad < 0:
            seen = see[i].clone()
            seen[at] = False
            check(got[i:i + 1], *attend(q[i:i + 1].double(), k[seen].double(), v[seen].double(), q.shape[1] ** -0.5, dtype))
        else:
            assert bool(got[i].isnan().all())


@pytest.mark.parametrize("bad", [INF, -INF])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
def test_window(d, dtype, bad, hip):
    g = torch.Generator().manual_seed(d)
    q, k, v = (torch.randn(1, 130, h, d, generator=g).to(DT[dtype]) for h in (2, 1, 1))
    p = torch.arange(130)
    see = (p[None] <= p[:, None]) & ((p[:, None] - p < 50) | (p < 3))
    for at in (1, 64, 100):
        x = k.clone()
        x[0, at, 0, 7] = bad
        got = ck.window_attention(q.cuda(), x.cuda(), v.cuda(), 50, 3).cpu()
        for h in range(2):
            judge(got[0, 2:, h], q[0, 2:, h], k[0, :, 0], v[0, :, 0], see[2:], at, bad, DT[dtype])


@pytest.mark.parametrize("bad", [INF, -INF])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("page", [16, 20])
def test_paged(page, dtype, bad, hip):
    g = torch.Generator().manual_seed(page)
    n, d = 700, 64
    q, k, v = (torch.randn(s, d, generator=g).to(DT[dtype]) for s in (16, n, n))
    need = -(-n // page)
    table = torch.randperm(need, generator=g).to(torch.int32)
    at = torch.arange(n)
    rows = table[at // page].long() * page + at % page
    for key in (0, 333, 699):
        x = k.clone()
        x[key, 7] = bad
        caches = []
        for t in (x, v):
            c = torch.zeros(need * page, d, dtype=DT[dtype])
            c[rows] = t
            caches.append(c.view(need, page, 1, d).cuda())
        got = ck.paged_attention(q[None].cuda(), *caches, table[None].cuda(), torch.tensor([n], dtype=torch.int32).cuda())[0].cpu()
        judge(got, q, k, v, torch.ones(16, n, dtype=torch.bool), key, bad, DT[dtype])
