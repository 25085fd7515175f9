"""Every key of a long sequence counts (attention_cells.py): none is left out or read twice by any
chunk, wave, range or join."""
import pytest
import torch

import attention_cells as cells
import comfy_kitchen as ck

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}


# lengths, query heads a key-value head, key-value heads, head_dim, page, query and cache types, window, sinks.
# One sequence in as many chunks as there are, in hundreds, two tiles in a wave, unlike ones together
PAGED = [([600001], 16, 1, 64, 64, "f16", "f16", 0, 0), ([70001], 16, 1, 64, 16, "bf16", "bf16", 0, 0),
         ([70001], 16, 2, 64, 20, "bf16", "e4m3", 0, 0), ([30000, 3, 45001], 5, 2, 128, 256, "f16", "f16", 0, 0),
         ([4000], 5, 8, 128, 16, "bf16", "bf16", 0, 0), ([9000, 4000, 1, 8999], 4, 8, 128, 8, "bf16", "bf16", 0, 0),
         ([1023, 1024, 1025], 16, 1, 96, 12, "f16", "e4m3", 0, 0), ([2500, 5000], 16, 1, 256, 32, "bf16", "bf16", 0, 0),
         ([50000, 20000], 8, 2, 128, 64, "bf16", "e4m3", 8192, 33), ([40007], 16, 2, 96, 20, "f16", "f16", 30001, 100),
         ([0, 1, 31, 33, 511, 513, 2500], 3, 2, 64, 1, "bf16", "bf16", 0, 0)]


@pytest.mark.parametrize("run", [1, 32, 5000])
@pytest.mark.parametrize("case", PAGED, ids=str)
def test_paged(case, run, hip):
    lengths, reps, kv_heads, dim, page, dtype, cache, window, sinks = case
    g = torch.Generator().manual_seed(1)
    need = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(need) + 2, generator=g).to(torch.int32).cuda()
    k, v = (torch.full((sum(need) + 2, page, kv_heads, dim), float("nan"), device="cuda").to(DT[cache]) for _ in range(2))
    table = torch.full((len(lengths), max(need)), -1, dtype=torch.int32, device="cuda")
    want, at = [], 0
    for b, n in enumerate(lengths):
        pages = order[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = pages
        t = torch.arange(n, device="cuda")
        see = (t >= n - window if window else t >= 0) | (t < sinks)
        rows = pages[t[see] // page].long() * page + t[see] % page
        count = cells.counts(see, reps, dim, run)
        for h in range(kv_heads):
            kk, vv = cells.keys_values(n, reps, dim, run, 2.0 ** h, "cuda")
            for x, y in ((k, kk), (v, vv)):
                x.view(-1, kv_heads, dim)[rows, h] = y[see].to(DT[cache])
            want.append(cells.shares(count, 2.0 ** h))
    q = cells.queries(reps, dim).repeat(len(lengths), kv_heads, 1).to(DT[dtype]).cuda()
    got = ck.paged_attention(q, k, v, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), 1.0, window, sinks)
    cells.check(got, torch.stack(want).view(q.shape), DT[dtype])


# batch, queries, keys, query heads a key-value head, key-value heads, head_dim, type, window, sinks
WINDOW = [(1, 1, 50001, 4, 2, 64, "bf16", 0, 0), (2, 3, 3333, 5, 1, 128, "f16", 2000, 40), (1, 40, 20000, 2, 1, 96, "bf16", 15000, 0),
          (1, 3001, 3001, 5, 1, 128, "bf16", 1000, 70), (1, 2500, 4100, 2, 2, 64, "f16", 0, 0), (1, 777, 777, 3, 8, 64, "f16", 256, 4),
          (1, 4096, 4096, 4, 1, 256, "bf16", 1500, 16), (3, 200, 1500, 16, 2, 128, "f16", 333, 65)]


@pytest.mark.parametrize("run", [1, 32, 700])
@pytest.mark.parametrize("case", WINDOW, ids=str)
def test_window(case, run, hip):
    batch, queries, keys, reps, kv_heads, dim, dtype, window, sinks = case
    lengths = [keys - 37 * b for b in range(batch)]
    p, j = torch.arange(queries, device="cuda")[:, None] + keys - queries, torch.arange(keys, device="cuda")
    q = cells.queries(reps, dim).repeat(kv_heads, 1).expand(batch, queries, -1, -1).to(DT[dtype]).cuda()
    k, v, want = [], [], []
    for h in range(kv_heads):
        kk, vv = cells.keys_values(keys, reps, dim, run, 2.0 ** h, "cuda")
        k.append(kk.to(DT[dtype])), v.append(vv.to(DT[dtype]))
    for n in lengths:
        see = (j <= p) & (j < n)
        if window:
            see &= (p - j < window) | (j < sinks)
        count = torch.cat([cells.counts(s, reps, dim, run) for s in see.split(256)])
        want.append(torch.stack([cells.shares(count, 2.0 ** h) for h in range(kv_heads)], 1).flatten(1, 2))
    k, v = (torch.stack(x, 1).expand(batch, keys, kv_heads, dim).contiguous() for x in (k, v))
    got = ck.window_attention(q, k, v, window, sinks, torch.tensor(lengths, dtype=torch.int32, device="cuda"), 1.0)
    cells.check(got, torch.stack(want), DT[dtype])
