"""Groups of sequences that were appended to, forked, trimmed, compacted and freed in any order, against a comparison of their
page lists, page by page; and what finding them costs the host."""
import random
import time

import pytest
import torch

import comfy_kitchen as ck


@pytest.fixture(autouse=True)
def copies(monkeypatch):
    monkeypatch.setattr(ck, "paged_copy", lambda *a: None)


def common(a, b):
    n = 0
    while n < min(len(a), len(b)) and a[n] == b[n] and a[n] >= 0:
        n += 1
    return n


def plain(c, order):
    """The rule of `groups`, on whole page lists."""
    pages, lengths = [c.pages(s) for s in order], [c.length(s) for s in order]
    bounds, firsts = [], []
    for i, p in enumerate(pages):
        same = common(firsts[-1], p) if bounds else 0
        if same:
            members, had = i - bounds[-1], len(firsts[-1])
            after = common(p, pages[i + 1]) if i + 1 < len(pages) else 0
            if members * same < (members - 1) * had or (2 * same < after and members * same < after):
                same = 0
        if same:
            firsts[-1] = firsts[-1][:same]
        else:
            bounds.append(i)
            firsts.append(p[:common(p, p)])
    bounds.append(len(order))
    tokens = [min(len(f) * c.page_size, *lengths[a:b]) if b - a > 1 else min(len(f) * c.page_size, lengths[a])
              for f, a, b in zip(firsts, bounds, bounds[1:])]
    saved = sum((b - a - 1) * n for n, a, b in zip(tokens, bounds, bounds[1:]))
    return None if saved == 0 else (bounds, tokens)


@pytest.mark.parametrize("seed", range(12))
def test_as_page_by_page(seed):
    rng = random.Random(seed)
    size = rng.choice([1, 2, 4, 16])
    c = ck.PagedKVCache(1, 600, size, 1, 16, device="cpu")
    live, seen = [], 0
    for _ in range(400):
        what = rng.random()
        if not live or what < 0.1:
            live.append(c.add())
        elif what < 0.5:
            some = rng.sample(live, rng.randint(1, len(live)))
            try:
                c.append(some, [rng.choice([0, 1, 1, size, 3 * size]) for _ in some])
            except ck.OutOfPages:
                c.free(live.pop(rng.randrange(len(live))))
        elif what < 0.75:
            live.append(c.fork(rng.choice(live)))
        elif what < 0.82:
            c.trim(rng.choice(live), rng.randint(1, 6 * size), rng.randint(0, 3 * size))
        elif what < 0.86:
            s = rng.choice(live)
            pages = c.pages(s)
            keep = [t for t in range(c.length(s)) if pages[t // size] >= 0 and rng.random() < 0.8]
            try:
                c.compact(s, keep)
            except ck.OutOfPages:
                pass
        elif what < 0.93 or len(live) > 30:
            c.free(live.pop(rng.randrange(len(live))))
        order = rng.sample(live, len(live)) if rng.random() < 0.3 else sorted(live, key=c.pages)
        want, got = plain(c, order), c.groups(order, 1)
        assert (None if got is None else (got[0].tolist(), got[1].tolist())) == want
        seen += want is not None
    assert seen > 100


def fastest(f):
    times = []
    for _ in range(7):
        begin = time.perf_counter()
        f()
        times.append(time.perf_counter() - begin)
    return min(times)


@pytest.mark.parametrize("forks", [True, False])
def test_finding_groups_costs_less_than_the_tables(forks):
    """A step asks for both; the tables hold every page's number, and groups come from a few of each sequence."""
    c = ck.PagedKVCache(1, 64 * 2048 + 64, 16, 1, 16, device="cpu")
    first = c.add()
    c.append([first], 16 * 2048 - 5)
    order = [first, *(c.fork(first) for _ in range(63))]
    if not forks:
        others = [c.add() for _ in range(63)]
        c.append(others, 16 * 2048 - 5)
        order = [first, *others]
    c.append(order)
    assert (c.groups(order, 1) is not None) == forks
    assert fastest(lambda: c.groups(order, 1)) < fastest(lambda: c.tables(order)) / 4
