"""The host side of PagedKVCache (no GPU): which pages sequences own, what is copied, and what is
refused without a change.  Copies are recorded instead of made."""
import random

import pytest
import torch

import comfy_kitchen as ck


@pytest.fixture
def moved(monkeypatch):
    log = []
    monkeypatch.setattr(ck, "paged_copy", lambda k, v, src, dst: log.append((src.tolist(), dst.tolist())))
    return log


def cache(pages=8, page=4):
    return ck.PagedKVCache(1, pages, page, 1, 16, torch.float16, device="cpu")


def test_append_and_free(moved):
    c = cache()
    a, b = c.add(), c.add()
    slots = c.append([a, b], [5, 0]).tolist()
    pages = c.pages(a)
    assert slots == [pages[t // 4] * 4 + t % 4 for t in range(5)] and c.pages(b) == []
    assert c.append([a]).tolist() == [pages[1] * 4 + 1] and c.length(a) == 6
    table, lengths = c.tables([b, a])
    assert table.tolist() == [[-1, -1], pages] and lengths.tolist() == [0, 6] and table.dtype == torch.int32
    c.free(a)
    assert c.free_pages == 8 and a not in c and b in c and not moved


def test_fork_copies_on_append(moved):
    c = cache()
    a = c.add()
    c.append([a], [6])
    first, last = c.pages(a)
    b = c.fork(a)
    assert c.pages(b) == [first, last] and c.free_pages == 6
    slot = c.append([b]).tolist()
    new = c.pages(b)[1]
    assert new != last and slot == [new * 4 + 2]
    assert moved == [([last * 4, last * 4 + 1], [new * 4, new * 4 + 1])]
    assert c.append([a]).tolist() == [last * 4 + 2] and len(moved) == 1  # the last owner keeps the page
    c.free(a)
    assert c.free_pages == 6  # the shared first page stays with b, and b has its copy of the last
    c.free(b)
    assert c.free_pages == 8


def test_owners_that_append_together(moved):
    c = cache()
    a = c.add()
    c.append([a], [2])
    b, d = c.fork(a), c.fork(a)
    c.append([a, b, d], 1)
    assert len({c.pages(s)[0] for s in (a, b, d)}) == 3 and len(moved) == 1 and len(moved[0][0]) == 4
    full = c.fork(a)
    c.append([a], [1])  # 3 -> 4 tokens: a fork shares it, so it is copied
    assert len(moved) == 2
    c.append([full], [1])
    again = c.fork(full)
    c.append([again], [1])  # a full page needs no copy
    assert len(moved) == 2 and c.pages(again)[0] == c.pages(full)[0]


def test_refused_without_a_change(moved):
    c = cache(pages=2)
    a = c.add()
    c.append([a], [6])
    b = c.fork(a)
    for call in (lambda: c.append([a], [3]), lambda: c.append([b], [1]), lambda: c.compact(a, [0, 3])):
        with pytest.raises(ck.OutOfPages):
            call()
    assert c.length(a) == c.length(b) == 6 and c.pages(a) == c.pages(b) and c.free_pages == 0 and not moved
    for call in (lambda: c.append([a, a], 1), lambda: c.append([a], [-1]), lambda: c.append([a], [1, 2]),
                 lambda: c.compact(a, [3, 3]), lambda: c.compact(a, [2, 6]), lambda: c.compact(a, [-1]),
                 lambda: c.trim(a, 0), lambda: c.trim(a, 4, -1), lambda: cache(pages=0)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(KeyError):
        c.free(99)


def test_trim_and_compact(moved):
    c = cache(pages=10)
    a = c.add()
    c.append([a], [22])
    pages = c.pages(a)
    assert c.trim(a, 5, 3) == 3  # sinks on page 0; tokens 17..21 on pages 4 and 5
    assert c.pages(a) == [pages[0], -1, -1, -1, *pages[4:]] and c.free_pages == 7 and c.trim(a, 5, 3) == 0
    with pytest.raises(ValueError, match="trim"):
        c.compact(a, [0, 8])
    c.compact(a, torch.tensor([0, 1, 2, 17, 18, 19, 20, 21]))
    new = c.pages(a)
    assert c.length(a) == 8 and len(new) == 2 and c.free_pages == 8
    assert moved == [([pages[0] * 4 + i for i in range(3)] + [pages[t // 4] * 4 + t % 4 for t in range(17, 22)],
                      [p * 4 + i for p in new for i in range(4)])]
    c.compact(a, [])
    assert c.length(a) == 0 and c.pages(a) == [] and c.free_pages == 10


def test_random_walk_keeps_the_books(moved):
    """Contents followed through every copy: each sequence's slots hold its tokens, no page is lost
    or owned twice, and no copy reads what it writes."""
    rng = random.Random(5)
    c = cache(pages=24, page=4)
    store, want, token = {}, {}, 0
    for _ in range(1500):
        live = list(want)
        what = rng.choice(["add", "fork", "free", "append", "append", "append", "trim", "compact"])
        try:
            if what == "add" and len(live) < 8:
                want[c.add()] = []
            elif not live:
                continue
            elif what == "fork" and len(live) < 8:
                s = rng.choice(live)
                want[c.fork(s)] = list(want[s])
            elif what == "free":
                s = rng.choice(live)
                c.free(s)
                del want[s]
            elif what == "append":
                some = rng.sample(live, rng.randint(1, min(4, len(live))))
                counts = [rng.choice([0, 1, 1, 1, 2, 5]) for _ in some]
                moved.clear()
                slots = iter(c.append(some, counts).tolist())
                for src, dst in moved:
                    assert not set(src) & set(dst) and len(set(dst)) == len(dst)
                    store.update(zip(dst, [store[x] for x in src]))
                for s, n in zip(some, counts):
                    for _ in range(n):
                        store[next(slots)] = token
                        want[s].append(token)
                        token += 1
            elif what == "trim":
                s = rng.choice(live)
                c.trim(s, rng.randint(1, 9), rng.randint(0, 5))
                want[s] = [t if c.pages(s)[i // 4] >= 0 else None for i, t in enumerate(want[s])]
            elif what == "compact":
                s = rng.choice(live)
                keep = [i for i, t in enumerate(want[s]) if t is not None and rng.random() < 0.6]
                moved.clear()
                c.compact(s, keep)
                for src, dst in moved:
                    assert not set(src) & set(dst)
                    store.update(zip(dst, [store[x] for x in src]))
                want[s] = [want[s][i] for i in keep]
        except ck.OutOfPages:
            pass
        owned = set()
        for s, tokens in want.items():
            pages = c.pages(s)
            owned |= {p for p in pages if p >= 0}
            assert c.length(s) == len(tokens)
            for i, t in enumerate(tokens):
                if t is not None:
                    assert store[pages[i // 4] * 4 + i % 4] == t
        assert c.free_pages == 24 - len(owned)


def test_plain_calls_of_ops_that_change_their_arguments():
    """They go past the custom op like the others, and count the change as it does."""
    from comfy_kitchen.ops import changed, untouched

    assert all(untouched(op) for op in ("paged_write", "paged_copy", "paged_attention"))
    x = torch.zeros(3)
    changed(x, x.view(3))
    assert x._version == 2
    with torch.inference_mode():
        y = torch.zeros(2)
        changed(y)
    changed(y)
