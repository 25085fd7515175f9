"""Groups of so many sequences that attention does not take them all with a group each (host only)."""
import ctypes

import pytest
import torch

import comfy_kitchen as ck
import comfy_kitchen.backends.hip as hb
from comfy_kitchen import paged


@pytest.fixture(autouse=True)
def copies(monkeypatch):
    monkeypatch.setattr(ck, "paged_copy", lambda *a: None)


def strangers(c, count):
    new = [c.add() for _ in range(count)]
    c.append(new)
    return new


def accepted(batch, groups):
    """Whether the operator takes that many (its arguments are checked before anything runs; the workspace's size last)."""
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    s = (ctypes.c_int64 * 8)(256, 64, 2048, 128, 64, 2048, 128, 64)
    lib = hb.load_library()
    assert lib.ckh_shared_attention(p, p, p, p, p, p, p, None, None, p, batch, 4, 2, 64, groups, 3, 16, 2, 2, s, 1.0, 2, 2, p, 1, 0) == 1
    return b"together at most" not in lib.ckh_last_error()


def test_the_limit_is_the_operators():
    assert accepted(paged.MOST_SPANS - 1, 1) and not accepted(paged.MOST_SPANS, 1)


@pytest.mark.parametrize("single", [1, 2046, 2047, 2100, 4000, 4093])
def test_a_pair_among_strangers(single):
    c = ck.PagedKVCache(1, 5000, 4, 1, 16, device="cpu")
    a = c.add()
    c.append([a], 12)
    b = c.fork(a)
    others = strangers(c, single)
    for at in (0, single // 2, single):
        order = [*others[:at], a, b, *others[at:]]
        got = c.groups(order, 1)
        if len(order) + 1 + (at > 0) + (at < single) > paged.MOST_SPANS:
            assert got is None
            continue
        starts, shared = got[0].tolist(), got[1].tolist()
        assert accepted(len(order), len(shared))
        assert starts[0] == 0 and starts[-1] == len(order) and starts == sorted(starts) and len(starts) == len(shared) + 1
        i = starts.index(at)
        assert starts[i + 1] == at + 2 and shared[i] == 12
        # what is in a group with strangers shares nothing
        assert all(n == 0 or q - p == 1 for j, (p, q, n) in enumerate(zip(starts, starts[1:], shared)) if j != i)


def test_more_than_the_operator_takes():
    c = ck.PagedKVCache(1, 3000, 4, 1, 16, device="cpu")
    first = strangers(c, 1400)
    order = [s for f in first for s in (f, c.fork(f), c.fork(f))]
    assert c.groups(order, 1) is None  # 4200 sequences
    assert c.groups(order[:3000], 1)[1].tolist() == [1] * 1000
    assert c.groups(order[:3090], 1) is None  # in 1030 groups


def test_pairs_that_are_too_many():
    c = ck.PagedKVCache(1, 3000, 4, 1, 16, device="cpu")
    order = [s for f in strangers(c, 1500) for s in (f, c.fork(f))]
    assert c.groups(order, 1) is None
    assert len(c.groups(order[:2730], 1)[1]) == 1365
