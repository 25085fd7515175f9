"""Which sequences of a cache begin with the same pages (host only)."""
import pytest
import torch

import comfy_kitchen as ck


@pytest.fixture(autouse=True)
def copies(monkeypatch):
    monkeypatch.setattr(ck, "paged_copy", lambda *a: None)


def cache(pages=100, page=4):
    return ck.PagedKVCache(1, pages, page, 1, 16, device="cpu")


def found(c, sequences, least=1):
    got = c.groups(sequences, least)
    return None if got is None else (got[0].tolist(), got[1].tolist())


def test_forks_of_one_sequence():
    c = cache()
    a = c.add()
    c.append([a], 11)
    b, d = c.fork(a), c.fork(a)
    assert found(c, [a, b, d]) == ([0, 3], [11])  # the last page too, while nobody has appended
    c.append([a, b, d])
    assert found(c, [a, b, d]) == ([0, 3], [8])
    c.append([a, b, d], [20, 1, 0])
    got = c.groups([a, b, d], 1)
    assert found(c, [a, b, d]) == ([0, 3], [8]) and got[0].dtype == got[1].dtype == torch.int32
    assert found(c, [a]) is None and found(c, []) is None


def test_several_groups_and_strangers():
    c = cache()
    a, x = c.add(), c.add()
    c.append([a, x], [20, 13])
    b, y, z = c.fork(a), c.fork(x), c.add()
    c.append([a, b, x, y, z], [1, 2, 3, 4, 5])
    assert found(c, [z, a, b, x, y]) == ([0, 1, 3, 5], [5, 20, 12])
    assert found(c, [a, x, b, y]) is None  # neighbours only
    row = 2 * 16 * 2
    assert found(c, [z, a, b, x, y], 32 * row) and found(c, [z, a, b, x, y], 32 * row + 1) is None


def test_one_that_shares_little_does_not_join():
    c = cache()
    a = c.add()
    c.append([a], 4)
    far = c.fork(a)  # shares one page of many
    c.append([far], 30)
    c.append([a], 40)
    b, d = c.fork(a), c.fork(a)
    assert found(c, [a, b, d, far]) == ([0, 3, 4], [44, 34])
    assert found(c, [far, a, b, d]) == ([0, 1, 4], [34, 44])
    assert found(c, [a, far]) == ([0, 2], [4])


def test_pages_given_back_are_not_shared():
    c = cache()
    a = c.add()
    c.append([a], 40)
    c.trim(a, 8, 4)
    b = c.fork(a)
    assert found(c, [a, b]) == ([0, 2], [4])


def test_a_window_and_groups():
    c = cache()
    with pytest.raises(ValueError, match="not both"):
        c.attend(0, torch.zeros(1, 1, 16), torch.zeros(1, 1), torch.zeros(1), window=4, groups=(torch.zeros(1), torch.zeros(1)))
