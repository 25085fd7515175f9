"""From where on groups are found without being told: what they save has to make up for the search too, which is the host's, once
for all layers."""
import pytest
import torch

import comfy_kitchen as ck

MB = 1 << 20


def saving(layers, members, tokens=64 * 1024):
    """(whether there are groups, the bytes of a layer that they save)"""
    c = ck.PagedKVCache(layers, tokens // 1024, 1024, 1, 16, device="cpu")
    first = c.add()
    c.append([first], tokens)
    order = [first, *(c.fork(first) for _ in range(members - 1))]
    row = 2 * 16 * 2  # bytes of a token
    return c.groups(order) is not None, (members - 1) * tokens * row


@pytest.mark.parametrize("layers", [1, 2, 10, 40])
def test_few_layers_have_to_save_more_each(layers):
    least = (80 + 400 / layers) * MB
    seen = set()
    for members in (2, 20, 22, 24, 25, 29, 31, 69, 71, 118, 122, 200):
        got, saved = saving(layers, members)
        assert got == (saved >= least), (members, saved / MB)
        seen.add(got)
    assert seen == {True, False}


def test_a_given_number_holds_as_it_is():
    c = ck.PagedKVCache(2, 4, 1024, 1, 16, device="cpu")
    first = c.add()
    c.append([first], 4096)
    order = [first, c.fork(first)]
    assert c.groups(order) is None and c.groups(order, 4096 * 64) is not None and c.groups(order, 4096 * 64 + 1) is None
