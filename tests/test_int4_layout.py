"""GroupInt4Layout without a GPU: weights with and without zero points copied into each other."""
import pytest
import torch

from comfy_kitchen.tensor import QuantizedTensor
from comfy_kitchen.tensor.int4 import GroupInt4Layout


def weight(zeros, seed, group=64, rows=4):
    g = torch.Generator().manual_seed(seed)
    groups = 128 // group
    codes = torch.randint(0, 256, (rows, 64), generator=g, dtype=torch.uint8)
    scale = torch.rand(rows, groups, generator=g).bfloat16()
    zero = torch.randint(0, 16, (rows, groups), generator=g, dtype=torch.uint8) if zeros else None
    params = GroupInt4Layout.Params(scale=scale, orig_dtype=torch.bfloat16, orig_shape=(rows, 128), group_size=group, zero=zero)
    return QuantizedTensor(codes, "GroupInt4Layout", params)


def tensors(w):
    return [t if t is None else t.clone() for t in GroupInt4Layout.get_plain_tensors(w)]


def equal(a, b):
    return all((x is None and y is None) or torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("to,of", [(False, False), (False, True), (True, False), (True, True)])
def test_copy(to, of):
    dst, src = weight(to, 1), weight(of, 2)
    codes, want = dst._qdata, tensors(src)
    assert dst.copy_(src) is dst and dst._qdata is codes and equal(tensors(dst), want)
    src._qdata.zero_(), src.params.scale.zero_()
    if of:
        src.params.zero.zero_()
    assert equal(tensors(dst), want)  # nothing is shared


@pytest.mark.parametrize("other", [dict(group=32), dict(rows=3)])
def test_a_copy_that_does_not_fit_changes_nothing(other):
    for zeros in (False, True):
        dst = weight(zeros, 1)
        before, params = tensors(dst), dst.params
        with pytest.raises(RuntimeError):
            dst.copy_(weight(zeros, 2, **other))
        assert equal(tensors(dst), before) and dst.params is params and params.group_size == 64
