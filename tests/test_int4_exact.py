"""What the exact inputs of 4-bit linears (int4_exact.py) tell apart: mistakes planted in the definition,
on the CPU."""
import pytest
import torch

from int4_exact import LONG_GROUPS, MANY_GROUPS, SHAPES, Linear, dense, far

DTYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])


@DTYPES
@pytest.mark.parametrize("m", [1, 20])
@pytest.mark.parametrize("k,group", LONG_GROUPS)
def test_a_block_in_the_next_group(k, group, m, dtype):
    c = Linear(m, 5, k, group, dtype, True, False)
    assert c.largest() < 2 ** 22
    last = (c.cols // 32) % (group // 32) == group // 32 - 1
    at = (c.cols // group + last).clamp(max=c.scales.shape[1] - 1)
    assert not torch.equal(c.want(c.weight_cols(at)), c.want())


@DTYPES
@pytest.mark.parametrize("zeros,bias", [(False, True), (True, False), (True, True)])
@pytest.mark.parametrize("m,n,k,group", SHAPES + MANY_GROUPS)
def test_mistakes(m, n, k, group, zeros, bias, dtype):
    """Nothing at all, the last 32 inputs, a step of 128 or a group missing, a zero point off by one and a
    neighbour's scale, in one group, first, middle and last: each gives another result, in the first
    rows and outputs already."""
    m, n = min(m, 8), min(n, 64)
    c = Linear(m, n, k, group, dtype, zeros, bias)
    assert c.largest() < 2 ** 22
    want, w, cols = c.want(), c.weight_cols(), c.cols
    groups = c.scales.shape[1]

    def differs(change, inputs):
        return not torch.equal(c.want(torch.where(inputs, change, w)), want)

    none = torch.zeros((), dtype=torch.float64)
    assert differs(none, cols >= 0)
    if n * m > 1:  # one output alone may round a term away
        assert differs(none, cols >= k - 32)
        for step in {0, k // 256, (k - 1) // 128}:
            assert differs(none, cols // 128 == step)
        for g in {0, groups // 2, groups - 1}:
            here = cols // group == g
            assert differs(none, here)
            off = w - c.scales.double()[:, cols // group]
            assert differs(off, here)
            if groups > 1:
                other = c.weight_cols(torch.where(here, (g + 1) % groups, cols // group))
                assert differs(other, here)


@DTYPES
@pytest.mark.parametrize("m,n,k,group", SHAPES[1:])
def test_dense_inputs_missing(m, n, k, group, dtype):
    """The norm sees the last 32 inputs missing, at every K."""
    (x, codes, scales, zeros), want = dense(min(m, 8), min(n, 64), k, group, dtype)
    assert far(want.to(dtype), want, dtype) < 0.6
    y = want.clone()
    for i in range(k - 32, k):
        q = codes[:, i // 2] // 16 if i % 2 else codes[:, i // 2] % 16
        y -= x[:, i:i + 1].double() * (q.double() - zeros[:, i // group].double()) * scales[:, i // group].double()
    assert far(y.to(dtype), want, dtype) > 1
