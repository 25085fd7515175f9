"""What the exact inputs of 4-bit linears (int4_exact.py) tell apart: mistakes planted in the definition,
on the CPU."""
import pytest
import torch

from int4_exact import LONG_GROUPS, Linear

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
