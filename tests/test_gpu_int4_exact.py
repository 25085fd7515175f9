"""linear_int4 on inputs whose sums are exact (int4_exact.py): equal to the definition, one rounding."""
import pytest
import torch

import comfy_kitchen as ck
from int4_exact import LONG_GROUPS, Linear

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def same(c: Linear):
    assert c.largest() < 2 ** 22
    got = ck.linear_int4(c.x.cuda(), c.codes.cuda(), c.scales.cuda(), None if c.zeros is None else c.zeros.cuda(),
                         None if c.bias is None else c.bias.cuda(), group_size=c.group)
    assert torch.equal(got.cpu(), c.want())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m", [1, 3, 9, 20])
@pytest.mark.parametrize("k,group", LONG_GROUPS)
def test_groups_of_millions(k, group, m, dtype, hip):
    """The last 32 inputs of a long group have its scale and zero point, not the next one's."""
    same(Linear(m, 5, k, group, DT[dtype], True, False))
