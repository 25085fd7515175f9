"""linear_int4 on inputs whose sums are exact (int4_exact.py): equal to the definition, one rounding."""
import pytest
import torch

import comfy_kitchen as ck
from int4_exact import LONG_GROUPS, MANY_GROUPS, SHAPES, Linear, dense, far

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def same(c: Linear):
    assert c.largest() < 2 ** 22
    got = ck.linear_int4(c.x.cuda(), c.codes.cuda(), c.scales.cuda(), None if c.zeros is None else c.zeros.cuda(),
                         None if c.bias is None else c.bias.cuda(), group_size=c.group)
    assert torch.equal(got.cpu(), c.want())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m,n,k,group", SHAPES)
def test_linear(m, n, k, group, dtype, hip):
    for seed, (zeros, bias) in enumerate(((False, True), (True, False), (True, True))):
        same(Linear(m, n, k, group, DT[dtype], zeros, bias, seed))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m,n,k,group", SHAPES[1:])
def test_dense(m, n, k, group, dtype, hip):
    (x, codes, scales, zeros), want = dense(m, n, k, group, DT[dtype], device="cuda")
    assert far(ck.linear_int4(x, codes, scales, zeros, group_size=group), want, DT[dtype]) < 1


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m", [1, 3, 9, 20])
@pytest.mark.parametrize("k,group", LONG_GROUPS)
def test_groups_of_millions(k, group, m, dtype, hip):
    """The last 32 inputs of a long group have its scale and zero point, not the next one's."""
    same(Linear(m, 5, k, group, DT[dtype], True, False))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m,n,k,group", MANY_GROUPS)
def test_many_groups_and_rows(m, n, k, group, dtype, hip):
    same(Linear(m, n, k, group, DT[dtype], False, True))
    same(Linear(m, n, k, group, DT[dtype], True, False, seed=1))


def test_many_groups_without_a_workspace(hip):
    c = Linear(40, 96, 6144, 32, torch.bfloat16, True, False)
    d = [t.cuda() for t in (c.x, c.codes, c.scales, c.zeros)]
    y = torch.empty(40, 96, dtype=torch.bfloat16, device="cuda")
    hip._launch("ckh_linear_int4", y, *(t.data_ptr() for t in d), None, y.data_ptr(), 40, 96, 6144, 6144, 32, 2, 2, 0, None, 0)
    assert torch.equal(y.cpu(), c.want())
