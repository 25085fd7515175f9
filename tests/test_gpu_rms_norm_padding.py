"""MXFP8 of a norm whose rows are padded: bit for bit the two calls, whatever a row's factor is."""
import pytest
import torch

import comfy_kitchen as ck

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def bits(t):
    return t.contiguous().view(torch.uint8)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows", [7, 300, 2300])
@pytest.mark.parametrize("cols", [1, 7, 33, 40, 95, 100, 257, 1003, 4101])
def test_padding_of_rows_that_are_not_finite(cols, rows, dtype, hip):
    """Columns behind the last are zeros for the two calls, also where the row's factor is NaN (a NaN, and with eps 0 a row of zeros
    and so an infinite one) or 0 (an infinity)."""
    g = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.randn(rows, cols, device="cuda", generator=g).to(DT[dtype])
    r = torch.randn(rows, cols, device="cuda", generator=g).to(DT[dtype])
    w = (1 + 0.3 * torch.randn(cols, device="cuda", generator=g)).to(DT[dtype])
    x[1, cols // 2], x[2, cols - 1], x[3, 0], x[4, cols - 1] = float("nan"), -float("nan"), float("inf"), -float("inf")
    x[5], r[5] = 0, 0
    for eps in (1e-6, 0.0):
        for weight, residual in ((w, r), (w, None), (None, None)):
            y = ck.rms_norm(x, weight, residual, eps)
            y = y if residual is None else y[0]
            codes, scales = ck.rms_norm_mxfp8(x, weight, residual, eps, pad_32x=True)[:2]
            q, s = ck.quantize_mxfp8(y, pad_32x=True)
            assert torch.equal(bits(scales), bits(s))
            assert torch.equal(bits(codes), bits(q)), (bits(codes) != bits(q)).nonzero()[:4].tolist()
