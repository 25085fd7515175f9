"""Norms of many rows in 8 bits, where a thread holds several pieces of a row: bit for bit the two calls."""
import pytest
import torch

import comfy_kitchen as ck

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def bits(t):
    return t.contiguous().view(torch.uint8)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols", [(8192, 1440), (8200, 1529), (8192, 1536), (9001, 1792), (8192, 1920), (8321, 2040), (8192, 2048), (8193, 2304),
                                       (8200, 5120), (8192, 9000)])
def test_codes_of_many_rows(rows, cols, dtype, hip):
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    x = torch.randn(rows, cols, device="cuda", generator=g).to(DT[dtype])
    r = (torch.randn(rows, cols, device="cuda", generator=g) * 3).to(DT[dtype])
    w = (1 + 0.3 * torch.randn(cols, device="cuda", generator=g)).to(DT[dtype])
    x[5], r[5] = 0, 0
    scale = torch.tensor(0.02, device="cuda")
    y, h = ck.rms_norm(x, w, r)
    plain = ck.rms_norm(x)
    for out in (torch.float8_e4m3fn, torch.float8_e5m2):
        codes, h8 = ck.rms_norm_fp8(x, scale, w, r, output_type=out)
        assert torch.equal(bits(codes), bits(ck.quantize_per_tensor_fp8(y, scale, out))) and torch.equal(bits(h), bits(h8))
        assert torch.equal(bits(ck.rms_norm_fp8(x, scale, output_type=out)), bits(ck.quantize_per_tensor_fp8(plain, scale, out)))
    codes, scales, h8 = ck.rms_norm_mxfp8(x, w, r, pad_32x=True)
    q, s = ck.quantize_mxfp8(y, pad_32x=True)
    assert torch.equal(bits(h), bits(h8)) and torch.equal(bits(codes), bits(q)) and torch.equal(bits(scales), bits(s))
    codes, scales = ck.rms_norm_mxfp8(x, pad_32x=True)
    q, s = ck.quantize_mxfp8(plain, pad_32x=True)
    assert torch.equal(bits(codes), bits(q)) and torch.equal(bits(scales), bits(s))


@pytest.mark.parametrize("rows", [1, 300, 8192])
@pytest.mark.parametrize("cols", [1536, 1920])
def test_a_row_among_many_is_a_row_alone(rows, cols, hip):
    g = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.randn(8192, cols, device="cuda", generator=g).bfloat16()
    scale = torch.tensor(0.02, device="cuda")
    whole, part = ck.rms_norm_fp8(x, scale), ck.rms_norm_fp8(x[:rows], scale)
    assert torch.equal(bits(whole[:rows]), bits(part))
