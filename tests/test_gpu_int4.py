"""Weight-only 4-bit linears against their definition in 64 bits.

Bounds.  linear_int4 rounds once to x's type (relative 2^-8 in bf16, 2^-11 in f16) after fp32 sums:
each of the about K/32 accumulations of a sum of terms x (B + q) s, B = 128 in bf16 and 1024 in
f16, errs by at most 2^-23 of their absolute sum, and so does the sum of x that is subtracted.
quantize_int4 and dequantize_int4 are exact to the bit."""
import pytest
import torch

import comfy_kitchen as ck

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def weight(n, k, group, zeros, scale_dtype, seed):
    g = torch.Generator().manual_seed(seed)
    groups = -(-k // group)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.int32).to(torch.uint8)
    scales = (torch.rand(n, groups, generator=g) * 0.02 + 1e-3).to(scale_dtype)
    z = torch.randint(0, 16, (n, groups), generator=g, dtype=torch.int32).to(torch.uint8) if zeros else None
    return codes, scales, z


def wide(codes, scales, zeros, group):
    """The weight in 64 bits."""
    n, half = codes.shape
    q = torch.stack((codes % 16, codes // 16), 2).reshape(n, 2 * half).double()
    at = torch.arange(2 * half) // group
    z = 8.0 if zeros is None else zeros.double()[:, at]
    return (q - z) * scales.double()[:, at]


def check(y, x, w, scales, group, bias=None):
    want = x.double() @ w.t()
    if bias is not None:
        want = want + bias.double()
    k = x.shape[1]
    base, unit = (128, 2.0 ** -8) if x.dtype == torch.bfloat16 else (1024, 2.0 ** -11)
    s = scales.double().abs()[:, torch.arange(k) // group]
    mass = x.double().abs() @ s.t() * (base + 16)
    bound = unit * want.abs() * 1.01 + (k / 32 + 64) * 2.0 ** -23 * mass + 1e-7
    y, top = y.cpu(), torch.finfo(x.dtype).max
    over = want.abs() > top + bound  # beyond the type: infinite, with its sign
    assert torch.equal(y[over].double(), torch.copysign(torch.full_like(want[over], float("inf")), want[over]))
    err = torch.where(over, 0.0, (y.double() - want).abs())
    assert y.dtype == x.dtype and y.shape == want.shape
    assert bool((err <= bound).all()), float((err / bound).max())


# rows at and past the 16-row tiles, N that ends inside a tile, K of one block, inside a step of
# 128, more steps than waves, groups of every alignment, a last group that is shorter
SHAPES = [(1, 1, 32, 32), (1, 16, 128, 128), (1, 1000, 5120, 128), (2, 33, 160, 64), (3, 77, 416, 96), (15, 50, 4096, 32),
          (16, 129, 1088, 128), (17, 64, 2080, 64), (31, 100, 96, 256), (32, 17, 992, 32), (33, 48, 1312, 160),
          (48, 250, 640, 128), (64, 31, 2016, 64), (65, 100, 512, 512), (130, 40, 288, 64), (1, 5000, 2048, 64),
          # more groups, or more activations, than are staged at a time; wide enough for the other tiles
          (1, 40, 16416, 32), (3, 40, 16416, 32), (4, 9000, 4256, 128), (2, 9000, 1056, 32), (20, 40, 16416, 32),
          (1, 20, 36864, 128), (2, 20, 36896, 256), (9, 9000, 544, 64), (40, 9000, 1056, 96),
          # more rows, with K in ranges: odd ones, one that ends inside a step, more groups than one range may hold
          (17, 200, 1696, 64), (24, 512, 5120, 128), (33, 100, 8224, 32), (64, 300, 14336, 128), (100, 70, 70016, 32),
          (45, 20000, 544, 128), (200, 65, 1120, 96)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m,n,k,group", SHAPES)
def test_linear(m, n, k, group, dtype, hip):
    g = torch.Generator().manual_seed(m * 7 + n + k)
    for zeros, scale_dtype, bias_dtype in ((False, dtype, None), (True, "f32", "f32"), (True, dtype, dtype)):
        codes, scales, z = weight(n, k, group, zeros, DT[scale_dtype], m + n + k)
        x = torch.randn(m, k, generator=g).to(DT[dtype])
        bias = None if bias_dtype is None else torch.randn(n, generator=g).to(DT[bias_dtype])
        y = ck.linear_int4(x.cuda(), codes.cuda(), scales.cuda(), None if z is None else z.cuda(),
                           None if bias is None else bias.cuda(), group_size=group)
        check(y, x, wide(codes, scales, z, group), scales, group, bias)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_strides_shapes_and_alignment(dtype, hip):
    codes, scales, z = weight(72, 256, 64, True, DT[dtype], 3)
    w = wide(codes, scales, z, 64)
    args = (codes.cuda(), scales.cuda(), z.cuda())
    g = torch.Generator().manual_seed(5)
    big = torch.randn(6, 5, 264, generator=g).to(DT[dtype])
    for x in (big[:, -1, :256], big[:, 2, 8:], big[:, 0, 3:259], big[:, :, 4:260], big[0, 0, :256],
              big.transpose(0, 1)[..., :256], torch.randn(256, 9, generator=g).to(DT[dtype]).t(), big[:0, 0, :256]):
        d = big.cuda()
        xd = x.cuda() if x.data_ptr() < big.data_ptr() or x.data_ptr() >= big.data_ptr() + big.nbytes else \
            torch.as_strided(d, x.shape, x.stride(), x.storage_offset())
        y = ck.linear_int4(xd, *args, group_size=64)
        assert y.shape == (*x.shape[:-1], 72)
        if x.numel():
            check(y.reshape(-1, 72), x.reshape(-1, 256), w, scales, 64)
    # a weight that is a view: rows of a larger one, and one off the 16-byte boundary
    x = big[:, 0, :256].contiguous()
    y = ck.linear_int4(x.cuda(), args[0][3:50], args[1][3:50], args[2][3:50], group_size=64)
    check(y, x, w[3:50], scales[3:50], 64)
    flat = torch.zeros(72 * 128 + 5, dtype=torch.uint8, device="cuda")
    flat[5:] = args[0].flatten()
    y = ck.linear_int4(x.cuda(), flat[5:].view(72, 128), args[1], args[2], group_size=64)
    check(y, x, w, scales, 64)


def test_values_at_the_ends(hip):
    """Codes 0 and 15 against every zero point, activations with a large common part, zero scales."""
    codes = torch.tensor([[0x00], [0xff], [0xf0], [0x0f]], dtype=torch.uint8).repeat(4, 64)
    scales = torch.tensor([1.0, 0.0, 2.0 ** -14, 100.0]).repeat_interleave(4)[:, None].repeat(1, 4)
    z = torch.arange(16, dtype=torch.uint8)[:, None].repeat(1, 4)
    w = wide(codes, scales, z, 32)
    for dtype in (torch.bfloat16, torch.float16):
        x = (torch.randn(5, 128, generator=torch.Generator().manual_seed(1)) + 20).to(dtype)
        y = ck.linear_int4(x.cuda(), codes.cuda(), scales.cuda(), z.cuda(), group_size=32)
        check(y, x, w, scales, 32)
    x = torch.zeros(3, 128, dtype=torch.bfloat16)
    x[1, 7] = float("inf")
    y = ck.linear_int4(x.cuda(), codes.cuda(), scales.cuda(), z.cuda(), group_size=32).cpu()
    assert bool((y[0] == 0).all()) and bool((y[2] == 0).all())  # its neighbours are untouched
    assert not bool(torch.isfinite(y[1][scales[:, 0] > 0]).any())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (5, 96, 64), (33, 1024, 128), (7, 2080, 96), (3, 288, 512)])
def test_quantize_and_dequantize(n, k, group, dtype, hip):
    g = torch.Generator().manual_seed(n + k)
    w = (torch.randn(n, k, generator=g) * torch.exp(torch.randn(n, 1, generator=g))).to(DT[dtype])
    w[0, :32] = 0
    groups = -(-k // group)
    pad = torch.nn.functional.pad(w.float(), (0, groups * group - k)).reshape(n, groups, group)
    scales = (pad.abs().amax(-1) / 7).to(DT[dtype])
    s = scales.float()[..., None]
    q = torch.where(s > 0, torch.round(pad / torch.where(s > 0, s, 1.0)), torch.zeros_like(pad)).clamp(-8, 7) + 8
    q = q.reshape(n, -1)[:, :k].to(torch.uint8)
    codes, got = ck.quantize_int4(w.cuda(), group)
    assert got.dtype == w.dtype and torch.equal(got.cpu(), scales)
    assert torch.equal(codes.cpu(), q[:, 0::2] | (q[:, 1::2] << 4))
    z = torch.randint(0, 16, (n, groups), generator=g, dtype=torch.int32).to(torch.uint8)
    for zeros in (None, z):
        for out in DT.values():
            back = ck.dequantize_int4(codes, got, None if zeros is None else zeros.cuda(), group, out)
            want = wide(codes.cpu(), scales, zeros, group).float().to(out)
            assert torch.equal(back.cpu(), want)


def test_streams_and_graph(hip):
    codes, scales, z = weight(300, 2048, 128, True, torch.bfloat16, 9)
    args = (codes.cuda(), scales.cuda(), z.cuda())
    x = torch.randn(4, 2048, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    want = ck.linear_int4(x, *args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ck.linear_int4(x, *args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)  # K is split over waves in a fixed order
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ck.linear_int4(static, *args)
    for i in range(3):
        static.copy_(x * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ck.linear_int4(x * (i + 1), *args))


def test_without_a_workspace(hip):
    """The C entry point without the workspace that splits K: the same result up to fp32 sums, for a
    K whose groups fit one range and one whose do not."""
    import comfy_kitchen.backends.hip as hb

    for k in (1024, 6144):
        codes, scales, _ = weight(96, k, 32, False, torch.bfloat16, 4)
        x = torch.randn(40, k, generator=torch.Generator().manual_seed(1)).bfloat16()
        d = [t.cuda() for t in (x, codes, scales)]
        y = torch.empty(40, 96, dtype=torch.bfloat16, device="cuda")
        assert hb._lib.ckh_linear_int4_workspace_bytes(40, 96, k, 32) > 0
        hb._launch("ckh_linear_int4", y, *(t.data_ptr() for t in d), None, None, y.data_ptr(), 40, 96, k, k, 32, 2, 2, 0, None, 0)
        check(y, x, wide(codes, scales, None, 32), scales, 32)


def test_refusals(hip):
    codes, scales, z = (t.cuda() for t in weight(8, 128, 32, True, torch.bfloat16, 1))
    x = torch.zeros(2, 128, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ck.NoCapableBackendError):
        ck.linear_int4(x.float(), codes, scales, z, group_size=32)
    with pytest.raises(ck.NoCapableBackendError):
        ck.linear_int4(x, codes.to(torch.int8), scales, z, group_size=32)
    with pytest.raises(ck.NoCapableBackendError):
        ck.linear_int4(x.cpu(), codes, scales, z, group_size=32)
    with pytest.raises(ValueError, match="inputs"):
        ck.linear_int4(x[:, :64], codes, scales, z, group_size=32)
    with pytest.raises(ValueError, match="scales must be"):
        ck.linear_int4(x, codes, scales, z, group_size=64)
    with pytest.raises(ValueError, match="zeros must be"):
        ck.linear_int4(x, codes, scales, z[:4], group_size=32)
    with pytest.raises(ValueError, match="group_size"):
        ck.linear_int4(x, codes, scales, z, group_size=48)
    with pytest.raises(ValueError, match="bias"):
        ck.linear_int4(x, codes, scales, z, torch.zeros(7, device="cuda"), group_size=32)
    with pytest.raises(ValueError, match="multiples of 32"):
        ck.quantize_int4(torch.zeros(4, 48, device="cuda"), 32)
    with pytest.raises(ValueError, match="multiples of 32"):
        ck.quantize_int4(torch.zeros(4, 64, device="cuda"), 16)
