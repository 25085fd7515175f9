"""The root-mean-square norm: against its definition in 64 bits, and in 8 bits bit for bit against the two
calls it stands for.

The bound: one rounding of the result, unit |y| (bf16 2^-8, f16 2^-11, f32 2^-24), and fp32 arithmetic: the
sum of squares is a sum of 8 terms, a tree of 6 levels and a sum of at most 128, each step 2^-24 off, half of which
the root passes on, with as much again of root and products: under 2^-17 |y| in all.  f16's results under 2^-14 have steps of 2^-24."""
import pytest
import torch

import comfy_kitchen as ck

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}


def make(rows, cols, dtype, seed=0, size=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g) * size).to(DT[dtype])
    r = (torch.randn(rows, cols, generator=g) * 3 * size).to(DT[dtype])
    w = (1 + 0.3 * torch.randn(cols, generator=g)).to(DT[dtype])
    return x, r, w


def want(h, w, eps=1e-6):
    h = h.double()
    y = h / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    return y if w is None else y * w.double()


def check(y, h, w, dtype, eps=1e-6):
    ref = want(h, w, eps)
    err = (y.cpu().double() - ref).abs()
    bound = (UNIT[dtype] + 2.0 ** -17) * ref.abs() + (2.0 ** -25 if dtype == "f16" else 1e-37)
    assert y.dtype == DT[dtype] and y.shape == h.shape
    assert bool((err <= bound).all()), float((err / bound.clamp_min(1e-300)).max())


def bits(t):
    return t.contiguous().cpu().view(torch.uint8)


SIZES = [(1, 1), (3, 7), (2, 8), (5, 100), (130, 256), (1, 4096), (7, 4104), (33, 5120), (2, 5121), (2, 16400), (1, 32768), (2, 40000), (1, 65536)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_plain(rows, cols, dtype, hip):
    x, r, w = make(rows, cols, dtype, rows + cols)
    check(ck.rms_norm(x.cuda(), w.cuda()), x, w, dtype)
    check(ck.rms_norm(x.cuda()), x, None, dtype)
    y, h = ck.rms_norm(x.cuda(), w.cuda(), r.cuda(), eps=0.01)
    total = (x.float() + r.float()).to(x.dtype)
    assert torch.equal(h.cpu(), total)
    check(y, total, w, dtype, 0.01)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_fp8_is_the_two_calls(rows, cols, dtype, hip):
    x, r, w = (t.cuda() for t in make(rows, cols, dtype, rows * cols + 1))
    scale = torch.tensor(0.02, device="cuda")
    for out in (torch.float8_e4m3fn, torch.float8_e5m2):
        y, h = ck.rms_norm(x, w, r)
        codes, h8 = ck.rms_norm_fp8(x, scale, w, r, output_type=out)
        assert codes.dtype == out and torch.equal(bits(codes), bits(ck.quantize_per_tensor_fp8(y, scale, out))) and torch.equal(h, h8)
        assert torch.equal(bits(ck.rms_norm_fp8(x, scale, output_type=out)), bits(ck.quantize_per_tensor_fp8(ck.rms_norm(x), scale, out)))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols,pad", [(1, 32, False), (3, 96, False), (128, 160, False), (129, 256, True), (777, 5120, False), (1, 5120, True),
                                           (5, 7, True), (40, 100, True), (2, 33, True), (300, 4096, False), (1025, 64, False), (2, 65536, False)])
def test_mxfp8_is_the_two_calls(rows, cols, pad, dtype, hip):
    x, r, w = (t.cuda() for t in make(rows, cols, dtype, rows * cols + 2))
    x[:, :32] = 0
    r[:, :32] = 0  # a block of zeros
    y, h = ck.rms_norm(x, w, r)
    codes, scales, h8 = ck.rms_norm_mxfp8(x, w, r, pad_32x=pad)
    q, s = ck.quantize_mxfp8(y, pad_32x=pad)
    assert codes.shape == q.shape and scales.shape == s.shape and codes.dtype == q.dtype and scales.dtype == s.dtype
    assert torch.equal(h, h8) and torch.equal(bits(codes), bits(q)) and torch.equal(bits(scales), bits(s))
    codes, scales = ck.rms_norm_mxfp8(x, pad_32x=pad)
    q, s = ck.quantize_mxfp8(ck.rms_norm(x), pad_32x=pad)
    assert torch.equal(bits(codes), bits(q)) and torch.equal(bits(scales), bits(s))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_rows_that_are_not_finite_stay_alone(dtype, hip):
    x, r, w = (t.cuda() for t in make(6, 320, dtype))
    clean = ck.rms_norm(x, w)
    x[1, 5], x[3, 7], x[4] = float("inf"), float("nan"), 0
    scale = torch.tensor(0.02, device="cuda")
    y = ck.rms_norm(x, w)
    assert torch.equal(y[[0, 2, 5]], clean[[0, 2, 5]]) and bool((y[4] == 0).all()) and bool(y[3].isnan().all())
    assert bool(y[1, 5].isnan()) and bool((y[1, :5] == 0).all())
    codes, (q, s) = ck.rms_norm_fp8(x, scale, w), ck.rms_norm_mxfp8(x, w)
    assert torch.equal(bits(codes), bits(ck.quantize_per_tensor_fp8(y, scale)))
    q2, s2 = ck.quantize_mxfp8(y)
    assert torch.equal(bits(q), bits(q2)) and torch.equal(bits(s), bits(s2))


def test_large_values_do_not_overflow_in_f16(hip):
    x = torch.full((2, 4096), 60000.0, dtype=torch.float16, device="cuda")
    assert bool((ck.rms_norm(x) == 1).all())
    y, h = ck.rms_norm(x, residual=x)
    assert bool(h.isinf().all()) and bool(y.isnan().all())  # the sum as it is stored


def test_strides_shapes_and_weight_types(hip):
    g = torch.Generator(device="cuda").manual_seed(4)
    wide = torch.randn(12, 1000, device="cuda", generator=g).bfloat16()
    for x in (wide[:, :640], wide[::2, 8:648], wide[:, 3:643], wide[:, ::2], wide.t(), wide[:1].expand(5, -1), wide[0], wide.view(3, 4, 1000),
              wide.view(3, 4, 1000).transpose(0, 1), wide[:, :640].unflatten(0, (3, 4))):
        for wt in (torch.float32, torch.float16, torch.bfloat16):
            w = (1 + torch.randn(x.shape[-1], device="cuda", generator=g)).to(wt)
            y, h = ck.rms_norm(x, w, x)
            total = (x.float() * 2).bfloat16().cpu()
            assert torch.equal(h.cpu(), total) and y.is_contiguous() and h.is_contiguous()
            check(y, total, w.cpu(), "bf16")


@pytest.mark.parametrize("cols", [64, 1000, 4104, 5120, 9000, 20000])
def test_a_row_alone_or_among_others(cols, hip):
    """The same row gives the same result: among many rows, alone, and where it does not lie on 16 bytes."""
    x, r, w = (t.cuda() for t in make(1100, cols, "bf16", cols))
    y, h = ck.rms_norm(x, w, r)
    off = torch.zeros(cols + 3, dtype=torch.bfloat16, device="cuda")
    for i in (0, 7, 1099):
        assert torch.equal(ck.rms_norm(x[i:i + 1], w, r[i:i + 1])[0], y[i:i + 1])
        off[3:] = h[i]
        assert torch.equal(ck.rms_norm(off[3:], w), y[i])


def test_nothing_to_do(hip):
    for shape in ((0, 64), (3, 0), (2, 0, 32)):
        x = torch.empty(shape, device="cuda", dtype=torch.bfloat16)
        w = torch.ones(shape[-1], device="cuda")
        y, h = ck.rms_norm(x, w, x)
        assert y.shape == x.shape == h.shape
        assert ck.rms_norm_fp8(x, torch.tensor(1.0), w).shape == x.shape
    for pad in (False, True):
        x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16)
        codes, scales = ck.rms_norm_mxfp8(x, pad_32x=pad)
        assert codes.shape == (0, 64) and scales.shape == (0, 4)


def test_through_the_custom_op_and_captured(hip):
    x, r, w = (t.cuda() for t in make(70, 5120, "bf16"))
    y, h = torch.ops.comfy_kitchen.rms_norm(x, w, r, 1e-6)
    assert torch.equal(y, ck.rms_norm(x, w, r)[0])
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        y, h = ck.rms_norm(x, w, r)
        q, s = ck.rms_norm_mxfp8(h, w)
    for i in range(3):
        x.mul_(1.5)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        y2, h2 = ck.rms_norm(x, w, r)
        q2, s2 = ck.rms_norm_mxfp8(h2, w)
        assert torch.equal(y, y2) and torch.equal(h, h2) and torch.equal(bits(q), bits(q2)) and torch.equal(bits(s), bits(s2))


def test_refusals(hip):
    x = torch.zeros(4, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="weights for rows"):
        ck.rms_norm(x, torch.ones(65, device="cuda"))
    with pytest.raises(ValueError, match="differ"):
        ck.rms_norm(x, None, x[:2])
    with pytest.raises(ValueError, match="differ"):
        ck.rms_norm_fp8(x, torch.tensor(1.0), None, x.float())
    with pytest.raises(ValueError, match="65536"):
        ck.rms_norm(torch.zeros(1, 65537, device="cuda"))
    with pytest.raises(ValueError, match="divisible by 32"):
        ck.rms_norm_mxfp8(x[:, :40])
    with pytest.raises(ck.NoCapableBackendError):
        ck.rms_norm(x.double())
    with pytest.raises(ck.NoCapableBackendError):
        ck.rms_norm_mxfp8(x[0])
    with pytest.raises(ck.NoCapableBackendError):
        ck.rms_norm(x.cpu())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols", [(2048, 8), (2049, 64), (4099, 72), (3001, 96), (9001, 128), (2500, 136), (2177, 200), (4096, 256)])
def test_many_short_rows(rows, cols, dtype, hip):
    """A head's norm: the same bits as a few rows at a time, in 8 bits as the two calls."""
    x, r, w = make(rows, cols, dtype, rows * cols + 3)
    x[7], r[7], x[11, 3] = 0, 0, float("nan")
    keep = torch.arange(rows) != 11
    xc, rc, wc = x.cuda(), r.cuda(), w.cuda()
    y, h = ck.rms_norm(xc, wc, rc)
    total = (x.float() + r.float()).to(x.dtype)
    assert torch.equal(bits(h[keep]), bits(total[keep])) and bool(h[11, 3].isnan()) and bool(y[11].isnan().all())
    check(y.cpu()[keep], total[keep], w, dtype)
    plain = ck.rms_norm(xc)
    check(plain.cpu()[keep], x[keep], None, dtype)
    for i in range(0, rows, 1000):
        a, b = ck.rms_norm(xc[i:i + 1000], wc, rc[i:i + 1000])
        assert torch.equal(bits(y[i:i + 1000]), bits(a)) and torch.equal(bits(h[i:i + 1000]), bits(b))
    scale = torch.tensor(0.02, device="cuda")
    for out in (torch.float8_e4m3fn, torch.float8_e5m2):
        codes, h8 = ck.rms_norm_fp8(xc, scale, wc, rc, output_type=out)
        assert torch.equal(bits(codes), bits(ck.quantize_per_tensor_fp8(y, scale, out))) and torch.equal(bits(h), bits(h8))
    codes, scales, h8 = ck.rms_norm_mxfp8(xc, wc, rc, pad_32x=True)
    q, s = ck.quantize_mxfp8(y, pad_32x=True)
    assert torch.equal(bits(h), bits(h8)) and torch.equal(bits(codes), bits(q)) and torch.equal(bits(scales), bits(s))
