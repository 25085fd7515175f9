"""The text-generation operators together: the sample's decoder against a plain forward pass in 32 bits
over the whole token sequence with the dequantized weights, and the int4 layout under F.linear."""
import sys
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "comfy-kitchen_amd" / "samples"))

import text_generation as tg  # noqa: E402

import comfy_kitchen as ck  # noqa: E402
from comfy_kitchen.tensor import QuantizedTensor  # noqa: E402

pytestmark = pytest.mark.gpu


def plain(model, tokens):
    """Logits behind every token, in 32 bits, without a cache."""
    c = model.config
    w = {k: v.dequantize().float() if isinstance(v, QuantizedTensor) else v.float() for k, v in model.weights.items()}
    n = len(tokens)

    def norm(x, name):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + c.eps) * w[name]

    f = tg.rope_matrices(torch.arange(n, device="cuda"), c.head_dim, c.rope_base)

    def rope(x):
        pairs = x.unflatten(-1, (-1, 1, 2))
        return (f[:, None] * pairs).sum(-1).flatten(-2)

    at = torch.arange(n, device="cuda")
    see = at[:, None] >= at
    if c.window:
        see &= (at[:, None] - at < c.window) | (at < c.sinks)
    x = w["embedding"][tokens]
    for i in range(c.layers):
        q, k, v = (norm(x, f"{i}.norm1") @ w[f"{i}.qkv"].t()).unflatten(-1, (-1, c.head_dim)).split((c.heads, c.kv_heads, c.kv_heads), 1)
        q, k = rope(q), rope(k)
        k, v = (t.repeat_interleave(c.heads // c.kv_heads, 1) for t in (k, v))
        s = torch.einsum("qhd,khd->hqk", q, k) * c.head_dim ** -0.5
        p = torch.softmax(s.masked_fill(~see, -float("inf")), -1)
        x = x + torch.einsum("hqk,khd->qhd", p, v).flatten(1) @ w[f"{i}.out"].t()
        gate, up = (norm(x, f"{i}.norm2") @ w[f"{i}.up"].t()).chunk(2, -1)
        x = x + (F.silu(gate) * up) @ w[f"{i}.down"].t()
    return norm(x, "norm") @ w["head"].t()


# a dozen 16-bit roundings a layer of about 2^-9 (bf16) each, the cache's 2^-4 of E4M3 codes on top
@pytest.mark.parametrize("window,sinks,cache,bound", [(0, 0, None, 0.04), (24, 3, None, 0.04), (24, 3, torch.float8_e4m3fn, 0.15)])
def test_decoder(window, sinks, cache, bound, hip):
    c = tg.Config(window=window, sinks=sinks)
    model = tg.TextDecoder(c, tg.TextDecoder.random_weights(c), pages=40, page_size=8, cache_dtype=cache,
                           cache_scale=None if cache is None else 1 / 64)
    g = torch.Generator(device="cuda").manual_seed(3)
    text = torch.randint(0, c.vocab, (3, 60), device="cuda", generator=g)
    text[:, :37] = text[0, :37]  # one prompt, three continuations
    want = [plain(model, t) for t in text]

    def near(got, ref):
        assert float((got.float() - ref).norm() / ref.norm()) < bound

    first, logits = model.prompt(text[0, :37])
    near(logits, want[0][36])
    sequences = [first, model.cache.fork(first), model.cache.fork(first)]
    for i in range(37, 60):
        logits = model.step(sequences, text[:, i])
        for b in range(3):
            near(logits[b], want[b][i])
    for s in sequences:
        model.cache.free(s)
    assert model.cache.free_pages == 40


def test_generate(hip):
    c = tg.Config(layers=1, window=32, sinks=2)
    model = tg.TextDecoder(c, tg.TextDecoder.random_weights(c), pages=64)
    prompt = torch.arange(50, device="cuda")
    runs = [model.generate(prompt, 12, 3, generator=torch.Generator(device="cuda").manual_seed(1)) for _ in range(2)]
    assert runs[0].shape == (3, 12) and torch.equal(*runs) and model.cache.free_pages == 64


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(96, 256), (50, 100)], ids=["whole", "padded"])
def test_layout(shape, dtype, hip):
    g = torch.Generator(device="cuda").manual_seed(1)
    w = (torch.randn(shape, generator=g, device="cuda") * 0.05).to(dtype)
    qw = QuantizedTensor.from_float(w, "GroupInt4Layout", group_size=64)
    assert qw.shape == w.shape and qw.dtype == dtype and set(qw.state_dict("w")) == {"w", "w_scale"}
    back = qw.dequantize()
    assert back.shape == w.shape
    exact = ck.dequantize_int4(qw._qdata, qw.params.scale, None, 64, torch.float32)[:, :shape[1]]  # before dequantize()'s rounding
    assert torch.equal(exact.to(dtype), back)
    assert bool(((exact - w.float()).abs() <= 0.51 * qw.params.scale.float().repeat_interleave(64, 1)[:, :shape[1]]).all())
    x = torch.randn(5, shape[1], generator=g, device="cuda").to(dtype)
    bias = torch.randn(shape[0], generator=g, device="cuda").to(dtype)
    want = F.linear(x.float(), back.float(), bias.float())
    # dequantize() rounds each weight to 16 bits, the product only its result
    tol = (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11) * (x.float().abs() @ back.float().abs().t() + want.abs())
    for y in (F.linear(x, qw, bias), torch.addmm(bias, x, qw.t()), torch.mm(x, qw.t()) + bias, F.linear(x[None, :2], qw, bias)[0]):
        assert y.dtype == dtype and bool(((y.float() - want[:y.shape[0]]).abs() <= 2 * tol[:y.shape[0]] + 1e-3).all())
    assert torch.equal(F.linear(x.float(), qw), F.linear(x.float(), back.float()))  # f32 activations: dequantized
    moved = qw.to("cpu").to("cuda")
    assert torch.equal(F.linear(x, moved, bias), F.linear(x, qw, bias))
    assert torch.equal(F.linear(x, qw.clone().t().t(), bias), F.linear(x, qw, bias))
    codes, scale = qw._qdata, qw.params.scale
    zero = torch.randint(0, 16, scale.shape, generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)
    shifted = QuantizedTensor(codes, "GroupInt4Layout", type(qw.params)(scale=scale, orig_dtype=dtype, orig_shape=tuple(shape),
                                                                        group_size=64, zero=zero))
    assert torch.equal(F.linear(x, shifted), ck.linear_int4(F.pad(x, (0, 2 * codes.shape[1] - shape[1])), codes, scale, zero, None, 64))
    assert set(shifted.state_dict("w")) == {"w", "w_scale", "w_zero"}


def test_operators_under_compile_and_modes(hip):
    """The custom ops (what anything that looks at the dispatcher sees) give the calls' results."""
    from torch.utils._python_dispatch import TorchDispatchMode

    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            if func.namespace == "comfy_kitchen":
                seen.append(func._schema.name.split("::")[1])
            return func(*args, **(kwargs or {}))

    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randn(64, 128, generator=g, device="cuda").bfloat16()
    q = torch.randn(2, 4, 64, generator=g, device="cuda").bfloat16()
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([20, 9], dtype=torch.int32, device="cuda")
    slots = torch.arange(8, 64, 8, device="cuda")

    def run():
        k, v = (torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        codes, scales = ck.quantize_int4(w, 64)
        x = ck.linear_int4(q.flatten(1)[:, :128], codes, scales, group_size=64)
        rows = torch.cos(torch.arange(7 * 128, device="cuda").reshape(7, 2, 64)).bfloat16()
        ck.paged_write(rows, rows * 2, k, v, slots)
        ck.paged_copy(k, v, slots, slots + 1)
        return [x, ck.dequantize_int4(codes, scales, None, 64), k, v, ck.paged_attention(q, k, v, table, lengths),
                ck.window_attention(q[None], q[None, :, :2], q[None, :, 2:], 1)]

    want = run()
    with Watch():
        got = run()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert seen == ["quantize_int4", "linear_int4", "paged_write", "paged_copy", "dequantize_int4", "paged_attention", "window_attention"]
    torch._dynamo.reset()
    for a, b in zip(torch.compile(run)(), want):
        assert torch.allclose(a.float(), b.float(), atol=1e-2, rtol=1e-2)
