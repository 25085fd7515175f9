"""The text-generation entry points refuse bad arguments with a message, without a GPU (arguments are
checked before any HIP call), and have nothing to do for empty calls."""
import ctypes

import pytest
import torch

import comfy_kitchen as ck
import comfy_kitchen.backends.hip as hb


@pytest.fixture(scope="module")
def lib():
    return hb.load_library()


@pytest.fixture(scope="module")
def mem():
    buf = ctypes.create_string_buffer(4096)
    yield (ctypes.addressof(buf) + 255) // 256 * 256
    del buf


def strides(*values):
    return (ctypes.c_int64 * len(values))(*values)


def refused(lib, status, text):
    assert status == 1 and text.encode() in lib.ckh_last_error(), lib.ckh_last_error()


def test_int4(lib, mem):
    p = mem
    refused(lib, lib.ckh_quantize_int4(p, p, p, 4, 48, 32, 2, 0), "multiple of 32")
    refused(lib, lib.ckh_quantize_int4(p, p, p, 4, 64, 16, 2, 0), "group size")
    refused(lib, lib.ckh_quantize_int4(p, p, p, 4, 64, 32, 5, 0), "unsupported input dtype")
    refused(lib, lib.ckh_quantize_int4(None, p, p, 4, 64, 32, 2, 0), "null pointer")
    refused(lib, lib.ckh_dequantize_int4(p, p, None, p + 2, 4, 64, 32, 2, 2, 0), "misaligned")
    refused(lib, lib.ckh_dequantize_int4(p, p, None, p, 4, 64, 32, 3, 2, 0), "unsupported scale dtype")

    def linear(x=p, m=2, n=4, k=64, stride=64, group=32, x_code=2, scale_code=2, bias=None, bias_code=0):
        return lib.ckh_linear_int4(x, p, p, None, bias, p, m, n, k, stride, group, x_code, scale_code, bias_code, None, 0, 0)

    refused(lib, linear(x_code=0), "unsupported activation dtype")
    refused(lib, linear(scale_code=5), "unsupported scale dtype")
    refused(lib, linear(bias=p, bias_code=6), "unsupported bias dtype")
    refused(lib, linear(stride=56), "rows overlap")
    refused(lib, linear(stride=68), "misaligned")
    refused(lib, linear(x=p + 8), "misaligned")
    refused(lib, linear(k=1 << 24), "multiple of 32")
    refused(lib, linear(m=1 << 21), "activation rows")
    refused(lib, linear(stride=1 << 24), "stride too large")
    assert linear(m=0) == 0 and linear(n=0) == 0 and lib.ckh_quantize_int4(None, None, None, 0, 64, 32, 2, 0) == 0
    assert lib.ckh_linear_int4_workspace_bytes(1, 4096, 4096, 128) == 0


def test_paged_attention(lib, mem):
    p = mem
    ok = strides(256, 64, 2048, 128, 64, 2048, 128, 64)

    def call(q=p, heads=4, kv_heads=2, dim=64, pages=3, page=16, most=2, s=ok, window=0, sinks=0, code=2, cache=2, batch=1):
        return lib.ckh_paged_attention(q, p, p, p, p, None, None, p, batch, heads, kv_heads, dim, pages, page, most, most, s, window,
                                       sinks, 1.0, code, cache, None, 0, 0)

    for kwargs, text in ((dict(code=0), "query dtype"), (dict(cache=1), "cache dtype"), (dict(dim=80), "head_dim"), (dict(heads=3), "heads"),
                         (dict(kv_heads=0), "heads"), (dict(pages=0), "pages"), (dict(page=0), "pages"), (dict(most=1 << 30), "pages"),
                         (dict(window=-1), "window"), (dict(sinks=1 << 40), "sinks"), (dict(q=None), "null pointer"), (dict(q=p + 4), "misaligned"),
                         (dict(s=strides(256, 64, 2048, 126, 64, 2048, 128, 64)), "stride 3"), (dict(s=strides(256, 64, 2048, 1 << 25, 64, 2048, 128, 64)), "too large"),
                         (dict(s=strides(-256, 64, 2048, 128, 64, 2048, 128, 64)), "stride 0")):
        refused(lib, call(**kwargs), text)
    assert call(batch=0) == 0 and call(heads=0) == 0
    f = lib.ckh_paged_attention_workspace_bytes
    assert f(1, 8, 8, 128, 16, 8) == 0 < f(1, 8, 8, 128, 16, 4000) and f(0, 8, 8, 128, 16, 8) == 0


def test_window_attention(lib, mem):
    p = mem
    ok = strides(4096, 256, 64, 4096, 128, 64, 4096, 128, 64)

    def call(q=p, batch=1, queries=4, keys=4, heads=4, kv_heads=2, dim=64, s=ok, window=0, sinks=0, code=2):
        return lib.ckh_window_attention(q, p, p, None, p, batch, queries, keys, heads, kv_heads, dim, s, window, sinks, 1.0, code, None, 0, 0)

    for kwargs, text in ((dict(code=5), "dtype"), (dict(dim=32), "head_dim"), (dict(heads=5), "heads"), (dict(keys=1 << 31), "keys"),
                         (dict(window=-2), "window"), (dict(q=None), "null pointer"), (dict(q=p + 8), "misaligned"),
                         (dict(s=strides(4096, 256, 64, 4096, 0, 64, 4096, 128, 64)), "overlap"), (dict(s=strides(4096, 250, 64, 4096, 128, 64, 4096, 128, 64)), "stride 1"),
                         (dict(s=strides(4096, 256, 64, 4096, 128, 64, 4096, 1 << 23, 64)), "too large")):
        refused(lib, call(**kwargs), text)
    assert call(batch=0) == 0 and call(queries=0) == 0


def test_pages(lib, mem):
    p = mem
    ok = strides(128, 64, 128, 64, 2048, 128, 64, 2048, 128, 64)

    def write(key=p, tokens=2, dim=64, pages=3, page=16, s=ok, code=2, cache=2, slots=p, wide=0):
        return lib.ckh_paged_write(key, p, p, p, slots, None, None, tokens, 2, dim, pages, page, s, code, cache, wide, 0)

    for kwargs, text in ((dict(code=0), "unsupported dtype"), (dict(cache=1), "cache dtype"), (dict(dim=24), "head_dim"), (dict(pages=0), "pages"),
                         (dict(pages=1 << 30, page=16), "pages"), (dict(key=None), "null pointer"), (dict(slots=p + 4, wide=1), "misaligned"),
                         (dict(tokens=1 << 30), "too many"), (dict(s=strides(128, 64, 128, 60, 2048, 128, 64, 2048, 128, 64)), "stride 3")):
        refused(lib, write(**kwargs), text)
    assert write(tokens=0) == 0
    ok8 = strides(0, 2048, 128, 64, 0, 2048, 128, 64)

    def copy(cache=p, layers=1, rows=2, dim=64, pages=3, page=16, s=ok8, size=2):
        return lib.ckh_paged_copy(cache, p, p, p, layers, rows, 2, dim, pages, page, s, size, 0, 0)

    for kwargs, text in ((dict(size=3), "elements of 3"), (dict(dim=12), "multiple of 16 bytes"), (dict(layers=70000), "layers"), (dict(page=0), "pages"),
                         (dict(cache=None), "null pointer"), (dict(rows=1 << 30), "too many"), (dict(s=strides(0, 2048, 128, 4, 0, 2048, 128, 64)), "stride 3")):
        refused(lib, copy(**kwargs), text)
    assert copy(rows=0) == 0 and copy(layers=0) == 0


def test_no_cpu_fallback_and_fake_shapes():
    with pytest.raises(ck.NoCapableBackendError):
        ck.linear_int4(torch.zeros(1, 32).bfloat16(), torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1).bfloat16())
    from torch._subclasses.fake_tensor import FakeTensorMode

    op = torch.ops.comfy_kitchen
    with FakeTensorMode():
        w, x = torch.empty(48, 320, dtype=torch.float16), torch.empty(2, 3, 320, dtype=torch.bfloat16)
        codes, scales = op.quantize_int4(w, 128)
        assert codes.shape == (48, 160) and codes.dtype == torch.uint8 and scales.shape == (48, 3) and scales.dtype == w.dtype
        assert op.linear_int4(x, codes, scales, None, None, 128).shape == (2, 3, 48)
        assert op.dequantize_int4(codes, scales, None, 128, 0).shape == (48, 320)
        q, cache = torch.empty(5, 8, 64, dtype=torch.bfloat16), torch.empty(9, 16, 2, 64, dtype=torch.bfloat16)
        i = torch.empty(5, 3, dtype=torch.int32)
        y = op.paged_attention(q, cache, cache, i, i[:, 0], None, 0, 0, None, None)
        assert y.shape == q.shape and y.dtype == q.dtype
        p = torch.empty(2, 7, 8, 64, dtype=torch.float16)
        assert op.window_attention(p, p, p, 4, 1, None, None).shape == p.shape
        assert op.paged_write(q[:, :2], q[:, :2], cache, cache.clone(), i[:, 0], None, None) is None
