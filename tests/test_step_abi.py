"""The entry points of a generation step's other operators refuse bad arguments with a message, without a GPU
(arguments are checked before any HIP call), and have nothing to do for empty calls; rope_rates; fake shapes."""
import ctypes
import math

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


def test_rms_norm(lib, mem):
    p = mem

    def call(x=p, r=None, w=p, scale=None, y=p, scales=None, h=None, rows=2, cols=64, out_rows=2, out_cols=64, step=64, r_step=0, code=2, w_code=2,
             out=2, mx=0):
        return lib.ckh_rms_norm(x, r, w, scale, y, scales, h, rows, cols, out_rows, out_cols, step, r_step, 1e-6, code, w_code, out, mx, 0)

    for kwargs, text in ((dict(code=5), "unsupported dtype"), (dict(w_code=5), "weight dtype"), (dict(out=1), "result of dtype"), (dict(out=6, mx=1), "result of dtype"),
                         (dict(rows=-1), "rows of"), (dict(rows=1 << 31), "rows of"), (dict(cols=65537), "65536 at most"), (dict(out_cols=32), "only MXFP8"),
                         (dict(out=5, mx=1, out_cols=48), "multiple of 32"), (dict(out=5, mx=1, out_rows=1), "multiple of 32"),
                         (dict(out=5, mx=1, out_rows=129), "multiple of 32"), (dict(out=5, mx=1), "null pointer"), (dict(out=5), "null pointer"),
                         (dict(r=p), "null pointer"), (dict(x=None), "null pointer"), (dict(x=p + 1), "misaligned"), (dict(w=p + 2, w_code=0), "misaligned"),
                         (dict(out=5, mx=1, scales=p, y=p + 4), "misaligned"), (dict(step=-64), "negative stride")):
        refused(lib, call(**kwargs), text)
    assert call(rows=0, out_rows=0, x=None) == 0 and call(cols=0, out_cols=0, x=None) == 0
    for rows, cols in ((1 << 26, 8), (1 << 26, 7), (1 << 19, 65536)):
        refused(lib, call(rows=rows, out_rows=rows, cols=cols, out_cols=cols, step=cols), "too many elements")


def test_paged_write_rope(lib, mem):
    p = mem
    ok = strides(256, 64, 128, 64, 128, 64, 2048, 128, 64, 2048, 128, 64)

    def call(q=p, out=p, tokens=2, heads=4, kv_heads=2, dim=64, rotary=64, pages=3, page=16, s=ok, code=2, cache=2, at=p, wide_at=0, slots=p, wide=0, rates=p,
             k_scale=None):
        return lib.ckh_paged_write_rope(q, p, p, at, rates, out, None, p, p, slots, k_scale, None, tokens, heads, kv_heads, dim, rotary, pages, page, s, 1, 1.0, code,
                                        cache, wide_at, wide, 0)

    for kwargs, text in ((dict(code=0), "unsupported dtype"), (dict(cache=1), "cache dtype"), (dict(dim=24), "multiple of 16"), (dict(rotary=66), "turned"),
                         (dict(rotary=63), "turned"), (dict(rotary=-2), "turned"), (dict(pages=0), "pages"), (dict(pages=1 << 30), "pages"),
                         (dict(k_scale=p), "scales with a cache"), (dict(tokens=1 << 31), "heads"), (dict(tokens=1 << 28), "too many"), (dict(q=None), "null pointer"),
                         (dict(rates=None), "null pointer"), (dict(q=p + 8), "misaligned"), (dict(at=p + 4, wide_at=1), "misaligned"),
                         (dict(slots=p + 4, wide=1), "misaligned"), (dict(s=strides(256, 60, 128, 64, 128, 64, 2048, 128, 64, 2048, 128, 64)), "stride 1"),
                         (dict(s=strides(256, 64, 128, 64, 128, 64, 2048, 128, 64, 2048, -128, 64)), "stride 10")):
        refused(lib, call(**kwargs), text)
    assert call(tokens=0, q=None) == 0 and call(heads=0, kv_heads=0) == 0


def test_sample(lib, mem):
    p = mem

    def call(x=p, u=p, t=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, rows=1, vocab=100, code=0, ws=p, nbytes=1 << 20):
        return lib.ckh_sample(x, u, t, None, None, None, temperature, top_k, top_p, min_p, p, rows, vocab, vocab, code, ws, nbytes, 0)

    nan = float("nan")
    for kwargs, text in ((dict(code=5), "dtype"), (dict(vocab=0), "logits"), (dict(vocab=(1 << 24) + 1), "logits"), (dict(rows=65536), "rows"),
                         (dict(temperature=-1.0), "temperature"), (dict(temperature=nan), "temperature"), (dict(top_k=-1), "top_k"), (dict(top_p=-0.5), "top_p"),
                         (dict(top_p=nan), "top_p"), (dict(min_p=1.1), "min_p"), (dict(min_p=nan), "min_p"), (dict(x=None), "null pointer"), (dict(ws=None), "null pointer"),
                         (dict(x=p + 2), "misaligned"), (dict(u=p + 2), "misaligned"), (dict(ws=p + 4), "misaligned"), (dict(t=p + 1), "misaligned"),
                         (dict(nbytes=100), "workspace")):
        refused(lib, call(**kwargs), text)
    assert call(rows=0, x=None) == 0
    f = lib.ckh_sample_workspace_bytes
    assert f(0, 5) == 0 < f(1, 1) == f(1, 8192) < f(1, 8193) == f(2, 1)


def test_shared_attention(lib, mem):
    p = mem
    ok = strides(256, 64, 2048, 128, 64, 2048, 128, 64)

    def call(q=p, heads=4, kv_heads=2, dim=64, groups=1, pages=3, page=16, most=2, s=ok, code=2, cache=2, batch=2, shared=p, ws=p, nbytes=1 << 40):
        return lib.ckh_shared_attention(q, p, p, p, p, p, shared, None, None, p, batch, heads, kv_heads, dim, groups, pages, page, most, most, s, 1.0, code, cache,
                                        ws, nbytes, 0)

    for kwargs, text in ((dict(code=0), "query dtype"), (dict(cache=1), "cache dtype"), (dict(dim=80), "head_dim"), (dict(heads=3), "heads"),
                         (dict(kv_heads=0), "heads"), (dict(pages=0), "pages"), (dict(page=0), "pages"), (dict(most=1 << 30), "pages"), (dict(groups=-1), "groups"),
                         (dict(batch=4096), "4096"), (dict(q=None), "null pointer"), (dict(shared=None), "null pointer"), (dict(ws=None), "null pointer"),
                         (dict(q=p + 4), "misaligned"), (dict(ws=p + 8), "misaligned"), (dict(nbytes=1000), "workspace"),
                         (dict(s=strides(256, 64, 2048, 126, 64, 2048, 128, 64)), "stride 3"),
                         (dict(s=strides(256, 64, 2048, 1 << 25, 64, 2048, 128, 64)), "too large"), (dict(heads=65532, kv_heads=65532, batch=4000), "too many")):
        refused(lib, call(**kwargs), text)
    assert call(batch=0) == 0 and call(heads=0) == 0
    f = lib.ckh_shared_attention_workspace_bytes
    assert f(0, 8, 8, 128, 1, 16, 8) == 0 < f(1, 8, 8, 128, 0, 16, 8) and f(4, 8, 0, 128, 1, 16, 8) == 0


def test_shared_attention_workspace(lib):
    """No more than the tables' tokens need, nor than a long context's chunks do."""
    small = lib.ckh_shared_attention_workspace_bytes(4, 40, 8, 128, 1, 16, 55)
    assert small < 4 << 20
    sizes = [lib.ckh_shared_attention_workspace_bytes(4, 40, 8, 128, 1, 16, n) for n in (1, 55, 1000, 10 ** 5, 10 ** 7)]
    assert sizes == sorted(sizes) and sizes[-1] == sizes[-2] < 64 << 20
    for tokens in (0, 1, 63, 64, 65):
        assert lib.ckh_shared_attention_workspace_bytes(1, 1, 1, 64, 0, 1, tokens) > 0


def test_rope_rates():
    plain = ck.rope_rates(64, 10000.0, device="cpu")
    assert plain.dtype == torch.float32 and plain.shape == (32,)
    want = [10000.0 ** (-2 * i / 64) for i in range(32)]
    assert torch.equal(plain, torch.tensor(want, dtype=torch.float64).float())
    assert torch.equal(ck.rope_rates(64, factor=4.0, device="cpu"), torch.tensor([w / 4 for w in want], dtype=torch.float64).float())
    got = ck.rope_rates(64, factor=8.0, context=4096, slow=1.0, fast=32.0, device="cpu")
    for i, w in enumerate(want):
        share = min(1.0, max(0.0, (4096 * w / (2 * math.pi) - 1) / 31))
        assert float(got[i]) == pytest.approx(w * (share + (1 - share) / 8), rel=1e-7)
    assert got[0] == plain[0] and got[-1] == plain[-1] / 8
    assert ck.rope_rates(0, device="cpu").shape == (0,)
    for kwargs in (dict(dim=3), dict(dim=-2), dict(dim=8, base=0.0), dict(dim=8, factor=0.0), dict(dim=8, context=-1), dict(dim=8, context=9, slow=2.0, fast=2.0)):
        with pytest.raises(ValueError):
            ck.rope_rates(device="cpu", **kwargs)


def test_no_cpu_fallback_and_fake_shapes():
    x = torch.zeros(2, 64).bfloat16()
    for call in (lambda: ck.rms_norm(x), lambda: ck.rms_norm_fp8(x, torch.tensor(1.0)), lambda: ck.rms_norm_mxfp8(x),
                 lambda: ck.sample_tokens(x, torch.zeros(2)), lambda: ck.sample_tokens(x, torch.zeros(2), torch.ones(2), 3)):
        with pytest.raises(ck.NoCapableBackendError):
            call()
    from torch._subclasses.fake_tensor import FakeTensorMode

    op = torch.ops.comfy_kitchen
    with FakeTensorMode():
        x, r = torch.empty(3, 5, 320, dtype=torch.float16), torch.empty(3, 5, 320, dtype=torch.float16)
        y, h = op.rms_norm(x, None, r, 1e-6)
        assert y.shape == h.shape == x.shape and y.dtype == x.dtype and op.rms_norm(x, None, None, 1e-6)[1].shape == (0,)
        y, h = op.rms_norm_fp8(x, torch.empty(()), None, r, 1e-6, 6)
        assert y.dtype == torch.float8_e5m2 and h.shape == x.shape
        q, s, h = op.rms_norm_mxfp8(x[0, :, :300], None, None, 1e-6, True)
        assert q.shape == (32, 320) and s.shape == (128, 12) and s.dtype == torch.float8_e8m0fnu and h.shape == (0,)
        assert op.sample_tokens(x[0], torch.empty(5), 1.0, 0, 1.0, 0.0, None, None, None, None).dtype == torch.int64
        q, cache = torch.empty(5, 8, 64, dtype=torch.bfloat16), torch.empty(9, 16, 2, 64, dtype=torch.bfloat16)
        i = torch.empty(5, 3, dtype=torch.int32)
        assert op.shared_attention(q, cache, cache, i, i[:, 0], i[:, 0], i[:4, 0], None, None, None).shape == q.shape
        for keep in (True, False):
            turned, key = op.paged_write_rope(q, q[:, :2], q[:, :2], i[:, 0], torch.empty(32), cache, cache.clone(), i[:, 0], True, 1.0, None, None, keep)
            assert turned.shape == q.shape and key.shape == (5 if keep else 0, 2, 64)
