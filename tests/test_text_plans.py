"""Strides that place no element (of dimensions of size 1, of empty tensors) do not matter to the
text-generation calls: what their checks answer, without a GPU."""
import pytest
import torch

import comfy_kitchen.backends.hip as hb


@pytest.fixture(scope="module", autouse=True)
def lib():
    hb.load_library()


def odd(*shape, dtype=torch.bfloat16):
    """Zeros of that shape whose leading strides are odd wherever the size is 1."""
    t = torch.zeros(shape, dtype=dtype)
    return t.as_strided(shape, [s if n > 1 else 2 * s + 3 for n, s in zip(shape[:-1], t.stride())] + [1])


def described(*tensors):
    return [x for t in tensors for x in (t.shape, t.stride(), t.dtype)]


def one_of_a_wider_projection(width=772):
    """The first row's heads cut from rows of a width that is no multiple of 16 bytes."""
    return torch.zeros(2, width, dtype=torch.bfloat16)[:, :256].unflatten(1, (4, 64))[:1]


@pytest.mark.parametrize("make", [one_of_a_wider_projection, lambda: odd(1, 4, 64), lambda: odd(3, 1, 64), lambda: odd(1, 1, 64),
                                  lambda: torch.zeros(4, 64, 1, dtype=torch.bfloat16).permute(2, 0, 1)])
def test_queries_keys_and_values(make):
    q = make()
    cache = torch.zeros(3, 16, q.shape[1], 64, dtype=torch.bfloat16)
    table, n = torch.zeros(q.shape[0], 2, dtype=torch.int32), q.shape[0]
    sizes, _ = hb._attention_plan(*described(q, cache, cache), table.shape, table.stride(), n, 0, 0, None)
    assert sizes[:4] == (n, q.shape[1], q.shape[1], 64) and all(s % 8 == 0 for s in sizes[8])
    assert hb._rows16(q) is q
    plan = hb._write_plan(*described(q, q, cache, cache), n, torch.int32)
    assert plan[:3] == tuple(q.shape) and all(s % 8 == 0 for s in plan[5])
    x = q[:, None]
    sizes, _ = hb._window_plan(*described(x, x, x), None, 4, 1, None)
    assert sizes[:3] == (n, 1, 1) and all(s % 8 == 0 for s in sizes[6])


def test_caches():
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    for shape in ((1, 16, 2, 64), (3, 1, 2, 64), (3, 16, 1, 64), (1, 1, 1, 64)):
        cache = odd(*shape)
        assert hb._attention_plan(*described(q, cache, cache), (2, 1), (1, 1), 2, 0, 0, None) is not None
        keys = q[:, :shape[2]]
        assert hb._write_plan(*described(keys, keys, cache, cache), 2, torch.int32) is not None
        assert hb._copy_plan(*described(cache, cache), (2,), torch.int32, (2,), torch.int32) is not None
        layers = odd(1, *shape)
        assert all(s % 8 == 0 for s in hb._copy_plan(*described(layers, layers), (2,), torch.int32, (2,), torch.int32)[6])


def test_copies_still_made():
    """Strides that do place elements are asked for as before, and a copy answers."""
    q = torch.zeros(3, 772, dtype=torch.bfloat16)[:, :256].unflatten(1, (4, 64))
    cache = torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16)
    rest = (torch.Size((3, 1)), (1, 1), 3, 0, 0, None)
    assert hb._attention_plan(*described(q, cache, cache), *rest) is None
    assert hb._attention_plan(*described(hb._rows16(q), cache, cache), *rest) is not None
    with pytest.raises(ValueError, match="16-byte"):
        bad = torch.zeros(3, 16, 2, 67, dtype=torch.bfloat16)[..., :64]
        hb._attention_plan(*described(hb._rows16(q), bad, bad), *rest)


def test_nothing_to_do():
    def linear(x):
        return hb._linear_plan(x.shape, x.stride(), x.dtype, (8, 64), (8, 1), torch.bfloat16, None, 128)

    whole = torch.zeros(128, 9, dtype=torch.bfloat16)
    assert linear(whole.t()) is None  # strides that place elements: copied
    for x in (whole.t()[:0], torch.zeros(2, 0, 128, dtype=torch.bfloat16)[:, :, :], whole.t()[:0].unflatten(0, (0, 3))):
        assert linear(x)[0] == (*x.shape[:-1], 8)
    for shape in ((0, 5, 4, 64), (2, 0, 4, 64)):
        q = torch.zeros(shape, dtype=torch.bfloat16)
        q = q.as_strided(shape, (3, 5, 7, 9))
        k = torch.zeros(shape[0], 9, 2, 64, dtype=torch.bfloat16)
        assert hb._window_plan(*described(q, k, k), None, 0, 0, None) is not None
    none = torch.zeros(0, 2, 64, dtype=torch.bfloat16).as_strided((0, 2, 64), (5, 3, 2))
    cache = torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16)
    assert hb._write_plan(*described(none, none, cache, cache), 0, torch.int64) is not None
    assert hb._attention_plan(*described(none, cache, cache), (0, 0), (1, 1), 0, 0, 0, None) is not None


def test_writes_with_scales_into_16_bits():
    """They are not scaled, so a scale there is refused (without a GPU: before any HIP call)."""
    import ctypes

    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    strides = (ctypes.c_int64 * 10)(128, 64, 128, 64, 2048, 128, 64, 2048, 128, 64)
    for scales in ((p, None), (None, p)):
        assert hb._lib.ckh_paged_write(p, p, p, p, p, *scales, 2, 2, 64, 3, 16, strides, 2, 2, 0, 0) == 1
        assert b"scales" in hb._lib.ckh_last_error()


def test_workspace_of_linears_does_not_grow_with_the_prompt():
    """Tiles that fill the GPU need no ranges of K, however many groups it has."""
    f = hb._lib.ckh_linear_int4_workspace_bytes
    for group in (32, 64, 96, 128, 1024):
        for k in (1024, 5120, 13824, 70016):
            for n in (256, 1024, 5120, 13824, 60000):
                sizes = [f(m, n, k, group) for m in (1, 16, 17, 24, 64, 100, 512, 2000, 16384, 100000)]
                assert max(sizes) <= 64 * 2 ** 20 and sizes[:2] == [0, 0] and sizes[-1] == 0, (group, k, n, sizes)
    assert f(16384, 5120, 13824, 32) == 0 < f(24, 5120, 13824, 32)


def test_page_tables_whose_tiles_pass_32_bits():
    """The kernel adds the tiles of 64 sequences in 32 bits; one sequence may have all that a table holds."""
    import ctypes

    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    strides = (ctypes.c_int64 * 8)(256, 64, 2 ** 26, 64, 64, 2 ** 26, 64, 64)

    def call(batch, most, q=p):
        return hb._lib.ckh_paged_attention(q, p, p, p, p, None, None, p, batch, 4, 1, 64, 3, 2 ** 20, most, most, strides, 0, 0, 1.0, 2, 2,
                                           None, 0, 0)

    for batch, most in ((64, 1024), (1000, 1024), (33, 2047)):
        assert call(batch, most) == 1 and b"page tables of" in hb._lib.ckh_last_error()
    for batch, most in ((64, 1023), (60000, 1000), (32, 2047), (1, 2047)):  # as far as the null pointer
        assert call(batch, most, None) == 1 and b"null pointer" in hb._lib.ckh_last_error()
