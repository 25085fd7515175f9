"""What PagedKVCache does where the device refuses a call, or would refuse every later one (no GPU)."""
import pytest
import torch

import comfy_kitchen as ck


def cache(pages=8, page=4, **kwargs):
    return ck.PagedKVCache(1, pages, page, 1, 16, torch.float16, device="cpu", **kwargs)


def state(c):
    return {s: (c.pages(s), c.length(s)) for s in range(20) if s in c}, c.free_pages, list(c._owners), list(c._free)


@pytest.mark.parametrize("broken", ["copy", "transfer"])
def test_a_refused_call_changes_nothing(broken, monkeypatch):
    moved = []
    monkeypatch.setattr(ck, "paged_copy", lambda k, v, src, dst: moved.append((src.tolist(), dst.tolist())))
    c = cache()
    a = c.add()
    c.append([a], [6])
    b = c.fork(a)
    before = state(c)

    def refuse(*args, **kwargs):
        raise RuntimeError("refused")

    with monkeypatch.context() as m:
        if broken == "copy":
            m.setattr(ck, "paged_copy", refuse)
        else:
            m.setattr(c, "_on_device", refuse)
        for call in (lambda: c.append([a, b], [1, 7]), lambda: c.append([b], [1]), lambda: c.compact(a, [0, 3, 5])):
            with pytest.raises(RuntimeError, match="refused"):
                call()
            assert state(c) == before
    # and the same calls go through afterwards, with the pages that were free
    slots = c.append([a, b], [1, 7]).tolist()
    pages = c.pages(a)[1:] + c.pages(b)[1:]
    assert len(moved) == 1 and len(set(pages)) == len(pages) == 4 and c.free_pages == 3
    assert slots == [c.pages(a)[1] * 4 + 2] + [c.pages(b)[t // 4] * 4 + t % 4 for t in range(6, 13)]
    c.free(a)
    c.free(b)
    assert c.free_pages == 8 and not any(c._owners)


def test_a_cache_that_no_call_takes():
    for change, match in ((dict(head_dim=72), "multiple of 16"), (dict(dtype=torch.float32), "float32"),
                          (dict(dtype=torch.float8_e5m2), "e5m2"), (dict(pages=2 ** 27, page_size=16), "32 bits")):
        args = dict(layers=1, pages=4, page_size=4, kv_heads=1, head_dim=16, dtype=torch.float16, device="meta")
        args.update(change)
        with pytest.raises(ValueError, match=match):
            ck.PagedKVCache(**args)


def test_scales_of_a_cache_that_is_not_scaled():
    """write leaves 16-bit rows as they are, so attend must not multiply them."""
    for scales in (dict(k_scale=0.5), dict(v_scale=2.0)):
        with pytest.raises(ValueError, match="float8_e4m3fn"):
            cache(**scales)
