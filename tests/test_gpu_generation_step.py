"""A generation step's operators together: the sample's decoder with attention over what its sequences share, with MXFP8
linears, and its choice of tokens."""
import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "comfy-kitchen_amd" / "samples"))

import text_generation as tg  # noqa: E402
from test_gpu_text_generation import plain  # noqa: E402

pytestmark = pytest.mark.gpu


# 16-bit roundings as in the test of the plain decoder (0.04; the cache's E4M3 codes 0.15).  MXFP8: nine linears whose
# activations are rounded to E4M3, each 2^-4 / sqrt(3) off at most in the mean, add up to 0.11 if none cancels any other.
@pytest.mark.parametrize("linears,cache,bound", [("int4", None, 0.04), ("int4", torch.float8_e4m3fn, 0.15), ("mxfp8", None, 0.15)])
def test_forks_read_their_prompt_once(linears, cache, bound, hip):
    c = tg.Config(linears=linears)
    model = tg.TextDecoder(c, tg.TextDecoder.random_weights(c), pages=80, page_size=8, cache_dtype=cache,
                           cache_scale=None if cache is None else 1 / 64, share_from=1)
    g = torch.Generator(device="cuda").manual_seed(3)
    text = torch.randint(0, c.vocab, (6, 60), device="cuda", generator=g)
    text[:4, :37] = text[0, :37]  # four answers to one prompt, two to another
    text[4:, :45] = text[4, :45]
    want = [plain(model, t) for t in text]

    def near(got, ref):
        assert float((got.float() - ref).norm() / ref.norm()) < bound

    a, logits = model.prompt(text[0, :37])
    near(logits, want[0][36])
    b, logits = model.prompt(text[4, :45])
    near(logits, want[4][44])
    sequences = [a, *(model.cache.fork(a) for _ in range(3)), b, model.cache.fork(b)]
    for i in range(15):
        at = [37 + i] * 4 + [45 + i] * 2
        if i:
            starts, shared = (t.tolist() for t in model.cache.groups(sequences, 1))
            assert starts == [0, 4, 6] and shared == [32, 40]
        logits = model.step(sequences, torch.stack([text[j, n] for j, n in enumerate(at)]))
        for j, n in enumerate(at):
            near(logits[j], want[j][n])
    for s in sequences:
        model.cache.free(s)
    assert model.cache.free_pages == 80


@pytest.mark.parametrize("linears", ["int4", "mxfp8"])
def test_generate(linears, hip):
    c = tg.Config(layers=1, linears=linears)
    model = tg.TextDecoder(c, tg.TextDecoder.random_weights(c), pages=64, share_from=1)
    prompt = torch.arange(50, device="cuda")
    how = dict(temperature=0.7, top_k=20, top_p=0.9, min_p=0.01)
    runs = [model.generate(prompt, 12, 3, generator=torch.Generator(device="cuda").manual_seed(1), **how) for _ in range(2)]
    assert runs[0].shape == (3, 12) and torch.equal(*runs) and model.cache.free_pages == 64
    assert bool(((runs[0] >= 0) & (runs[0] < c.vocab)).all())
    greedy = [model.generate(prompt, 12, n, temperature=0.0) for n in (1, 3)]
    assert torch.equal(greedy[1][0], greedy[1][1])
    # the first token of every run is one of the kept ones
    sequence, logits = model.prompt(prompt)
    model.cache.free(sequence)
    assert bool(torch.isin(runs[0][:, 0], logits.float().topk(20).indices).all()) and greedy[0][0, 0] == logits.argmax()


def test_a_captured_step(hip):
    """One layer's step as a graph: replayed with other tokens, lengths, slots and random numbers it gives what eager calls do."""
    import comfy_kitchen as ck

    g = torch.Generator(device="cuda").manual_seed(5)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g).bfloat16()

    b, heads, hk, d, hidden, vocab = 6, 8, 2, 64, 512, 3000
    cache = [[randn(20, 16, hk, d) for _ in range(2)] for _ in range(2)]
    cache[1] = [t.clone() for t in cache[0]]
    w, wo, head = randn((heads + 2 * hk) * d, hidden) * 0.05, randn(hidden, heads * d) * 0.05, randn(vocab, hidden)
    norm, rates = 1 + 0.1 * randn(hidden), ck.rope_rates(d)
    x, r, u = randn(b, hidden), randn(b, hidden), torch.rand(b, device="cuda", generator=g)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    table = i32([[0, 1, 2, 3 + i, 9 + i] for i in range(b)])
    lengths, groups, shared = i32([50 + i for i in range(b)]), i32([0, 4, 6]), i32([48, 48])

    def step(k, v):
        y, h = ck.rms_norm(x, norm, r)
        q, key, value = (y @ w.t()).unflatten(-1, (-1, d)).split((heads, hk, hk), 1)
        at = lengths - 1
        page = torch.gather(table, 1, (at // 16)[:, None].long())[:, 0]
        q = ck.paged_write_rope(q, key, value, at, rates, k, v, page * 16 + at % 16)
        o = ck.shared_attention(q, k, v, table, lengths, groups, shared)
        y, h = ck.rms_norm(o.flatten(1) @ wo.t(), norm, h)
        return ck.sample_tokens(y @ head.t(), u, 0.8, 50, 0.95), h

    step(*cache[0])
    step(*cache[1])
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        tokens, h = step(*cache[0])
    for i in range(4):
        x.copy_(randn(b, hidden))
        u.copy_(torch.rand(b, device="cuda", generator=g))
        lengths.add_(1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want, want_h = step(*cache[1])
        assert torch.equal(tokens, want) and torch.equal(h, want_h)
        assert all(torch.equal(s, t) for s, t in zip(*cache))
