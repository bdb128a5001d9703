"""The decoder operators together, as examples/beam_decode.py uses them: a beam
search on the paged caches must score its hypotheses as a plain decoder without a
cache does, and must not depend on where its pages lie.

The plain decoder recomputes each hypothesis from the start in float64 on the same
bf16 weights; the framework's keeps activations in bf16 between products. A logit is
a product of the last normed activation (norm sqrt(d)) with an embedding row (norm
2): rounding the activation alone moves it by 2^-9 x 2 x sqrt(d) / sqrt(d) x 20 / 20
= 0.004, the two layers' dozen roundings before it by some four times that. The
summed log probability of n tokens is held to 0.1 n, a few times what they make
together; scores that lost a beam's history, read another clip's frames or a page
late are off by whole units a token.
"""
import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))

pytestmark = pytest.mark.gpu


def plain_score(W, features, tokens, start):
    """Sum of log probabilities of `tokens` (n,) after `start` over one clip's
    features (frames, d), all in float64."""
    d = features.shape[1]
    heads = d // 64
    lin = lambda x, w: x @ w[0].double().T + w[1].double()  # noqa: E731
    norm = lambda x, ln: torch.nn.functional.layer_norm(  # noqa: E731
        x, (d,), ln[0].double(), ln[1].double())
    inputs = torch.cat([torch.tensor([start], device=tokens.device), tokens[:-1]])
    n = len(inputs)
    x = W["embed"][inputs].double() + W["pos"][:n].double()
    f = features.to(torch.bfloat16).double()
    split = lambda t: t.view(-1, heads, 64).transpose(0, 1)  # noqa: E731
    causal = torch.full((n, n), float("-inf"), dtype=torch.float64, device=x.device).triu(1)

    def attend(q, k, v, mask=None):
        s = split(q) @ split(k).transpose(1, 2) / 8
        p = torch.softmax(s if mask is None else s + mask, -1)
        return (p @ split(v)).transpose(0, 1).reshape(-1, d)

    for w in W["layers"]:
        q, k, v = lin(norm(x, w["ln1"]), w["qkv"]).chunk(3, 1)
        x = x + lin(attend(q, k, v, causal), w["out"])
        k, v = lin(f, w["kv2"]).chunk(2, 1)
        x = x + lin(attend(lin(norm(x, w["ln2"]), w["q2"]), k, v), w["out2"])
        x = x + lin(torch.nn.functional.gelu(lin(norm(x, w["ln3"]), w["fc1"])), w["fc2"])
    logits = norm(x, W["ln"]) @ W["embed"].double().T
    return torch.log_softmax(logits, -1).gather(1, tokens[:, None]).sum().item()


@pytest.fixture(scope="module")
def setup(cuda):
    import beam_decode as B
    gen = torch.Generator(device="cuda").manual_seed(3)
    features = torch.randn(3, 150, 384, generator=gen, device="cuda")
    return B, B.decoder_weights(n_text=40), features


@pytest.mark.parametrize("beams,steps,page", [(1, 12, 16), (5, 30, 8), (4, 17, 16)])
def test_beam_search_scores_its_hypotheses(setup, beams, steps, page):
    B, W, features = setup
    decoder = B.BeamDecoder(W, features, beams, page_size=page)
    tokens, total = B.beam_search(decoder, 1, steps)
    assert tokens.shape == (3, beams, steps) and total.isfinite().all()
    assert (total[:, :-1] >= total[:, 1:]).all()
    assert decoder.cache.lens.tolist() == [steps] * (3 * beams)
    for c in range(3):
        rows = [tuple(r) for r in tokens[c].tolist()]
        assert len(set(rows)) == beams
        for b in range(beams):
            want = plain_score(W, features[c], tokens[c, b], 1)
            assert abs(total[c, b].item() - want) < 0.1 * steps, (c, b, total[c, b].item(), want)


def test_beam_search_does_not_depend_on_where_pages_lie(setup):
    """The same search with the pool made dense half way: the same bits."""
    B, W, features = setup
    a = B.beam_search(B.BeamDecoder(W, features, 5, page_size=4), 1, 24)
    b = B.beam_search(B.BeamDecoder(W, features, 5, page_size=4), 1, 24, compact_at=11)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_cache_refuses_bad_sizes(cuda):
    from wxb200.kvcache import PagedKVCache
    with pytest.raises(ValueError):
        PagedKVCache(1, 0, 16, 2, 64, 1, 10)
    cache = PagedKVCache(2, 5, 16, 2, 64, 2, 40, dtype=torch.float32)
    cache.step(grow=torch.tensor([17, 33], dtype=torch.int32, device="cuda"))
    assert cache.lens.tolist() == [17, 33] and cache.status.tolist() == [0, 0]
    cache.step(parents=torch.tensor([-1, 1], dtype=torch.int32, device="cuda"))
    assert cache.lens.tolist() == [0, 33] and cache.status.tolist() == [2, 0]
