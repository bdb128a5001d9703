"""The decoder operators where their device arrays contradict one another or a call
meets a rare path: what is written, what is left out and what is reported."""
import math

import pytest
import torch

import decoder_ref as R
from test_decoder_ops_gpu import check_fork, dev, make_cache, make_pool, randn
from wxb200 import _lib as L
from wxb200 import ops
from wxb200.kvcache import PagedKVCache

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float32]
INT_MIN, INT_MAX = -2 ** 31, 2 ** 31 - 1


@pytest.fixture(autouse=True)
def no_device_error(cuda):
    L.device_error()
    yield
    assert L.device_error() == 0


# ------------------------------------------------------------------ append


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["token", "head", "padded"])
@pytest.mark.parametrize("count", [4, 5, 9, 10, 12, INT_MAX, -1, INT_MIN])
def test_append_counts_out_of_range(cuda, dtype, layout, count):
    """Three rows where ten positions end at len 10 and `count` are announced: row t at
    10 - count + t where that is one, a neighbour written as ever, and a report."""
    page, tokens, lens = 4, 3, [10, 7]
    k, v, table, n, gen = make_cache(lens, page, 2, 64, dtype, seed=1, layout=layout, spoil=False)
    new = randn(gen, 2, tokens, 2, 64, dtype=dtype)
    ek, ev = k.clone(), v.clone()
    for i, c in enumerate((count, tokens)):
        for t in range(min(c, tokens)):
            pos = lens[i] - c + t
            if pos >= 0:
                at = table[i, pos // page].long()
                ek[at, pos % page], ev[at, pos % page] = new[i, t], -new[i, t]
    ops.kv_append(new, -new, k, v, table, n, counts=dev([count, tokens]))
    assert L.device_error() == L.WX_DEVERR_PAGE
    assert torch.equal(k, ek) and torch.equal(v, ev)


@pytest.mark.parametrize("length", [INT_MIN, -1, 0, 2])
def test_append_lengths_before_the_first_row(cuda, length):
    """Positions below 0 are left out whatever length and count they come from."""
    k, v, table, n, gen = make_cache([8], 4, 2, 64, torch.bfloat16, seed=2, spoil=False)
    ek, ev = k.clone(), v.clone()
    new = randn(gen, 1, 3, 2, 64, dtype=torch.bfloat16)
    if length == 2:                     # rows 1 and 2 have a position, row 0 none
        at = table[0, 0].long()
        ek[at, :2], ev[at, :2] = new[0, 1:], -new[0, 1:]
    ops.kv_append(new, -new, k, v, table, dev([length]), counts=dev([3]))
    assert L.device_error() == L.WX_DEVERR_PAGE
    assert torch.equal(k, ek) and torch.equal(v, ev)


def test_cache_append_of_fewer_rows_than_granted(cuda):
    """One row after a step of three: it is the first of the three, and reported."""
    cache = PagedKVCache(1, 6, 4, 2, 64, 2, 12)
    gen = torch.Generator(device="cuda").manual_seed(3)
    prompt = randn(gen, 2, 2, 2, 64, dtype=torch.bfloat16)
    cache.step(grow=dev([2, 2]))
    cache.append(0, prompt, -prompt)
    cache.step(grow=dev([3, 1]))
    cache.k.zero_()
    row = randn(gen, 2, 2, 64, dtype=torch.bfloat16)
    cache.append(0, row, -row)
    assert L.device_error() == L.WX_DEVERR_PAGE
    want = torch.zeros_like(cache.k)
    for i in range(2):
        want[0, cache.table[i, 0].long(), 2] = row[i]     # position 2 of either
    assert torch.equal(cache.k, want)


# ------------------------------------------------------------------ scores


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("rows,vocab", [(2, 1500), (4, 9001), (300, 1003), (3, 50001)])
def test_scores_nan_at_the_first_token(cuda, dtype, offset, rows, vocab):
    """Token 0 is NaN in a row where more logits tie than a list holds: NaN stands
    above all, and among NaNs the lowest token comes first."""
    wide = torch.full((rows, vocab + 8), -math.inf, dtype=dtype, device="cuda")
    x = wide[:, offset:offset + vocab]
    x[:, 0] = math.nan                          # the others masked
    x[1] = math.nan                             # no number at all
    none = torch.full((rows,), -1, device="cuda")
    lp, entropy, top, index = ops.token_logprobs(x, none, top_k=8)
    assert index.tolist() == [list(range(8))] * rows
    assert top.isnan().all() and entropy.isnan().all() and (lp == 0).all()
    x[0, 0], x[0, 7] = -math.inf, math.nan      # and one that is not the first
    index = ops.token_logprobs(x, none, top_k=8)[3]
    assert index[0].tolist() == [7, 0, 1, 2, 3, 4, 5, 6]


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_at_the_least_temperature(cuda, dtype):
    """As temperature goes to 0 the largest logit takes all."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    x = randn(gen, 3, 5003, dtype=dtype)
    tokens = x.argmax(1)
    x[torch.arange(3, device="cuda"), tokens] = 8.0     # alone at the top
    for t in (4.5e-39, 1e-38, 1e-30):
        lp, entropy, top, index = ops.token_logprobs(x, tokens, top_k=2, temperature=t)
        assert (lp == 0).all() and (entropy == 0).all()
        assert (top[:, 0] == 0).all() and torch.equal(index[:, 0].long(), tokens)
        assert (top[:, 1] < -1e28).all()


# ------------------------------------------------------------------ compact


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_pages", [12, 20000])
def test_compact_entries_that_the_counts_call_free(cuda, dtype, n_pages):
    """An entry whose page nobody counts has no tokens: it is left out and reported,
    wherever the page lies, and does not end up naming another sequence's page."""
    gen = torch.Generator(device="cuda").manual_seed(n_pages)
    k = make_pool(gen, n_pages, 4, 2, 64, dtype, layers=2)
    v = make_pool(gen, n_pages, 4, 2, 64, dtype, layers=2)
    last = n_pages - 1
    # used: 0, 2, last - 1, last; free below their number: 1 and 3
    good = [[2, last], [0, last - 1]]
    refs = [0] * n_pages
    for p in (0, 2, last - 1, last):
        refs[p] = 1
    for bad, count in ((1, 0), (3, 0), (last - 2, 0), (3, -1), (5, -7), (n_pages, 0)):
        table = [good[0] + [-1], good[1] + [bad]]
        r = list(refs)
        if bad < n_pages:
            r[bad] = count
        pools = k.clone(), v.clone()
        got = ops.kv_compact(*pools, dev(table), dev(r))
        assert L.device_error() == L.WX_DEVERR_PAGE
        assert got[0].tolist() == [[2, 3, -1], [0, 1, -1]]
        assert got[1].tolist() == [1] * 4 + [0] * (n_pages - 4) and got[2].tolist() == [4, 2]
        for new, old in zip(pools, (k, v)):
            assert torch.equal(new[:, 3], old[:, last]) and torch.equal(new[:, 1], old[:, last - 1])
            assert torch.equal(new[:, [0, 2]], old[:, [0, 2]])


# ------------------------------------------------------------------ copies of large pages


@pytest.mark.parametrize("layout", ["token", "head", "padded"])
@pytest.mark.parametrize("dtype,page,heads,hd", [(torch.bfloat16, 16, 20, 64),
                                                 (torch.float32, 33, 5, 128)])
def test_fork_copies_large_pages(cuda, dtype, layout, page, heads, hd):
    """Pages of 2560 and 5280 vectors, which go in two and three parts, the last one not
    full: copies that end in the first part, on either side of its end and in a later
    one, more parts in all than there are CTAs."""
    clips, beams, layers = 12, 6, 4
    gen = torch.Generator(device="cuda").manual_seed(page)
    filled = [m for m in (1, 12, 13, 15, 25, 26, 32) if m < page]
    lens = [page + filled[c % len(filled)] for c in range(clips) for _ in range(beams)]
    n_pages = 2 * clips + clips * beams
    table = [[2 * c + 1, 2 * c, -1] for c in range(clips) for _ in range(beams)]
    refs = [beams] * (2 * clips) + [0] * (clips * beams)
    k = make_pool(gen, n_pages, page, heads, hd, dtype, layout, layers=layers)
    v = make_pool(gen, n_pages, page, heads, hd, dtype, layout, layers=layers)
    parents = [c * beams + (7 * b) % beams for c in range(clips) for b in range(beams)]
    t, n, r, grown = check_fork(k, v, table, lens, refs, parents, [1] * (clips * beams), page)
    assert sum(x > 0 for x in r) == clips + clips * beams and min(grown) == 1


@pytest.mark.parametrize("layout", ["token", "head", "padded"])
@pytest.mark.parametrize("dtype,page,heads,hd", [(torch.bfloat16, 16, 20, 64),
                                                 (torch.float32, 33, 5, 128)])
def test_compact_moves_large_pages(cuda, dtype, layout, page, heads, hd):
    """As above, whole pages."""
    layers, n_pages, n_used = 4, 150, 70
    gen = torch.Generator(device="cuda").manual_seed(page)
    k = make_pool(gen, n_pages, page, heads, hd, dtype, layout, layers=layers)
    v = make_pool(gen, n_pages, page, heads, hd, dtype, layout, layers=layers)
    used = torch.randperm(n_pages, generator=torch.Generator().manual_seed(page))[:n_used]
    table = used.view(7, 10).tolist()
    refs = [0] * n_pages
    for p in used.tolist():
        refs[p] = 1
    t, r, st, moves = R.compact_ref(table, refs)
    src, dst = (torch.tensor(x, device="cuda") for x in zip(*moves))
    ek, ev = k.clone(), v.clone()
    ek[:, dst], ev[:, dst] = k[:, src], v[:, src]
    got = ops.kv_compact(k, v, dev(table), dev(refs))
    assert got[0].tolist() == t and got[1].tolist() == r and got[2].tolist() == st
    assert torch.equal(k, ek) and torch.equal(v, ev)


# ------------------------------------------------------------------ rows that share memory


def test_outputs_that_share_memory_are_refused(cuda):
    """Read, such a cache is one key-value head for several; written, or as a result, it
    is refused."""
    k, v, table, n, gen = make_cache([9, 30], 8, 1, 64, torch.bfloat16, seed=1, spoil=False)
    q = randn(gen, 2, 4, 64, dtype=torch.bfloat16)
    row = torch.empty(2, 1, 64, dtype=torch.bfloat16, device="cuda")
    for out in (row.expand(2, 4, 64), row.transpose(0, 1).repeat(1, 2, 1).expand(2, 4, 64)):
        with pytest.raises(ValueError, match="share memory"):
            ops.paged_attention(q, k, v, table, n, out=out)
    k2, v2 = k.expand(-1, -1, 2, 64), v.expand(-1, -1, 2, 64)
    assert torch.equal(ops.paged_attention(q, k2, v2, table, n),
                       ops.paged_attention(q, k2.contiguous(), v2.contiguous(), table, n))
    refs = torch.zeros(k.shape[0], dtype=torch.int32, device="cuda")
    for call in (lambda: ops.kv_append(q[:, :2], q[:, 2:], k2, v2, table, n),
                 lambda: ops.kv_fork(k2[None], v2[None], table, n, refs, grow=n),
                 lambda: ops.kv_compact(k2[None], v2[None], table, refs),
                 lambda: ops.kv_compact(k.expand(2, -1, -1, 1, 64), v.expand(2, -1, -1, 1, 64),
                                        table, refs)):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------ arguments


def test_return_lse_without_a_truth_value(cuda):
    """The caller's own error, and nothing launched."""
    k, v, table, n, gen = make_cache([9], 8, 2, 64, torch.bfloat16, seed=1)
    q = randn(gen, 1, 2, 64, dtype=torch.bfloat16)
    out = torch.full_like(q, 5.0)
    with pytest.raises(RuntimeError, match="ambiguous"):
        ops.paged_attention(q, k, v, table, n, out=out, return_lse=torch.zeros(2))
    assert (out == 5).all()


# ------------------------------------------------------------------ a captured step


def test_cache_step_replayed_from_a_graph(cuda):
    """A step captured with its new tables copied back is the same step, replay after
    replay, as one that is called."""
    page, beams, steps = 4, 3, 9
    gen = torch.Generator(device="cuda").manual_seed(4)
    rows = randn(gen, steps + 1, beams, 2, 64, dtype=torch.bfloat16)
    order = [dev([(b * (t + 1)) % beams for b in range(beams)]) for t in range(steps)]
    parents, grow, row = dev([0, 1, 2]), dev([1] * beams), rows[0].clone()

    def begin():
        cache = PagedKVCache(1, 20, page, 2, 64, beams, 12)
        cache.step(grow=grow)
        cache.append(0, rows[0], -rows[0])
        return cache

    def step(cache):
        cache.step(parents, grow)
        cache.append(0, row, -row)
        return cache.attend(0, row)

    plain, want = begin(), []
    for t in range(steps):
        parents.copy_(order[t])
        row.copy_(rows[t + 1])
        want.append((step(plain).clone(), plain.table.clone(), plain.lens.clone()))
    cache = begin()
    held = cache.table, cache.lens, cache.refs
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache)
        for old, new in zip(held, (cache.table, cache.lens, cache.refs)):
            old.copy_(new)
    cache.table, cache.lens, cache.refs = held
    for t in range(steps):
        parents.copy_(order[t])
        row.copy_(rows[t + 1])
        graph.replay()
        assert torch.equal(out, want[t][0])
        assert torch.equal(cache.table, want[t][1]) and torch.equal(cache.lens, want[t][2])
        assert cache.grown.tolist() == [1] * beams
