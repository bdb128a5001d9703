"""The decoder operators on the GPU against plain restatements (decoder_ref):
attention over the paged cache and token scores against their definitions in 64
bits, within bounds derived from the arithmetic; the cache's page plans and
copies exactly."""
import math
import random

import pytest
import torch

import decoder_ref as R
from wxb200 import _lib as L
from wxb200 import ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float32]


@pytest.fixture(autouse=True)
def no_device_error(cuda):
    yield
    assert L.device_error() == 0


def randn(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def make_pool(gen, n_pages, page, heads, hd, dtype, layout="token", layers=None):
    lead = () if layers is None else (layers,)
    if layout == "token":
        return randn(gen, *lead, n_pages, page, heads, hd, dtype=dtype)
    if layout == "head":
        return randn(gen, *lead, n_pages, heads, page, hd, dtype=dtype).transpose(-3, -2)
    # rows padded: neither tokens nor heads side by side
    return randn(gen, *lead, n_pages, page, heads, hd + 16, dtype=dtype)[..., :hd]


def make_cache(lens, page, heads, hd, dtype, seed=0, layout="token", width=None, spoil=True):
    """A cache that holds `lens` tokens on pages in random order. spoil: every slot
    that no sequence holds is NaN."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n = [-(-x // page) for x in lens]
    total = sum(n)
    width = width or max(1, max(n))
    ids = torch.randperm(total + 2, generator=torch.Generator().manual_seed(seed))
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for i, m in enumerate(n):
        table[i, :m] = ids[at:at + m]
        at += m
    k = make_pool(gen, total + 2, page, heads, hd, dtype, layout)
    v = make_pool(gen, total + 2, page, heads, hd, dtype, layout)
    if spoil:
        held = torch.zeros(total + 2, page, dtype=torch.bool)
        for i, x in enumerate(lens):
            for s in range(n[i]):
                held[table[i, s], :min(page, x - s * page)] = True
        k[~held.cuda()] = math.nan
        v[~held.cuda()] = math.nan
    return k, v, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), gen


def check_attend(q, k, v, table, lens, starts=None, scale=None, **kw):
    hd = q.shape[-1]
    q4 = q if q.dim() == 4 else q.unflatten(1, (k.shape[2], -1))
    got, lse = ops.paged_attention(q, k, v, table, lens, starts=starts, scale=scale,
                                   return_lse=True, **kw)
    assert got.shape == q.shape and got.dtype == q.dtype and lse.shape == q.shape[:-1]
    o, l, o_tol, l_tol = R.attend64(q4, k, v, table, lens, hd ** -0.5 if scale is None else scale,
                                    starts)
    o, l, o_tol, l_tol = (t.reshape(s) for t, s in ((o, q.shape), (l, q.shape[:-1]),
                                                   (o_tol, q.shape), (l_tol, q.shape[:-1])))
    empty = l == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert (got[empty] == 0).all()
    over = ((got.double() - o).abs() - o_tol)[~empty]
    assert over.numel() == 0 or over.max() <= 0, over.max()
    over = ((lse.double() - l).abs() - l_tol)[~empty]
    assert over.numel() == 0 or over.max() <= 0, over.max()
    return got, lse


# ------------------------------------------------------------------ attention


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group", [1, 2, 3, 5, 8, 9, 16, 21])
def test_attend_groups(cuda, dtype, hd, group):
    lens = [0, 1, 2, 15, 16, 17, 63, 129, 200]
    k, v, table, n, gen = make_cache(lens, 16, 3, hd, dtype, seed=group)
    check_attend(randn(gen, len(lens), 3 * group, hd, dtype=dtype), k, v, table, n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [1, 3, 8, 16, 20, 64, 100, 256])
@pytest.mark.parametrize("layout", ["token", "head", "padded"])
def test_attend_pages_and_layouts(cuda, dtype, page, layout):
    lens = [page, page + 1, 3 * page - 1, 333, 1]
    k, v, table, n, gen = make_cache(lens, page, 2, 64, dtype, seed=page, layout=layout)
    check_attend(randn(gen, len(lens), 8, 64, dtype=dtype), k, v, table, n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens", [[5000], [1, 4097, 0, 2048], [1023, 1024, 1025], [20011, 3]])
@pytest.mark.parametrize("hd,group", [(64, 1), (128, 4)])
def test_attend_long(cuda, dtype, lens, hd, group):
    """The cache's length split over CTAs and joined."""
    k, v, table, n, gen = make_cache(lens, 32, 2, hd, dtype, seed=len(lens))
    check_attend(randn(gen, len(lens), 2 * group, hd, dtype=dtype), k, v, table, n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("seqs,width", [(130, 2048), (128, 300), (3, 5000)])
def test_attend_long_tables(cuda, dtype, seqs, width):
    """Tables that could hold far more than they do: the split goes by the keys there
    are, and by the bound alone where sequences are many."""
    lens = [9000, 0, 4100] + [(7 * i) % 90 for i in range(seqs - 3)]
    k, v, table, n, gen = make_cache(lens, 64, 2, 64, dtype, seed=seqs, width=width)
    check_attend(randn(gen, seqs, 6, 64, dtype=dtype), k, v, table, n)
    check_attend(randn(gen, seqs, 6, 64, dtype=dtype), k, v, table, n, max_len=9000)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,group", [(10, 3), (7, 11), (9, 1)])
def test_attend_many_short_sequences(cuda, dtype, heads, group):
    """Enough short items that each has a warp, in either type."""
    lens = [(37 * i) % 120 for i in range(301)]
    k, v, table, n, gen = make_cache(lens, 16, heads, 64, dtype, seed=heads)
    check_attend(randn(gen, 301, heads * group, 64, dtype=dtype), k, v, table, n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group", [1, 2, 3, 8, 13])
def test_attend_many_tiny_sequences(cuda, dtype, hd, group):
    """A warp for each item of at most 16 keys; q and out where no vector fits."""
    lens = [i % 17 for i in range(301)]
    k, v, table, n, gen = make_cache(lens, 16, 4, hd, dtype, seed=group)
    wide = randn(gen, 301, 4 * group * hd + 3, dtype=dtype)
    q = wide[:, 1:-2].unflatten(1, (4 * group, hd))
    out = torch.empty_like(wide)[:, 1:-2].unflatten(1, (4 * group, hd))
    got, _ = check_attend(q, k, v, table, n, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert torch.equal(ops.paged_attention(q.contiguous(), k, v, table, n), got)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_window(cuda, dtype):
    lens = [40, 40, 40, 40, 700, 700, 0, 2500]
    starts = torch.tensor([0, 7, 39, 40, 16, 699, 3, 2100], dtype=torch.int32, device="cuda")
    k, v, table, n, gen = make_cache(lens, 16, 2, 64, dtype, seed=3)
    q = randn(gen, len(lens), 4, 64, dtype=dtype)
    got, lse = check_attend(q, k, v, table, n, starts=starts)
    assert (lse[3] == -math.inf).all() and (got[6] == 0).all()
    # what lies outside the window does not matter, NaN neither
    for i in range(len(lens)):
        for p in range(min(lens[i], int(starts[i]))):
            k[table[i, p // 16].long(), p % 16] = math.nan
            v[table[i, p // 16].long(), p % 16] = math.inf
    again = ops.paged_attention(q, k, v, table, n, starts=starts)
    assert torch.equal(again, got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("beams", [1, 5, 7])
def test_attend_beams_share_a_clip(cuda, dtype, beams):
    """Beams over one clip's keys as one group, q and out as strided views."""
    clips, heads, hd = 3, 4, 64
    k, v, table, n, gen = make_cache([100, 37, 64], 16, heads, hd, dtype, seed=beams)
    x = randn(gen, clips * beams, heads * hd, dtype=dtype)
    q = x.view(clips, beams, heads, hd).transpose(1, 2)
    got, _ = check_attend(q, k, v, table, n)
    assert got.stride() == q.stride()
    for b in range(beams):
        one = ops.paged_attention(x.view(clips, beams, heads, hd)[:, b], k, v, table, n)
        if dtype == torch.float32:
            assert (one - got[:, :, b]).abs().max() < 1e-5
        else:
            assert (one.float() - got[:, :, b].float()).abs().max() < 0.05


@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_strides_and_out(cuda, dtype):
    """q a column slice at an odd offset, out a slice of a wider buffer."""
    lens = [33, 70]
    k, v, table, n, gen = make_cache(lens, 16, 2, 64, dtype, seed=9)
    wide = randn(gen, 2, 3 + 4 * 64 + 5, dtype=dtype)
    q = wide[:, 3:3 + 256].unflatten(1, (4, 64))
    dest = torch.full((2, 9 + 256 + 7), 5.0, dtype=dtype, device="cuda")
    out = dest[:, 9:9 + 256].unflatten(1, (4, 64))
    assert ops.paged_attention(q, k, v, table, n, out=out) is out
    plain = ops.paged_attention(q.contiguous(), k, v, table, n)
    assert torch.equal(out, plain)
    assert (dest[:, :9] == 5).all() and (dest[:, 265:] == 5).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [50, 3000])
def test_attend_large_scores_and_scales(cuda, dtype, n):
    k, v, table, lens, gen = make_cache([n], 16, 1, 64, dtype, seed=4)
    q = randn(gen, 1, 4, 64, dtype=dtype)
    check_attend(q * 30, k, v, table, lens)
    check_attend(q, k, v, table, lens, scale=0.0)
    check_attend(q, k, v, table, lens, scale=-2.0)
    check_attend(q, k, v, table, lens, max_len=table.shape[1] * 16)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [40, 2000])
def test_attend_infinite_scores(cuda, dtype, n):
    """Scores of -inf weigh nothing (all of them: an empty row); +inf and NaN among
    the keys attended to give NaN."""
    k, v, table, lens, gen = make_cache([n, n, n, n], 16, 1, 64, dtype, seed=5)
    q = torch.ones(4, 1, 64, dtype=dtype, device="cuda")
    at = lambda i, p: (table[i, p // 16].long(), p % 16)  # noqa: E731
    k[at(0, 7)] = -math.inf                       # one key masked by its score
    for p in range(n):
        k[at(1, p)] = -math.inf                   # all keys
    k[at(2, 3)] = math.inf
    k[at(3, 5)] = math.nan
    got, lse = ops.paged_attention(q, k, v, table, lens, return_lse=True)
    keep = [p for p in range(n) if p != 7]
    rows = torch.stack([k[at(0, p)] for p in keep])[:, 0].double()
    vals = torch.stack([v[at(0, p)] for p in keep])[:, 0].double()
    p = torch.softmax(rows.sum(1) / 8, 0)
    assert (got[0, 0].double() - p @ vals).abs().max() < (1e-4 if dtype == torch.float32 else 0.02)
    assert (got[1] == 0).all() and (lse[1] == -math.inf).all()
    assert got[2].isnan().all() and got[3].isnan().all()
    assert lse[2:].isnan().all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group", [5, 8, 9, 16])
@pytest.mark.parametrize("lens", [[1, 0, 17, 777, 4096], [6000, 0, 300]])
def test_attend_fp32_many_rows(cuda, hd, group, lens):
    """Groups that the tensor cores take in fp32, over a cluster and in chunks, with a
    window that begins inside a tile."""
    k, v, table, n, gen = make_cache(lens, 16, 2, hd, torch.float32, seed=hd + group)
    q = randn(gen, len(lens), 2 * group, hd)
    check_attend(q, k, v, table, n)
    starts = torch.tensor([x // 3 for x in lens], dtype=torch.int32, device="cuda")
    check_attend(q, k, v, table, n, starts=starts)


@pytest.mark.parametrize("group", [2, 5, 16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("ks,qs", [(1e37, 1e-36), (1e-37, 1e37), (1e-30, 1e30), (1.0, 1e-38)])
def test_attend_fp32_extremes(cuda, hd, group, ks, qs):
    """Numbers near the ends of fp32's range, whose products are ordinary."""
    k, v, table, n, gen = make_cache([300, 33], 16, 2, hd, torch.float32, seed=group, spoil=False)
    k *= ks
    check_attend(randn(gen, 2, 2 * group, hd) * qs, k, v, table, n)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group", [1, 4, 5, 16])
@pytest.mark.parametrize("n", [40, 2000])
def test_attend_fp32_infinite_values(cuda, hd, group, n):
    """An infinite or NaN number of V shows in its dimension alone."""
    k, v, table, lens, gen = make_cache([n], 16, 2, hd, torch.float32, seed=group)
    q = randn(gen, 1, 2 * group, hd)
    want = ops.paged_attention(q, k, v, table, lens).unflatten(1, (2, group))
    at = table[0, (n - 5) // 16].long(), (n - 5) % 16
    v[at][0, 3] = math.inf
    v[at][1, 7] = -math.inf
    v[at][1, 62] = math.nan
    got = ops.paged_attention(q, k, v, table, lens).unflatten(1, (2, group))
    assert (got[:, 0, :, 3] == math.inf).all() and (got[:, 1, :, 7] == -math.inf).all()
    assert got[:, 1, :, 62].isnan().all()
    for h, d in ((0, [3]), (1, [7, 62])):
        keep = [x for x in range(hd) if x not in d]
        torch.testing.assert_close(got[:, h][..., keep], want[:, h][..., keep], rtol=0, atol=1e-5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_same_result_each_time_and_anywhere_in_a_batch(cuda, dtype):
    lens = [4000, 17, 900, 4000]
    k, v, table, n, gen = make_cache(lens, 16, 2, 128, dtype, seed=6)
    q = randn(gen, 4, 8, 128, dtype=dtype)
    a, la = ops.paged_attention(q, k, v, table, n, return_lse=True)
    for _ in range(3):
        b, lb = ops.paged_attention(q, k, v, table, n, return_lse=True)
        assert torch.equal(a, b) and torch.equal(la, lb)
    flip = torch.arange(3, -1, -1, device="cuda")
    c = ops.paged_attention(q[flip].contiguous(), k, v, table[flip].contiguous(),
                            n[flip].contiguous())
    assert torch.equal(c[flip], a)


def test_attend_offsets_past_32_bits(cuda):
    """A pool of more than 2^31 elements: pages at its far end."""
    page, heads, hd = 16, 8, 128
    n_pages = 2 ** 31 // (page * heads * hd) + 64
    k = torch.zeros(n_pages, page, heads, hd, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for t in (k, v):
        t[-8:] = randn(gen, 8, page, heads, hd, dtype=torch.bfloat16)
    table = torch.arange(n_pages - 8, n_pages, dtype=torch.int32, device="cuda")[None]
    n = torch.tensor([8 * page - 3], dtype=torch.int32, device="cuda")
    check_attend(randn(gen, 1, heads, hd, dtype=torch.bfloat16), k, v, table, n)
    new = randn(gen, 1, heads, hd, dtype=torch.bfloat16)
    n += 1
    ops.kv_append(new, -new, k, v, table, n)
    assert torch.equal(k[-1, page - 3], new[0]) and torch.equal(v[-1, page - 3], -new[0])
    assert k[:n_pages - 8].any().item() is False


def test_attend_on_a_side_stream_and_in_a_graph(cuda):
    lens = [3000, 5]
    k, v, table, n, gen = make_cache(lens, 16, 2, 64, torch.bfloat16, seed=8)
    q = randn(gen, 2, 4, 64, dtype=torch.bfloat16)
    want = ops.paged_attention(q, k, v, table, n)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = ops.paged_attention(q, k, v, table, n)
    s.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    out = torch.empty_like(q)
    with torch.cuda.graph(g, stream=s):
        ops.paged_attention(q, k, v, table, n, out=out)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    q.copy_(randn(gen, 2, 4, 64, dtype=torch.bfloat16))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ops.paged_attention(q, k, v, table, n))


def test_attend_bad_pages_are_left_out_and_reported(cuda):
    k, v, table, n, gen = make_cache([40, 40], 16, 1, 64, torch.bfloat16, seed=2, spoil=False)
    q = randn(gen, 2, 1, 64, dtype=torch.bfloat16)
    good = ops.paged_attention(q, k, v, table, n)
    bad = table.clone()
    bad[0, 1] = k.shape[0]          # past the pool
    got = ops.paged_attention(q, k, v, bad, n)
    assert L.device_error() == L.WX_DEVERR_PAGE
    assert torch.equal(got[1], good[1]) and got[0].isfinite().all()
    two = torch.tensor([24, 40], dtype=torch.int32, device="cuda")
    only = table.clone()
    only[0, 1] = table[0, 2]        # tokens 0..15 and 32..39 as 24 in a row
    want = ops.paged_attention(q, k, v, only, two)
    assert (got[0].float() - want[0].float()).abs().max() < 0.05
    n[0] = 100                      # longer than the table
    ops.paged_attention(q, k, v, table, n)
    assert L.device_error() == L.WX_DEVERR_PAGE


# ------------------------------------------------------------------ append


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["token", "head", "padded"])
@pytest.mark.parametrize("tokens,page", [(1, 16), (5, 3), (40, 16), (7, 64)])
def test_append(cuda, dtype, layout, tokens, page):
    lens = [tokens, tokens + 1, tokens + 30, 2 * tokens, 200]
    counts = torch.tensor([tokens, 0, max(0, tokens - 1), 1, tokens], dtype=torch.int32,
                          device="cuda")
    k, v, table, n, gen = make_cache(lens, page, 3, 64, dtype, seed=page, layout=layout,
                                     spoil=False)
    kn, vn = (randn(gen, 5, tokens, 3, 64, dtype=dtype) for _ in range(2))
    for c in (None, counts):
        ek, ev = k.clone(), v.clone()
        for i, x in enumerate(lens):
            m = tokens if c is None else int(c[i])
            for t in range(m):
                pos = x - m + t
                at = table[i, pos // page].long()
                ek[at, pos % page], ev[at, pos % page] = kn[i, t], vn[i, t]
        ops.kv_append(kn, vn, k, v, table, n, counts=c)
        assert torch.equal(k, ek) and torch.equal(v, ev)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0, 1, 8])
def test_append_from_a_qkv_buffer(cuda, dtype, offset):
    """Column slices of one QKV buffer, aligned and not."""
    k, v, table, n, gen = make_cache([9, 30], 8, 2, 64, dtype, seed=1, spoil=False)
    qkv = randn(gen, 2, 3 * 128 + 16, dtype=dtype)
    kn = qkv[:, offset + 128:offset + 256].unflatten(1, (2, 64))
    vn = qkv[:, offset + 256:offset + 384].unflatten(1, (2, 64))
    ops.kv_append(kn, vn, k, v, table, n)
    for i, pos in enumerate([8, 29]):
        at = table[i, pos // 8].long()
        assert torch.equal(k[at, pos % 8], kn[i]) and torch.equal(v[at, pos % 8], vn[i])


def test_append_bad_positions_are_left_out_and_reported(cuda):
    k, v, table, n, gen = make_cache([9, 30], 8, 2, 64, torch.float32, seed=1, spoil=False)
    before = k.clone()
    new = randn(gen, 2, 2, 64)
    n[0] = 0                        # no room before the first position
    n[1] = 33                       # on a page that the table does not name
    ops.kv_append(new, new, k, v, table, n)
    assert L.device_error() == L.WX_DEVERR_PAGE
    assert torch.equal(k, before)


# ------------------------------------------------------------------ fork, compact


def dev(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def check_fork(k, v, table, lens, refs, parents, grow, page):
    """One fork against fork_ref, pools included. Returns the new lists."""
    t, n, r, g, st, copies = R.fork_ref(table, lens, refs, parents, grow, page)
    ek, ev = k.clone(), v.clone()
    for s, d, m in copies:
        ek[:, d, :m], ev[:, d, :m] = k[:, s, :m], v[:, s, :m]
    got = ops.kv_fork(k, v, dev(table), dev(lens), dev(refs),
                      parents=None if parents is None else dev(parents),
                      grow=None if grow is None else dev(grow))
    for name, x, y in zip(("table", "lens", "refs", "grown", "status"), got, (t, n, r, g, st)):
        assert x.tolist() == y, name
    assert torch.equal(k, ek) and torch.equal(v, ev)
    return t, n, r, g


@pytest.mark.parametrize("dtype,layout", [(torch.bfloat16, "token"), (torch.float32, "head"),
                                          (torch.bfloat16, "padded")])
@pytest.mark.parametrize("page,seqs,seed", [(1, 3, 0), (4, 7, 1), (16, 5, 2), (5, 40, 3)])
def test_fork_append_attend_over_many_steps(cuda, dtype, layout, page, seqs, seed):
    """A random run of forks, ends, starts and growth: every plan equals the
    restatement's, and each sequence's cache always holds the tokens that its
    history appended."""
    rng = random.Random(seed)
    width = 60 // page + 1
    n_pages = seqs * width // 3 + 2          # short at times
    gen = torch.Generator(device="cuda").manual_seed(seed)
    k = make_pool(gen, n_pages, page, 2, 64, dtype, layout, layers=2)
    v = make_pool(gen, n_pages, page, 2, 64, dtype, layout, layers=2)
    table, lens, refs = [[-1] * width for _ in range(seqs)], [0] * seqs, [0] * n_pages
    history = [[] for _ in range(seqs)]      # (step, row, token) of each position
    written = {}
    for step in range(25):
        parents = [rng.choice([-1] + [i] * 6 + list(range(seqs))) for i in range(seqs)]
        grow = [rng.choice([0, 1, 1, 1, 2, 9]) for _ in range(seqs)]
        if step % 6 == 5:
            parents = None
        if step % 7 == 6:
            grow = None
        table, lens, refs, grown = check_fork(k, v, table, lens, refs, parents, grow, page)
        tokens = max(1, max(grown))
        new = randn(gen, 2, seqs, tokens, 2, 64, dtype=dtype)
        for layer in range(2):
            ops.kv_append(new[layer], -new[layer], k[layer], v[layer], dev(table), dev(lens),
                          counts=dev(grown))
        par = list(range(seqs)) if parents is None else parents
        history = [list(history[p]) if p >= 0 else [] for p in par]
        for i in range(seqs):
            for t in range(grown[i]):
                history[i].append((step, i, t))
                written[step, i, t] = new[:, i, t]
            assert len(history[i]) == lens[i]
            if lens[i]:
                want = torch.stack([written[h] for h in history[i]], 1)
                pos = torch.arange(lens[i], device="cuda")
                at = dev(table[i]).long()[pos // page]
                assert torch.equal(k[:, at, pos % page], want)
                assert torch.equal(v[:, at, pos % page], -want)


def test_fork_larger_table(cuda):
    """More sequences and pages than one pass of the planning threads."""
    rng = random.Random(5)
    seqs, width, page, n_pages = 300, 40, 4, 12000
    gen = torch.Generator(device="cuda").manual_seed(5)
    k = make_pool(gen, n_pages, page, 1, 64, torch.float32, layers=1)
    v = make_pool(gen, n_pages, page, 1, 64, torch.float32, layers=1)
    lens = [rng.randint(0, (width - 2) * page) for _ in range(seqs)]
    ids = list(range(n_pages))
    rng.shuffle(ids)
    table, refs = [], [0] * n_pages
    for n in lens:
        m = -(-n // page)
        row = [ids.pop() for _ in range(m)]
        for p in row:
            refs[p] = 1
        table.append(row + [-1] * (width - m))
    for step in range(3):
        parents = [rng.choice([i, i, rng.randint(0, seqs - 1), -1]) for i in range(seqs)]
        grow = [rng.choice([0, 1, 3]) for _ in range(seqs)]
        table, lens, refs, _ = check_fork(k, v, table, lens, refs, parents, grow, page)


def test_fork_all_beams_from_one(cuda):
    """Every beam goes on as the last: one keeps the page, the others copy it."""
    page, beams = 16, 5
    gen = torch.Generator(device="cuda").manual_seed(0)
    k = make_pool(gen, 12, page, 2, 64, torch.bfloat16, layers=3)
    v = make_pool(gen, 12, page, 2, 64, torch.bfloat16, layers=3)
    table, lens = [[7, i] + [-1] for i in range(beams)], [20] * beams
    refs = [1] * 5 + [0, 0, 5] + [0] * 4
    t, n, r, g = check_fork(k, v, table, lens, refs, [4] * beams, [1] * beams, page)
    assert t[0][:2] == [7, 4] and sorted(x[1] for x in t[1:]) == [0, 1, 2, 3]
    assert n == [21] * beams and g == [1] * beams


def test_fork_pool_and_table_too_small(cuda):
    page = 4
    gen = torch.Generator(device="cuda").manual_seed(0)
    k = make_pool(gen, 4, page, 1, 64, torch.float32, layers=1)
    v = make_pool(gen, 4, page, 1, 64, torch.float32, layers=1)
    table, lens = [[0, 1], [2, -1], [-1, -1], [-1, -1]], [8, 3, 0, 0]
    refs = [1, 1, 1, 0]
    # sequence 0 is at the table's width, 1 needs no page, 2 takes the last, 3 is short
    t, n, r, g = check_fork(k, v, table, lens, refs, None, [1, 1, 2, 2], page)
    assert g == [0, 1, 2, 0] and n == [8, 4, 2, 0]


@pytest.mark.parametrize("dtype,layout", [(torch.bfloat16, "token"), (torch.float32, "head"),
                                          (torch.bfloat16, "padded")])
@pytest.mark.parametrize("n_pages,share", [(5, 0.5), (64, 0.0), (64, 1.0), (700, 0.3),
                                           (20000, 0.6)])
def test_compact(cuda, dtype, layout, n_pages, share):
    rng = random.Random(n_pages)
    gen = torch.Generator(device="cuda").manual_seed(n_pages)
    page = 4 if n_pages > 1000 else 16
    k = make_pool(gen, n_pages, page, 2, 64, dtype, layout, layers=2)
    v = make_pool(gen, n_pages, page, 2, 64, dtype, layout, layers=2)
    used = rng.sample(range(n_pages), int(n_pages * share))
    seqs = 6
    table = [used[i::seqs] for i in range(seqs)]
    width = max(1, max(map(len, table)))
    if used:
        table[0] = [used[0]] + table[0][1:]
        table[1] = [used[0]] + table[1][1:] if table[1] else [used[0]]
    table = [r + [-1] * (width - len(r)) for r in table]
    refs = [0] * n_pages
    for r in table:
        for p in r:
            if p >= 0:
                refs[p] += 1
    t, r, st, moves = R.compact_ref(table, refs)
    ek, ev = k.clone(), v.clone()
    if moves:
        src, dst = (torch.tensor(x, device="cuda") for x in zip(*moves))
        ek[:, dst], ev[:, dst] = k[:, src], v[:, src]
    got = ops.kv_compact(k, v, dev(table), dev(refs))
    assert got[0].tolist() == t and got[1].tolist() == r and got[2].tolist() == st
    assert torch.equal(k, ek) and torch.equal(v, ev)


def test_plans_in_a_graph(cuda):
    """A captured step of forks replays on the buffers' current contents."""
    page, beams = 8, 4
    gen = torch.Generator(device="cuda").manual_seed(0)
    k = make_pool(gen, 20, page, 2, 64, torch.bfloat16, layers=2)
    v = make_pool(gen, 20, page, 2, 64, torch.bfloat16, layers=2)
    table = dev([[0, 1, -1], [0, 2, -1], [0, 3, -1], [0, 4, -1]])
    lens, refs = dev([11] * beams), dev([4, 1, 1, 1, 1] + [0] * 15)
    parents, grow = dev([0, 1, 2, 3]), dev([1] * beams)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.kv_fork(k, v, table, lens, refs, parents=parents, grow=grow)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = ops.kv_fork(k, v, table, lens, refs, parents=parents, grow=grow)
    for p in ([3, 3, 3, 3], [1, 0, -1, 2]):
        parents.copy_(dev(p))
        g.replay()
        torch.cuda.synchronize()
        want = R.fork_ref(table.tolist(), lens.tolist(), refs.tolist(), p, [1] * beams, page)
        assert [x.tolist() for x in out] == list(want[:5])


# ------------------------------------------------------------------ scores


def check_score(x, tokens, top_k, temperature):
    got = ops.token_logprobs(x, tokens, top_k=top_k, temperature=temperature)
    want = R.score64(x, tokens, top_k, temperature)
    for y, name, tol in zip(got, ("logprob", "entropy", "top_logprob"),
                            ("logprob_tol", "entropy_tol", "top_tol")):
        w = want[name]
        fine = w.isfinite()
        assert torch.equal(y[~fine].double(), w[~fine]), name
        over = (y.double() - w).abs()[fine] - want[tol][fine]
        assert over.numel() == 0 or over.max() <= 0, (name, over.max())
    assert torch.equal(got[3].long(), want["top_index"])
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 31), (5, 257), (1, 5000), (7, 50001),
                                        (2, 131072), (300, 1003), (700, 4099)])
@pytest.mark.parametrize("top_k", [0, 1, 10, 32])
def test_scores(cuda, dtype, rows, vocab, top_k):
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    x = (randn(gen, rows, vocab) * 4).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    check_score(x, tokens, min(top_k, vocab), 1.0)
    check_score(x, tokens, min(top_k, vocab), 0.3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_masked_tokens_and_no_token(cuda, dtype):
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = (randn(gen, 6, 3001) * 3).to(dtype)
    x[:, ::2] = -math.inf
    x[1, 2990:] = torch.finfo(dtype).min       # masked by the type's lowest value
    x[2, :-1] = -math.inf                      # one token left
    tokens = torch.tensor([1, 2, 3000, -1, 3001, 2999], device="cuda")
    x[2, -1] = 1.0
    got = check_score(x, tokens, 8, 1.0)
    assert got[0][2] == 0 and got[0][1] == -math.inf and got[0][3] == 0
    assert got[0][4] == -math.inf and got[1][2] == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [40, 9001])
def test_scores_rows_without_a_token_and_without_numbers(cuda, dtype, vocab):
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = randn(gen, 6, vocab).to(dtype)
    x[0] = -math.inf                           # every token masked
    x[1] = torch.finfo(dtype).min              # all at the type's lowest value: even
    x[2, 5] = math.nan
    x[3, 7] = math.inf
    x[4] = torch.finfo(dtype).max
    tokens = torch.full((6,), 5, device="cuda")
    lp, ent, top, index = ops.token_logprobs(x, tokens, top_k=4)
    assert lp[0] == -math.inf and ent[0] == 0 and (top[0] == -math.inf).all()
    assert index[0].tolist() == [0, 1, 2, 3]
    for r in (1, 4):
        # n equal terms: log n, within the sum's bound and the logarithm's last bits
        tol = (vocab / 256 + 64) * R.U32 + 2.0 ** -22 * (1 + math.log(vocab)) + 1e-7
        assert abs(lp[r].item() + math.log(vocab)) < tol and abs(ent[r].item()
                                                                 - math.log(vocab)) < tol
        assert index[r].tolist() == [0, 1, 2, 3]
    for r in (2, 3):
        assert lp[r].isnan() and ent[r].isnan() and top[r].isnan().any()
    assert index[2][0] == 5 and index[3][0] == 7
    one = slice(5, 6)
    assert torch.equal(lp[one], check_score(x[one], tokens[one], 4, 1.0)[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_ties_go_to_the_lowest_token(cuda, dtype):
    x = torch.zeros(3, 20011, dtype=dtype, device="cuda")
    x[1, 100::7] = 2.0
    x[2, 19000:] = -0.0
    x[2, 5] = -1.0
    tokens = torch.tensor([0, 100, 5], device="cuda")
    index = check_score(x, tokens, 32, 1.0)[3]
    assert index[0].tolist() == list(range(32))
    assert index[1].tolist() == list(range(100, 100 + 7 * 32, 7))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_scores_of_strided_rows(cuda, dtype, offset):
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = (randn(gen, 9, 2111) * 3).to(dtype)[:, offset:offset + 2003]
    tokens = torch.randint(0, 2003, (9,), generator=gen, device="cuda")
    check_score(x, tokens, 7, 1.0)


def test_scores_of_many_rows(cuda):
    """More rows than a grid's second dimension."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = randn(gen, 65600, 37)
    tokens = torch.randint(0, 37, (65600,), generator=gen, device="cuda")
    check_score(x, tokens, 3, 1.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_of_large_logits(cuda, dtype):
    """Logits that rise and fall by far more than a power of two's range."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    x = torch.linspace(-3000, 3000, 30011, device="cuda").repeat(3, 1)
    x[1] = x[1].flip(0)
    x[2] = x[2, torch.randperm(30011, generator=gen, device="cuda")]
    x = x.to(dtype)
    tokens = torch.randint(0, 30011, (3,), generator=gen, device="cuda")
    check_score(x, tokens, 20, 1.0)
    check_score(x, tokens, 20, 0.01)


def test_scores_same_each_time(cuda):
    gen = torch.Generator(device="cuda").manual_seed(6)
    x = (randn(gen, 4, 50001) * 3).to(torch.bfloat16)
    tokens = torch.randint(0, 50001, (4,), generator=gen, device="cuda")
    a = ops.token_logprobs(x, tokens, top_k=20)
    for _ in range(3):
        b = ops.token_logprobs(x, tokens, top_k=20)
        assert all(torch.equal(p, q) for p, q in zip(a, b))


# ------------------------------------------------------------------ refusals


def test_refusals(cuda):
    k, v, table, n, gen = make_cache([20, 3], 16, 2, 64, torch.bfloat16, seed=1)
    q = randn(gen, 2, 4, 64, dtype=torch.bfloat16)
    bad = [
        lambda: ops.paged_attention(q.float(), k, v, table, n),
        lambda: ops.paged_attention(q.cpu(), k, v, table, n),
        lambda: ops.paged_attention(q[:, :3], k, v, table, n),
        lambda: ops.paged_attention(q[:1], k, v, table, n),
        lambda: ops.paged_attention(q.transpose(1, 2), k, v, table, n),
        lambda: ops.paged_attention(q, k, v[:, :, :1], table, n),
        lambda: ops.paged_attention(q, k.half(), v.half(), table, n),
        lambda: ops.paged_attention(q, k, v, table.long(), n),
        lambda: ops.paged_attention(q, k, v, table, n.long()),
        lambda: ops.paged_attention(q, k, v, table, n[:1]),
        lambda: ops.paged_attention(q, k, v, table, n, max_len=100),
        lambda: ops.paged_attention(q, k, v, table, n, max_len=-1),
        lambda: ops.paged_attention(q, k, v, table, n, starts=n.long()),
        lambda: ops.paged_attention(q, k, v, table, n, out=torch.empty_like(q).float()),
        lambda: ops.kv_append(q, q, k, v, table, n),
        lambda: ops.kv_append(q[:, :2], q[:, 2:], k, v, table, n[:1]),
        lambda: ops.kv_append(q[:, :2].float(), q[:, 2:].float(), k, v, table, n),
        lambda: ops.kv_append(q[:, :2], q[:, 2:].contiguous(), k, v, table, n),
        lambda: ops.kv_fork(k, v, table, n, n),
        lambda: ops.kv_fork(k[None], v[None], table, n, n),
        lambda: ops.kv_fork(k[None], v[None], table, n, dev([0] * k.shape[0]), parents=n.long()),
        lambda: ops.kv_fork(k[None], v[None], table[0], n, dev([0] * k.shape[0])),
        lambda: ops.kv_compact(k, v, table, n),
        lambda: ops.kv_compact(k[None], v[None], table, n),
        lambda: ops.token_logprobs(q[:, 0].half(), n.long()),
        lambda: ops.token_logprobs(q[:, 0], n),
        lambda: ops.token_logprobs(q[:, 0], n[:1].long()),
        lambda: ops.token_logprobs(q[:, 0], n.long(), top_k=33),
        lambda: ops.token_logprobs(q[:, 0, :8], n.long(), top_k=9),
        lambda: ops.token_logprobs(q[:, 0], n.long(), top_k=-1),
        lambda: ops.token_logprobs(q[:, 0], n.long(), temperature=0.0),
        lambda: ops.token_logprobs(q[:, 0], n.long(), temperature=math.nan),
        lambda: ops.token_logprobs(q[:, 0, ::2], n.long()),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")
    wide = torch.zeros(4, 16, 1, 96, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(L.WxError):
        ops.paged_attention(q[:, :1, :32].repeat(1, 1, 3), wide, wide, table, n)
    assert ops.token_logprobs(q[:0, 0], n[:0].long(), top_k=3)[2].shape == (0, 3)
