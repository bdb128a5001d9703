"""The decoder operators' entry points refuse bad arguments on the host, before any
CUDA call (so these run without a GPU), and the tests' restatements of the page plans
keep the cache's invariants."""
import ctypes
import random

import pytest

import decoder_ref as R

P = ctypes.c_void_p(4096)     # aligned, never dereferenced
ODD = ctypes.c_void_p(4097)
NUL = ctypes.c_void_p(0)


@pytest.fixture
def lib(wxlib):
    from wxb200 import _lib
    return wxlib, _lib


def attend(l, **kw):
    a = dict(q=P, qs=(64, 64, 64), k=P, v=P, ks=(1024, 64, 64), table=P, ld=4, lens=P, starts=NUL,
             out=P, os=(64, 64, 64), lse=NUL, n=2, heads=1, group=1, hd=64, pages=10, page=16,
             max_len=64, scale=0.125, dtype=0, ws=NUL, space=0)
    assert not set(kw) - set(a)
    a.update(kw)
    return l.wx_paged_attention(a["q"], *a["qs"], a["k"], a["v"], *a["ks"], a["table"], a["ld"],
                                a["lens"], a["starts"], a["out"], *a["os"], a["lse"], a["n"],
                                a["heads"], a["group"], a["hd"], a["pages"], a["page"],
                                a["max_len"], a["scale"], a["dtype"], a["ws"], a["space"], NUL)


@pytest.mark.parametrize("bad", [
    dict(n=-1), dict(n=70000), dict(heads=0), dict(group=0), dict(max_len=-1), dict(max_len=65),
    dict(dtype=2), dict(pages=0), dict(page=0), dict(k=NUL), dict(v=ODD), dict(ks=(1024, 60, 64)),
    dict(ks=(1020, 64, 64)), dict(ks=(-1024, 64, 64)), dict(q=NUL), dict(out=NUL), dict(lens=NUL),
    dict(table=NUL), dict(ld=0), dict(q=ODD), dict(max_len=8192, ld=600),
    dict(max_len=8192, ld=600, ws=P, space=16)])
def test_paged_attention_refuses(lib, bad):
    l, L = lib
    assert attend(l, **bad) == L.WX_ERR_INVALID
    assert L.last_error()


def test_paged_attention_head_dim_and_no_sequences(lib):
    l, L = lib
    assert attend(l, hd=96) == L.WX_ERR_UNSUPPORTED
    assert "head dim 96" in L.last_error()
    assert attend(l, n=0, q=NUL, out=NUL, lens=NUL, table=NUL) == L.WX_OK


def test_paged_attention_workspace(lib):
    l, L = lib
    space = l.wx_paged_attention_workspace
    assert space(4, 2, 4, 64, 1000, 0) == 0               # one launch, joined on chip
    big = space(1, 2, 4, 64, 100000, 0)
    assert big > 8 * 64 * 4 and space(2, 2, 4, 64, 100000, 0) >= big
    assert space(1, 2, 4, 65, 1000, 0) == L.WX_ERR_UNSUPPORTED
    assert space(1, 0, 4, 64, 1000, 0) == L.WX_ERR_INVALID


def append(l, **kw):
    a = dict(k=P, v=P, s=(64, 64, 64), kc=P, vc=P, ks=(1024, 64, 64), table=P, ld=4, lens=P,
             counts=NUL, n=2, tokens=1, heads=1, hd=64, pages=10, page=16, dtype=0)
    a.update(kw)
    return l.wx_kv_append(a["k"], a["v"], *a["s"], a["kc"], a["vc"], *a["ks"], a["table"], a["ld"],
                          a["lens"], a["counts"], a["n"], a["tokens"], a["heads"], a["hd"],
                          a["pages"], a["page"], a["dtype"], NUL)


@pytest.mark.parametrize("bad", [
    dict(k=NUL), dict(kc=NUL), dict(vc=ODD), dict(table=NUL), dict(lens=NUL), dict(ld=0),
    dict(n=-1), dict(n=70000), dict(tokens=-1), dict(heads=0), dict(hd=0), dict(hd=60),
    dict(pages=0), dict(page=0), dict(dtype=9), dict(tokens=1 << 26), dict(ks=(1024, 4, 64))])
def test_kv_append_refuses(lib, bad):
    l, L = lib
    assert append(l, **bad) == L.WX_ERR_INVALID
    assert L.last_error()


def test_kv_append_of_nothing(lib):
    l, L = lib
    assert append(l, n=0) == L.WX_OK and append(l, tokens=0, k=NUL) == L.WX_OK


def at(i):
    return ctypes.c_void_p(4096 * (i + 1))


def fork(l, **kw):
    a = dict(k=P, v=P, layers=2, ks=(16384, 1024, 64, 64), heads=1, hd=64, pages=10, page=16,
             dtype=0, table=at(1), lens=at(2), refs=at(3), parents=NUL, grow=NUL, n=2, width=4,
             table_out=at(4), lens_out=at(5), refs_out=at(6), grown=at(7), status=at(8), ws=at(9),
             space=1 << 20)
    a.update(kw)
    return l.wx_kv_fork(a["k"], a["v"], a["layers"], *a["ks"], a["heads"], a["hd"], a["pages"],
                        a["page"], a["dtype"], a["table"], a["lens"], a["refs"], a["parents"],
                        a["grow"], a["n"], a["width"], a["table_out"], a["lens_out"],
                        a["refs_out"], a["grown"], a["status"], a["ws"], a["space"], NUL)


@pytest.mark.parametrize("bad", [
    dict(layers=0), dict(ks=(16388, 1024, 64, 64)), dict(n=0), dict(width=0), dict(ws=NUL),
    dict(ws=ODD), dict(space=16), dict(table=NUL), dict(lens=NUL), dict(refs=NUL),
    dict(table_out=NUL), dict(lens_out=NUL), dict(refs_out=NUL), dict(status=NUL),
    dict(table_out=at(1)), dict(lens_out=at(2)), dict(refs_out=at(3)), dict(dtype=5),
    dict(page=1 << 16, width=1 << 16, space=1 << 40)])
def test_kv_fork_refuses(lib, bad):
    l, L = lib
    assert fork(l, **bad) == L.WX_ERR_INVALID
    assert L.last_error()


@pytest.mark.parametrize("bad", [
    dict(table=NUL), dict(refs=NUL), dict(table_out=NUL), dict(refs_out=NUL), dict(status=NUL),
    dict(refs_out=at(3)), dict(space=0), dict(k=NUL), dict(layers=-1)])
def test_kv_compact_refuses(lib, bad):
    l, L = lib
    a = dict(k=P, v=P, layers=2, table=at(1), refs=at(3), table_out=at(4), refs_out=at(6),
             status=at(8), space=1 << 20)
    a.update(bad)
    assert l.wx_kv_compact(a["k"], a["v"], a["layers"], 16384, 1024, 64, 64, 1, 64, 10, 16, 0,
                           a["table"], a["refs"], 2, 4, a["table_out"], a["refs_out"],
                           a["status"], at(9), a["space"], NUL) == L.WX_ERR_INVALID
    assert L.last_error()


def score(l, **kw):
    a = dict(x=P, dtype=1, rows=2, vocab=100, ld=100, tokens=P, top_k=4, t=1.0, lp=P, ent=P,
             top=P, index=P)
    a.update(kw)
    return l.wx_token_logprobs(a["x"], a["dtype"], a["rows"], a["vocab"], a["ld"], a["tokens"],
                               a["top_k"], a["t"], a["lp"], a["ent"], a["top"], a["index"], NUL)


@pytest.mark.parametrize("bad", [
    dict(x=NUL), dict(x=ODD), dict(dtype=3), dict(rows=-1), dict(vocab=0), dict(ld=99),
    dict(tokens=NUL), dict(top_k=-1), dict(top_k=33), dict(vocab=3), dict(t=0.0), dict(t=-1.0),
    dict(t=float("nan")), dict(t=float("inf")), dict(t=1e-45), dict(top=NUL), dict(index=NUL)])
def test_token_logprobs_refuses(lib, bad):
    l, L = lib
    assert score(l, **bad) == L.WX_ERR_INVALID
    assert L.last_error()


def test_token_logprobs_of_no_rows(lib):
    l, L = lib
    assert score(l, rows=0, x=NUL) == L.WX_OK


@pytest.mark.parametrize("page,seed", [(1, 0), (4, 1), (16, 2)])
def test_plans_keep_the_invariants(page, seed):
    """References count the table's entries, a sequence holds exactly the pages of its
    tokens, and no page that two sequences share is written by either."""
    rng = random.Random(seed)
    seqs, width, n_pages = 6, 48 // page, 200 // page
    table, lens, refs = [[-1] * width for _ in range(seqs)], [0] * seqs, [0] * n_pages
    for _ in range(60):
        parents = [rng.choice([-1, i, i, i, rng.randrange(seqs)]) for i in range(seqs)]
        grow = [rng.choice([0, 1, 1, 5]) for _ in range(seqs)]
        table, lens, refs, grown, status, copies = R.fork_ref(table, lens, refs, parents, grow,
                                                              page)
        count = [0] * n_pages
        for row, n in zip(table, lens):
            held = -(-n // page)
            assert all(p >= 0 for p in row[:held]) and all(p == -1 for p in row[held:])
            for p in row[:held]:
                count[p] += 1
        assert count == refs and status[0] == sum(r == 0 for r in refs)
        for i in range(seqs):
            for pos in range(lens[i] - grown[i], lens[i]):      # positions to be written
                for j in range(seqs):
                    shared = j != i and table[j][pos // page] == table[i][pos // page]
                    assert not shared or lens[j] <= pos
        assert not {d for _, d, _ in copies} & {s for s, _, _ in copies}
        if rng.random() < 0.3:
            table, refs, (used, _), moves = R.compact_ref(table, refs)
            assert all(r > 0 for r in refs[:used]) and not any(refs[used:])
