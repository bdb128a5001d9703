"""The decoder operators' host side and sources: what can be checked without a GPU."""
import re
from pathlib import Path

import pytest
import torch

from test_decoder_capi import NUL, P, append, at, attend, fork, lib, score  # noqa: F401
from wxb200 import _build
from wxb200.kvcache import PagedKVCache

CSRC = Path(__file__).resolve().parents[1] / "whisper-xdna_b200" / "csrc"


def compact(l, **kw):
    a = dict(layers=1, ks=(16384, 1024, 64, 64), heads=1, pages=10, page=16)
    a.update(kw)
    return l.wx_kv_compact(P, P, a["layers"], *a["ks"], a["heads"], 64, a["pages"], a["page"], 0,
                           at(1), at(3), 2, 4, at(4), at(6), at(8), at(9), 1 << 20, NUL)


@pytest.mark.parametrize("name", ["paged_attention.cu", "kvcache.cu", "kvcache.cuh", "score.cu"])
def test_no_read_only_loads(name):
    """These kernels start as programmatic dependents: while they already live, the
    kernel before them may still write what they read, a fork the page table say. A
    read-only load promises that nobody does."""
    text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    assert not re.findall(r"__ldg\b|ld\.global(?:\.\w+)*\.nc\b|__restrict__", text)


@pytest.mark.parametrize("device,want", [(None, 1), ("cuda", 1), (torch.device("cuda"), 1),
                                         ("cuda:0", 0), (torch.device("cuda", 2), 2)])
def test_cache_device(monkeypatch, device, want):
    """A device without an index is the current one."""
    seen = set()
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    for name in ("empty", "full", "zeros", "tensor"):
        monkeypatch.setattr(torch, name, lambda *a, device, **kw: seen.add(device))
    PagedKVCache(1, 4, 16, 2, 64, 1, 40, device=device)
    assert seen == {torch.device("cuda", want)}


def test_cache_refuses_other_devices():
    for device in ("cpu", torch.device("meta")):
        with pytest.raises(ValueError, match="CUDA"):
            PagedKVCache(1, 4, 16, 2, 64, 1, 40, device=device)


@pytest.mark.parametrize("kw", [dict(os=(0, 64, 64)), dict(os=(63, 64, 64)), dict(os=(-63, 64, 64)),
                                dict(heads=2, os=(128, 0, 64)), dict(group=2, os=(128, 64, 1))])
def test_attention_refuses_an_out_on_itself(lib, kw):
    """Rows of out that share memory would be written by several CTAs at once."""
    l, L = lib
    assert attend(l, **kw) == L.WX_ERR_INVALID
    assert "share memory" in L.last_error()


@pytest.mark.parametrize("call", [append, fork, compact])
@pytest.mark.parametrize("pages,page,heads,ks", [(2, 1, 1, (0, 64, 64)), (1, 2, 1, (128, 0, 64)),
                                                 (1, 1, 2, (128, 128, 0)),
                                                 (2, 1, 1, (56, 64, 64))])
def test_writers_refuse_a_cache_on_itself(lib, call, pages, page, heads, ks):
    l, L = lib
    if call is not append:
        ks = (16384,) + ks
    assert call(l, pages=pages, page=page, heads=heads, ks=ks) == L.WX_ERR_INVALID
    assert "share memory" in L.last_error()


@pytest.mark.parametrize("call", [fork, compact])
def test_plans_refuse_layers_on_one_another(lib, call):
    l, L = lib
    assert call(l, layers=2, ks=(0, 1024, 64, 64)) == L.WX_ERR_INVALID


@pytest.mark.parametrize("t", [3e-39, 4.2e-39])
def test_scores_refuse_a_temperature_past_the_exponents(lib, t):
    """log2(e) / t is what logits are multiplied by: infinite, it makes every score NaN."""
    l, L = lib
    assert score(l, t=t) == L.WX_ERR_INVALID
    assert "temperature" in L.last_error()


def test_binding_is_built_again_for_another_torch(monkeypatch, tmp_path):
    """It is linked against torch's C++ interface, which no source file's time tells of."""
    ran = []

    def run(cmd, **kw):
        ran.append(cmd)
        (tmp_path / "_decoder.so").write_bytes(b"")
        return type("Done", (), {"returncode": 0, "stdout": "", "stderr": ""})

    monkeypatch.setattr(_build, "BUILD", tmp_path)
    monkeypatch.setattr(_build, "BINDING", tmp_path / "_decoder.so")
    monkeypatch.setattr(_build.subprocess, "run", run)
    _build.build_binding()
    _build.build_binding()
    assert len(ran) == 1
    monkeypatch.setattr(torch, "__version__", torch.__version__ + "1")
    _build.build_binding()
    _build.build_binding()
    assert len(ran) == 2
    _build.build_binding(force=True)
    assert len(ran) == 3


@pytest.mark.parametrize("n,width", [(1 << 20, 1 << 11), (1 << 20, (1 << 10) + 1)])
def test_fork_refuses_a_table_that_its_sums_do_not_hold(lib, n, width):
    """The pages asked for are summed in 32 bits: past them a sum below 0 would pass for
    one that the pool holds."""
    l, L = lib
    assert fork(l, n=n, width=width, page=1, space=1 << 40) == L.WX_ERR_INVALID
    assert "page table" in L.last_error()
