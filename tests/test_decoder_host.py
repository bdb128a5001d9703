"""The decoder operators' host side and sources: what can be checked without a GPU."""
import re
from pathlib import Path

import pytest
import torch

from wxb200.kvcache import PagedKVCache

CSRC = Path(__file__).resolve().parents[1] / "whisper-xdna_b200" / "csrc"


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
