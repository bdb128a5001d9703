"""The decoder operators' host side and sources: what can be checked without a GPU."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "whisper-xdna_b200" / "csrc"


@pytest.mark.parametrize("name", ["paged_attention.cu", "kvcache.cu", "kvcache.cuh", "score.cu"])
def test_no_read_only_loads(name):
    """These kernels start as programmatic dependents: while they already live, the
    kernel before them may still write what they read, a fork the page table say. A
    read-only load promises that nobody does."""
    text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    assert not re.findall(r"__ldg\b|ld\.global(?:\.\w+)*\.nc\b|__restrict__", text)
