"""Edges of the decoder-attention operators that need no GPU: what the kernels'
sources may not do, and refusals before any launch."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "tenstorrent-wh-blockspmm_b200", "csrc")


def _code(name):
    """A source file without its comments."""
    text = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


@pytest.mark.parametrize("name", ["rope.cu", "rope.cuh", "append.cu", "decode.cu", "prompt.cu"])
def test_early_kernels_read_no_memory_as_constant(name):
    """These kernels are resident while the kernel before them still writes, so
    nothing they read is constant for as long as they live: no ld.global.nc."""
    assert not re.search(r"__ldg\s*\(|ld\.global\.nc|__restrict__", _code(name))
    assert name == "rope.cuh" or "stream_wait()" in _code(name)
