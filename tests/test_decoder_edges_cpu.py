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


# ------------------------------------------------------------------ devices --
torch = pytest.importorskip("torch")
import bsp  # noqa: E402


class OnGpu:
    """Looks like a CUDA tensor on GPU `index`; has no memory there."""

    def __init__(self, shape, dtype, index):
        self._t = torch.zeros(shape, dtype=dtype)
        self.shape, self.dtype, self.device = self._t.shape, dtype, torch.device("cuda", index)
        self.is_cuda = True

    def __getattr__(self, name):
        return getattr(self._t, name)


def test_cache_on_one_gpu():
    """All four tensors of a cache are on one GPU, which the cache knows."""
    parts = [((3, 2, 16, 64), torch.uint8), ((3, 2, 16, 64), torch.uint8), ((3, 2), torch.float32), ((3, 2), torch.float32)]
    assert bsp.KvCache(*(OnGpu(*p, 1) for p in parts)).ordinal == 1
    for other in range(4):
        with pytest.raises(bsp.BspError) as e:
            bsp.KvCache(*(OnGpu(*p, int(i == other)) for i, p in enumerate(parts)))
        assert e.value.status == bsp.BSP_ERR_INVALID_ARG and "cuda:1" in str(e.value)
