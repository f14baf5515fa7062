"""What the decoder-attention calls refuse before any kernel or GPU is asked for."""
import os
import sys

import pytest

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tenstorrent-wh-blockspmm_b200"))
import bsp  # noqa: E402


def _refused(f):
    with pytest.raises(bsp.BspError) as e:
        f()
    assert e.value.status == bsp.BSP_ERR_INVALID_ARG
    return str(e.value)


def test_operands_that_are_no_cuda_tensors():
    x, i = torch.zeros(2, 1, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    assert "x must be a cuda tensor" in _refused(lambda: bsp.rope(x, i, x.float()))
    assert "x must be a torch tensor" in _refused(lambda: bsp.rope([1], i, x.float(), out=x))
    assert "3 dimensions" in _refused(lambda: bsp.rope(x[0], i, x.float()))
    assert "layout" in _refused(lambda: bsp.rope(x, i, x.float(), layout="thirds"))


def test_plans_and_caches_that_are_none():
    """A closed plan has no handle; anything that is no plan or cache has no such attribute."""
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    calls = bsp._calls or bsp._load_calls()

    class Closed:
        handle = None

    _refused(lambda: calls.prompt(Closed(), 0, x, x, x, x, 1.0, None, None))
    _refused(lambda: calls.decode(Closed(), 0, None, x, x, x, x, 1.0, None, None))
    with pytest.raises(AttributeError):
        calls.prompt(None, 0, x, x, x, x, 1.0, None, None)
    with pytest.raises(AttributeError):
        bsp.kv_append(None, x, x, x, x, x)
    with pytest.raises(TypeError):
        calls.rope(x)
