"""Decoder attention on the GPU where it is easiest to get wrong: calls right
behind one another, value scales far apart, masked places that are not finite,
pages that begin with zeros, other streams.  Gold: decoder_ref.py."""
import numpy as np
import pytest

import decoder_ref as ref
from test_decoder_gpu import bsp, check_attention, cuda, host, i32, page_table, torch_  # noqa: F401

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------- ordering --
@pytest.mark.parametrize("page,d", [(16, 64), (64, 128)])
def test_calls_see_what_the_call_before_wrote(bsp, page, d):  # noqa: F811
    """Appends that grow the pages' scales, rotations and single-token attention
    in turn, lengths counted on the device: the bits of a run that waits for the
    GPU after every call."""
    torch = torch_()
    n, hq, hk, steps = 40, 8, 2, 40
    g = torch.Generator(device="cuda").manual_seed(7)
    x = [torch.randn((steps, n, h, d), device="cuda", generator=g) for h in (hq, hk, hk)]
    grow = 2.0 ** (torch.arange(steps, device="cuda") % 7).float()[:, None, None, None]  # within a page, too
    q, k, v = x[0].bfloat16(), (x[1] * grow).bfloat16(), (x[2] * grow).bfloat16()
    table = bsp.rope_table(256, d)
    first = [3 * s % 50 for s in range(n)]
    per = -(-(max(first) + steps) // page)
    pages = cuda(np.random.default_rng(1).permutation(n * per).reshape(n, per).astype(np.int32))
    starts = i32(np.arange(n + 1))
    plan = bsp.DecodePlan(bsp.device(), n, hq, hk, d, page)

    def run(wait):
        cache = bsp.KvCache.empty(n * per, hk, page, d)
        cache.k.copy_((torch.arange(cache.k.numel(), device="cuda") % 126).to(torch.uint8).view(cache.k.shape))
        cache.v.copy_(cache.k)
        before = i32(first)
        lens = before + 1
        out = torch.empty_like(q)
        turned = torch.empty_like(q)
        qr, again = torch.empty_like(q[0]), torch.empty_like(q[0])
        torch.cuda.synchronize()
        for t in range(steps):
            for call in (lambda: bsp.kv_append(cache, k[t], v[t], starts, before, pages, table=table, q=q[t], q_out=qr),
                         lambda: plan.execute(cache, qr, lens, pages, out[t]),
                         lambda: bsp.rope(out[t], before, table, out=again),
                         lambda: bsp.rope(again, lens, table, out=turned[t]),
                         lambda: before.add_(1), lambda: lens.add_(1)):
                call()
                if wait:
                    torch.cuda.synchronize()
        bsp.device().synchronize()
        return out, turned, cache.k, cache.v, cache.k_scale, cache.v_scale

    gold = run(True)
    assert bool(torch.isfinite(gold[0]).all())
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(run(False), gold))


# ------------------------------------------------------------------ devices --
def test_cache_of_another_gpu_is_refused(bsp):  # noqa: F811
    """A cache says on which GPU it is; the calls compare that with their tensors
    before anything is launched.  (The stand-in's memory is this GPU's, so that the
    call could do no harm if it went on.)"""
    torch = torch_()
    cache = bsp.KvCache.empty(2, 1, 16, 64)
    assert cache.ordinal == torch.cuda.current_device() and cache.k.device.index == cache.ordinal

    class Elsewhere:
        address, ordinal = cache.address, cache.ordinal + 1

    x = torch.ones((1, 1, 64), device="cuda", dtype=torch.bfloat16)
    o = torch.zeros_like(x)
    plan = bsp.DecodePlan(bsp.device(), 1, 1, 1, 64, 16)
    for call in (lambda c: bsp.kv_append(c, x, x, i32([0, 1]), i32([0]), i32([[0]])),
                 lambda c: plan.execute(c, x, i32([1]), i32([[0]]), o)):
        with pytest.raises(bsp.BspError, match="cache is on cuda:1, not on GPU 0") as e:
            call(Elsewhere)
        assert e.value.status == bsp.BSP_ERR_INVALID_ARG
        call(cache)
    bsp.device().synchronize()
    assert bool((o == 1).all()) and bool(cache.k.any())
