"""Decoder attention on the GPU where it is easiest to get wrong: calls right
behind one another, value scales far apart, masked places that are not finite,
pages that begin with zeros, other streams.  Gold: decoder_ref.py."""
import numpy as np
import pytest

import decoder_ref as ref
from test_decoder_gpu import bsp, check_attention, cuda, host, i32, page_table, prompt_gold, torch_  # noqa: F401

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


# ------------------------------------------------------- value scales far apart --
def _pages_of(kind, size, n, page, hk, d, rng):
    """Values [n, hk, d] whose pages have scales far apart."""
    v = rng.normal(0, 1, (n, hk, d)) * size
    at = np.arange(n)[:, None, None]
    if kind == "zeros":           # the first page holds zeros: scale 1
        v[: min(page, n)] = 0
    elif kind == "zeros_last":
        v[-(n % page or page):] = 0
    elif kind == "outlier":       # one token far larger than all others
        v[n // 3] = 1e3
    elif kind == "turns":         # three sizes in turn
        v = v * np.choose(at // page % 3, [1.0, 2.0 ** 20, 2.0 ** -20])
    elif kind == "falling":
        v = v * 2.0 ** (-2.0 * (at // page))
    elif kind == "rising":
        v = v * 2.0 ** (2.0 * (at // page))
    return v


FAR = [("zeros", 1e-3), ("zeros", 1e-4), ("zeros", 1e-5), ("zeros", 1e-12), ("zeros", 1e-25), ("zeros_last", 1e-5),
       ("outlier", 1e-4), ("outlier", 1e-20), ("turns", 1.0), ("falling", 1e6), ("rising", 1e-6), ("plain", 1.0)]


@pytest.mark.parametrize("kind,size", FAR, ids=[f"{k}_{s:g}" for k, s in FAR])
@pytest.mark.parametrize("hq,hk,d,page", [(8, 2, 64, 16), (16, 1, 128, 16), (4, 1, 128, 64), (20, 1, 64, 32)])
def test_decode_value_scales(bsp, kind, size, hq, hk, d, page):  # noqa: F811
    """The output's error is that of the weights (2^-11, rounded to fp16) times
    sum p |v|, whatever the scales of the pages; weights below 2^-14 of the largest
    are off by up to 2^-25 of it."""
    torch = torch_()
    rng = np.random.default_rng(11)
    lens = [640, 100, 17]
    per = [-(-n // page) for n in lens]
    pages = page_table(rng, lens, page, sum(per))
    cache = bsp.KvCache.empty(sum(per), hk, page, d)
    k = rng.normal(0, 1, (sum(lens), hk, d))
    v = np.concatenate([_pages_of(kind, size, n, page, hk, d, rng) for n in lens])
    bsp.kv_append(cache, *(cuda(ref.bf16(x), torch.bfloat16) for x in (k, v)), i32(np.concatenate([[0], np.cumsum(lens)])),
                  i32([0] * 3), cuda(pages))
    q = ref.bf16(rng.normal(0, 1, (3, hq, d)))
    codes, scales = [cache.k.cpu().numpy(), cache.v.cpu().numpy()], [host(cache.k_scale), host(cache.v_scale)]
    keys, values = ([(ref.VALUES[c[pages[s][: per[s]]]] * x[pages[s][: per[s]]][:, :, None, None])
                     .transpose(1, 0, 2, 3).reshape(hk, -1, d)[:, :n] for s, n in enumerate(lens)]
                    for c, x in zip(codes, scales))
    gold, lse = np.zeros(q.shape), np.zeros(q.shape[:2])
    weight, size_, most = np.zeros(q.shape), np.zeros(q.shape[:2] + (1,)), np.zeros(q.shape)
    for s in range(3):
        for h in range(hq):
            qq, kk, vv = q[s, h][None].astype(float), keys[s][h // (hq // hk)], values[s][h // (hq // hk)]
            gold[s, h], lse[s, h], weight[s, h] = (x[0] for x in ref.attention(qq, kk, vv, d ** -0.5, [lens[s]]))
            size_[s, h, 0] = d ** -0.5 * (np.abs(qq) @ np.abs(kk).T).max()
            top = np.exp(d ** -0.5 * (qq @ kk.T).max() - lse[s, h])  # the largest weight
            most[s, h] = 2.0 ** -25 * top * np.abs(vv).sum(0)
    weight = weight + most / (2 * ref.UH)
    for ctas in (0, 1, 5):
        plan = bsp.DecodePlan(bsp.device(), 3, hq, hk, d, page, opts=bsp.make_opts(max_ctas=ctas))
        o, l = torch.full(q.shape, float("nan"), device="cuda").bfloat16(), torch.full(q.shape[:2], float("nan"), device="cuda")
        plan.execute(cache, cuda(q, torch.bfloat16), i32(lens), cuda(pages), o, lse=l)
        bsp.device().synchronize()
        # (the 1e-30 of the check is far below every value here but those of 1e-25)
        check_attention(o, l, gold, lse, weight, size_, 2 * ref.UH)


@pytest.mark.parametrize("d,hq", [(64, 4), (128, 16)])
def test_decode_scales_at_the_ends(bsp, d, hq):  # noqa: F811
    """Pages at the two ends of the scales' range, 2^-100 and 2^119: the large
    values are the output, and the sum of the weights is not touched by them."""
    torch = torch_()
    rng = np.random.default_rng(2)
    page, n = 16, 96
    cache = bsp.KvCache.empty(n // page, 1, page, d)
    v = np.ones((n, 1, d)) * np.where(np.arange(n) // page % 2, 3e38, 1e-30)[:, None, None]
    k = rng.normal(0, 1, (n, 1, d))
    pages = i32(np.arange(n // page)[None])
    bsp.kv_append(cache, cuda(ref.bf16(k), torch.bfloat16), cuda(ref.bf16(v), torch.bfloat16), i32([0, n]), i32([0]), pages)
    assert {float(x) for x in cache.v_scale.flatten()} == {2.0 ** -100, 2.0 ** 119}
    q = ref.bf16(rng.normal(0, 1, (1, hq, d)))
    o, l = torch.empty((1, hq, d), device="cuda").bfloat16(), torch.empty((1, hq), device="cuda")
    kk, vv = (ref.VALUES[c.cpu().numpy()[:, 0]].reshape(n, d) * host(s)[:, 0].repeat(page)[:, None]
              for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    gold, lse, weight = ref.attention(q[0].astype(float), kk, vv, d ** -0.5, [n] * hq)
    size = d ** -0.5 * (np.abs(q[0].astype(float)) @ np.abs(kk).T).max(1, keepdims=True)
    for ctas in (1, 0):
        plan = bsp.DecodePlan(bsp.device(), 1, hq, 1, d, page, opts=bsp.make_opts(max_ctas=ctas))
        plan.execute(cache, cuda(q, torch.bfloat16), i32([n]), pages, o, lse=l)
        bsp.device().synchronize()
        check_attention(o[0], l[0], gold, lse, weight, size, 2 * ref.UH)


@pytest.mark.parametrize("d,page", [(64, 16), (128, 64)])
def test_decode_many_small_weights_beside_a_large_one(bsp, d, page):  # noqa: F811
    """One token takes nearly all the weight and its value is zero; 20000 tokens of
    2^-22 each, of one key, are the output."""
    torch = torch_()
    n, hq = 20001, 4
    per = -(-n // page)
    cache = bsp.KvCache.empty(per, 1, page, d)
    rng = np.random.default_rng(3)
    k = np.zeros((n, 1, d))
    k[0, 0, 0] = 2.0
    v = rng.normal(0.5, 1, (n, 1, d))
    v[0] = 0
    v[:: page, 0, :: 7] = 4.0  # the pages have one scale
    v[0] = 0
    v[1, 0, 3] = 4.0
    pages = i32(np.arange(per)[None])
    bsp.kv_append(cache, cuda(ref.bf16(k), torch.bfloat16), cuda(ref.bf16(v), torch.bfloat16), i32([0, n]), i32([0]), pages)
    q = np.zeros((1, hq, d), np.float32)
    q[0, :, 0] = ref.bf16([7.5, 7.6, 7.7, 7.8])  # scores of 15 to 15.6 at scale 1: weights of 2^-22 beside it
    o, l = torch.empty((1, hq, d), device="cuda").bfloat16(), torch.empty((1, hq), device="cuda")
    kk, vv = (ref.VALUES[c.cpu().numpy()[:, 0]].reshape(-1, d)[:n] * host(s)[:, 0].repeat(page)[:n, None]
              for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    gold, lse, weight = ref.attention(q[0].astype(float), kk, vv, 1.0, [n] * hq)
    size = (np.abs(q[0].astype(float)) @ np.abs(kk).T).max(1, keepdims=True)
    top = np.exp((q[0].astype(float) @ kk.T).max(1) - lse)
    weight = weight + 2.0 ** -32 * top[:, None] * np.abs(vv).sum(0) / (2 * ref.UH)
    for ctas in (0, 1):  # one: a quarter of the tokens is in the warp of the large one
        plan = bsp.DecodePlan(bsp.device(), 1, hq, 1, d, page, opts=bsp.make_opts(max_ctas=ctas))
        plan.execute(cache, cuda(q, torch.bfloat16), i32([n]), pages, o, scale=1.0, lse=l)
        bsp.device().synchronize()
        check_attention(o[0], l[0], gold, lse, weight, size, 2 * ref.UH)


# ------------------------------------------------------------ masked values --
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 1)])
def test_prompt_hidden_values_weigh_nothing(bsp, d, hq, hk):  # noqa: F811
    """Values near the type's largest and lowest at keys that the causal mask hides,
    at each place of a step: exactly nothing of them in the rows before."""
    torch = torch_()
    n = 300
    rng = np.random.default_rng(12)
    q = ref.bf16(rng.normal(0, 1, (n, hq, d)))
    k, v = (ref.bf16(rng.normal(0, 1, (n, hk, d))) for _ in range(2))
    qt, kt, vt = (cuda(x, torch.bfloat16) for x in (q, k, v))
    gold = prompt_gold(q.astype(float), k.astype(float), v.astype(float), [n], [n], hk, d ** -0.5, True)
    plan = bsp.PromptPlan(bsp.device(), [n], [n], hq, hk, d)
    o, lse = torch.empty_like(qt), torch.empty((n, hq), device="cuda")
    for at in (1, 30, 64, 127, 130, 200, 290):
        v2 = vt.clone()
        v2[at:, :, ::2] = 3.3e38
        v2[at:, :, 1::2] = -3.3e38
        plan.execute(qt, kt, v2, o, lse=lse)
        bsp.device().synchronize()
        check_attention(o[:at], lse[:at], *(x[:at] for x in gold), ref.U16)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 3.3e38])
@pytest.mark.parametrize("cut", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_rows_without_a_key_are_zero(bsp, bad, cut, d):  # noqa: F811
    """Queries that see no key get O = 0 and lse = -inf, whatever V holds."""
    torch = torch_()
    n, m = (2100, 1500) if cut else (257, 200)
    q, k, v = (torch.randn((x, h, d), device="cuda").bfloat16() for x, h in ((n, 2), (m, 1), (m, 1)))
    v[:] = bad
    plan = bsp.PromptPlan(bsp.device(), [n], [m], 2, 1, d)
    assert (plan.info()["workspace_bytes"] > 0) == cut
    o, lse = torch.full_like(q, float("nan")), torch.full((n, 2), float("nan"), device="cuda")
    plan.execute(q, k, v, o, lse=lse)
    bsp.device().synchronize()
    assert bool((o[: n - m] == 0).all()) and bool(torch.isneginf(lse[: n - m]).all())
    assert not bool((o[n - m:] == 0).any()) and bool(torch.isfinite(lse[n - m:]).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("hq,hk,d", [(1, 1, 128), (4, 1, 64), (3, 3, 128)])
def test_prompt_value_that_is_not_finite(bsp, bad, hq, hk, d):  # noqa: F811
    """A NaN or infinity in V: not finite where it is seen, in its column alone;
    rows of tiles that do not run its step of 128 keys, and other columns, keep
    their bits."""
    torch = torch_()
    n, more = 500, 60
    q, k, v = (torch.randn((x, h, d), device="cuda").bfloat16() for x, h in ((n, hq), (n + more, hk), (n + more, hk)))
    plan = bsp.PromptPlan(bsp.device(), [n], [n + more], hq, hk, d)
    tokens = 128 // plan.info()["packed_heads"]
    o, o2 = torch.empty_like(q), torch.empty_like(q)
    lse, lse2 = (torch.empty((n, hq), device="cuda") for _ in range(2))
    plan.execute(q, k, v, o, lse=lse)
    for at in (0, 59, 128, 187, 300, n + more - 1):
        v2 = v.clone()
        v2[at, 0, 3] = bad
        plan.execute(q, k, v2, o2, lse=lse2)
        bsp.device().synchronize()
        seen = torch.arange(n, device="cuda") + more >= at
        heads = slice(0, hq // hk)
        assert not bool(torch.isfinite(o2[seen][:, heads, 3]).any())
        # the last query of a row's tile, and the keys that the tile's steps cover
        last = (torch.arange(n, device="cuda") // tokens * tokens + tokens - 1).clamp(max=n - 1)
        runs = (last + more + 1 + 127) // 128 * 128 > at // 128 * 128
        same = torch.ones_like(o, dtype=torch.bool)
        same[runs.nonzero()[:, 0], heads, 3] = False
        assert torch.equal(o2[same], o[same]) and torch.equal(lse2, lse)


# ------------------------------------------------------------------- zeros --
@pytest.mark.parametrize("page,d,hk,zeros,after", [(16, 64, 1, 1, 1), (16, 128, 2, 15, 1), (64, 128, 3, 7, 40),
                                                   (128, 64, 2, 100, 28), (128, 128, 1, 127, 1)])
@pytest.mark.parametrize("size", [1e-2, 1e-4, 1e-12])
def test_append_small_values_behind_zeros(bsp, page, d, hk, zeros, after, size):  # noqa: F811
    """A page that begins with zeros takes the scale of the values that follow, as
    if they stood alone; a page that holds one code at scale 1 keeps it."""
    torch = torch_()
    rng = np.random.default_rng(page + zeros)
    x = ref.bf16(rng.normal(0, size, (after, hk, d)))
    xt = cuda(x, torch.bfloat16)
    nothing = torch.zeros((zeros, hk, d), device="cuda", dtype=torch.bfloat16)
    nothing[:, :, 1] = -0.0
    cache = bsp.KvCache.empty(2, hk, page, d)
    pages = i32([[1]])
    bsp.kv_append(cache, nothing, nothing, i32([0, zeros]), i32([0]), pages)
    assert bool((cache.k_scale[1] == 1).all()) and not bool((cache.k[1] & 127).any())
    bsp.kv_append(cache, xt, xt, i32([0, after]), i32([zeros]), pages)
    bsp.device().synchronize()
    e = np.array([ref.exponent(np.abs(x[:, h]).max()) for h in range(hk)])
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        assert np.array_equal(host(scale)[1], 2.0 ** e)
        got = codes.cpu().numpy()[1]
        for h in range(hk):
            assert np.array_equal(got[h, zeros: zeros + after], ref.e4m3(x[:, h].astype(float) * 2.0 ** -e[h]))
        assert not (got[:, :zeros] & 127).any()
    # the smallest code of one earlier token is a value that has to stay
    cache = bsp.KvCache.empty(2, hk, page, d)
    bsp.kv_append(cache, nothing, nothing, i32([0, zeros]), i32([0]), pages)
    cache.k[1, hk - 1, zeros // 2, d - 1] = 129
    bsp.kv_append(cache, xt, xt, i32([0, after]), i32([zeros]), pages)
    bsp.device().synchronize()
    assert float(cache.k_scale[1, hk - 1]) == 1.0 and int(cache.k[1, hk - 1, zeros // 2, d - 1]) == 129
    assert np.array_equal(cache.k.cpu().numpy()[1, hk - 1, zeros: zeros + after], ref.e4m3(x[:, hk - 1].astype(float)))
    assert np.array_equal(host(cache.v_scale)[1], 2.0 ** e)


# ----------------------------------------------------------------- streams --
@pytest.mark.parametrize("as_number", [False, True])
def test_outputs_belong_to_the_calls_stream(bsp, as_number):  # noqa: F811
    """What rope and rope_table allocate comes from the memory of the stream that
    they run on, and goes back to it: the current stream's kernels never had it."""
    torch = torch_()
    s = torch.cuda.Stream()
    given = s.cuda_stream if as_number else s
    x, pos = torch.randn((4099, 3, 64), device="cuda"), i32(np.arange(4099))
    turned = bsp.rope_table(4099, 64)
    torch.cuda.synchronize()
    table = bsp.rope_table(4099, 64, stream=given)
    y = bsp.rope(x, pos, table, stream=given)
    s.synchronize()
    assert torch.equal(y, bsp.rope(x, pos, table)) and torch.equal(table, bsp.rope_table(4099, 64))
    del table, y
    for make in (lambda: bsp.rope_table(4099, 64, stream=given), lambda: bsp.rope(x, pos, turned, stream=given)):
        made = make()
        s.synchronize()
        at, shape = made.data_ptr(), made.shape
        del made
        here = torch.empty(shape, device="cuda")
        with torch.cuda.stream(torch.cuda.ExternalStream(s.cuda_stream)):
            there = torch.empty(shape, device="cuda")
        assert here.data_ptr() != at and there.data_ptr() == at
    bsp.device().synchronize()


def test_first_appends_of_a_device_from_several_threads(bsp):  # noqa: F811
    """The first append on a device sets the kernels up, whichever thread makes it:
    eight at once (each has its stream, cache and tensors) give what one gives."""
    import threading

    torch = torch_()
    x = torch.randn((300, 2, 128), device="cuda").bfloat16()
    pages, starts, before = i32(np.arange(19)[None]), i32([0, 300]), i32([0])
    one = bsp.KvCache.empty(19, 2, 16, 128)
    bsp.kv_append(one, x, x, starts, before, pages)
    torch.cuda.synchronize()
    for _ in range(5):
        dev = bsp.Device(0)
        caches, streams = [bsp.KvCache.empty(19, 2, 16, 128) for _ in range(8)], [torch.cuda.Stream() for _ in range(8)]
        torch.cuda.synchronize()
        together, failed = threading.Barrier(8), []

        def call(i):
            try:
                together.wait(30)
                bsp.kv_append(caches[i], x, x, starts, before, pages, dev=dev, stream=streams[i])
            except Exception as e:
                failed.append(e)

        threads = [threading.Thread(target=call, args=(i,)) for i in range(8)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        dev.synchronize()
        torch.cuda.synchronize()
        assert not failed
        assert all(torch.equal(c.k, one.k) and torch.equal(c.v_scale, one.v_scale) for c in caches)
        dev.close()
