"""Rotary positions, the paged 8-bit cache, prompt attention and single-token
attention on the GPU against plain 64-bit forms (decoder_ref.py).

Tolerances, from the arithmetic:
  rotary f32    two products and a sum: 2^-23 (|a c| + |b s|); bf16 adds 2^-8 of
                the result;
  cache         codes equal those of the 64-bit form except where its value is
                within 2^-20 of a rounding boundary (32-bit rotation before it);
  attention     O is rounded to bf16 (2^-8 |o|); each weight to bf16 (prompt) or
                fp16 (decode): u sum(p |v|); scores in fp32: a relative error of
                the weights of 2^-16 (1 + scale sum |q k|), the same for lse.
"""
import numpy as np
import pytest

import decoder_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def bsp():
    import bsp as b

    return b


def torch_():
    import torch

    return torch


def cuda(x, dtype=None):
    torch = torch_()
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t if dtype is None else t.to(dtype)


def host(t):
    return t.detach().double().cpu().numpy()


def i32(x):
    return cuda(np.asarray(x, np.int32))


def spread(x, rng, pad_heads=1, pad_tokens=0):
    """The same values as a view with larger strides; NaN between."""
    torch = torch_()
    t, h, d = x.shape
    big = torch.full((t, h + pad_heads, d + 8), float("nan"), dtype=x.dtype, device="cuda")
    big[:, :h, :d] = x
    return big[:, :h, :d]


# ------------------------------------------------------------------ rotary --
@pytest.mark.parametrize("kind,kw", [("none", {}), ("linear", dict(factor=4.0)), ("base", dict(factor=8.0)),
                                     ("parts", dict(factor=8.0, context=4096.0, slow=1.0, fast=32.0, magnitude=1.2))])
@pytest.mark.parametrize("rot", [16, 64, 128])
def test_rope_table(bsp, kind, kw, rot):
    n = 3001
    t = host(bsp.rope_table(n, rot, base=10000.0, kind=kind, **kw))
    a = np.arange(n)[:, None] * ref.frequencies(rot, 10000.0, kind, **{k: v for k, v in kw.items() if k != "magnitude"})
    gold = np.stack([np.cos(a), np.sin(a)], -1) * kw.get("magnitude", 1.0)
    # one rounding to 32 bits, and the 64-bit angle's own error (2^-50 of up to 3000)
    assert np.abs(t - gold).max() <= 2.0 ** -24 * 1.2 + 1e-11


def test_rope_table_far_position(bsp):
    t = bsp.rope_table(1 << 20, 16)
    a = float((1 << 20) - 1) * ref.frequencies(16)
    assert np.abs(host(t[-1]) - np.stack([np.cos(a), np.sin(a)], -1)).max() <= 2.0 ** -24 + 1e-9


ROPE = [(1, 1, 16, 16), (3, 5, 64, 64), (7, 8, 128, 64), (33, 3, 96, 32), (300, 4, 128, 128), (2, 2, 512, 512), (129, 40, 256, 128)]


@pytest.mark.parametrize("tokens,heads,d,rot", ROPE)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("transpose", [False, True])
def test_rope(bsp, tokens, heads, d, rot, layout, dtype, transpose):
    torch = torch_()
    rng = np.random.default_rng(tokens * 7 + d)
    x = rng.normal(0, 1, (tokens, heads, d)).astype(np.float32)
    x = x if dtype == "f32" else ref.bf16(x)
    pos = rng.integers(0, 5000, tokens).astype(np.int32)
    table = bsp.rope_table(5000, rot)
    xt = cuda(x, torch.float32 if dtype == "f32" else torch.bfloat16)
    gold = ref.rotate(x, host(table), pos, layout, transpose)
    size = ref.rotate(np.abs(x), np.abs(host(table)) * [1, -1], pos, layout, False)  # |a c| + |b s| of the first of a pair
    size = np.maximum(np.abs(size), np.abs(ref.rotate(np.abs(x), np.abs(host(table)), pos, layout, False)))
    tol = 2.0 ** -23 * 2 * size + (0 if dtype == "f32" else ref.U16 * np.abs(gold)) + 1e-30
    out = bsp.rope(xt, i32(pos), table, layout=layout, transpose=transpose)
    assert (np.abs(host(out) - gold) <= tol).all()
    strided = spread(xt, rng)
    out2 = spread(torch.zeros_like(xt), rng)
    bsp.rope(strided, i32(pos), table, layout=layout, transpose=transpose, out=out2)
    assert torch.equal(out2, out)
    assert torch.isnan(torch.as_strided(out2, (tokens, heads + 1, d + 8), ((heads + 1) * (d + 8), d + 8, 1))[:, heads]).all()
    bsp.rope(xt, i32(pos), table, layout=layout, transpose=transpose, out=xt)  # in place
    assert torch.equal(xt, out)
    bsp.device().synchronize()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_gradient(bsp, layout):
    """The transposed rotation is the gradient: against differences of
    sum(g * rope(x)), which is linear in x, so they have only rounding errors
    (2^-23 of the 64 terms of the sum, over the step)."""
    torch = torch_()
    rng = np.random.default_rng(5)
    x, g = (rng.normal(0, 1, (2, 1, 64)).astype(np.float32) for _ in range(2))
    pos, table = i32([3, 77]), bsp.rope_table(100, 32, kind="parts", factor=4.0, context=64.0, magnitude=1.3)
    grad = host(bsp.rope(cuda(g), pos, table, layout=layout, transpose=True))
    f = lambda y: float((host(bsp.rope(cuda(y), pos, table, layout=layout)) * g).sum())  # noqa: E731
    for k in range(x.size):
        e = np.zeros(x.size, np.float32)
        e[k] = 0.5
        e = e.reshape(x.shape)
        d = (f(x + e) - f(x - e)) / 1.0
        assert abs(d - grad.reshape(-1)[k]) <= 2.0 ** -23 * 8 * 64


def test_rope_nothing_and_bad_position(bsp):
    torch = torch_()
    table = bsp.rope_table(8, 16)
    x = torch.ones((0, 2, 16), device="cuda", dtype=torch.bfloat16)
    assert bsp.rope(x, i32(np.zeros(0)), table).shape == (0, 2, 16)
    x = torch.ones((3, 2, 16), device="cuda", dtype=torch.bfloat16)
    y = torch.full_like(x, 7)
    bsp.rope(x, i32([0, 8, -1]), table, out=y)
    with pytest.raises(bsp.BspError, match="outside its table"):
        bsp.device().synchronize()
    assert (y[0] == 1).all() and (y[1:] == 7).all()
    bsp.device().synchronize()


# ------------------------------------------------------------------- cache --
def make_cache(bsp, rng, n_pages, hk, page, d, strided=False):
    torch = torch_()
    codes = [ref.e4m3(np.clip(rng.normal(0, 100, (n_pages, hk, page, d)), -448, 448)) for _ in range(2)]
    scales = [(2.0 ** rng.integers(-9, -5, (n_pages, hk))).astype(np.float32) for _ in range(2)]
    if strided:  # K and V of a page side by side
        both = torch.full((n_pages, 2, hk, page, d), 127, dtype=torch.uint8, device="cuda")
        k, v = both[:, 0], both[:, 1]
        k.copy_(cuda(codes[0]))
        v.copy_(cuda(codes[1]))
    else:
        k, v = cuda(codes[0]), cuda(codes[1])
    cache = bsp.KvCache(k, v, cuda(scales[0]), cuda(scales[1]))
    return cache, codes, [s.astype(np.float64) for s in scales]


def page_table(rng, tokens, page, n_pages):
    per = [-(-t // page) for t in tokens]
    order = rng.permutation(n_pages)[: sum(per)]
    width = max(per + [1]) + 1
    t, at = np.full((len(per), width), -1, np.int32), 0
    for s, n in enumerate(per):
        t[s, :n] = order[at: at + n]
        at += n
    return t


def near_boundary(x, e):
    """Where 2^-20 of x decides the code of x 2^-e."""
    y = x * 2.0 ** -e
    return ref.e4m3(y * (1 - 2.0 ** -20)) != ref.e4m3(y * (1 + 2.0 ** -20))


APPEND = [
    # new, before, kv heads, query heads, page, d, rot
    ([1], [0], 1, 1, 16, 64, 64),
    ([1, 1, 1], [0, 15, 16], 2, 4, 16, 128, 128),
    ([1, 0, 5, 16, 17], [31, 7, 30, 16, 15], 3, 3, 16, 128, 64),
    ([70, 1, 0, 64], [3, 63, 0, 0], 2, 10, 64, 128, 128),
    ([33, 200], [95, 0], 1, 8, 32, 64, 32),
    ([129, 300, 1], [127, 1, 255], 2, 2, 128, 128, 128),
    ([1] * 40, list(range(40)), 8, 32, 64, 128, 128),
    ([1] * 30 + [150], [5] * 30 + [37], 2, 6, 64, 128, 64),   # a prompt among single tokens
    ([1] * 20 + [200, 17], [100] * 20 + [90, 0], 1, 3, 128, 64, 64),
    # more sequences than blocks fit at once, no more tokens than sequences
    ([1] * 310, [7 * i % 70 for i in range(310)], 1, 2, 16, 128, 128),
    ([0] * 220 + [70, 0, 40, 3] + [1] * 170, [3] * 394, 2, 3, 128, 128, 64),
    ([0] * 200 + [100] + [1] * 190, [30] * 391, 1, 1, 128, 64, 64),
]


@pytest.mark.parametrize("new,before,hk,hq,page,d,rot", APPEND, ids=[f"n{sum(c[0])}_p{c[4]}_d{c[5]}_h{c[2]}" for c in APPEND])
@pytest.mark.parametrize("layout", ["half", "interleaved", "none"])
def test_append(bsp, new, before, hk, hq, page, d, rot, layout):
    torch = torch_()
    rng = np.random.default_rng(sum(new) + page + d)
    tokens = sum(new)
    n_pages = sum(-(-(a + b) // page) for a, b in zip(new, before)) + 2
    cache, codes, scales = make_cache(bsp, rng, n_pages, hk, page, d, strided=layout == "interleaved")
    pages = page_table(rng, [a + b for a, b in zip(new, before)], page, n_pages)
    q, k, v = (ref.bf16(rng.normal(0, 1, (tokens, h, d)) * 3) for h in (hq, hk, hk))
    k[:, :, ::16] *= 8  # strong channels; some pages grow, some do not
    starts = np.concatenate([[0], np.cumsum(new)])
    tt = [cuda(x, torch.bfloat16) for x in (q, k, v)]
    kw = {}
    if layout != "none":
        table = bsp.rope_table(1000, rot)
        pos = np.concatenate([np.arange(b, b + n) for n, b in zip(new, before)]).astype(int)
        gq, gk = (ref.rotate(x, host(table), pos, layout) for x in (q, k))
        kw = dict(table=table, layout=layout, q=spread(tt[0], rng), q_out=torch.empty_like(tt[0]),
                  k_out=torch.empty_like(tt[1]))
    else:
        gk = k.astype(np.float64)
    bsp.kv_append(cache, spread(tt[1], rng), spread(tt[2], rng), i32(starts), i32(before), cuda(pages), **kw)
    bsp.device().synchronize()
    if layout != "none":
        for out, gold in ((kw["q_out"], gq), (kw["k_out"], gk)):
            assert (np.abs(host(out) - gold) <= ref.U16 * np.abs(gold) + 2.0 ** -22 * 40).all()
    for c, s, x, got, gots in ((codes[0], scales[0], gk, cache.k, cache.k_scale),
                               (codes[1], scales[1], v.astype(np.float64), cache.v, cache.v_scale)):
        ref.append(c, s, x, starts, before, pages)
        assert np.array_equal(host(gots), s)
        differ = got.cpu().numpy() != c
        if differ.any():  # only new tokens whose 64-bit value sits on a boundary
            ok = np.zeros_like(differ)
            at = 0
            for i, n in enumerate(new):
                for j in range(n):
                    p, slot = pages[i][(before[i] + j) // page], (before[i] + j) % page
                    ok[p, :, slot] = near_boundary(x[at], np.log2(s[p])[:, None])
                    at += 1
            assert not (differ & ~ok).any()


def test_append_in_place_and_growth(bsp):
    """Token by token with rising size: every append re-rounds the page; then
    k_out and q_out on top of k and q."""
    torch = torch_()
    rng = np.random.default_rng(3)
    cache = bsp.KvCache.empty(3, 1, 16, 64)
    codes, scales = np.zeros((3, 1, 16, 64), np.uint8), np.ones((3, 1))
    pages = np.array([[2, 0]], np.int32)
    for t in range(20):
        x = ref.bf16(rng.normal(0, 1, (1, 1, 64)) * 2.0 ** (t - 3))
        xt = cuda(x, torch.bfloat16)
        bsp.kv_append(cache, xt, xt, i32([0, 1]), i32([t]), cuda(pages))
        ref.append(codes, scales, x.astype(np.float64), [0, 1], [t], pages)
        assert np.array_equal(cache.k.cpu().numpy(), codes) and np.array_equal(cache.v.cpu().numpy(), codes)
        assert np.array_equal(host(cache.k_scale), scales)
    table = bsp.rope_table(64, 64)
    q, k = (cuda(ref.bf16(rng.normal(0, 1, (12, 2, 64))), torch.bfloat16) for _ in range(2))
    k = k[:, :1]
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    a = (k, k, i32([0, 12]), i32([16]), cuda(np.array([[2, 0, 1]], np.int32)))
    bsp.kv_append(cache, *a, table=table, q=q, q_out=qo, k_out=ko)
    was = cache.k.clone()
    v = k.clone()
    bsp.kv_append(cache, k, v, *a[2:], table=table, q=q, q_out=q, k_out=k)
    assert torch.equal(q, qo) and torch.equal(k, ko) and torch.equal(cache.k, was)
    bsp.device().synchronize()


def test_append_values_that_are_not_finite(bsp):
    torch = torch_()
    x = np.zeros((16, 1, 64), np.float32)
    x[:] = ref.bf16(np.random.default_rng(1).normal(0, 1, x.shape))
    x[3, 0, 5], x[4, 0, 6], x[5, 0, 7], x[6, 0, 8] = np.inf, -np.inf, np.nan, 3e38
    cache = bsp.KvCache.empty(1, 1, 16, 64)
    xt = cuda(x, torch.bfloat16)
    bsp.kv_append(cache, xt, xt, i32([0, 16]), i32([0]), i32([[0]]))
    codes, scales = np.zeros((1, 1, 16, 64), np.uint8), np.ones((1, 1))
    ref.append(codes, scales, host(xt), [0, 16], [0], [[0]])
    got = cache.k.cpu().numpy()
    assert np.array_equal(got & 127, codes & 127) and np.array_equal(host(cache.k_scale), scales)
    assert [got[0, 0, t, 2 + t] & 127 for t in (3, 4, 5)] == [127] * 3
    # zeros alone keep scale 1; subnormal and huge values have a scale in range
    for size in (0.0, 1e-40, 3e38):
        y = torch.full((16, 1, 64), size, device="cuda").bfloat16()
        bsp.kv_append(cache, y, y, i32([0, 16]), i32([0]), i32([[0]]))
        s = float(cache.k_scale[0, 0])
        assert s == 2.0 ** ref.exponent(float(y[0, 0, 0])) and (size != 0 or s == 1.0)
    bsp.device().synchronize()


def test_append_bad_indices(bsp):
    """Pages, starts, lengths and positions outside their tables write nothing."""
    torch = torch_()
    cache = bsp.KvCache.empty(2, 1, 16, 64)
    x = torch.ones((4, 1, 64), device="cuda", dtype=torch.bfloat16)
    table = bsp.rope_table(8, 64)
    for starts, before, pages, kw in (([0, 4], [0], [[2]], {}), ([0, 4], [0], [[-1]], {}), ([0, 4], [16], [[0]], {}),
                                      ([0, 5], [0], [[0]], {}), ([3, 1], [0], [[0]], {}), ([-4, 0], [0], [[0]], {}),
                                      ([0, 4], [-3], [[0]], {}), ([0, 4], [5], [[0]], dict(table=table)),
                                      ([0, 2 ** 31 - 1], [0], [[0]], {}), ([0, 4], [2 ** 31 - 1], [[0]], {})):
        bsp.kv_append(cache, x, x, i32(starts), i32(before), cuda(np.array(pages, np.int32)), **kw)
        with pytest.raises(bsp.BspError, match="outside its table"):
            bsp.device().synchronize()
        assert not cache.k.any() and not cache.v.any() and (cache.k_scale == 1).all()


# ------------------------------------------------------------------ prompt --
def check_attention(o, lse, gold, glse, weight, size, u):
    o, lse = host(o), host(lse)
    assert np.isfinite(o).all()
    tol = ref.U16 * np.abs(gold) + (u + 2.0 ** -16 * (1 + size)) * 1.05 * weight + 1e-30
    bad = np.abs(o - gold) > tol
    assert not bad.any(), (int(bad.sum()), float((np.abs(o - gold) / tol).max()))
    assert np.array_equal(np.isneginf(lse), np.isneginf(glse))
    fin = np.isfinite(glse)
    assert (np.abs(lse[fin] - glse[fin]) <= 2.0 ** -16 * (1 + size[..., 0][fin])).all()


def prompt_gold(q, k, v, ql, kl, hk, scale, causal):
    group = q.shape[1] // hk
    gold, lse = np.zeros(q.shape), np.zeros(q.shape[:2])
    weight, size = np.zeros(q.shape), np.zeros(q.shape[:2] + (1,))
    a = b = 0
    for n, m in zip(ql, kl):
        for h in range(q.shape[1]):
            qq, kk, vv = q[a: a + n, h], k[b: b + m, h // group], v[b: b + m, h // group]
            sees = np.arange(n) + m - n + 1 if causal else np.full(n, m)
            gold[a: a + n, h], lse[a: a + n, h], weight[a: a + n, h] = ref.attention(qq, kk, vv, scale, sees)
            if m:
                size[a: a + n, h, 0] = scale * (np.abs(qq) @ np.abs(kk).T).max(1)
        a, b = a + n, b + m
    return gold, lse, weight, size


PROMPT = [
    # q lengths, kv lengths, heads, kv heads, d
    ([1], [1], 1, 1, 64),
    ([1], [129], 8, 1, 128),
    ([37], [37], 8, 2, 64),
    ([128, 129, 127], [128, 129, 127], 4, 4, 128),
    ([0, 5, 0, 300, 1], [3, 5, 0, 300, 700], 6, 2, 128),
    ([257, 40], [200, 10], 5, 1, 64),           # more queries than keys: the first see nothing
    ([40], [0], 2, 1, 128),                     # no key at all
    ([1, 1, 1, 1], [1, 64, 128, 1000], 32, 2, 128),
    ([513], [1100], 16, 16, 64),
    ([2, 700, 33], [2, 800, 33], 40, 8, 128),
    ([3000], [3000], 3, 1, 128),
    ([90], [90], 64, 1, 64),
]


@pytest.mark.parametrize("ql,kl,hq,hk,d", PROMPT, ids=[f"q{sum(c[0])}_kv{sum(c[1])}_h{c[2]}_{c[3]}_d{c[4]}" for c in PROMPT])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt(bsp, ql, kl, hq, hk, d, causal):
    torch = torch_()
    rng = np.random.default_rng(sum(ql) * 3 + sum(kl) + hq)
    q = ref.bf16(rng.normal(0, 1, (sum(ql), hq, d)))
    k, v = (ref.bf16(rng.normal(0, 1, (sum(kl), hk, d))) for _ in range(2))
    plan = bsp.PromptPlan(bsp.device(), ql, kl, hq, hk, d, causal=causal)
    qt, kt, vt = (cuda(x, torch.bfloat16) for x in (q, k, v))
    o = torch.full_like(qt, float("nan"))
    lse = torch.full((sum(ql), hq), float("nan"), device="cuda")
    plan.execute(qt, kt, vt, o, lse=lse)
    bsp.device().synchronize()
    gold, glse, weight, size = prompt_gold(q.astype(float), k.astype(float), v.astype(float), ql, kl, hk,
                                           1 / np.sqrt(d), causal)
    check_attention(o, lse, gold, glse, weight, size, ref.U16)
    # strided operands and no lse: the same bits
    o2 = spread(torch.zeros_like(o), rng)
    plan.execute(spread(qt, rng), spread(kt, rng), spread(vt, rng), o2)
    assert torch.equal(o2, o)
    # another stream, few CTAs
    small = bsp.PromptPlan(bsp.device(), ql, kl, hq, hk, d, causal=causal, opts=bsp.make_opts(max_ctas=3))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    o3 = torch.zeros_like(o)
    small.execute(qt, kt, vt, o3, lse=lse, stream=s)
    s.synchronize()
    check_attention(o3, lse, gold, glse, weight, size, ref.U16)
    bsp.device().synchronize()


CUT = [
    ([16], [5000], 8, 2, 128, True),
    ([1], [20011], 4, 4, 64, True),
    ([3, 1, 130], [700, 9001, 130], 6, 2, 64, True),
    ([2100], [1500], 2, 1, 128, True),          # the first 600 queries see no key
    ([1500], [1500], 5, 1, 128, True),          # rows that see keys of the first parts only
    ([40, 200], [4097, 3000], 3, 1, 128, False),
    ([1500], [1500], 4, 1, 64, False),
]


@pytest.mark.parametrize("ql,kl,hq,hk,d,causal", CUT, ids=[f"q{sum(c[0])}_kv{sum(c[1])}_d{c[4]}_{c[5]}" for c in CUT])
def test_prompt_cut_keys(bsp, ql, kl, hq, hk, d, causal):
    """Few rows of many keys: the keys are cut into parts that a second kernel
    joins.  The same values as the whole up to rounding, the same bits again."""
    torch = torch_()
    rng = np.random.default_rng(sum(kl))
    q = ref.bf16(rng.normal(0, 1, (sum(ql), hq, d)))
    k, v = (ref.bf16(rng.normal(0, 1, (sum(kl), hk, d))) for _ in range(2))
    k *= np.float32(1 + 3 * (np.arange(len(k)) % 997 > 900))[:, None, None]  # parts of different weight
    k = ref.bf16(k)
    plan = bsp.PromptPlan(bsp.device(), ql, kl, hq, hk, d, causal=causal)
    assert plan.info()["workspace_bytes"] > 0
    qt, kt, vt = (cuda(x, torch.bfloat16) for x in (q, k, v))
    gold = prompt_gold(q.astype(float), k.astype(float), v.astype(float), ql, kl, hk, 1 / np.sqrt(d), causal)
    o, lse = torch.full_like(qt, float("nan")), torch.full((sum(ql), hq), float("nan"), device="cuda")
    plan.execute(qt, kt, vt, o, lse=lse)
    bsp.device().synchronize()
    check_attention(o, lse, *gold, ref.U16)
    o2, lse2 = spread(torch.zeros_like(o), rng), torch.zeros_like(lse)
    for _ in range(3):
        plan.execute(spread(qt, rng), spread(kt, rng), spread(vt, rng), o2, lse=lse2)
        assert torch.equal(o2, o) and torch.equal(lse2, lse)
    plan.execute(qt, kt, vt, o2)  # no lse
    assert torch.equal(o2, o)
    # few CTAs, so other parts; and whole
    for kw in (dict(max_ctas=20), dict(group_rows=-1)):
        other = bsp.PromptPlan(bsp.device(), ql, kl, hq, hk, d, causal=causal, opts=bsp.make_opts(**kw))
        other.execute(qt, kt, vt, o2, lse=lse2)
        bsp.device().synchronize()
        check_attention(o2, lse2, *gold, ref.U16)
    assert other.info()["workspace_bytes"] == 0


@pytest.mark.parametrize("at", [0, 127, 128, 1000, 2999])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_prompt_cut_bad_key(bsp, at, bad):
    """A bad key in one part makes the joined rows that see it NaN, and no other."""
    torch = torch_()
    n, m, d = 600, 3000, 128
    rng = np.random.default_rng(5)
    q = ref.bf16(np.abs(rng.normal(0, 1, (n, 1, d))) + 0.1)
    k, v = (ref.bf16(rng.normal(0, 1, (m, 1, d))) for _ in range(2))
    plan = bsp.PromptPlan(bsp.device(), [n], [m], 1, 1, d)
    assert plan.info()["workspace_bytes"] > 0
    gold = prompt_gold(q.astype(float), k.astype(float), v.astype(float), [n], [m], 1, 1 / np.sqrt(d), True)
    qt, kt, vt = (cuda(x, torch.bfloat16) for x in (q, k, v))
    kt[at, 0, 5] = bad
    o, lse = torch.empty_like(qt), torch.empty((n, 1), device="cuda")
    plan.execute(qt, kt, vt, o, lse=lse)
    bsp.device().synchronize()
    first = max(0, at - (m - n))  # the first query that sees the key
    if first:
        check_attention(o[:first], lse[:first], *(x[:first] for x in gold), ref.U16)
    assert torch.isnan(o[first:]).all() and torch.isnan(lse[first:]).all()


@pytest.mark.parametrize("scale", [1e-3, 30.0])
def test_prompt_scales_and_rising_scores(bsp, scale):
    """Flat and one-hot softmax, and scores that rise along the keys so that
    the running maximum moves on every step."""
    torch = torch_()
    n, d = 700, 128
    rng = np.random.default_rng(2)
    q = ref.bf16(np.abs(rng.normal(0, 1, (n, 2, d))))
    k = ref.bf16(np.arange(n)[:, None, None] / 64.0 * np.ones((n, 1, d)) / 16)
    v = ref.bf16(rng.normal(0, 1, (n, 1, d)))
    plan = bsp.PromptPlan(bsp.device(), [n], [n], 2, 1, d)
    o, lse = torch.empty((n, 2, d), device="cuda", dtype=torch.bfloat16), torch.empty((n, 2), device="cuda")
    plan.execute(cuda(q, torch.bfloat16), cuda(k, torch.bfloat16), cuda(v, torch.bfloat16), o, scale=scale, lse=lse)
    bsp.device().synchronize()
    gold, glse, weight, size = prompt_gold(q.astype(float), k.astype(float), v.astype(float), [n], [n], 1, scale, True)
    check_attention(o, lse, gold, glse, weight, size, ref.U16)


def test_prompt_huge_scores(bsp):
    """Scores of 10^10, far above 2^24: the largest key takes all."""
    torch = torch_()
    n, d = 200, 64
    q = torch.full((n, 1, d), 1e5, device="cuda").bfloat16()
    k = (torch.arange(n, device="cuda")[:, None, None] * 100.0 * torch.ones((n, 1, d), device="cuda")).bfloat16()
    v = torch.randn((n, 1, d), device="cuda").bfloat16()
    plan = bsp.PromptPlan(bsp.device(), [n], [n], 1, 1, d)
    o = torch.empty_like(q)
    plan.execute(q, k, v, o, scale=1.0)
    bsp.device().synchronize()
    # k is rounded to bf16, so neighbours may tie: the mean of the tied values
    kk = k[:, 0, 0].float()
    gold = torch.stack([v[: i + 1, 0][kk[: i + 1] == kk[: i + 1].max()].float().mean(0) for i in range(n)])
    assert (o[:, 0].float() - gold).abs().max() <= 2 * ref.U16 * v.abs().max().float()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_prompt_neighbours_do_not_leak(bsp, bad):
    """Infinities and NaN in the keys, values and queries of one sequence
    change nothing in the others."""
    torch = torch_()
    ql, d = [100, 60, 200], 128
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn((sum(ql), h, d), device="cuda", generator=g).bfloat16() for h in (4, 2, 2))
    plan = bsp.PromptPlan(bsp.device(), ql, ql, 4, 2, d)
    o, o2 = torch.empty_like(q), torch.empty_like(q)
    plan.execute(q, k, v, o)
    for x in (q, k, v):
        x[100:160] = bad
    plan.execute(q, k, v, o2)
    bsp.device().synchronize()
    keep = torch.ones(sum(ql), dtype=torch.bool)
    keep[100:160] = False
    assert torch.equal(o2[keep], o[keep]) and torch.isnan(o2[~keep]).any()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_prompt_bad_key_makes_its_rows_nan(bsp, d, bad):
    """A key that is NaN (or gives an infinite score) makes the rows that see
    it NaN, at whichever place of a step it stands; the rows before are right."""
    torch = torch_()
    n = 300
    rng = np.random.default_rng(3)
    q = ref.bf16(np.abs(rng.normal(0, 1, (n, 2, d))) + 0.1)
    k, v = (ref.bf16(rng.normal(0, 1, (n, 1, d))) for _ in range(2))
    gold = prompt_gold(q.astype(float), k.astype(float), v.astype(float), [n], [n], 1, 1 / np.sqrt(d), True)
    plan = bsp.PromptPlan(bsp.device(), [n], [n], 2, 1, d)
    qt, kt, vt = (cuda(x, torch.bfloat16) for x in (q, k, v))
    o, lse = torch.empty_like(qt), torch.empty((n, 2), device="cuda")
    for at in list(range(0, 20)) + [31, 32, 63, 64, 77, 96, 127, 128, 129, 200, 299]:
        k2 = kt.clone()
        k2[at, 0, 5] = bad
        plan.execute(qt, k2, vt, o, lse=lse)
        if at:
            check_attention(o[:at], lse[:at], *(x[:at] for x in gold), ref.U16)
        assert torch.isnan(o[at:]).all() and torch.isnan(lse[at:]).all(), at
    bsp.device().synchronize()


def test_plans_outlive_their_device(bsp):
    """A plan destroyed after its device was closed frees its memory."""
    dev = bsp.Device(0)
    plans = [bsp.PromptPlan(dev, [5], [5], 2, 1, 64), bsp.DecodePlan(dev, 3, 2, 1, 64, 16)]
    dev.close()
    for p in plans:
        p.close()
    torch_().cuda.synchronize()


# ------------------------------------------------------------------ decode --
DECODE = [
    # lengths, heads, kv heads, d, page
    ([1], 1, 1, 64, 16),
    ([1, 0, 15, 16, 17, 63, 64, 65, 0], 8, 2, 128, 16),
    ([127, 128, 129, 300, 1000], 5, 1, 128, 64),
    ([33, 70, 500], 16, 1, 64, 32),
    ([257, 4000], 20, 1, 128, 128),             # more than 16 query heads share a key/value head
    ([999] * 3 + [1], 32, 32, 64, 16),
    ([20000], 8, 1, 128, 64),                   # one row over many CTAs
    ([5, 9000, 31], 24, 3, 128, 32),
    ([64, 3] * 50, 4, 2, 64, 128),
]


def decode_gold(q, codes, scales, lens, pages, hk, scale):
    group = q.shape[1] // hk
    n, hq, d = q.shape
    gold, lse, weight, size = np.zeros(q.shape), np.zeros((n, hq)), np.zeros(q.shape), np.zeros((n, hq, 1))
    page = codes[0].shape[2]
    for s, m in enumerate(lens):
        use = pages[s][: -(-m // page)]
        k, v = ((ref.VALUES[c[use]] * x[use][:, :, None, None]).transpose(1, 0, 2, 3).reshape(hk, -1, d)[:, :m]
                for c, x in zip(codes, scales))
        for h in range(hq):
            qq, kk = q[s, h][None], k[h // group]
            gold[s, h], lse[s, h], weight[s, h] = (x[0] for x in ref.attention(qq, kk, v[h // group], scale, [m]))
            if m:
                size[s, h, 0] = scale * (np.abs(qq) @ np.abs(kk).T).max()
    return gold, lse, weight, size


@pytest.mark.parametrize("lens,hq,hk,d,page", DECODE, ids=[f"n{len(c[0])}_t{sum(c[0])}_h{c[1]}_{c[2]}_d{c[3]}_p{c[4]}" for c in DECODE])
@pytest.mark.parametrize("strided", [False, True])
def test_decode(bsp, lens, hq, hk, d, page, strided):
    torch = torch_()
    rng = np.random.default_rng(sum(lens) + hq)
    n_pages = sum(-(-t // page) for t in lens) + 2
    cache, codes, scales = make_cache(bsp, rng, n_pages, hk, page, d, strided)
    pages = page_table(rng, lens, page, n_pages)
    # behind the last token the page holds whatever it held: NaN codes here
    for s, m in enumerate(lens):
        if m % page:
            for c in (cache.k, cache.v):
                c[int(pages[s][m // page]), :, m % page:] = 127
    q = ref.bf16(rng.normal(0, 1, (len(lens), hq, d)))
    qt = cuda(q, torch.bfloat16)
    o, lse = torch.full_like(qt, float("nan")), torch.full((len(lens), hq), float("nan"), device="cuda")
    gold, glse, weight, size = decode_gold(q.astype(float), codes, scales, lens, pages, hk, 1 / np.sqrt(d))
    for ctas in (0, 1, 7, 50):  # the rows are cut in different places
        plan = bsp.DecodePlan(bsp.device(), len(lens) + 3, hq, hk, d, page, opts=bsp.make_opts(max_ctas=ctas))
        for again in range(2):
            o.fill_(float("nan"))
            lse.fill_(float("nan"))
            plan.execute(cache, spread(qt, rng) if strided else qt, i32(lens), cuda(pages), o, lse=lse)
            bsp.device().synchronize()
            check_attention(o, lse, gold, glse, weight, size, 2 * ref.UH)
            if again:  # the same bits, whichever CTA finishes last
                assert torch.equal(o, first)
            first = o.clone()
    o2 = spread(torch.zeros_like(o), rng)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    plan.execute(cache, qt, i32(lens), cuda(pages), o2, stream=s)
    s.synchronize()
    assert torch.equal(o2, o)


def test_decode_scales_far_apart(bsp):
    """Pages whose value scales differ by 2^12, keys whose scales differ too,
    and one-hot rows."""
    torch = torch_()
    rng = np.random.default_rng(9)
    lens, hq, hk, d, page = [500, 100], 4, 2, 128, 16
    n_pages = 40
    cache, codes, scales = make_cache(bsp, rng, n_pages, hk, page, d)
    scales = [(2.0 ** rng.integers(-16, -4, (n_pages, hk))) for _ in range(2)]
    cache.k_scale.copy_(cuda(scales[0].astype(np.float32)))
    cache.v_scale.copy_(cuda(scales[1].astype(np.float32)))
    pages = page_table(rng, lens, page, n_pages)
    q = ref.bf16(rng.normal(0, 1, (2, hq, d)) * np.array([1e-6, 1.0, 300.0, 1e4])[None, :, None])
    o, lse = torch.empty((2, hq, d), device="cuda", dtype=torch.bfloat16), torch.empty((2, hq), device="cuda")
    plan = bsp.DecodePlan(bsp.device(), 2, hq, hk, d, page)
    plan.execute(cache, cuda(q, torch.bfloat16), i32(lens), cuda(pages), o, lse=lse)
    bsp.device().synchronize()
    gold, glse, weight, size = decode_gold(q.astype(float), codes, scales, lens, pages, hk, 1 / np.sqrt(d))
    # weights below 2^-14 of the largest (weight x value scale) lose bits: 2^-24 of it
    top = np.array([448 * scales[1][pages[s][: -(-m // page)]].max() for s, m in enumerate(lens)])
    weight = weight + 2.0 ** -13 * top[:, None, None]
    check_attention(o, lse, gold, glse, weight, size, 2 * ref.UH)


def test_decode_nan_stays_in_its_row(bsp):
    """A NaN code in a key or a value reaches the heads and sequences that read
    it (a value: its column) and no others."""
    torch = torch_()
    rng = np.random.default_rng(6)
    lens, hq, hk, d, page = [200, 300, 150], 4, 2, 64, 32
    cache, _, _ = make_cache(bsp, rng, 30, hk, page, d)
    pages = page_table(rng, lens, page, 30)
    q = cuda(ref.bf16(rng.normal(0, 1, (3, hq, d))), torch.bfloat16)
    plan = bsp.DecodePlan(bsp.device(), 3, hq, hk, d, page)
    o, o2 = torch.empty_like(q), torch.empty_like(q)
    plan.execute(cache, q, i32(lens), cuda(pages), o)
    k = cache.k.clone()
    cache.k[int(pages[1][4]), 1, 7, 3] = 127
    plan.execute(cache, q, i32(lens), cuda(pages), o2)
    assert torch.isnan(o2[1, 2:]).all() and torch.equal(o2[1, :2], o[1, :2]) and torch.equal(o2[[0, 2]], o[[0, 2]])
    cache.k.copy_(k)
    cache.v[int(pages[1][4]), 1, 7, 3] = 127
    plan.execute(cache, q, i32(lens), cuda(pages), o2)
    hit = torch.zeros_like(o, dtype=torch.bool)
    hit[1, 2:, 3] = True
    assert torch.isnan(o2[hit]).all() and torch.equal(o2[~hit], o[~hit])
    bsp.device().synchronize()


def test_decode_far_pages(bsp):
    """A cache whose pages lie more than 2^32 bytes from its start."""
    torch = torch_()
    rng = np.random.default_rng(4)
    hk, page, d, far = 1, 16, 64, 1 << 28
    n_pages = 20
    big = [torch.zeros(far * n_pages, dtype=torch.uint8, device="cuda") for _ in range(2)]
    k, v = (torch.as_strided(b, (n_pages, hk, page, d), (far, page * d, d, 1)) for b in big)
    codes = [ref.e4m3(np.clip(rng.normal(0, 100, (n_pages, hk, page, d)), -448, 448)) for _ in range(2)]
    k.copy_(cuda(codes[0]))
    v.copy_(cuda(codes[1]))
    scales = [np.full((n_pages, hk), 2.0 ** -7) for _ in range(2)]
    cache = bsp.KvCache(k, v, *(cuda(s.astype(np.float32)) for s in scales))
    pages = rng.permutation(n_pages)[None].astype(np.int32)
    x = ref.bf16(rng.normal(0, 1, (3, 1, d)))
    bsp.kv_append(cache, cuda(x, torch.bfloat16), cuda(x, torch.bfloat16), i32([0, 3]), i32([300]), cuda(pages))
    for c, s in zip(codes, scales):
        ref.append(c, s, x.astype(float), [0, 3], [300], pages)
    assert np.array_equal(k.cpu().numpy(), codes[0]) and np.array_equal(v.cpu().numpy(), codes[1])
    q = ref.bf16(rng.normal(0, 1, (1, 2, d)))
    o, lse = torch.empty((1, 2, d), device="cuda", dtype=torch.bfloat16), torch.empty((1, 2), device="cuda")
    plan = bsp.DecodePlan(bsp.device(), 1, 2, 1, d, page)
    plan.execute(cache, cuda(q, torch.bfloat16), i32([303]), cuda(pages), o, lse=lse)
    bsp.device().synchronize()
    check_attention(o, lse, *decode_gold(q.astype(float), codes, scales, [303], pages, hk, 1 / 8.0), 2 * ref.UH)


def test_decode_bad_indices(bsp):
    """Lengths beyond the page table count as 0, pages outside the cache as
    zeros; both are reported."""
    torch = torch_()
    cache = bsp.KvCache.empty(4, 1, 16, 64)
    q = torch.ones((1, 1, 64), device="cuda", dtype=torch.bfloat16)
    plan = bsp.DecodePlan(bsp.device(), 1, 1, 1, 64, 16)
    for lens, pages in (([33], [[0, 1]]), ([-1], [[0, 1]]), ([20], [[0, 4]]), ([20], [[-7, 1]])):
        o = torch.full_like(q, 5)
        plan.execute(cache, q, i32(lens), i32(pages), o)
        with pytest.raises(bsp.BspError, match="outside its table"):
            bsp.device().synchronize()
        assert (o == 0).all()


# ---------------------------------------------------------------- together --
def test_prompt_then_tokens(bsp):
    """A prompt, then tokens one by one: decode over the cache agrees with
    prompt attention over the same keys and values within the cache's 8 bits."""
    torch = torch_()
    rng = np.random.default_rng(8)
    n, steps, hq, hk, d, page = 150, 5, 8, 2, 128, 64
    q, k, v = (cuda(ref.bf16(rng.normal(0, 1, (n + steps, h, d))), torch.bfloat16) for h in (hq, hk, hk))
    table = bsp.rope_table(512, d)
    cache, pages = bsp.KvCache.empty(4, hk, page, d), i32([[3, 1, 0]])
    qr, kr = torch.empty_like(q), torch.empty_like(k)
    bsp.kv_append(cache, k[:n], v[:n], i32([0, n]), i32([0]), pages, table=table, q=q[:n], q_out=qr[:n], k_out=kr[:n])
    plan = bsp.DecodePlan(bsp.device(), 1, hq, hk, d, page)
    o = torch.empty((steps, hq, d), device="cuda", dtype=torch.bfloat16)
    for i in range(steps):
        a = slice(n + i, n + i + 1)
        bsp.kv_append(cache, k[a], v[a], i32([0, 1]), i32([n + i]), pages, table=table, q=q[a], q_out=qr[a], k_out=kr[a])
        plan.execute(cache, qr[a], i32([n + i + 1]), pages, o[i:i + 1])
    full = torch.empty_like(q)
    bsp.PromptPlan(bsp.device(), [n + steps], [n + steps], hq, hk, d).execute(qr, kr, v, full)
    bsp.device().synchronize()
    # a key's code is off by up to 2^-4 of its value: scores by 2^-4 |q| |k| / sqrt(d) / sqrt(d) at random
    # (about 0.04 here); values by 2^-4: the norm of the difference stays under a tenth of the norm
    a, b = o.double(), full[n:].double()
    assert float((a - b).norm() / b.norm()) <= 0.1


def test_example(bsp):
    """examples/serve_attention.py: prompts, then tokens, checked at its end."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "serve_attention.py")
    spec = importlib.util.spec_from_file_location("serve_attention", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    assert m.main(["--steps", "5"]) < 0.1


def test_graph_capture(bsp):
    """Every execute is captured in one graph and replayed on new inputs."""
    torch = torch_()
    rng = np.random.default_rng(8)
    hq, hk, d, page = 4, 2, 64, 16
    table, pages = bsp.rope_table(64, d), i32([[0, 1, 2]])
    plan, prompt = bsp.DecodePlan(bsp.device(), 1, hq, hk, d, page), bsp.PromptPlan(bsp.device(), [5], [5], hq, hk, d)
    x = [torch.zeros((5, h, d), device="cuda", dtype=torch.bfloat16) for h in (hq, hk, hk)]
    cache = bsp.KvCache.empty(3, hk, page, d)
    starts, before, lens, pos = i32([0, 5]), i32([20]), i32([25]), i32(np.arange(20, 25))

    def step(out):
        bsp.kv_append(cache, x[1], x[2], starts, before, pages, table=table, q=x[0], q_out=out[0], k_out=out[1])
        bsp.rope(x[0], pos, table, out=out[4])
        prompt.execute(out[0], out[1], x[2], out[2])
        plan.execute(cache, out[0][4:], lens, pages, out[3])

    outs = [[torch.zeros((n, h, d), device="cuda", dtype=torch.bfloat16) for n, h in ((5, hq), (5, hk), (5, hq), (1, hq), (5, hq))]
            for _ in range(2)]
    step(outs[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(outs[0])
    for seed in range(2):
        for t in x:
            t.copy_(cuda(ref.bf16(rng.normal(0, 1, tuple(t.shape))), torch.bfloat16))
        cache.k.zero_()
        cache.v.zero_()
        graph.replay()
        torch.cuda.synchronize()
        cache.k.zero_()
        cache.v.zero_()
        step(outs[1])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(*outs)) and torch.equal(outs[0][0], outs[0][4])
    bsp.device().synchronize()


def test_graph_capture_of_cut_prompt(bsp):
    """A plan that is cut, captured with its joining kernel and replayed on other inputs."""
    torch = torch_()
    q, k, v = (torch.zeros((n, h, 64), device="cuda", dtype=torch.bfloat16) for n, h in ((9, 4), (4000, 2), (4000, 2)))
    plan = bsp.PromptPlan(bsp.device(), [9], [4000], 4, 2, 64)
    assert plan.info()["workspace_bytes"] > 0
    o = [torch.zeros_like(q) for _ in range(2)]
    plan.execute(q, k, v, o[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.execute(q, k, v, o[0])
    for _ in range(3):
        for t in (q, k, v):
            t.normal_()
        graph.replay()
        plan.execute(q, k, v, o[1])
        torch.cuda.synchronize()
        assert torch.equal(o[0], o[1]) and bool(o[0].any())
    bsp.device().synchronize()


# ---------------------------------------------------------------- refusals --
def test_refusals(bsp):
    torch = torch_()
    dev = bsp.device()
    z = lambda *s, dt=torch.bfloat16: torch.zeros(s, dtype=dt, device="cuda")  # noqa: E731
    table = bsp.rope_table(16, 64)
    cache = bsp.KvCache.empty(4, 2, 16, 64)
    pages, one = i32([[0, 1]]), i32([0, 2])
    bad = [
        lambda: bsp.rope_table(16, 24), lambda: bsp.rope_table(0, 64), lambda: bsp.rope_table(16, 64, base=-1.0),
        lambda: bsp.rope_table(16, 64, kind="linear", factor=0.0), lambda: bsp.rope_table(16, 64, kind="odd"),
        lambda: bsp.rope_table(16, 64, kind="parts", factor=2.0), lambda: bsp.rope_table(16, 64, base=float("nan")),
        lambda: bsp.rope(z(2, 1, 32), i32([0, 1]), table),                    # rot > d
        lambda: bsp.rope(z(2, 1, 72), i32([0, 1]), table),                    # d % 16
        lambda: bsp.rope(z(2, 1, 64), i32([0]), table),
        lambda: bsp.rope(z(2, 1, 64), cuda(np.zeros(2, np.int64)), table),
        lambda: bsp.rope(z(2, 1, 64), i32([0, 1]), table, layout="other"),
        lambda: bsp.rope(z(2, 1, 64, dt=torch.float16), i32([0, 1]), table),
        lambda: bsp.rope(z(2, 1, 68)[:, :, 4:], i32([0, 1]), table),          # misaligned
        lambda: bsp.rope(z(2, 1, 64), i32([0, 1]), table, out=z(2, 1, 64, dt=torch.float32)),
        lambda: bsp.rope(z(2, 64, 1).transpose(1, 2), i32([0, 1]), table, out=z(2, 1, 32)),
        lambda: bsp.KvCache.empty(4, 2, 16, 96).desc and bsp.kv_append(
            bsp.KvCache.empty(4, 2, 16, 96), z(2, 2, 96), z(2, 2, 96), one, i32([0]), pages),
        lambda: bsp.kv_append(bsp.KvCache.empty(4, 2, 24, 64), z(2, 2, 64), z(2, 2, 64), one, i32([0]), pages),
        lambda: bsp.kv_append(cache, z(2, 1, 64), z(2, 2, 64), one, i32([0]), pages),
        lambda: bsp.kv_append(cache, z(2, 2, 64), z(3, 2, 64), one, i32([0]), pages),
        lambda: bsp.kv_append(cache, z(2, 2, 64), z(2, 2, 64), i32([0]), i32([0]), pages),
        lambda: bsp.kv_append(cache, z(2, 2, 64), z(2, 2, 64), one, i32([0]), pages, q=z(2, 2, 64), q_out=z(2, 2, 64)),
        lambda: bsp.kv_append(cache, z(2, 2, 64), z(2, 2, 64), one, i32([0]), pages, table=table, q=z(2, 2, 64)),
        lambda: bsp.kv_append(cache, z(2, 2, 64), z(2, 2, 64), one, i32([0]), pages, table=bsp.rope_table(4, 128)),
        lambda: bsp.KvCache(z(2, 1, 16, 64), z(2, 1, 16, 64), z(2, 1), z(2, 1)),
        lambda: bsp.KvCache(cache.k, cache.v, cache.k_scale, z(3, 2, dt=torch.float32)),
        lambda: bsp.KvCache(cache.k, cache.v[:2], cache.k_scale, cache.v_scale),
        lambda: bsp.PromptPlan(dev, [4], [4], 4, 3, 64), lambda: bsp.PromptPlan(dev, [4], [4], 4, 2, 96),
        lambda: bsp.PromptPlan(dev, [4], [4, 4], 4, 2, 64), lambda: bsp.PromptPlan(dev, [-4], [4], 4, 2, 64),
        lambda: bsp.PromptPlan(dev, [2 ** 31 - 1, 2 ** 31 - 1], [4, 4], 4, 2, 64),
        lambda: bsp.DecodePlan(dev, -1, 4, 2, 64, 16), lambda: bsp.DecodePlan(dev, 1, 4, 2, 64, 20),
        lambda: bsp.DecodePlan(dev, 1, 5, 2, 64, 16),
    ]
    plan = bsp.PromptPlan(dev, [4], [6], 4, 2, 64)
    q, k = z(4, 4, 64), z(6, 2, 64)
    bad += [lambda: plan.execute(q, k, k, z(4, 4, 128)), lambda: plan.execute(z(5, 4, 64), k, k, q),
            lambda: plan.execute(q, k[:5], k, z(4, 4, 64)), lambda: plan.execute(q, k, k, z(4, 4, 64), scale=0.0),
            lambda: plan.execute(q, k, k, z(4, 4, 64), scale=float("inf")),
            lambda: plan.execute(q, k, k, z(4, 4, 64), lse=z(4, 3, dt=torch.float32)),
            lambda: plan.execute(q.float(), k, k, z(4, 4, 64)),
            lambda: plan.execute(z(4, 4, 68)[:, :, 4:], k, k, z(4, 4, 64))]
    dp = bsp.DecodePlan(dev, 1, 4, 2, 64, 16)
    q1 = z(1, 4, 64)
    bad += [lambda: dp.execute(cache, z(2, 4, 64), i32([1, 1]), i32([[0], [0]]), z(2, 4, 64)),
            lambda: dp.execute(cache, q1, i32([1, 1]), pages, z(1, 4, 64)),
            lambda: dp.execute(bsp.KvCache.empty(4, 2, 32, 64), q1, i32([1]), pages, z(1, 4, 64)),
            lambda: dp.execute(cache, q1, i32([1]), pages, z(1, 4, 64), scale=-1.0),
            lambda: dp.execute(cache, q1, i32([1]), pages, z(1, 2, 64)),
            lambda: dp.execute(cache, q1.cpu(), i32([1]), pages, z(1, 4, 64))]
    for i, f in enumerate(bad):
        with pytest.raises(bsp.BspError) as e:
            f()
        assert e.value.status in (bsp.BSP_ERR_INVALID_ARG, bsp.BSP_ERR_UNSUPPORTED), i
    dev.synchronize()
