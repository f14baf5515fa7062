"""Workloads of the decoder-attention operators: rotary positions, the paged
8-bit key/value cache, attention over whole prompts and attention of single
tokens over that cache.

`own = False` runs every operator in elementary torch operations in 32 bits;
`own = True` makes the calls a user makes of libbsp's binding (bsp.py).

Conventions of all operators
  x [tokens, heads, d]; tokens of all sequences packed one after the other.
  rotary table: float32 [positions, rot / 2, 2] of (cos, sin).
  cache: pages of `page` tokens, k and v [pages, kv_heads, page, d] in e4m3 with
  one power-of-two scale per (page, head): value = code * scale.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "tenstorrent-wh-blockspmm_b200")


def _bsp():
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    import bsp

    return bsp


# ------------------------------------------------------------------- cases --
def _mix(rng, n, low, high):
    """n lengths spread over the logarithm of [low, high], as text."""
    return " ".join(str(int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))) for _ in range(n))


def listed():
    r = random.Random(11)
    return [
        # one decoding step's queries of a few requests: latency
        dict(name="rope_step", op="rope", tokens=16, heads=32, d=128, rot=128, layout="half", dtype="bf16",
             transpose=False, scaling="none"),
        # gradient of the rotation of half of each head over a training batch, in float32
        dict(name="rope_grad", op="rope", tokens=8191, heads=32, d=128, rot=64, layout="interleaved", dtype="f32",
             transpose=True, scaling="linear"),
        # one token of each of 64 running requests goes into the cache
        dict(name="append_step", op="append", new=" ".join(["1"] * 64), before=_mix(r, 64, 1, 2000), heads=32,
             kv_heads=8, d=128, page=64, rot=128, layout="half", scaling="none"),
        # prompts of very different lengths, one of them the second part of a longer prompt
        dict(name="append_prompt", op="append", new="5003 1 2777 64 6100 333", before="0 17 0 0 1999 0", heads=32,
             kv_heads=8, d=128, page=16, rot=128, layout="half", scaling="parts"),
        # a short question: latency
        dict(name="prompt_short", op="prompt", q="37", kv="37", heads=8, kv_heads=2, d=64, causal=True),
        # a scheduler's packed batch: new prompts and the continuations of two
        dict(name="prompt_packed", op="prompt", q="2048 513 1 1290 96 2001 777", kv="2048 513 600 1290 96 3001 777",
             heads=32, kv_heads=8, d=128, causal=True),
        # every head with keys of its own, heads of 64
        dict(name="prompt_heads64", op="prompt", q="1999 3001 1025", kv="1999 3001 1025", heads=16, kv_heads=16,
             d=64, causal=True),
        # one long document, the sequence length of the block-sparse attention benchmark
        dict(name="prompt_long", op="prompt", q="16384", kv="16384", heads=8, kv_heads=2, d=128, causal=True),
        # one running request: latency
        dict(name="decode_one", op="decode", kv="1000", heads=32, kv_heads=8, d=128, page=64),
        # a busy server: 64 requests of mixed lengths
        dict(name="decode_batch", op="decode", kv=_mix(r, 64, 500, 8000), heads=32, kv_heads=8, d=128, page=64),
        # two long contexts, few rows: the keys' axis has to be split
        dict(name="decode_long", op="decode", kv="100003 131072", heads=40, kv_heads=8, d=128, page=128),
        # small pages, heads of 64, every head with keys of its own
        dict(name="decode_heads64", op="decode", kv=_mix(r, 24, 100, 9000), heads=16, kv_heads=16, d=64, page=16),
    ]


def draw(rng):
    def log(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    op = rng.choice(["rope", "append", "prompt", "decode"])
    d = rng.choice([64, 128, 128])
    if op == "rope":
        rot = rng.choice([d, d, d // 2])
        return dict(op=op, tokens=log(1, 8192), heads=rng.choice([1, 5, 8, 24, 32]), d=d, rot=rot,
                    layout=rng.choice(["half", "interleaved"]), dtype=rng.choice(["bf16", "bf16", "f32"]),
                    transpose=rng.random() < 0.4, scaling=rng.choice(["none", "linear", "parts"]))
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 4, 5, 8])
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        n = log(1, 64)
        steps = rng.random() < 0.5
        new = " ".join(["1"] * n) if steps else _mix(rng, n, 1, max(1, 9000 // n))
        return dict(op=op, new=new, before=_mix(rng, n, 1, 2000), heads=kv_heads * group, kv_heads=kv_heads, d=d,
                    page=page, rot=rng.choice([d, d, d // 2]), layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "parts"]))
    if op == "prompt":
        n = log(1, 8)
        total = log(16, 7000)
        q = _mix(rng, n, 1, max(1, total // n))
        kv = " ".join(str(int(x) + (log(1, 700) if rng.random() < 0.3 else 0)) for x in q.split())
        return dict(op=op, q=q, kv=kv, heads=kv_heads * group if kv_heads * group <= 32 else kv_heads * 4,
                    kv_heads=kv_heads, d=d, causal=rng.random() < 0.85)
    n = log(1, 64)
    kv = _mix(rng, n, 1, min(60000, max(2, 250000 // n)))
    return dict(op=op, kv=kv, heads=kv_heads * group, kv_heads=kv_heads, d=d, page=page)


def _ints(text):
    return [int(x) for x in text.split()]


def _pairs(q, kv, causal):
    """(query, key) pairs that attend; with causal the last query sees every key."""
    if not causal:
        return sum(a * b for a, b in zip(q, kv))
    return sum(a * b - a * (a - 1) // 2 for a, b in zip(q, kv))


def work(case):
    d = case["d"]
    if case["op"] == "rope":
        size = 2 if case["dtype"] == "bf16" else 4
        n = case["tokens"] * case["heads"] * d
        return {"bytes": 2 * n * size + case["tokens"] * (4 + 4 * case["rot"]),
                "flops": 3 * case["tokens"] * case["heads"] * case["rot"]}
    if case["op"] == "append":
        new, hq, hk = sum(_ints(case["new"])), case["heads"], case["kv_heads"]
        # q, k, v in, rotated q and k out, k and v codes out, one table row a token, scales of the pages
        return {"bytes": new * d * (4 * hq + 4 * hk + 2 * hk + 2 * hk) + new * 4 * case["rot"]
                + 16 * hk * sum(1 + a // case["page"] for a in _ints(case["new"])),
                "flops": 3 * new * case["rot"] * (hq + hk) + 4 * new * hk * d}
    if case["op"] == "prompt":
        q, kv = _ints(case["q"]), _ints(case["kv"])
        return {"bytes": 2 * d * (2 * sum(q) * case["heads"] + 2 * sum(kv) * case["kv_heads"])
                + 4 * sum(q) * case["heads"],
                "flops": 4 * d * case["heads"] * _pairs(q, kv, case["causal"])}
    kv = _ints(case["kv"])
    return {"bytes": sum(kv) * case["kv_heads"] * d * 2 + 4 * len(kv) * case["heads"] * d,
            "flops": 4 * sum(kv) * case["heads"] * d}


# ------------------------------------------------------------------ inputs --
CONTEXT = 1 << 17   # positions of a long context's rotary table


def _table(rot, scaling, positions):
    """cos and sin of position * frequency, frequencies of base 10000, made in 64 bits."""
    i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    freq = 10000.0 ** (-2.0 * i / rot)
    size = 1.0
    if scaling == "linear":  # positions squeezed four times
        freq = freq / 4.0
    elif scaling == "parts":  # slow dimensions squeezed eight times, fast ones kept, a ramp between
        turns = 4096.0 * freq / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        freq = freq * keep + freq / 8.0 * (1 - keep)
        size = 0.1 * math.log(8.0) + 1.0
    a = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * freq
    return (torch.stack([a.cos(), a.sin()], -1) * size).float().contiguous()


def _two(e):
    """2 ** e in float32 for whole e in [-126, 127], exactly."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _exponent(amax):
    """Smallest e with amax <= 448 * 2 ** e (448: the largest e4m3), within [-100, 119]; 0 for amax 0."""
    m, x = torch.frexp(amax)
    e = torch.where(m <= 0.875, x - 9, x - 8)
    return torch.where(amax > 0, e.clamp(-100, 119), torch.zeros_like(e)).to(torch.int32)


def _pages(n_seqs_tokens, page):
    return [-(-n // page) for n in n_seqs_tokens]


def _cache(g, tokens, kv_heads, d, page):
    """A cache in use: shuffled pages, keys with a few strong channels, and its page table."""
    per = _pages(tokens, page)
    n = sum(per) + 3
    order = torch.randperm(n, device="cuda", generator=g)[: sum(per)].to(torch.int32)
    width = max(max(per), 1)
    rows = torch.repeat_interleave(torch.arange(len(per), device="cuda"), torch.tensor(per, device="cuda"))
    first = torch.tensor(np.concatenate([[0], np.cumsum(per)[:-1]]), device="cuda")
    cols = torch.arange(sum(per), device="cuda") - first[rows]
    table = torch.zeros((len(per), width), dtype=torch.int32, device="cuda")
    table[rows, cols] = order
    out = []
    for strong in (4.0, 1.0):
        x = torch.randn((n, kv_heads, page, d), device="cuda", generator=g)
        x[..., :: 32] *= strong
        e = _exponent(x.abs().amax((2, 3)))
        out += [(x * _two(-e)[:, :, None, None]).to(torch.float8_e4m3fn), _two(e)]
        del x
    return out[0], out[2], out[1], out[3], table


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case)
    d = case["d"]
    if case["op"] == "rope":
        dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        t, h = case["tokens"], case["heads"]
        s["x"] = torch.randn((t, h, d), device="cuda", generator=g).to(dt)
        s["y"] = torch.empty_like(s["x"])
        s["positions"] = (torch.randint(0, 40000, (t,), device="cuda", generator=g) if t < 64 else
                          torch.arange(t, device="cuda")).to(torch.int32)
        s["table"] = _table(case["rot"], case["scaling"], CONTEXT if t < 64 else 16384)
        return s
    hq, hk = case["heads"], case["kv_heads"]
    if case["op"] == "append":
        new, before = _ints(case["new"]), _ints(case["before"])
        t = sum(new)
        # q, k and v are parts of one projection's output
        qkv = torch.randn((t, hq + 2 * hk, d), device="cuda", generator=g).bfloat16()
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        s["q_out"] = torch.empty((t, hq, d), dtype=torch.bfloat16, device="cuda")
        s["k_out"] = torch.empty((t, hk, d), dtype=torch.bfloat16, device="cuda")
        s["k8"], s["v8"], s["k_scale"], s["v_scale"], s["pages"] = _cache(
            g, [a + b for a, b in zip(new, before)], hk, d, case["page"])
        s["starts"] = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")
        s["before"] = torch.tensor(before, dtype=torch.int32, device="cuda")
        s["table"] = _table(case["rot"], case["scaling"], 16384)
    elif case["op"] == "prompt":
        q, kv = _ints(case["q"]), _ints(case["kv"])
        s["q_lens"], s["kv_lens"] = q, kv
        s["seq_q"] = torch.repeat_interleave(torch.arange(len(q), device="cuda"), torch.tensor(q, device="cuda"))
        s["seq_kv"] = torch.repeat_interleave(torch.arange(len(kv), device="cuda"), torch.tensor(kv, device="cuda"))
        start_q = torch.tensor(np.concatenate([[0], np.cumsum(q)[:-1]]), device="cuda")
        start_kv = torch.tensor(np.concatenate([[0], np.cumsum(kv)[:-1]]), device="cuda")
        shift = torch.tensor([b - a for a, b in zip(q, kv)], device="cuda")
        s["pos_q"] = torch.arange(sum(q), device="cuda") - start_q[s["seq_q"]] + shift[s["seq_q"]]
        s["pos_kv"] = torch.arange(sum(kv), device="cuda") - start_kv[s["seq_kv"]]
        s["q"] = torch.randn((sum(q), hq, d), device="cuda", generator=g).bfloat16()
        kvx = torch.randn((sum(kv), 2 * hk, d), device="cuda", generator=g).bfloat16()
        s["k"], s["v"] = kvx[:, :hk], kvx[:, hk:]
        s["o"] = torch.empty((sum(q), hq, d), dtype=torch.bfloat16, device="cuda")
        s["lse"] = torch.empty((sum(q), hq), dtype=torch.float32, device="cuda")
        if own:
            bsp = _bsp()
            s["plan"] = bsp.PromptPlan(bsp.device(), q, kv, hq, hk, d, causal=case["causal"])
    else:
        kv = _ints(case["kv"])
        s["k8"], s["v8"], s["k_scale"], s["v_scale"], s["pages"] = _cache(g, kv, hk, d, case["page"])
        s["lens"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
        s["q"] = torch.randn((len(kv), hq, d), device="cuda", generator=g).bfloat16()
        s["o"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty((len(kv), hq), dtype=torch.float32, device="cuda")
        if own:
            bsp = _bsp()
            s["plan"] = bsp.DecodePlan(bsp.device(), len(kv), hq, hk, d, case["page"])
    if own and "k8" in s:
        s["cache"] = _bsp().KvCache(s["k8"], s["v8"], s["k_scale"], s["v_scale"])
    return s


# ------------------------------------------------------------- plain forms --
def _rotate(x, cos_sin, layout, transpose):
    """x [tokens, heads, d] float, cos_sin [tokens, rot / 2, 2]."""
    c, s = cos_sin[:, None, :, 0], cos_sin[:, None, :, 1]
    if transpose:
        s = -s
    half = c.shape[-1]
    y = x.clone()
    if layout == "half":
        a, b = x[..., :half], x[..., half:2 * half]
        y[..., :half], y[..., half:2 * half] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * c - b * s, b * c + a * s
    return y


def _append_plain(s):
    page = s["page"]
    starts, before, pages = s["starts"].long(), s["before"].long(), s["pages"].long()
    t = s["k"].shape[0]
    seq = torch.searchsorted(starts[1:].contiguous(), torch.arange(t, device="cuda"), right=True)
    pos = torch.arange(t, device="cuda") - starts[seq] + before[seq]
    cs = s["table"][pos]
    q = _rotate(s["q"].float(), cs, s["layout"], False)
    k = _rotate(s["k"].float(), cs, s["layout"], False)
    pid, slot = pages[seq, pos // page], pos % page
    # the pages that already hold earlier tokens of their sequence
    n_new = starts[1:] - starts[:-1]
    held = pages.gather(1, (before // page).clamp(max=pages.shape[1] - 1)[:, None])[:, 0]
    keep = (before % page > 0) & (n_new > 0)
    outs = []
    for x, codes, scale in ((k, s["k8"], s["k_scale"]), (s["v"].float(), s["v8"], s["v_scale"])):
        amax = torch.zeros_like(scale)
        amax.scatter_reduce_(0, pid[:, None].expand(-1, scale.shape[1]), x.abs().amax(-1), "amax")
        e = _exponent(amax)
        old = _exponent(448.0 * scale[held])
        both = torch.where(keep[:, None], torch.maximum(old, e[held]), e[held])
        grown = torch.where((torch.arange(page, device="cuda") < (before % page)[:, None])[:, None, :, None]
                            & keep[:, None, None, None] & (both > old)[:, :, None, None],
                            (codes[held].float() * _two(old - both)[:, :, None, None]), codes[held].float())
        # a sequence without new tokens writes nothing
        some = n_new > 0
        codes[held[some]] = grown[some].to(codes.dtype)
        e[held[some]] = both[some]
        scale[pid] = _two(e)[pid]
        codes[pid, :, slot] = (x * _two(-e[pid])[:, :, None]).to(codes.dtype)
        outs += [codes, scale]
    s["q_out"].copy_(q)
    s["k_out"].copy_(k)
    return {"q": s["q_out"], "k": s["k_out"], "k8": outs[0], "k_scale": outs[1], "v8": outs[2], "v_scale": outs[3]}


def _softmax_rows(x):
    """In place: exp(x - max) of the last axis; (weights, their sums, log of the sum of exponentials)."""
    m = x.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    x.sub_(m).exp_()
    l = x.sum(-1, keepdim=True)
    return x, l, (m + l.log())[..., 0]


def _prompt_plain(s):
    hk, d = s["kv_heads"], s["d"]
    t, hq, _ = s["q"].shape
    q = s["q"].float().view(t, hk, hq // hk, d).permute(1, 2, 0, 3)
    k, v = s["k"].float().permute(1, 2, 0)[:, None], s["v"].float().permute(1, 0, 2)[:, None]
    x = torch.matmul(q, k)
    x *= 1.0 / math.sqrt(d)
    away = s["seq_q"][:, None] != s["seq_kv"]
    if s["causal"]:
        away |= s["pos_kv"] > s["pos_q"][:, None]
    x.masked_fill_(away, -math.inf)
    p, l, lse = _softmax_rows(x)
    o = torch.matmul(p, v) / l
    return {"o": o.permute(2, 0, 1, 3).reshape(t, hq, d).bfloat16(), "lse": lse.permute(2, 0, 1).reshape(t, hq)}


def _decode_plain(s):
    hk, d, page = s["kv_heads"], s["d"], s["page"]
    n, hq, _ = s["q"].shape
    pages = s["pages"].long()
    k = s["k8"][pages].float() * s["k_scale"][pages][..., None, None]
    v = s["v8"][pages].float() * s["v_scale"][pages][..., None, None]
    k = k.permute(0, 2, 1, 3, 4).reshape(n, hk, -1, d)
    v = v.permute(0, 2, 1, 3, 4).reshape(n, hk, -1, d)
    q = s["q"].float().view(n, hk, hq // hk, d)
    x = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    x.masked_fill_((torch.arange(k.shape[2], device="cuda") >= s["lens"][:, None])[:, None, None], -math.inf)
    p, l, lse = _softmax_rows(x)
    o = torch.matmul(p, v) / l
    return {"o": o.reshape(n, hq, d).bfloat16(), "lse": lse.reshape(n, hq)}


def run(state):
    s = state
    op = s["op"]
    if not own:
        if op == "rope":
            y = _rotate(s["x"].float(), s["table"][s["positions"].long()], s["layout"], s["transpose"])
            return y.to(s["x"].dtype)
        return {"append": _append_plain, "prompt": _prompt_plain, "decode": _decode_plain}[op](s)
    bsp = _bsp()
    if op == "rope":
        return bsp.rope(s["x"], s["positions"], s["table"], layout=s["layout"], transpose=s["transpose"], out=s["y"])
    if op == "append":
        bsp.kv_append(s["cache"], s["k"], s["v"], s["starts"], s["before"], s["pages"], table=s["table"],
                      layout=s["layout"], q=s["q"], q_out=s["q_out"], k_out=s["k_out"])
        return {"q": s["q_out"], "k": s["k_out"], "k8": s["k8"], "k_scale": s["k_scale"], "v8": s["v8"],
                "v_scale": s["v_scale"]}
    if op == "prompt":
        s["plan"].execute(s["q"], s["k"], s["v"], s["o"], lse=s["lse"])
    else:
        s["plan"].execute(s["cache"], s["q"], s["lens"], s["pages"], s["o"], lse=s["lse"])
    return {"o": s["o"], "lse": s["lse"]}


# ------------------------------------------------------------------- exact --
def _e4m3(x):
    """x (64 bits) to the nearest e4m3 value, ties to even, |x| <= 448."""
    _, e = torch.frexp(x)
    step = _two64((e - 4).clamp(min=-9))
    return torch.round(x / step) * step


def _two64(e):
    """2 ** e in 64 bits for whole e, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        x, cs = s["x"].double(), s["table"].double()[s["positions"].long()]
        z = torch.complex(cs[..., 0], -cs[..., 1] if case["transpose"] else cs[..., 1])[:, None]
        half = case["rot"] // 2
        y = x.clone()
        if case["layout"] == "half":
            w = torch.complex(x[..., :half], x[..., half:2 * half]) * z
            y[..., :half], y[..., half:2 * half] = w.real, w.imag
        else:
            w = torch.complex(x[..., 0:2 * half:2], x[..., 1:2 * half:2]) * z
            y[..., 0:2 * half:2], y[..., 1:2 * half:2] = w.real, w.imag
        return y
    d, hq, hk = case["d"], case["heads"], case["kv_heads"]
    if case["op"] == "append":
        new, before, page = _ints(case["new"]), _ints(case["before"]), case["page"]
        if s["k8"].numel() > 1 << 28:
            return None
        tables = s["table"].double()
        pages = s["pages"].cpu().numpy()
        half = case["rot"] // 2
        pos = torch.tensor(np.concatenate([np.arange(b, b + n) for n, b in zip(new, before)]), device="cuda")
        z = torch.complex(tables[pos][..., 0], tables[pos][..., 1])[:, None]
        rotated = []
        for x in (s["q"].double(), s["k"].double()):
            first, second = ((slice(0, half), slice(half, 2 * half)) if case["layout"] == "half" else
                             (slice(0, 2 * half, 2), slice(1, 2 * half, 2)))
            w = torch.complex(x[..., first], x[..., second]) * z
            y = x.clone()
            y[..., first], y[..., second] = w.real, w.imag
            rotated.append(y)
        out = {"q": rotated[0], "k": rotated[1]}
        for name, x in (("k", rotated[1]), ("v", s["v"].double())):
            codes, scale = s[name + "8"].double(), s[name + "_scale"].double()
            at = 0
            for i, (n, b) in enumerate(zip(new, before)):
                done = 0
                while done < n:
                    p, slot = int(pages[i, (b + done) // page]), (b + done) % page
                    m = min(n - done, page - slot)
                    part = x[at + done: at + done + m].permute(1, 0, 2)
                    e = _exponent(part.abs().amax((1, 2)))
                    if slot:
                        was = torch.frexp(scale[p])[1] - 1
                        e = torch.maximum(e, was)
                        codes[p, :, :slot] = _e4m3(codes[p, :, :slot] * _two64(was - e)[:, None, None])
                    codes[p, :, slot: slot + m] = _e4m3(part * _two64(-e)[:, None, None])
                    scale[p] = _two64(e)
                    done += m
                at += n
            out[name + "8"], out[name + "_scale"] = codes, scale
        return out
    if case["op"] == "prompt":
        q, kv = _ints(case["q"]), _ints(case["kv"])
        o = torch.empty((sum(q), hq, d), dtype=torch.float64, device="cuda")
        lse = torch.empty((sum(q), hq), dtype=torch.float64, device="cuda")
        at_q = at_kv = 0
        for n, m in zip(q, kv):
            for h in range(hq):
                kh = h // (hq // hk)
                k, v = s["k"][at_kv: at_kv + m, kh].double(), s["v"][at_kv: at_kv + m, kh].double()
                for a in range(0, n, 4096):
                    b = min(n, a + 4096)
                    x = s["q"][at_q + a: at_q + b, h].double() @ k.T / math.sqrt(d)
                    if case["causal"]:
                        see = torch.arange(m, device="cuda") <= torch.arange(a, b, device="cuda")[:, None] + (m - n)
                        x = torch.where(see, x, torch.full_like(x, -math.inf))
                    o[at_q + a: at_q + b, h] = torch.softmax(x, -1) @ v
                    lse[at_q + a: at_q + b, h] = torch.logsumexp(x, -1)
            at_q, at_kv = at_q + n, at_kv + m
        return {"o": o, "lse": lse}
    o = torch.empty((len(_ints(case["kv"])), hq, d), dtype=torch.float64, device="cuda")
    lse = torch.empty((o.shape[0], hq), dtype=torch.float64, device="cuda")
    for i, n in enumerate(_ints(case["kv"])):
        use = s["pages"][i, : -(-n // case["page"])].long()
        k, v = ((s[c][use].double() * s[c[0] + "_scale"][use].double()[..., None, None])
                .permute(1, 0, 2, 3).reshape(hk, -1, d)[:, :n] for c in ("k8", "v8"))
        x = s["q"][i].double().view(hk, hq // hk, d) @ k.transpose(1, 2) / math.sqrt(d)
        o[i] = (torch.softmax(x, -1) @ v).reshape(hq, d)
        lse[i] = torch.logsumexp(x, -1).reshape(hq)
    return {"o": o, "lse": lse}
