"""The attention of one decoder layer, served: several requests of different
lengths send their prompts, then all of them take tokens one by one.

    python examples/serve_attention.py [--steps 16]

Prompts: one bsp.kv_append rotates queries and keys and fills the 8-bit cache,
one PromptPlan.execute attends within each prompt.  Each further token: one
kv_append for all requests, one DecodePlan.execute over their caches.  The last
token is checked against prompt attention over the whole context (16-bit keys
and values; the cache holds 8 bits).
"""
import argparse
import itertools
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tenstorrent-wh-blockspmm_b200"))
import bsp  # noqa: E402


class DecoderAttention:
    """Projections, rotary table and paged cache of one layer, and the pages of
    each running request."""

    def __init__(self, model, heads, kv_heads, d, n_pages, page=64, context=4096, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.kv_heads, self.d, self.page = heads, kv_heads, d, page
        self.w_in = (torch.randn((model, (heads + 2 * kv_heads) * d), device="cuda", generator=g) / model ** 0.5).bfloat16()
        self.w_out = (torch.randn((heads * d, model), device="cuda", generator=g) / (heads * d) ** 0.5).bfloat16()
        self.table = bsp.rope_table(context, d)
        self.cache = bsp.KvCache.empty(n_pages, kv_heads, page, d)
        self.free = list(range(n_pages))
        self.pages, self.lens = [], []

    def _project(self, x):
        qkv = (x @ self.w_in).view(x.shape[0], -1, self.d)
        return qkv.split([self.heads, self.kv_heads, self.kv_heads], 1)

    def _append(self, x, new):
        """Rotate and store the `new` tokens of each request; rotated q, k, and v."""
        before = list(self.lens)
        for s, n in enumerate(new):
            self.lens[s] += n
            while len(self.pages[s]) * self.page < self.lens[s]:
                self.pages[s].append(self.free.pop())
        width = max(len(p) for p in self.pages)
        i32 = dict(dtype=torch.int32, device="cuda")
        self.page_table = torch.tensor([p + [-1] * (width - len(p)) for p in self.pages], **i32)
        starts = torch.tensor([0, *itertools.accumulate(new)], **i32)
        q, k, v = self._project(x)
        q_rot = torch.empty_like(q, memory_format=torch.contiguous_format)
        k_rot = torch.empty_like(k, memory_format=torch.contiguous_format)
        bsp.kv_append(self.cache, k, v, starts, torch.tensor(before, **i32), self.page_table, table=self.table, q=q,
                      q_out=q_rot, k_out=k_rot)
        return q_rot, k_rot, v

    def prompts(self, x, lens):
        """x: the prompts of new requests, one after the other."""
        self.pages, self.lens = [[] for _ in lens], [0] * len(lens)
        q, k, v = self._append(x, lens)
        o = torch.empty_like(q)
        bsp.PromptPlan(bsp.device(), lens, lens, self.heads, self.kv_heads, self.d).execute(q, k, v, o)
        self.decode = bsp.DecodePlan(bsp.device(), len(lens), self.heads, self.kv_heads, self.d, self.page)
        return o.flatten(1) @ self.w_out, (k, v)

    def tokens(self, x):
        """x: one token of each request."""
        q, k, v = self._append(x, [1] * x.shape[0])
        o = torch.empty_like(q)
        self.decode.execute(self.cache, q, torch.tensor(self.lens, dtype=torch.int32, device="cuda"), self.page_table, o)
        return o.flatten(1) @ self.w_out, (q, k, v, o)


def main(argv=None):
    a = argparse.ArgumentParser()
    a.add_argument("--steps", type=int, default=16)
    a = a.parse_args(argv)
    lens, model = [700, 33, 1, 256, 1201], 1024
    layer = DecoderAttention(model, heads=16, kv_heads=4, d=128, n_pages=64)
    x = torch.randn((sum(lens), model), device="cuda").bfloat16()
    y, (k, v) = layer.prompts(x, lens)
    keys, values = [list(t.split(lens)) for t in (k, v)]
    for _ in range(a.steps):
        y, (q, k1, v1, o) = layer.tokens(torch.randn((len(lens), model), device="cuda").bfloat16())
        for s in range(len(lens)):
            keys[s], values[s] = torch.cat([keys[s], k1[s:s + 1]]), torch.cat([values[s], v1[s:s + 1]])
    whole = torch.empty_like(o)
    bsp.PromptPlan(bsp.device(), [1] * len(lens), layer.lens, 16, 4, 128).execute(q, torch.cat(keys), torch.cat(values), whole)
    bsp.device().synchronize()
    off = float((o.double() - whole.double()).norm() / whole.double().norm())
    print(f"{len(lens)} requests, {sum(lens)} prompt tokens, {a.steps} steps: 8-bit cache against 16-bit keys and values "
          f"{off:.4f} of the norm; output {tuple(y.shape)}")
    return off


if __name__ == "__main__":
    # e4m3 keeps 4 bits of a key or value: each is off by up to 1/16
    sys.exit(0 if main() < 0.1 else 1)
