"""One attention layer of a decoder on low-bit weights and a low-bit key/value cache: a prompt, then tokens one by one.

    python -m comp_amd.examples.cached_attention [--prompt 300] [--steps 8] [--cache q4_0]

Each step multiplies the activations with the Q4_0 projections for queries, keys and values (host.gemv_multi, or host.gemm
for the prompt), writes the new keys and values into the quantized cache (kv.write), attends over all of it (kv.attend) and
multiplies with the output projection.  Weights and inputs are random; the layer has 32 query and 8 kv heads of 128 channels.
The last line says how far the step's attention is from plain attention over what the cache holds."""

from __future__ import annotations

import argparse

import torch

from comp_amd import host, kv

HEADS, KV_HEADS, DIM, WIDTH = 32, 8, 128, 4096


def random_weight(rows, cols, seed):
    """Q4_0 split planes of random codes and scales."""
    g = torch.Generator().manual_seed(seed)
    wq = torch.randint(0, 256, (rows, cols // 2), dtype=torch.uint8, generator=g)
    ws = (0.002 + 0.002 * torch.rand((rows, cols // 32), generator=g)).half().view(torch.int16)
    return wq.cuda(), ws.cuda(), rows


class Layer:
    """The projections, and one sequence's pages of a cache."""

    def __init__(self, tokens, cache_format="q4_0", page=64):
        pages = -(-tokens // page)
        self.cache = kv.KVCache(pages, KV_HEADS, DIM, cache_format, cache_format, page)
        self.table = torch.randperm(pages, generator=torch.Generator().manual_seed(7)).to(torch.int32)[None].cuda()
        self.qkv = [random_weight(h * DIM, WIDTH, i) for i, h in enumerate((HEADS, KV_HEADS, KV_HEADS))]
        self.out = random_weight(WIDTH, HEADS * DIM, 3)
        self.length = 0

    def slots(self, first, count):
        j = torch.arange(first, first + count, device="cuda")
        return self.table[0].long()[j // self.cache.page] * self.cache.page + j % self.cache.page

    def step(self, x):
        """x f32 [tokens][WIDTH], the sequence's next tokens -> (the layer's output, queries, attention)."""
        t = x.shape[0]
        xq, xd = host.quantize("q4_0", x)
        q, k, v = (host.gemv("q4_0", wq, ws, xq, xd, n, WIDTH, block_n=None, mode=2)[0] for wq, ws, n in self.qkv) if t > 3 else (
            host.gemv_multi("q4_0", self.qkv, WIDTH, xq=xq, xd=xd))  # fmt: skip
        kv.write(self.cache, k.view(t, KV_HEADS, DIM), v.view(t, KV_HEADS, DIM), self.slots(self.length, t))
        self.length += t
        lengths = torch.tensor([self.length], dtype=torch.int32, device="cuda")
        starts = None if t == 1 else torch.tensor([0, t], dtype=torch.int32, device="cuda")
        q = q.view(t, HEADS, DIM)
        a = kv.attend(self.cache, q, self.table, lengths, starts, max_length=self.length)
        aq, ad = host.quantize("q4_0", a.view(t, HEADS * DIM))
        y, _ = host.gemv("q4_0", self.out[0], self.out[1], aq, ad, WIDTH, HEADS * DIM, block_n=None, mode=2)
        return y, q, a

    def plain(self, q):
        """Attention of the last rows' queries over what the cache holds, in plain f64 operations."""
        k, v = (x.double().repeat_interleave(HEADS // KV_HEADS, dim=1) for x in kv.read(self.cache, self.slots(0, self.length)))
        s = (q.double()[:, :, None] * k.transpose(0, 1)[None]).sum(-1) / DIM**0.5
        t, n = q.shape[0], self.length
        s = s.masked_fill(torch.arange(n, device="cuda") > torch.arange(n - t, n, device="cuda")[:, None, None], -torch.inf)
        return (torch.softmax(s, -1)[..., None] * v.transpose(0, 1)[None]).sum(2)


def run(prompt=300, steps=8, cache_format="q4_0"):
    """A prompt and `steps` single tokens -> the largest relative distance of an attention from plain()'s."""
    layer, worst = Layer(prompt + steps, cache_format), 0.0
    g = torch.Generator().manual_seed(11)
    x = torch.randn((prompt, WIDTH), generator=g).cuda()
    for i in range(steps + 1):
        y, q, a = layer.step(x)
        rows = slice(-4, None)  # of a prompt, the last rows
        want = layer.plain(q[rows])
        worst = max(worst, float((a[rows].double() - want).norm() / want.norm()))
        x = y[-1:] / y[-1:].square().mean().sqrt()
    return worst


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--prompt", type=int, default=300)
    p.add_argument("--steps", type=int, default=8)
    p.add_argument("--cache", choices=("q4_0", "q8_0"), default="q4_0")
    a = p.parse_args()
    print(f"{a.prompt} + {a.steps} tokens, {a.cache} cache: attention off by {run(a.prompt, a.steps, a.cache):.2e} of plain attention's")


if __name__ == "__main__":
    main()
