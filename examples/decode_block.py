"""The attention blocks of a quantized decoder, decoding with parallel samples.

Per layer: int8 projection to q, k, v -> rotary positions and the store into
cache pages (one launch) -> attention over the pages -> int8 output
projection.  Prompts run token by token, fork into samples that share their
pages, finished samples are freed and the pool is compacted; no length, page
or slot visits the host.

    python examples/decode_block.py [--layers 4] [--prompts 4] [--samples 8]
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from ubridge_amd import int8, kvcache, moe, rope  # noqa: E402


class Block:
    """Random weights of one layer's projections."""

    def __init__(self, hidden, Hq, Hkv, D, generator, device="cuda"):
        def linear(n, k):
            w = torch.randint(-127, 128, (n, k), generator=generator, dtype=torch.int8)
            return int8.Linear(w.to(device), torch.full((n,), 1 / (73 * k ** 0.5), device=device))
        self.Hq, self.Hkv, self.D = Hq, Hkv, D
        self.qkv, self.out = linear((Hq + 2 * Hkv) * D, hidden), linear(hidden, Hq * D)

    def __call__(self, x, cache, layer, turn, positions, slots, tables, lens):
        """x [B, hidden], one new token of each sequence."""
        q, k, v = (y.unflatten(1, (-1, self.D)) for y in self.qkv(x).split(
            [self.Hq * self.D, self.Hkv * self.D, self.Hkv * self.D], 1))
        q = cache.append(layer, q, k, v, slots, positions=positions, rope=turn)
        return self.out(cache.attend(layer, q, tables, lens).flatten(1))


def grow(cache, rows):
    """A place for one more token of each row (all different): (positions,
    slots).  A row whose pages are full gets the lowest free one.  Where none is
    left, or the row has its width of pages, the slot is negative (the token is
    stored nowhere) and attention reports the row."""
    r = rows.long()
    at = cache.lens[r].long()
    full = at >= cache.width * cache.S
    i = (at // cache.S).clamp(max=cache.width - 1)
    need = (at % cache.S == 0) & ~full
    used = cache.refs != 0
    rank = torch.cumsum(need, 0) - 1
    got = need & (rank < (~used).sum())
    free = torch.argsort(used.int(), stable=True)[rank.clamp(0, len(used) - 1)].int()
    held = cache.tables[r, i]
    page = torch.where(need, torch.where(got, free, -1), held)
    cache.tables[r, i] = page
    cache.refs.index_add_(0, page.clamp(min=0).long(), got.int())
    cache.lens[r] += 1
    return at, torch.where(full | (page < 0), -1, page.long() * cache.S + at % cache.S)


def step(blocks, x, cache, turn, rows):
    positions, slots = grow(cache, rows)
    tables, lens = cache.tables[rows.long()], cache.lens[rows.long()]
    for layer, block in enumerate(blocks):
        x = x + block(x, cache, layer, turn, positions, slots, tables, lens)
    return x


def main():
    p = argparse.ArgumentParser()
    for name, default in (("layers", 4), ("hidden", 4096), ("heads", 32), ("kv_heads", 8), ("dim", 128),
                          ("prompts", 4), ("samples", 8), ("prompt", 200), ("tokens", 100)):
        p.add_argument("--" + name, type=int, default=default)
    a = p.parse_args()
    g = torch.Generator().manual_seed(0)
    blocks = [Block(a.hidden, a.heads, a.kv_heads, a.dim, g) for _ in range(a.layers)]
    S, n = 16, a.prompts * a.samples
    width = -(-(a.prompt + a.tokens) // S) + 1
    kv = torch.zeros(a.layers, 2, (a.prompts + n) * width, a.kv_heads, S, a.dim, dtype=torch.bfloat16, device="cuda")
    cache = kvcache.PagedCache(kv, rows=a.prompts + n, width=width)
    turn = rope.Rope(a.dim, base=500000.0)
    rows = lambda lo, hi: torch.arange(lo, hi, dtype=torch.int32, device="cuda")
    prompts, samples = rows(0, a.prompts), rows(a.prompts, a.prompts + n)
    noise = lambda b: torch.randn(b, a.hidden, device="cuda").bfloat16()
    for _ in range(a.prompt):
        step(blocks, noise(a.prompts), cache, turn, prompts)
    cache.fork(torch.arange(n, dtype=torch.int32, device="cuda") % a.prompts, samples)
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(a.tokens):
        y = step(blocks, noise(n), cache, turn, samples)
    torch.cuda.synchronize()
    t = (time.perf_counter() - t) / a.tokens
    cache.free(samples[::2].contiguous())
    used = int(cache.compact())
    y = step(blocks, noise(n // 2), cache, turn, samples[1::2].contiguous())
    moe.device_error()
    assert bool(torch.isfinite(y).all())
    print(f"{n} samples, {a.layers} layers: {t * 1e6:.0f} us a token step, {n / t:.0f} tokens/s; "
          f"{used} pages in use after half the samples left")


if __name__ == "__main__":
    main()
