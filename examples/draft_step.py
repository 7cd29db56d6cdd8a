"""A draft model's steps on pages of K and V heads: a toy model (random weights) whose attention and cache are real.

Prompts of different lengths go in at once (`gqa_insert`, `gqa_prefill`: a sliding window and the first tokens); then every step drafts a token per request (`gqa_insert`,
`gqa_decode` with the attention every entry gets added up, `sample`), and requests whose cache has grown past a budget give up the entries that got the least
attention (`kv_evict`), with the pages behind them.  All layers share one block table.

    python examples/draft_step.py [--requests 6] [--steps 40] [--cache bf16|e4m3]
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import dsv4_attn_b200 as d  # noqa: E402

LAYERS, KV_HEADS, HEADS, DIM, WIDTH, VOCAB = 2, 2, 8, 64, 256, 1024
WINDOW, FIRST = 96, 4                # the prompt's attention
BUDGET, SLACK, RECENT = 160, 32, 48  # of a request's entries: kept, let grow beyond that, and kept in any case


class Cache:
    """K and V pages [layers, pages, 64, heads, dim], one table for all layers, and the attention that the entries have got."""

    def __init__(self, requests, longest, dtype):
        dev = dict(device="cuda")
        width = (longest + 63) // 64 + 1
        self.k, self.v = (torch.zeros(LAYERS, requests * width, 64, KV_HEADS, DIM, dtype=dtype, **dev) for _ in "kv")
        self.scale = torch.full((KV_HEADS,), 0.02, **dev) if dtype == torch.float8_e4m3fn else None
        self.table = torch.full((requests, width), -1, dtype=torch.int32, **dev)
        self.kv_len = torch.zeros(requests, dtype=torch.int32, **dev)
        self.refs = torch.zeros(requests * width, dtype=torch.int32, **dev)
        self.weights = torch.zeros(requests, width * 64, **dev)
        self.tokens = torch.full((requests, width * 64), -1, dtype=torch.int64, **dev)     # the place in its request's text of every entry

    def scales(self):
        return dict(k_scale=self.scale, v_scale=self.scale)

    def grow(self, new):
        """Pages for `new` entries more of each request, free ones in ascending order."""
        slot = torch.arange(self.table.shape[1], device="cuda")
        need = (slot < ((self.kv_len + new + 63) // 64)[:, None]) & (self.table < 0)
        free = torch.sort((self.refs > 0).int(), stable=True).indices.to(torch.int32)
        nth = need.flatten().long().cumsum(0).reshape(need.shape) - 1
        self.table = torch.where(need, free[nth.clamp(min=0)], self.table)
        self.refs.index_add_(0, torch.where(need, self.table, 0).flatten().long(), need.int().flatten())


class Model:
    def __init__(self, gen):
        dev = dict(device="cuda", generator=gen)
        self.embed = torch.randn(VOCAB, WIDTH, **dev)
        self.qkv = torch.randn(LAYERS, WIDTH, (HEADS + 2 * KV_HEADS) * DIM, **dev) / WIDTH ** 0.5
        self.out = torch.randn(LAYERS, HEADS * DIM, WIDTH, **dev) / (HEADS * DIM) ** 0.5

    def layers(self, x, attention):
        """attention(layer, q, k, v) -> the heads' outputs; rows of the fused projection are handed on as they lie."""
        for layer in range(LAYERS):
            rows = (x @ self.qkv[layer]).bfloat16().unflatten(-1, (HEADS + 2 * KV_HEADS, DIM))
            q, k, v = rows.split([HEADS, KV_HEADS, KV_HEADS], dim=-2)
            x = x + attention(layer, q, k, v).flatten(-2).float() @ self.out[layer]
        return x @ self.embed.T / WIDTH ** 0.5


def prompt(model, cache, tokens, start, status):
    """The prompts' tokens, packed; returns the logits behind the last token of each request."""
    new = start[1:] - start[:-1]
    cache.grow(new)
    pos, length = cache.kv_len.clone(), cache.kv_len + new

    def attention(layer, q, k, v):
        d.gqa_insert(k, v, cache.k[layer], cache.v[layer], cache.table, pos, q_start=start, status=status, **cache.scales())
        return d.gqa_prefill(q, start, cache.k[layer], cache.v[layer], cache.table, length, DIM ** -0.5, window=WINDOW, first=FIRST, status=status, **cache.scales())[0]

    logits = model.layers(model.embed[tokens], attention)
    place = torch.arange(cache.tokens.shape[1], device="cuda")
    cache.tokens = torch.where(place < length[:, None], place, -1)
    cache.kv_len = length
    return logits[start[1:].long() - 1]


def step(model, cache, token, text_len, status):
    """One token per request; returns its logits."""
    one = torch.ones_like(cache.kv_len)
    cache.grow(one)
    pos, length = cache.kv_len.clone(), cache.kv_len + one
    cache.tokens.scatter_(1, pos[:, None].long(), text_len[:, None])

    def attention(layer, q, k, v):
        d.gqa_insert(k, v, cache.k[layer], cache.v[layer], cache.table, pos, status=status, **cache.scales())
        return d.gqa_decode(q, cache.k[layer], cache.v[layer], cache.table, length, DIM ** -0.5, weights=cache.weights, status=status, **cache.scales())[0]

    logits = model.layers(model.embed[token][:, None], attention)[:, 0]
    cache.kv_len = length
    return logits


def evict(cache, status):
    """Requests that have grown past the budget and its slack go back to the budget."""
    keep = torch.where(cache.kv_len > BUDGET + SLACK, BUDGET, cache.kv_len)
    cache.table, cache.kv_len, cache.refs, cache.weights, kept = d.kv_evict((cache.k, cache.v), cache.table, cache.kv_len, cache.refs, cache.weights, keep, first=FIRST, recent=RECENT,
                                                                            status=status)
    cache.tokens = torch.where(kept >= 0, cache.tokens.gather(1, kept.clamp(min=0).long()), -1)
    return kept


def run(requests=6, steps=40, dtype=torch.bfloat16, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    model, status = Model(gen), d.new_status("cuda")
    lengths = torch.randint(30, 250, (requests,), generator=gen, device="cuda", dtype=torch.int32)
    cache = Cache(requests, 250 + SLACK + 64, dtype)
    start = torch.zeros(requests + 1, dtype=torch.int32, device="cuda")
    start[1:] = lengths.cumsum(0)
    tokens = torch.randint(0, VOCAB, (int(start[-1]),), generator=gen, device="cuda")
    logits, text_len = prompt(model, cache, tokens, start, status), lengths.long()
    drafted, held = [], []
    for i in range(steps):
        token, _ = d.sample(logits.contiguous(), torch.rand(requests, generator=gen, device="cuda"), temperature=torch.full((requests,), 0.8, device="cuda"))
        drafted.append(token)
        logits = step(model, cache, token.long(), text_len, status)
        text_len = text_len + 1
        if i % 8 == 7:
            evict(cache, status)
        held.append(cache.kv_len.clone())
    return cache, torch.stack(drafted), torch.stack(held), status


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--requests", type=int, default=6)
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--cache", choices=("bf16", "e4m3"), default="bf16")
    a = ap.parse_args()
    cache, drafted, held, status = run(a.requests, a.steps, dict(bf16=torch.bfloat16, e4m3=torch.float8_e4m3fn)[a.cache])
    print("entries held:", held[0].tolist(), "->", held[-1].tolist(), "| pages in use", int((cache.refs > 0).sum()), "| status", status.tolist())


if __name__ == "__main__":
    main()
