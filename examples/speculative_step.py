"""Speculative decoding on the library's operators: a toy model (random weights, one projection per layer and head) whose attention is real.

Every step verifies a tree of drafted tokens per request in one pass: the drafts' cache rows are written behind the committed ones of the window, all
nodes attend with `hca_tree_decode`, `sample` draws a token at every node, the longest path of drafts that the draws agree with is accepted, and
`kv_entries_move` takes its rows to their places in the window, in all layers at once.  Now and then the worst requests are given up for copies of the best
(`kv_pages_free`, `kv_pages_fork`) and the pool is packed (`kv_pages_compact`).

    python examples/speculative_step.py [--requests 8] [--steps 12]
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import dsv4_attn_b200 as d  # noqa: E402
from dsv4_attn_b200 import layout  # noqa: E402

LAYERS, HEADS, VOCAB, WINDOW = 2, 16, 4096, 128
PARENTS = (-1, 0, 0, 1, 1, 3)            # node 0 is the last token drawn; the others are drafts
NODES = len(PARENTS)


class Cache:
    """Compressed entries in pages shared by all layers' tables, and a window of the last tokens with room for the drafts behind them."""

    def __init__(self, requests, pages, entries, gen):
        dev = dict(device="cuda")
        self.pool = layout.pack_entries(*torch.randn(LAYERS, pages, 64, 576, generator=gen, **dev).split([512, 64], dim=-1))
        width = (entries + 63) // 64 + 1
        self.table = torch.full((requests, width), -1, dtype=torch.int32, **dev)
        self.kv_len = torch.randint(1, entries + 1, (requests,), generator=gen, **dev).to(torch.int32)
        self.refs = torch.zeros(pages, dtype=torch.int32, **dev)
        used = ((self.kv_len + 63) // 64).tolist()
        order = torch.randperm(pages, generator=gen, **dev).to(torch.int32)
        at = 0
        for b, n in enumerate(used):
            self.table[b, :n] = order[at:at + n]
            self.refs[order[at:at + n].long()] = 1
            at += n
        # the window of a request is three pages of 64 rows, so that rows can be inserted as into any cache
        self.window = torch.zeros(LAYERS, requests, 192, layout.ENTRY_BYTES, dtype=torch.uint8, **dev)
        self.window_table = torch.arange(requests * 3, dtype=torch.int32, **dev).reshape(requests, 3)
        self.committed = torch.zeros(requests, dtype=torch.int64, **dev)


class Model:
    def __init__(self, gen):
        dev = dict(device="cuda")
        self.embed = torch.randn(VOCAB, 64, generator=gen, **dev)
        self.to_q = torch.randn(LAYERS, 64, HEADS * 576, generator=gen, **dev) / 8
        self.to_kv = torch.randn(LAYERS, 64, 576, generator=gen, **dev) / 8
        self.to_logits = torch.randn(LAYERS, HEADS * 512, VOCAB, generator=gen, **dev) / 12

    def logits(self, cache, tokens, positions, sees, window_len, status):
        """Logits of all nodes [B, T, VOCAB]; writes the nodes' rows into the windows."""
        B, T = tokens.shape
        x = self.embed[tokens]
        mask, total = layout.pack_tree_mask(sees), 0.0
        first = torch.full((B,), WINDOW, dtype=torch.int32, device="cuda")
        for layer in range(LAYERS):
            rows = d.rope_norm((x @ self.to_kv[layer]).bfloat16().reshape(B * T, 1, 576), positions).reshape(B, T, 576)
            d.kv_quantize_insert(rows, cache.window[layer].view(B * 3, 64, layout.ENTRY_BYTES), cache.window_table, first, status=status)
            q = d.rope_norm((x @ self.to_q[layer]).bfloat16().reshape(B * T, HEADS, 576), positions).reshape(B, T, HEADS, 576)
            out, _ = d.hca_tree_decode(q, cache.pool[layer], cache.table, cache.kv_len, cache.window[layer], window_len, mask, 576 ** -0.5, status=status)
            total = total + out.reshape(B, T, HEADS * 512).float() @ self.to_logits[layer]
        return total


def visible(cache, parents):
    """What the nodes see of the windows: tokens at places of their position modulo WINDOW, a node's ancestors, itself."""
    B = cache.committed.shape[0]
    drafts = layout.tree_sees(parents, 0)
    depth = drafts.sum(-1) - 1
    place = torch.arange(WINDOW, device="cuda")
    last = cache.committed[:, None] - 1                             # position of the newest committed token; a place holds the newest one that is alike
    position = last - (last - place) % WINDOW
    seen = (position[:, None] >= 0) & (position[:, None] > cache.committed[:, None, None] + depth[..., None] - WINDOW)
    return torch.cat([seen, drafts, torch.zeros(B, NODES, 64 - NODES, dtype=torch.bool, device="cuda")], dim=-1)


def accept(tokens, parents, drawn):
    """The longest path from node 0 whose drafts are the tokens drawn at their parents: nodes [B, T] (-1 behind its end), its length, and the token after it."""
    B, T = tokens.shape
    path = torch.full((B, T), -1, dtype=torch.int64, device="cuda")
    path[:, 0] = 0
    node, length = torch.zeros(B, dtype=torch.int64, device="cuda"), torch.ones(B, dtype=torch.int64, device="cuda")
    for depth in range(1, T):
        child = (parents == node[:, None]) & (tokens == drawn.gather(1, node[:, None]))
        found = child.any(1) & (length == depth)
        node = torch.where(found, child.int().argmax(1), node)
        path[:, depth] = torch.where(found, node, -1)
        length = length + found
    return path, length, drawn.gather(1, node[:, None])[:, 0]


def run(requests=8, steps=12, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cache, model = Cache(requests, requests * 6, 300, gen), Model(gen)
    status = d.new_status("cuda")
    parents = torch.tensor([PARENTS], device="cuda").expand(requests, NODES)
    window_len = torch.full((requests,), 192, dtype=torch.int32, device="cuda")
    last = torch.randint(0, VOCAB, (requests,), generator=gen, device="cuda")
    score = torch.zeros(requests, device="cuda")
    taken = []
    for step in range(steps):
        tokens = torch.randint(0, VOCAB, (requests, NODES), generator=gen, device="cuda")
        tokens[:, 0] = last
        depth = layout.tree_sees(parents, 0).sum(-1) - 1
        positions = (cache.committed[:, None] + depth).to(torch.int32).reshape(-1).contiguous()
        u = torch.rand(requests, NODES, generator=gen, device="cuda").reshape(-1)
        t, k, p = torch.full((requests * NODES,), 0.8, device="cuda"), torch.full((requests * NODES,), 40, dtype=torch.int32, device="cuda"), torch.full((requests * NODES,), 0.95, device="cuda")
        for proposing in (True, False):     # (a first pass stands in for the draft model: what it draws is drafted, and some of it accepted)
            logits = model.logits(cache, tokens, positions, visible(cache, parents), window_len, status)
            drawn, logprob = d.sample(logits.reshape(-1, VOCAB), u, temperature=t, top_k=k, top_p=p)
            drawn = drawn.reshape(requests, NODES).long()
            if proposing:
                tokens[:, 1::2] = drawn.gather(1, parents[:, 1::2])
        path, length, last = accept(tokens, parents, drawn)
        # accepted rows go to the places of their positions
        base = torch.arange(requests, device="cuda")[:, None] * 192
        place = (cache.committed[:, None] + torch.arange(NODES, device="cuda")) % WINDOW
        src = torch.where(path >= 0, base + WINDOW + path, -1).to(torch.int32).reshape(-1).contiguous()
        dst = torch.where(path >= 0, base + place, -1).to(torch.int32).reshape(-1).contiguous()
        d.kv_entries_move(cache.window, src, dst, status=status)
        cache.committed += length
        score += logprob.reshape(requests, NODES)[:, 0]
        taken.append(length.float().mean())
        if step % 4 == 3:               # the worst two requests become copies of the best two
            order = score.argsort().to(torch.int32)
            worst, best = order[:2].contiguous(), order[-2:].flip(0).contiguous()
            d.kv_pages_free(cache.table, cache.kv_len, cache.refs, worst, status=status)
            d.kv_pages_fork(cache.pool, cache.table, cache.kv_len, cache.refs, best, worst, status=status)
            w, g = worst.long(), best.long()
            cache.window[:, w], cache.committed[w], last[w], score[w] = cache.window[:, g], cache.committed[g], last[g], score[g]
            cache.table, cache.refs, live = d.kv_pages_compact(cache.pool, cache.table, cache.refs, status=status)
    return cache, torch.stack(taken), status


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--steps", type=int, default=12)
    a = ap.parse_args()
    cache, taken, status = run(a.requests, a.steps)
    print("tokens a step and request:", " ".join(f"{x:.2f}" for x in taken.tolist()), "| status", status.tolist(), "| pages in use", int((cache.refs > 0).sum()))


if __name__ == "__main__":
    main()
