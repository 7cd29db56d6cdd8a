"""What a draft model next to the compressed layers needs of its cache, as calls that can be timed and compared: pages of ordinary K and V heads, the
attention of new tokens over them (all of the cache, or a sliding window and the first tokens), prompts, and eviction of the entries that got
the least attention.

`own` false: the operators in plain torch operations, 32-bit arithmetic; true: the library's kernels.  Cases name sizes only;
`prepare` makes what a serving engine holds before the call (pools, tables, queries, weights), `run` is one call."""
import math

import torch

own = False

PAGE = 64                                                   # entries a page
TYPES = dict(bf16=torch.bfloat16, f16=torch.float16, e4m3=torch.float8_e4m3fn)


def listed():
    return [
        # ── new tokens' K and V into the pages ──
        # a decode step of a batch: one token each, from the rows of a fused projection
        dict(name="insert_step", kind="insert", B=64, T=1, Hkv=8, G=4, D=128, kv=2000, dtype="bf16", packed=False),
        # prompts of different lengths, packed one behind the other, into an 8-bit cache
        dict(name="insert_prompts_e4m3", kind="insert", B=6, T=4096, Hkv=8, G=4, D=128, kv=4096, dtype="e4m3", packed=True),
        # ── attention of one new token, or a few drafted ones ──
        # one user's next token
        dict(name="decode_one_request", kind="decode", B=1, T=1, Hkv=8, G=4, D=128, kv=1000, window=0, first=0, dtype="bf16", ragged=False, sink=False, weights=False),
        # a batch of requests of very different lengths
        dict(name="decode_batch_ragged", kind="decode", B=64, T=1, Hkv=8, G=4, D=128, kv=16384, window=0, first=0, dtype="bf16", ragged=True, sink=False, weights=False),
        # long contexts in 8 bits, five drafted tokens verified at once
        dict(name="decode_drafts_e4m3", kind="decode", B=12, T=5, Hkv=8, G=8, D=128, kv=32768, window=0, first=0, dtype="e4m3", ragged=False, sink=True, weights=False),
        # a sliding window and the first tokens, for a large batch; odd group
        dict(name="decode_window_first", kind="decode", B=256, T=1, Hkv=8, G=5, D=64, kv=8000, window=1024, first=4, dtype="f16", ragged=True, sink=False, weights=False),
        # ── with the attention every entry gets added up ──
        dict(name="decode_weights_one", kind="decode", B=1, T=1, Hkv=4, G=4, D=64, kv=2100, window=0, first=0, dtype="f16", ragged=False, sink=False, weights=True),
        dict(name="decode_weights_batch", kind="decode", B=32, T=1, Hkv=8, G=4, D=128, kv=8192, window=0, first=0, dtype="bf16", ragged=True, sink=False, weights=True),
        # ── prompts: a sliding window and the first tokens; a piece of a long prompt behind what is cached ──
        dict(name="prefill_window_ragged", kind="prefill", B=5, T=4096, Hkv=8, G=4, D=128, kv=4096, window=1024, first=4, dtype="bf16", sink=False),
        dict(name="prefill_piece_long", kind="prefill", B=1, T=4096, Hkv=8, G=4, D=128, kv=16384, window=0, first=0, dtype="bf16", sink=True),
        # ── eviction ──
        # one request back to its budget
        dict(name="evict_one_request", kind="evict", L=2, B=1, Hkv=4, D=64, kv=2176, keep=2048, first=4, recent=256, dtype="f16", ragged=False),
        # a batch through all layers of a cache
        dict(name="evict_batch_layers", kind="evict", L=8, B=24, Hkv=8, D=128, kv=4608, keep=4096, first=4, recent=512, dtype="bf16", ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("insert", "decode", "decode", "decode", "prefill", "prefill", "evict"))
    heads = dict(Hkv=rng.choice((1, 2, 3, 4, 8, 16)), G=rng.choice((1, 2, 4, 5, 7, 8, 16)), D=rng.choice((64, 128, 128, 256)))
    if kind == "insert":
        while True:
            c = dict(kind=kind, B=_log(rng, 1, 128), T=_log(rng, 1, 4096), **heads, kv=0, dtype=rng.choice(tuple(TYPES)), packed=rng.random() < 0.5)
            c["kv"] = c["T"] + rng.randint(0, 4000)
            if c["B"] * c["T"] * c["Hkv"] * c["D"] <= 25_000_000 and c["B"] * c["kv"] * c["Hkv"] * c["D"] <= 500_000_000:
                return c
    if kind == "decode":
        while True:
            c = dict(kind=kind, B=_log(rng, 1, 256), T=rng.choice((1, 1, 1, 1, 2, 3, 5, 8, 16)), **heads, kv=_log(rng, 1, 100_000),
                     window=rng.choice((0, 0, 0, 100, 512, 4096)), first=rng.choice((0, 1, 4, 70)), dtype=rng.choice(tuple(TYPES)), ragged=rng.random() < 0.5,
                     sink=rng.random() < 0.3, weights=rng.random() < 0.3)
            if c["B"] * c["kv"] * c["Hkv"] * c["D"] <= 500_000_000 and c["B"] * c["kv"] * c["Hkv"] * c["G"] * c["T"] <= 100_000_000:
                return c
    if kind == "prefill":
        while True:
            c = dict(kind=kind, B=_log(rng, 1, 16), T=_log(rng, 16, 8192), **heads, kv=0, window=rng.choice((0, 0, 128, 1000, 4096)), first=rng.choice((0, 1, 4, 70)),
                     dtype=rng.choice(tuple(TYPES)), sink=rng.random() < 0.3)
            c["kv"] = c["T"] + rng.choice((0, 0, _log(rng, 1, 16384)))
            if c["B"] * c["kv"] * c["T"] * c["Hkv"] * c["G"] <= 2_000_000_000 and c["D"] <= 128 * (1 + (c["kv"] < 4096)):
                return c
    while True:
        c = dict(kind=kind, L=_log(rng, 1, 32), B=_log(rng, 1, 64), Hkv=heads["Hkv"], D=heads["D"], kv=0, keep=_log(rng, 32, 16384), first=rng.choice((0, 1, 4, 16)),
                 recent=0, dtype=rng.choice(tuple(TYPES)), ragged=rng.random() < 0.5)
        c["kv"] = c["keep"] + _log(rng, 1, c["keep"])
        c["recent"] = rng.randint(0, c["keep"] // 2)
        if c["L"] * c["B"] * c["kv"] * c["Hkv"] * c["D"] <= 900_000_000:
            return c


# ── inputs ──
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, by=1.0):
    out = torch.empty(shape, device="cuda", dtype=dtype)
    rows = out.reshape(-1, shape[-1])
    step = max(1, (1 << 26) // shape[-1])
    for at in range(0, rows.shape[0], step):
        part = rows[at:at + step]
        part.copy_((torch.randn(part.shape, device="cuda", generator=g) * by).to(dtype))
    return out


def _scales(c, g):
    """The scales of an 8-bit cache's heads: values of deviation 1 reach up to some 100 of e4m3's 448."""
    if c["dtype"] != "e4m3":
        return None, None
    return tuple(0.04 + 0.02 * torch.rand(c["Hkv"], device="cuda", generator=g) for _ in "kv")


def _pools(c, g, B, kv, lead=()):
    """Pools of K and V heads, every place filled, and a table of pages in random order with room for `kv` entries and one page more."""
    pages = (kv + PAGE - 1) // PAGE + 1
    k_scale, v_scale = _scales(c, g)
    P = B * pages + 3
    shape = (*lead, P, PAGE, c["Hkv"], c["D"])
    by = 20.0 if c["dtype"] == "e4m3" else 1.0
    pools = [_randn(g, *shape, dtype=TYPES[c["dtype"]], by=by) for _ in "kv"]
    table = torch.randperm(P, device="cuda", generator=g)[:B * pages].int().reshape(B, pages)
    return dict(k_pool=pools[0], v_pool=pools[1], table=table, k_scale=k_scale, v_scale=v_scale)


def _lengths(c, g, B, kv, low):
    n = torch.full((B,), kv, device="cuda", dtype=torch.int32)
    if B > 1:
        n = (low + (kv - low) * torch.rand(B, device="cuda", generator=g) ** 0.7).int()
        n[0] = kv
    return n


def _shares(B, T, seed):
    """Lengths of prompts: T and parts of it, the same ones in another order for another seed."""
    part = (torch.arange(1, B + 1, device="cuda", dtype=torch.float64) * 0.6180339887498949) % 1
    new = (T * part ** 0.7).int().clamp(min=1)
    new[0] = T
    return new.roll(seed % B)


def _query_type(c):
    return torch.bfloat16 if c["dtype"] == "e4m3" else TYPES[c["dtype"]]


def prepare(case, seed):
    c, g = dict(case), _gen(seed)
    kind, B = c["kind"], c["B"]
    if kind == "evict":
        s = _pools(c, g, B, c["kv"], (c["L"],))
        n = _lengths(c, g, B if c["ragged"] else 1, c["kv"], c["keep"] - c["keep"] // 8).expand(B).contiguous()
        pages = s["table"].shape[1]
        held = torch.arange(pages, device="cuda") < ((n + PAGE - 1) // PAGE)[:, None]
        s["table"] = torch.where(held, s["table"], -1)
        refs = torch.zeros(s["k_pool"].shape[1] + 1, device="cuda", dtype=torch.int32)
        refs[torch.where(held, s["table"].long(), refs.numel() - 1)] = 1
        # attention adds up very unevenly: a few entries get most of it
        weights = torch.exp(2.5 * torch.randn(B, pages * PAGE, device="cuda", generator=g))
        weights *= torch.arange(pages * PAGE, device="cuda") < n[:, None]
        return dict(case=c, **s, kv_len=n, refs=refs[:-1].contiguous(), weights=weights)
    s = _pools(c, g, B, c["kv"])
    H, D, T, kv = c["Hkv"] * c["G"], c["D"], c["T"], c["kv"]
    dtype = _query_type(c)
    if kind == "decode":
        n = _lengths(c, g, B if c["ragged"] else 1, kv, min(kv, T)).expand(B).contiguous()
        s |= dict(q=_randn(g, B, T, H, D, dtype=dtype, by=2.0), kv_len=n, sink=torch.randn(H, device="cuda", generator=g) if c["sink"] else None, scale=D ** -0.5)
        if c["weights"]:
            s["weights"] = torch.rand(B, s["table"].shape[1] * PAGE, device="cuda", generator=g) * (torch.arange(s["table"].shape[1] * PAGE, device="cuda") < (n - T)[:, None])
        return dict(case=c, **s)
    # new tokens of prompts: T of the first request, fewer of the others, behind what their requests hold already
    new = _shares(B, T, seed)
    start = torch.zeros(B + 1, device="cuda", dtype=torch.int32)
    start[1:] = new.cumsum(0)
    past = (torch.rand(B, device="cuda", generator=g) * (kv - T + 1)).int()
    past[seed % B] = kv - T
    if kind == "prefill":
        N = int(start[-1])
        return dict(case=c, **s, q=_randn(g, N, H, D, dtype=dtype, by=2.0), start=start, kv_len=past + new, sink=torch.randn(H, device="cuda", generator=g) if c["sink"] else None,
                    scale=D ** -0.5)
    # the projection gives queries, keys and values of a token in one row
    rows = int(start[-1]) if c["packed"] else B * T
    qkv = _randn(g, rows, H + 2 * c["Hkv"], D, dtype=dtype)
    if not c["packed"]:
        qkv = qkv.reshape(B, T, H + 2 * c["Hkv"], D)
    k, v = qkv[..., H:H + c["Hkv"], :], qkv[..., H + c["Hkv"]:, :]
    return dict(case=c, **s, k=k, v=v, start=start if c["packed"] else None, past=past)


# ── the plain forms ──
def _quantised(x, scale, dtype):
    if scale is None:
        return x.to(dtype)
    return (x.float() / scale[:, None]).clamp(-448, 448).to(dtype)


def _plain_insert(s):
    c, table = s["case"], s["table"]
    k, v, past = s["k"].flatten(0, -3), s["v"].flatten(0, -3), s["past"].long()
    row = torch.arange(k.shape[0], device="cuda")
    if c["packed"]:
        b = torch.searchsorted(s["start"][1:].long(), row, right=True)
        at = past[b] + row - s["start"].long()[b]
    else:
        b = row // c["T"]
        at = past[b] + row % c["T"]
    entry = table[b, at // PAGE].long() * PAGE + at % PAGE
    for pool, x, scale in ((s["k_pool"], k, s["k_scale"]), (s["v_pool"], v, s["v_scale"])):
        width = pool.element_size()
        flat = pool.view(torch.uint8 if width == 1 else torch.int16).view(-1, c["Hkv"], c["D"])
        flat[entry] = _quantised(x, scale, pool.dtype).view(flat.dtype)
    return dict(k_pool=s["k_pool"], v_pool=s["v_pool"])


def _rows(pool, table, scale):
    """The entries of every request, [B, Hkv, N, D] in 32 bits."""
    x = pool.view(torch.uint8)[table.long().clamp(min=0)].view(pool.dtype).float()
    x = x.flatten(1, 2).transpose(1, 2)
    return x if scale is None else x * scale[:, None, None]


def _plain_attend(s, q, at):
    """Tokens q [B, T, H, D] at the places `at` [B, T] of their requests (negative: a token that sees nothing).  Returns out [B, T, H, D], lse [B, T, H]
    and the weights of the entries, added up over tokens and heads, [B, N]."""
    c = s["case"]
    B, T, H, D = q.shape
    k, v = _rows(s["k_pool"], s["table"], s["k_scale"]), _rows(s["v_pool"], s["table"], s["v_scale"])
    N = k.shape[2]
    j = torch.arange(N, device="cuda")
    back = at[..., None] - j                                                    # [B, T, N]
    seen = (back >= 0) & ((back < c["window"]) | (j < c["first"]) if c["window"] else True)
    x = torch.matmul(q.float().reshape(B, T, c["Hkv"], c["G"], D).permute(0, 2, 1, 3, 4).reshape(B, c["Hkv"], T * c["G"], D), k.transpose(2, 3)) * s["scale"]
    x = x.reshape(B, c["Hkv"], T, c["G"], N).masked_fill_(~seen[:, None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = x.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    below = total if s["sink"] is None else total + torch.exp(s["sink"].reshape(c["Hkv"], 1, c["G"], 1) - top)
    e /= torch.where(total == 0, torch.ones_like(below), below)
    weights = e.sum((1, 2, 3))
    out = torch.matmul(e.reshape(B, c["Hkv"], T * c["G"], N), v).reshape(B, c["Hkv"], T, c["G"], D).permute(0, 2, 1, 3, 4).reshape(B, T, H, D)
    lse = (top + torch.log(total))[..., 0].permute(0, 2, 1, 3).reshape(B, T, H)
    return out.to(q.dtype), lse, weights


def _plain_decode(s):
    T = s["case"]["T"]
    at = (s["kv_len"] - T)[:, None] + torch.arange(T, device="cuda")
    out, lse, weights = _plain_attend(s, s["q"], at)
    return dict(out=out, lse=lse, **(dict(weights=s["weights"] + weights) if s["case"]["weights"] else {}))


def _plain_prefill(s):
    c, q, start = s["case"], s["q"], s["start"].long()
    new = start[1:] - start[:-1]
    t = torch.arange(c["T"], device="cuda")
    there = t < new[:, None]                                                    # requests padded to the longest
    row = torch.where(there, start[:-1, None] + t, 0)
    at = torch.where(there, (s["kv_len"] - new)[:, None] + t, -1)
    out, lse, _ = _plain_attend(s, q[row], at)
    b = torch.searchsorted(start[1:], torch.arange(q.shape[0], device="cuda"), right=True)
    place = torch.arange(q.shape[0], device="cuda") - start[b]
    return dict(out=out[b, place], lse=lse[b, place])


def _plain_evict(s):
    c, table, n, weights = s["case"], s["table"], s["kv_len"].long(), s["weights"]
    B, pages = table.shape
    keep, cap = c["keep"], pages * PAGE
    j = torch.arange(cap, device="cuda")
    there = j < n[:, None]
    always = (j < c["first"]) | (j >= (n - c["recent"])[:, None])
    order = torch.sort(torch.where(there, torch.where(always, math.inf, weights), -math.inf), dim=1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(1, order, j.expand(B, cap))
    stays = there & (rank < keep)
    kept = torch.sort(torch.where(stays, j, cap), dim=1).values
    there = kept < cap
    kept = torch.where(there, kept, -1)
    length = there.sum(1)
    slots = torch.arange(pages, device="cuda")
    goes = (slots >= ((length + PAGE - 1) // PAGE)[:, None]) & (table >= 0)
    refs = s["refs"].clone()
    refs.index_add_(0, torch.where(goes, table, 0).long().reshape(-1), -goes.int().reshape(-1))
    b, to = torch.nonzero(there & (kept != j), as_tuple=True)
    src, dst = (table[b, i // PAGE].long() * PAGE + i % PAGE for i in (kept[b, to], to))
    for pool in (s["k_pool"], s["v_pool"]):
        flat = pool.view(torch.uint8).reshape(c["L"], -1, c["Hkv"] * c["D"] * pool.element_size())
        flat[:, dst] = flat[:, src]
    return dict(k_pool=s["k_pool"], v_pool=s["v_pool"], table=torch.where(goes, -1, table), kv_len=length.int(), refs=refs,
                weights=torch.where(there, weights.gather(1, kept.clamp(min=0)), 0), kept=kept.int())


def run(state):
    s = state
    c = s["case"]
    if own:
        import dsv4_attn_b200 as d
        if c["kind"] == "insert":
            d.gqa_insert(s["k"], s["v"], s["k_pool"], s["v_pool"], s["table"], s["past"], q_start=s["start"], k_scale=s["k_scale"], v_scale=s["v_scale"])
            return dict(k_pool=s["k_pool"], v_pool=s["v_pool"])
        if c["kind"] == "evict":
            table, kv_len, refs, weights, kept = d.kv_evict((s["k_pool"], s["v_pool"]), s["table"], s["kv_len"], s["refs"], s["weights"], c["keep"], first=c["first"],
                                                            recent=c["recent"])
            return dict(k_pool=s["k_pool"], v_pool=s["v_pool"], table=table, kv_len=kv_len, refs=refs, weights=weights, kept=kept)
        how = dict(window=c["window"], first=c["first"], k_scale=s["k_scale"], v_scale=s["v_scale"], attn_sink=s["sink"])
        if c["kind"] == "prefill":
            out, lse = d.gqa_prefill(s["q"], s["start"], s["k_pool"], s["v_pool"], s["table"], s["kv_len"], s["scale"], **how)
            return dict(out=out, lse=lse)
        weights = s["weights"].clone() if c["weights"] else None        # (added to in place)
        out, lse = d.gqa_decode(s["q"], s["k_pool"], s["v_pool"], s["table"], s["kv_len"], s["scale"], weights=weights, **how)
        return dict(out=out, lse=lse, **(dict(weights=weights) if c["weights"] else {}))
    if c["kind"] == "insert":
        return _plain_insert(s)
    if c["kind"] == "evict":
        return _plain_evict(s)
    return _plain_decode(s) if c["kind"] == "decode" else _plain_prefill(s)


def work(case):
    c = case
    width = 1 if c["dtype"] == "e4m3" else 2
    entry = 2 * c["Hkv"] * c["D"] * width                                       # bytes of an entry's K and V in one layer
    if c["kind"] == "insert":
        rows = c["B"] * c["T"] * (0.6 if c["packed"] and c["B"] > 1 else 1.0)
        return dict(bytes=rows * (entry + 4 * c["Hkv"] * c["D"]), flops=0)
    if c["kind"] == "evict":
        n = c["kv"] if not c["ragged"] else c["keep"] * 0.875 + (c["kv"] - c["keep"] * 0.875) * 0.6
        share = 1.0 if not c["ragged"] else min(1.0, 0.2 + 0.8 * (n > c["keep"]))
        return dict(bytes=c["B"] * (share * 2 * entry * c["L"] * (c["keep"] - c["first"]) + 12 * n), flops=0)
    H = c["Hkv"] * c["G"]
    if c["kind"] == "decode":
        kv = c["kv"] * (0.6 if c["ragged"] and c["B"] > 1 else 1.0)
        kv = min(kv, c["window"] + c["T"] + c["first"]) if c["window"] else kv
        rows = c["B"] * c["T"] * H
        return dict(bytes=c["B"] * kv * (entry + (8 if c["weights"] else 0)) + rows * (4 * c["D"] + 4), flops=4.0 * rows * kv * c["D"])
    T, B = c["T"], c["B"]
    mean = 1.0 if B == 1 else 0.6
    past = (c["kv"] - T) * (1.0 if B == 1 else 0.5)
    new = T * mean
    seen = past + new / 2                                                       # by a token, on average
    if c["window"]:
        seen = min(seen, c["window"] + c["first"])
    return dict(bytes=B * (new * H * (4 * c["D"] + 4) + (past + new) * entry), flops=4.0 * B * new * H * seen * c["D"])


# ── the definitions in 64 bits ──
def exact(case, seed):
    c = case
    if c["kind"] in ("insert", "evict"):
        return None             # values that move, whole numbers, and a rounding to the cache's type
    s = prepare(case, seed)
    start = s["start"].tolist() if c["kind"] == "prefill" else [b * c["T"] for b in range(c["B"] + 1)]
    q = s["q"].flatten(0, -3)
    lens, G = s["kv_len"].tolist(), c["G"]
    if sum((b - a) * n for a, b, n in zip(start, start[1:], lens)) * c["Hkv"] * G * c["D"] > 6e12:
        return None
    sink = None if s["sink"] is None else s["sink"].double()
    out = torch.zeros(q.shape, device="cuda", dtype=torch.float64)
    lse = torch.full(q.shape[:2], -math.inf, device="cuda", dtype=torch.float64)
    weights = s["weights"].double() if c.get("weights") else None
    for b, n in enumerate(lens):
        pages = s["table"][b, :(n + PAGE - 1) // PAGE].long()
        k, v = (s[name][pages].double().flatten(0, 1)[:n] for name in ("k_pool", "v_pool"))
        if c["dtype"] == "e4m3":
            k, v = k * s["k_scale"].double()[:, None], v * s["v_scale"].double()[:, None]
        T = start[b + 1] - start[b]
        for lo in range(0, T, 1024):
            hi = min(T, lo + 1024)
            place = n - T + torch.arange(lo, hi, device="cuda")[:, None]
            j = torch.arange(n, device="cuda")
            hidden = j > place
            if c["window"]:
                hidden |= (j <= place - c["window"]) & (j >= c["first"])
            rows = slice(start[b] + lo, start[b] + hi)
            for h in range(c["Hkv"] * G):
                x = (q[rows, h].double() @ k[:, h // G].T * s["scale"]).masked_fill(hidden, -math.inf)
                total = torch.logsumexp(x, -1)
                whole = total if sink is None else torch.logaddexp(total, sink[h])
                p = torch.exp(x - whole[:, None]).nan_to_num(0.0)
                out[rows, h] = p @ v[:, h // G]
                lse[rows, h] = total
                if weights is not None:
                    weights[b, :n] += p.sum(0)
    shape = s["q"].shape
    return dict(out=out.reshape(shape), lse=lse.reshape(shape[:-1]), **({} if weights is None else dict(weights=weights)))
