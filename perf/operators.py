"""A speculative decoding step on the paged latent cache, as calls that can be timed and compared: attention of a tree of
drafted tokens, sampling from given random numbers, and the pages of the cache around them (fork, free, compact, copy, move).

`own` false: the operators in plain torch operations, 32-bit arithmetic; true: the library's kernels.  Cases name sizes only;
`prepare` makes what a serving engine holds before the call (cache, tables, logits, random numbers), `run` is one call."""
import math

import torch

own = False

LATENT, ROPE, QK, ENTRY, PAGE = 512, 64, 576, 656, 64      # a cache entry: 512 e4m3 | 4 FP32 scales | 64 BF16; 64 entries a page
FIXED = 2.0 ** 40                                           # sampling weights are integers: floor(2^40 exp((l - max) / T))


def listed():
    return [
        # ── a tree of T drafted tokens per request over HCA's compressed entries and a window of 128 tokens + the drafts ──
        # one request, few heads per GPU: what one user waits for
        dict(name="tree_one_request", kind="tree", B=1, T=6, H=16, kv=300, window=128, ragged=False, sink=True),
        # a batch at 100k context (782 entries), 16 drafts
        dict(name="tree_batch_100k", kind="tree", B=64, T=16, H=128, kv=782, window=128, ragged=False, sink=True),
        # ragged requests (some without a compressed entry), odd head and draft counts: heads of a tensor-parallel shard
        dict(name="tree_ragged_odd", kind="tree", B=23, T=11, H=40, kv=3000, window=101, ragged=True, sink=False),
        # few requests, long contexts, wide trees
        dict(name="tree_long_wide", kind="tree", B=4, T=32, H=128, kv=25000, window=128, ragged=True, sink=True),
        # ── sampling ──
        # one request's next token, usual settings
        dict(name="sample_one_row", kind="sample", N=1, V=32000, dtype="f32", settings="usual", pad=0, masked=False),
        # a batch of 64, every request with settings of its own, some greedy, grammar masks on some rows
        dict(name="sample_batch", kind="sample", N=64, V=131072, dtype="f32", settings="mixed", pad=0, masked=True),
        # temperature only, odd vocabulary: rows start at any alignment
        dict(name="sample_temperature_odd", kind="sample", N=301, V=50257, dtype="f16", settings="temperature", pad=0, masked=False),
        # all nodes of 64 trees of 16, BF16 logits in a padded buffer
        dict(name="sample_tree_nodes", kind="sample", N=1024, V=131072, dtype="bf16", settings="mixed", pad=128, masked=False),
        # ── pages ──
        # four beams of one request replaced by forks of the others
        dict(name="pages_fork_beams", kind="pages", op="fork", L=1, B=8, kv=782, P=128, n=4),
        # half a batch forked through all layers of a cache
        dict(name="pages_fork_layers", kind="pages", op="fork", L=16, B=96, kv=4000, P=7000, n=48),
        # a fragmented pool packed to its front
        dict(name="pages_compact", kind="pages", op="compact", L=8, B=64, kv=2500, P=4600, n=0),
        # accepted drafts moved to their places in every layer's window
        dict(name="pages_accept_rows", kind="pages", op="move", L=16, B=64, kv=144, P=64, n=5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("tree", "tree", "sample", "sample", "pages"))
    if kind == "tree":
        while True:
            c = dict(kind="tree", B=_log(rng, 1, 64), T=_log(rng, 1, 64), H=rng.choice((8, 16, 20, 40, 64, 100, 128)), kv=_log(rng, 64, 25000),
                     window=rng.randint(64, 160), ragged=rng.random() < 0.5, sink=rng.random() < 0.5)
            if c["B"] * c["T"] * c["H"] * (c["kv"] + c["window"]) <= 4 * 32 * 128 * 16000:
                return c
    if kind == "sample":
        while True:
            c = dict(kind="sample", N=_log(rng, 1, 1024), V=_log(rng, 1000, 200000), dtype=rng.choice(("f32", "bf16", "f16")),
                     settings=rng.choice(("usual", "mixed", "temperature")), pad=rng.choice((0, 0, 3, 64)), masked=rng.random() < 0.3)
            if c["N"] * c["V"] <= 1 << 26:
                return c
    op = rng.choice(("fork", "compact", "copy", "move"))
    while True:
        c = dict(kind="pages", op=op, L=_log(rng, 1, 32), B=_log(rng, 4, 128), kv=_log(rng, 64, 6000), P=0, n=0)
        c["P"] = c["B"] * (c["kv"] // PAGE + 2) + rng.randint(1, 200)
        c["n"] = {"fork": max(1, c["B"] // 2), "compact": 0, "copy": rng.randint(1, max(1, c["P"] // 4)), "move": rng.randint(1, 8)}[op]
        if op == "move":
            c["kv"], c["P"] = 128 + 2 * c["n"], c["B"]
            return c
        if c["L"] * c["P"] <= 40000:
            return c


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ── inputs ──
def _entries(g, lead):
    """Random entries in the cache's byte layout, [*lead, 656]."""
    n = math.prod(lead)
    out = torch.empty(n, ENTRY, dtype=torch.uint8, device="cuda")
    for at in range(0, n, 1 << 18):
        m = min(n, at + (1 << 18)) - at
        x = torch.randn(m, 4, 128, device="cuda", generator=g)
        scale = x.abs().amax(-1) / 448
        out[at:at + m, :LATENT] = (x / scale[..., None]).to(torch.float8_e4m3fn).view(torch.uint8).reshape(m, LATENT)
        out[at:at + m, LATENT:LATENT + 16] = scale.view(torch.uint8).reshape(m, 16)
        out[at:at + m, LATENT + 16:] = torch.randn(m, ROPE, device="cuda", generator=g).bfloat16().view(torch.uint8).reshape(m, 2 * ROPE)
    return out.reshape(*lead, ENTRY)


def _pack_bits(seen):
    """bool [B, T, W] -> int32 [B, T, ceil(W / 32)], bit w % 32 of word w / 32."""
    B, T, W = seen.shape
    bits = torch.nn.functional.pad(seen, (0, -W % 32)).reshape(B, T, -1, 32).long() << torch.arange(32, device=seen.device)
    word = bits.sum(-1)
    return torch.where(word >= 1 << 31, word - (1 << 32), word).int()


def _prepare_tree(c, g):
    B, T, H, kv, win = c["B"], c["T"], c["H"], c["kv"], c["window"]
    kv_len = torch.full((B,), kv, device="cuda", dtype=torch.int32)
    if c["ragged"]:
        kv_len = (kv_len * torch.rand(B, device="cuda", generator=g) ** 0.7).int()
        kv_len[0], kv_len[-1] = kv, (0 if B > 2 else kv)
    pages = (kv + PAGE - 1) // PAGE
    table = torch.randperm(B * pages, device="cuda", generator=g).int().reshape(B, pages)
    # a random tree: node 0 is the last token, every other node hangs on one of the few before it; a node of depth d sees the
    # window without its d oldest tokens, its ancestors and itself
    back = torch.randint(1, 5, (B, T), device="cuda", generator=g)
    seen = torch.zeros(B, T, T, dtype=torch.bool, device="cuda")
    depth = torch.zeros(B, T, dtype=torch.long, device="cuda")
    seen[:, 0, 0] = True
    rows = torch.arange(B, device="cuda")
    for t in range(1, T):
        up = (t - back[:, t]).clamp(min=0)
        seen[:, t] = seen[rows, up]
        seen[:, t, t] = True
        depth[:, t] = depth[rows, up] + 1
    mask = torch.cat([torch.arange(win, device="cuda") >= depth[..., None], seen], dim=-1)
    return dict(q=torch.randn(B, T, H, QK, device="cuda", generator=g).bfloat16(), pool=_entries(g, (B * pages, PAGE)), table=table, kv_len=kv_len,
                win_pool=_entries(g, (B, win + T)), win_len=torch.full((B,), win + T, device="cuda", dtype=torch.int32), mask=_pack_bits(mask),
                sink=torch.randn(H, device="cuda", generator=g) if c["sink"] else None, scale=QK ** -0.5)


def _prepare_sample(c, g):
    N, V = c["N"], c["V"]
    # logits that fall with the logarithm of the rank, at a rate of the row's own, with noise; tokens in random order
    rate = 1.1 + 1.1 * torch.rand(N, 1, device="cuda", generator=g)
    logits = torch.empty(N, V + c["pad"], device="cuda", dtype=dict(f32=torch.float32, bf16=torch.bfloat16, f16=torch.float16)[c["dtype"]])
    logits.fill_(0.0)
    for at in range(0, N, 256):
        m = min(N, at + 256) - at
        rank = torch.rand(m, V, device="cuda", generator=g) * V + 1       # the rank of a token, as its expectation
        logits[at:at + m, :V] = (12 - rate[at:at + m] * torch.log(rank) + 0.5 * torch.randn(m, V, device="cuda", generator=g)).to(logits.dtype)
    logits = logits[:, :V]
    if c["masked"]:
        rows = torch.arange(N, device="cuda") % 4 == 1
        allowed = torch.rand(V, device="cuda", generator=g) < 0.02
        allowed[V // 2] = True
        logits.masked_fill_(rows[:, None] & ~allowed, -math.inf)
    s = dict(logits=logits, u=torch.rand(N, device="cuda", generator=g))
    pick = lambda *v: torch.tensor(v, device="cuda")[torch.randint(0, len(v), (N,), device="cuda", generator=g)]  # noqa: E731
    if c["settings"] == "temperature":
        s |= dict(temperature=0.6 + 0.6 * torch.rand(N, device="cuda", generator=g), top_k=None, top_p=None, min_p=None)
    elif c["settings"] == "usual":
        s |= dict(temperature=torch.full((N,), 0.8, device="cuda"), top_k=torch.full((N,), 50, device="cuda", dtype=torch.int32),
                  top_p=torch.full((N,), 0.95, device="cuda"), min_p=None)
    else:
        s |= dict(temperature=pick(0.0, 0.5, 0.7, 0.8, 1.0, 1.0, 1.2), top_k=pick(0, 0, 20, 40, 50, 100, 1000).int(), top_p=pick(0.8, 0.9, 0.95, 0.99, 1.0),
                  min_p=pick(0.0, 0.0, 0.02, 0.1))
    return s


def _prepare_pages(c, g):
    L, B, kv, P, n, op = c["L"], c["B"], c["kv"], c["P"], c["n"], c["op"]
    if op == "move":        # B windows of kv rows, n accepted drafts each, from the drafts' rows to places in the window
        pool = torch.randint(0, 256, (L, B, kv, ENTRY), device="cuda", dtype=torch.uint8, generator=g)
        first = torch.arange(B, device="cuda")[:, None] * kv
        src = first + 128 + torch.rand(B, kv - 128, device="cuda", generator=g).argsort(1)[:, :n].sort(1).values
        dst = first + (torch.randint(0, 128, (B, 1), device="cuda", generator=g) + torch.arange(n, device="cuda")) % 128
        take = torch.arange(n, device="cuda") < torch.randint(1, n + 1, (B, 1), device="cuda", generator=g)
        return dict(pool=pool, src=torch.where(take, src, -1).int().reshape(-1), dst=torch.where(take, dst, -1).int().reshape(-1))
    pool = torch.randint(0, 256, (L, P, PAGE, ENTRY), device="cuda", dtype=torch.uint8, generator=g)
    if op == "copy":
        order = torch.randperm(P, device="cuda", generator=g).int()
        return dict(pool=pool, src=order[:n].contiguous(), dst=order[n:2 * n].contiguous())
    kv_len = (kv - torch.randint(0, kv // 2 + 1, (B,), device="cuda", generator=g)).int()
    width = kv // PAGE + 2
    held = torch.arange(width, device="cuda") < ((kv_len + PAGE - 1) // PAGE)[:, None]
    where = torch.randperm(P, device="cuda", generator=g)[:B * width].reshape(B, width)
    table = torch.where(held, where, -1).int()
    refs = torch.zeros(P + 1, dtype=torch.int32, device="cuda").index_add_(0, torch.where(held, where, P).reshape(-1), torch.ones(B * width, dtype=torch.int32, device="cuda"))[:P].contiguous()
    s = dict(pool=pool, table=table, kv_len=kv_len, refs=refs)
    if op == "fork":
        order = torch.randperm(B, device="cuda", generator=g).int()
        s |= dict(parent=order[n:][torch.randint(0, B - n, (n,), device="cuda", generator=g)].contiguous(), child=order[:n].contiguous())
    return s


def prepare(case, seed):
    c = dict(case)
    made = dict(tree=_prepare_tree, sample=_prepare_sample, pages=_prepare_pages)[c["kind"]](c, _gen(seed))
    return dict(case=c, **made)


# ── the plain forms ──
def _dequantised(entries, dtype):
    lead = entries.shape[:-1]
    lat = entries[..., :LATENT].contiguous().view(torch.float8_e4m3fn).to(dtype)
    scale = entries[..., LATENT:LATENT + 16].contiguous().view(torch.float32).to(dtype)
    rope = entries[..., LATENT + 16:].contiguous().view(torch.bfloat16).to(dtype)
    return torch.cat([(lat.reshape(*lead, 4, 128) * scale[..., None]).reshape(*lead, LATENT), rope], dim=-1)


def _plain_tree(s):
    q, table, kv_len, win_len = s["q"].float(), s["table"], s["kv_len"], s["win_len"]
    B, T, H, _ = q.shape
    W = s["win_pool"].shape[1]
    k = torch.cat([_dequantised(s["pool"][table.long()].reshape(B, -1, ENTRY), torch.float32), _dequantised(s["win_pool"], torch.float32)], dim=1)
    n = table.shape[1] * PAGE
    at, w = torch.arange(n, device="cuda"), torch.arange(W, device="cuda")
    bits = (s["mask"].repeat_interleave(32, dim=-1)[..., :W] >> (w % 32)) & 1
    seen = torch.cat([(at < kv_len[:, None])[:, None].expand(B, T, n), (bits != 0) & (w < win_len[:, None])[:, None]], dim=-1)
    x = torch.matmul(q.reshape(B, T * H, QK), k.transpose(1, 2)).reshape(B, T, H, -1) * s["scale"]
    x.masked_fill_(~seen[:, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = x.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    below = total if s["sink"] is None else total + torch.exp(s["sink"][:, None] - top)
    out = torch.matmul(e.reshape(B, T * H, -1), k[..., :LATENT]).reshape(B, T, H, LATENT) / torch.where(total == 0, torch.ones_like(below), below)
    return dict(out=out.bfloat16(), lse=(top + torch.log(total)).squeeze(-1))


def _share(total, m):
    """floor(total * m / 2^24) of 64-bit integers, m <= 2^24."""
    return (total >> 24) * m + (((total & 0xFFFFFF) * m) >> 24)


def _plain_sample(s):
    l = s["logits"].float()
    N, V = l.shape
    l = torch.where(torch.isnan(l), -math.inf, l)
    top = l.amax(1, keepdim=True)
    t = s["temperature"]
    t = torch.ones(N, device="cuda") if t is None else t
    greedy = ~(t > 0)
    per = (1 / torch.where(greedy, torch.ones_like(t), t))[:, None]
    x = torch.where(l == top, torch.zeros_like(l), (l - top) * per)
    e = torch.exp(x)
    w = torch.where(l == -math.inf, 0, (e * FIXED).to(torch.int64))
    order = torch.sort(l, dim=1, descending=True, stable=True).indices
    place = torch.arange(V, device="cuda")
    w, e = w.gather(1, order), e.gather(1, order)
    if s["top_k"] is not None:
        k = torch.where(s["top_k"] <= 0, V, s["top_k"])[:, None]
        w = torch.where(place < k, w, 0)
    if s["top_p"] is not None:
        upto = w.cumsum(1)
        p = s["top_p"][:, None]
        most = _share(upto[:, -1:], (p.clamp(0, 1) * 2 ** 24).to(torch.int64)).clamp(min=1)
        w = torch.where((upto - w < most) | ~(p < 1), w, 0)
    if s["min_p"] is not None:
        w = torch.where(e < s["min_p"][:, None].clamp(max=1), 0, w)
    w = torch.where(greedy[:, None] & (place > 0), 0, w)
    upto = torch.zeros_like(w).scatter_(1, order, w).cumsum(1)
    total = upto[:, -1:]
    at = _share(total, (s["u"][:, None] * 2 ** 24).to(torch.int64).clamp(0, 2 ** 24 - 1))
    token = (upto <= at).sum(1)
    chosen = x.gather(1, token.clamp(max=V - 1)[:, None])
    logprob = (chosen - torch.log(total.float() / FIXED))[:, 0]
    none = total[:, 0] == 0
    return dict(token=torch.where(none, -1, token).int(), logprob=torch.where(none, -math.inf, logprob))


def _plain_free(s, requests):
    table, kv_len, refs = s["table"], s["kv_len"], s["refs"]
    r = requests.long()
    pages = table[r].long()
    held = (torch.arange(table.shape[1], device="cuda") < ((kv_len[r] + PAGE - 1) // PAGE)[:, None]) & (pages >= 0)
    refs.index_add_(0, torch.where(held, pages, 0).reshape(-1), -held.reshape(-1).int())
    table[r] = -1
    kv_len[r] = 0


def _plain_fork(s, parent, child):
    pool, table, kv_len, refs = s["pool"], s["table"], s["kv_len"], s["refs"]
    p, c = parent.long(), child.long()
    n, width = p.numel(), table.shape[1]
    length = kv_len[p]
    full, rest = (length // PAGE).long(), (length % PAGE).long()
    nth = (rest > 0).long().cumsum(0) - 1
    free = torch.sort((refs > 0).int(), stable=True).indices                # free pages first, in ascending order
    page = free[nth.clamp(min=0)]
    slot = torch.arange(width, device="cuda")
    shared = slot < full[:, None]
    rows = torch.where(shared, table[p].long(), -1)
    refs.index_add_(0, rows.clamp(min=0).reshape(-1), (rows >= 0).reshape(-1).int())
    rows = torch.where((slot == full[:, None]) & (rest[:, None] > 0), page[:, None], rows)
    refs.index_add_(0, page, (rest > 0).int())
    table[c] = rows.int()
    kv_len[c] = length
    old = table[p].long().gather(1, full.clamp(max=width - 1)[:, None])[:, 0]
    taken = torch.arange(PAGE, device="cuda") < rest[:, None]               # entries of the partly filled page
    child_at, entry = torch.nonzero(taken, as_tuple=True)
    pool[:, page[child_at], entry] = pool[:, old[child_at], entry]


def _plain_compact(s):
    pool, table, refs = s["pool"], s["table"], s["refs"]
    P = refs.numel()
    live = refs > 0
    count = live.sum()
    at = torch.arange(P, device="cuda")
    src = torch.nonzero(live & (at >= count))[:, 0]
    dst = torch.nonzero(~live & (at < count))[:, 0]
    to = at.clone()
    to[src] = dst
    pool[:, dst] = pool[:, src]
    new_refs = refs.clone()
    new_refs[dst] = refs[src]
    new_refs[src] = 0
    new_table = torch.where(table >= 0, to[table.clamp(min=0).long()].int(), table)
    return new_table, new_refs, count.int().reshape(1)


def _plain_move(s):
    pool, src, dst = s["pool"], s["src"].long(), s["dst"].long()
    flat = pool.reshape(pool.shape[0], -1, ENTRY)
    take = (src >= 0) & (dst >= 0)
    flat[:, dst[take]] = flat[:, src[take]]


def run(state):
    s = state
    if own:
        import dsv4_attn_b200 as d
    kind, op = s["case"]["kind"], s["case"].get("op")
    if kind == "tree":
        if not own:
            return _plain_tree(s)
        out, lse = d.hca_tree_decode(s["q"], s["pool"], s["table"], s["kv_len"], s["win_pool"], s["win_len"], s["mask"], s["scale"], attn_sink=s["sink"])
        return dict(out=out, lse=lse)
    if kind == "sample":
        if not own:
            return _plain_sample(s)
        token, logprob = d.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
        return dict(token=token, logprob=logprob)
    if op == "fork":        # the children's pages are given back, then the children become copies of their parents
        if own:
            d.kv_pages_free(s["table"], s["kv_len"], s["refs"], s["child"])
            d.kv_pages_fork(s["pool"], s["table"], s["kv_len"], s["refs"], s["parent"], s["child"])
        else:
            _plain_free(s, s["child"])
            _plain_fork(s, s["parent"], s["child"])
        return dict(pool=s["pool"], table=s["table"], kv_len=s["kv_len"], refs=s["refs"])
    if op == "compact":
        table, refs, count = d.kv_pages_compact(s["pool"], s["table"], s["refs"]) if own else _plain_compact(s)
        return dict(pool=s["pool"], table=table, refs=refs, count=count)
    if op == "copy":
        if own:
            d.kv_pages_copy(s["pool"], s["src"], s["dst"])
        else:
            s["pool"][:, s["dst"].long()] = s["pool"][:, s["src"].long()]
        return dict(pool=s["pool"])
    if own:
        d.kv_entries_move(s["pool"], s["src"], s["dst"])
    else:
        _plain_move(s)
    return dict(pool=s["pool"])


def work(case):
    c = case
    if c["kind"] == "tree":
        entries = c["kv"] * (0.6 if c["ragged"] else 1.0) + c["window"] + c["T"]
        rows = c["B"] * c["T"] * c["H"]
        return dict(bytes=rows * (2 * QK + 2 * LATENT + 4) + c["B"] * entries * ENTRY, flops=2.0 * rows * entries * (QK + LATENT))
    if c["kind"] == "sample":
        return dict(bytes=c["N"] * (c["V"] * (4 if c["dtype"] == "f32" else 2) + 28), flops=4.0 * c["N"] * c["V"])
    if c["op"] == "move":
        return dict(bytes=c["B"] * (c["n"] + 1) / 2 * (2 * ENTRY * c["L"] + 8), flops=0)
    if c["op"] == "copy":
        return dict(bytes=c["n"] * (2 * PAGE * ENTRY * c["L"] + 8), flops=0)
    width = c["kv"] // PAGE + 2
    if c["op"] == "fork":       # half a page per child and layer on average, the reference counts, the children's table rows read and written
        return dict(bytes=c["n"] * (PAGE * ENTRY * c["L"] + 16 * width) + 4 * c["P"], flops=0)
    live = min(c["P"], c["B"] * (0.75 * c["kv"] / PAGE + 0.5))
    return dict(bytes=live * (1 - live / c["P"]) * 2 * PAGE * ENTRY * c["L"] + 8 * c["P"] + 8 * c["B"] * width, flops=0)


# ── the definitions in 64 bits ──
def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["kind"] == "pages":
        return None             # bytes and whole numbers
    if c["kind"] == "sample":
        return _exact_sample(s)
    out, lse = [], []
    for b in range(c["B"]):
        n, m = int(s["kv_len"][b]), int(s["win_len"][b])
        pages = s["table"][b, :(n + PAGE - 1) // PAGE].long()
        k = _dequantised(torch.cat([s["pool"][pages].reshape(-1, ENTRY)[:n], s["win_pool"][b, :m]]), torch.float64)
        w = torch.arange(m, device="cuda")
        seen = (s["mask"][b].long()[:, w // 32] >> (w % 32)) & 1
        seen = torch.cat([torch.ones(c["T"], n, device="cuda", dtype=torch.long), seen], dim=1).bool()
        x = (s["q"][b].double() @ k.T * s["scale"]).masked_fill(~seen[:, None], -math.inf)
        total = torch.logsumexp(x, -1)
        whole = total if s["sink"] is None else torch.logaddexp(total, s["sink"].double())
        out.append(torch.exp(x - whole[..., None]) @ k[:, :LATENT])
        lse.append(total)
    return dict(out=torch.stack(out), lse=torch.stack(lse))


def _exact_sample(s):
    logprob = []
    one = lambda v, i, other: other if v is None else float(v[i])  # noqa: E731
    for i in range(s["logits"].shape[0]):
        l = s["logits"][i].double()
        t, k, p, m = one(s["temperature"], i, 1.0), int(one(s["top_k"], i, 0)), one(s["top_p"], i, 1.0), one(s["min_p"], i, 0.0)
        if t <= 0:
            logprob.append(torch.zeros((), device="cuda", dtype=torch.float64))
            continue
        weight = torch.exp((l - l.max()) / t)
        ranked, order = torch.sort(l, descending=True, stable=True)
        take = torch.zeros_like(weight)
        r = weight[order]
        if k > 0:
            r[k:] = 0
        if p < 1:
            r = r * (r.cumsum(0) - r < max(p, 1e-30) * r.sum())
        take[order] = r * (weight[order] >= m)
        upto = take.cumsum(0)
        token = torch.searchsorted(upto, float(s["u"][i]) * upto[-1], right=True).clamp(max=l.numel() - 1)
        logprob.append(torch.log(take[token] / upto[-1]))
    return dict(token=None, logprob=torch.stack(logprob))
