"""Eviction by attention weight and insertion into K and V pages against plain code.  Run with `-m gpu` on a B200."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

PAGE = 64


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import dsv4_attn_b200 as d
    return d


def state(kv_len, shapes, dtype=torch.bfloat16, layers=2, width=0, seed=0, weights=None, extra=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B = len(kv_len)
    pages = max(max((n + PAGE - 1) // PAGE for n in kv_len), width, 1)
    P = B * pages + 5
    pools = [torch.randint(0, 256, (layers, P, PAGE, *s[:-1], s[-1] * dtype.itemsize), device="cuda", dtype=torch.uint8, generator=g).view(dtype) for s in shapes]
    order = torch.randperm(P, device="cuda", generator=g).int()
    table = torch.full((B, pages), -1, device="cuda", dtype=torch.int32)
    refs = torch.zeros(P, device="cuda", dtype=torch.int32)
    for b, n in enumerate(kv_len):
        held = (n + PAGE - 1) // PAGE
        table[b, :held] = order[b * pages:b * pages + held]
        refs[table[b, :held].long()] = 1
    if weights is None:
        weights = torch.exp(2.5 * torch.randn(B, pages * PAGE + extra, device="cuda", generator=g))
    return pools, table, torch.tensor(kv_len, device="cuda", dtype=torch.int32), refs, weights


def expected(pools, table, kv_len, refs, weights, keep, first, recent):
    """One request at a time, on the CPU."""
    pools = [p.view(torch.uint8).cpu().clone() for p in pools]
    old = [p.clone() for p in pools]
    table, lens, refs, w = table.cpu().clone(), kv_len.tolist(), refs.cpu().clone(), weights.cpu()
    cap = table.shape[1] * PAGE
    new_w, kept = torch.zeros_like(w), torch.full((len(lens), cap), -1, dtype=torch.int32)
    keeps = [keep] * len(lens) if isinstance(keep, int) else keep
    for b, n in enumerate(lens):
        k = keeps[b]
        lo = min(first, k)
        hi = n - min(recent, k - lo)
        stay = list(range(n))
        if n > k:
            key = [(-float("inf") if x != x else x) for x in w[b, :n].tolist()]
            others = sorted(range(lo, hi), key=lambda j: (-key[j], j))[:k - lo - (n - hi)]
            stay = list(range(lo)) + sorted(others) + list(range(hi, n))
            for s in range((k + 63) // 64, (n + 63) // 64):
                refs[table[b, s]] -= 1
        for i, j in enumerate(stay):
            kept[b, i] = j
            new_w[b, i] = w[b, j]
            if i != j:
                for p, o in zip(pools, old):
                    p[:, table[b, i // 64], i % 64] = o[:, table[b, j // 64], j % 64]
        if n > k:
            table[b, (k + 63) // 64:(n + 63) // 64] = -1
        lens[b] = len(stay)
    return pools, table, lens, refs, new_w, kept


def same(pools, got, want):
    table, lens, refs, w, kept = got
    for p, q in zip(pools, want[0]):
        assert torch.equal(p.view(torch.uint8).cpu(), q)
    assert torch.equal(table.cpu(), want[1]) and lens.tolist() == want[2] and torch.equal(refs.cpu(), want[3])
    assert torch.equal(w.cpu().view(torch.int32), want[4].view(torch.int32)) and torch.equal(kept.cpu(), want[5])


@pytest.mark.parametrize("keep,first,recent", [(100, 0, 0), (100, 4, 32), (64, 1, 63), (1, 0, 0), (1, 1, 0), (0, 0, 0), (0, 3, 3), (128, 200, 10), (128, 100, 100), (5000, 4, 4)])
def test_budgets(lib, keep, first, recent):
    s = state([0, 1, 63, 64, 65, 100, 101, 128, 129, 700, 5000], [(2, 64), (2, 64)], seed=keep)
    want = expected(*s, keep, first, recent)
    st = lib.new_status("cuda")
    before = [t.clone() for t in s[1:]]
    same(s[0], lib.kv_evict(s[0], *s[1:], keep, first=first, recent=recent, status=st), want)
    assert st.tolist() == [0, 0, 0, 0]
    assert all(torch.equal(a, b) for a, b in zip(before, s[1:]))


@pytest.mark.parametrize("shapes,dtype,layers", [([(1, 8)], torch.bfloat16, 1), ([(656,)], torch.uint8, 3), ([(8, 128), (8, 128)], torch.float8_e4m3fn, 2), ([(3, 64), (5, 128), (16,)], torch.float16, 1),
                                                ([(1, 256)] * 4, torch.float16, 5)])
def test_pools(lib, shapes, dtype, layers):
    s = state([300, 1000, 40], shapes, dtype=dtype, layers=layers)
    want = expected(*s, 200, 2, 30)
    same(s[0], lib.kv_evict(s[0] if len(s[0]) > 1 else s[0][0], *s[1:], 200, first=2, recent=30), want)


def test_a_budget_for_each_request_in_place(lib):
    s = state([500, 500, 77, 300], [(2, 64), (2, 64)], extra=9)
    keep = [100, 499, 100, 0]
    want = expected(*s, keep, 1, 5)
    pools, table, lens, refs, w = s
    got = lib.kv_evict(pools, table, lens, refs, w, torch.tensor(keep, device="cuda", dtype=torch.int32), first=1, recent=5, new_table=table, new_len=lens, new_refs=refs, new_weights=w)
    assert got[0] is table and got[1] is lens and got[2] is refs and got[3] is w
    same(pools, got, want)


def test_ties_signs_and_values_that_are_not_numbers(lib):
    n = 5000
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randint(-2, 3, (4, 79 * 64), device="cuda", generator=g).float()
    w[1] = 0.0
    w[1, ::2] = -0.0
    w[2, ::3] = float("nan")
    w[2, 1::3] = float("inf")
    w[2, 2::7] = -float("inf")
    w[3] = torch.randn(79 * 64, device="cuda", generator=g) * 1e-40               # subnormal
    s = state([n] * 4, [(1, 16)], weights=w)
    for keep in (1, 700, 1700, 2500, 4999):
        t = state([n] * 4, [(1, 16)], weights=w)
        want = expected(*t, keep, 0, 0)
        same(t[0], lib.kv_evict(t[0], *t[1:], keep), want)
    del s


def test_a_long_request(lib):
    s = state([100_000, 5], [(1, 16)], layers=1)
    want = expected(*s, 60_000, 4, 1000)
    same(s[0], lib.kv_evict(s[0], *s[1:], 60_000, first=4, recent=1000), want)


def test_shared_pages_and_pages_out_of_range(lib):
    s = state([500, 500, 500, 500], [(2, 64)])
    pools, table, lens, refs, w = s
    refs[table[0, 2].long()] = 2                      # among those that are written
    refs[table[1, 7].long()] = 2                      # behind the new end: given back
    refs[table[2, 0].long()] = 3                      # before the first change
    w[2, :64] = 1e9
    table[3, 5] = refs.numel() + 3
    other = [t.clone() for t in (table, lens, refs, w)]
    st = lib.new_status("cuda")
    keep = torch.tensor([200, 200, 200, 200], device="cuda", dtype=torch.int32)
    old = [p.clone() for p in pools]
    got = lib.kv_evict(pools, table, lens, refs, w, keep, status=st)
    assert st[0].item() in (7, 12)
    assert got[1].tolist() == [500, 200, 200, 500]
    for b in (0, 3):
        assert torch.equal(got[0][b], table[b]) and got[4][b, :500].tolist() == list(range(500)) and torch.equal(got[3][b, :500], w[b, :500])
        for p, o in zip(pools, old):
            own = table[b][(table[b] >= 0) & (table[b] < refs.numel())].long()
            assert torch.equal(p[:, own].view(torch.uint8), o[:, own].view(torch.uint8))
    want = expected(old, *[t[1:3] if t.dim() == 2 or t.numel() == 4 else t for t in other], [200, 200], 0, 0)
    for b in (1, 2):
        assert torch.equal(got[0][b].cpu(), want[1][b - 1]) and torch.equal(got[4][b].cpu(), want[5][b - 1])
        for p, q in zip(pools, want[0]):
            own = table[b].long()
            assert torch.equal(p.view(torch.uint8).cpu()[:, own.cpu()], q[:, own.cpu()])
    assert torch.equal(got[2].cpu(), want[3])
    # one alone
    for code, b in ((12, 0), (7, 3)):
        st.zero_()
        lib.kv_evict(pools, table[b:b + 1].contiguous(), lens[b:b + 1].contiguous(), refs, w[b:b + 1].contiguous(), 200, status=st)
        assert st[0].item() == code
    # a length beyond the table
    st.zero_()
    r = lib.kv_evict(pools, table[1:2].contiguous(), torch.tensor([10_000], device="cuda", dtype=torch.int32), refs, w[1:2].contiguous(), 200, status=st)
    assert st[0].item() == 7 and r[1].item() == 10_000


def test_captured_and_replayed(lib):
    s = state([500, 300, 100], [(2, 64), (2, 64)])
    pools, table, lens, refs, w = s
    fresh = [t.clone() for t in (*pools, table, lens, refs, w)]
    want = expected(*s, 150, 2, 20)
    new = dict(new_table=table, new_len=lens, new_refs=refs, new_weights=w)
    lib.kv_evict(pools, table, lens, refs, w, 150, first=2, recent=20, **new)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = lib.kv_evict(pools, table, lens, refs, w, 150, first=2, recent=20, **new)
    for t, f in zip((*pools, table, lens, refs, w), fresh):
        t.copy_(f)
    graph.replay()
    same(pools, got, want)


# ── insertion ──
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("Hkv,D", [(1, 64), (3, 128), (8, 256), (5, 40)])
def test_insert(lib, dtype, packed, Hkv, D):
    g = torch.Generator(device="cuda").manual_seed(D)
    B, T, pages = 40, 7, 4
    src = torch.float16 if dtype == torch.float16 else torch.bfloat16
    pools = [torch.randint(0, 120, (B * pages + 3, PAGE, Hkv, D * dtype.itemsize), device="cuda", dtype=torch.uint8, generator=g).view(dtype) for _ in "kv"]
    table = torch.randperm(B * pages + 3, device="cuda", generator=g)[:B * pages].int().reshape(B, pages)
    pos = torch.randint(0, pages * PAGE - T, (B,), device="cuda", generator=g).int()
    new = torch.randint(0, T + 1, (B,), device="cuda", generator=g)
    new[3] = 0
    start = torch.zeros(B + 1, device="cuda", dtype=torch.int32)
    start[1:] = new.cumsum(0)
    scales = [0.01 + torch.rand(Hkv, device="cuda", generator=g) for _ in "kv"] if dtype == torch.float8_e4m3fn else [None, None]
    rows = int(start[-1]) + 4 if packed else B * T                 # four rows behind the last request
    qkv = (torch.randn(rows, 3 * Hkv, D, device="cuda", generator=g) * 50).to(src)
    qkv[0, :, 0] = 1e4
    if not packed:
        qkv = qkv.unflatten(0, (B, T))
    k, v = qkv[..., Hkv:2 * Hkv, :], qkv[..., 2 * Hkv:, :]
    want = [p.clone() for p in pools]
    for b in range(B):
        for t in range(int(new[b])):
            at = int(pos[b]) + t
            for p, x, s in zip(want, (k, v), scales):
                row = x[int(start[b]) + t] if packed else x[b, t]
                row = row if s is None else (row.float() / s[:, None]).clamp(-448, 448)
                p[int(table[b, at // PAGE]), at % PAGE] = row.to(dtype)
    st = lib.new_status("cuda")
    lib.gqa_insert(k, v, *pools, table, pos, **(dict(q_start=start) if packed else dict(n_rows=new.int())), k_scale=scales[0], v_scale=scales[1], status=st)
    for p, q in zip(pools, want):
        assert torch.equal(p.view(torch.uint8), q.view(torch.uint8))
    assert st.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
def test_every_value_over_scales_of_all_sizes(lib, src):
    x = torch.arange(65536, device="cuda", dtype=torch.int32).to(torch.int16).view(src).reshape(1, 256, 1, 256)
    table = torch.arange(4, device="cuda", dtype=torch.int32)[None]
    at = torch.zeros(1, device="cuda", dtype=torch.int32)
    for s in (1.0, 0.37, 3.0, 1 / 448, 0.0123, 117.3, 6e4, 1e-7, 1e-24, 1e-26, 1e-38, 1e24, 1e30):
        pools = [torch.zeros(4, PAGE, 1, 256, device="cuda", dtype=torch.float8_e4m3fn) for _ in "kv"]
        scale = torch.tensor([s], device="cuda")
        lib.gqa_insert(x, x.flip(1), *pools, table, at, k_scale=scale, v_scale=scale)
        want = (x.float() / scale).clamp(-448, 448).to(torch.float8_e4m3fn).reshape(256, 256)
        for p, w in zip(pools, (want, want.flip(0))):
            p = p.reshape(256, 256)
            nan = w.float().isnan()
            assert torch.equal(p.float().isnan(), nan) and torch.equal(p.view(torch.uint8)[~nan], w.view(torch.uint8)[~nan])


def test_insert_out_of_range(lib):
    pools = [torch.zeros(4, PAGE, 1, 64, device="cuda", dtype=torch.float16) for _ in "kv"]
    k = torch.ones(3, 2, 1, 64, device="cuda", dtype=torch.float16)
    table = torch.tensor([[0, 9], [1, -1], [2, 3]], device="cuda", dtype=torch.int32)
    for pos, filled in (([63, 0, 0], 5), ([0, 63, 0], 5), ([0, 0, 127], 5), ([0, 0, -1], 5), ([0, 0, 1 << 30], 4), ([0, 0, (1 << 31) - 1], 4)):
        st = lib.new_status("cuda")
        for p in pools:
            p.zero_()
        lib.gqa_insert(k, k, *pools, table, torch.tensor(pos, device="cuda", dtype=torch.int32), status=st)
        assert st[0] == 16 and int(pools[0].any(-1).sum()) == filled and int(pools[1].any(-1).sum()) == filled
