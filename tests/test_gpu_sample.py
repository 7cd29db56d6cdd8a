"""Sampling against the definition: integer weights in 64 bits, in plain torch (tokens have to be equal), and the distribution in FP64.  Run with
`-m gpu` on a B200.

The log-probability is a difference of two FP32 numbers, (l - l_max) / t of at most 28 (below, a weight is 0) and a logarithm of at
most 2^22: 28 x 2 roundings of 2^-24 and the logarithm's own 2 of 2^-24 x 16 stay below 6e-6."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

INF = math.inf


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import dsv4_attn_b200 as d
    return d


def share(total, m):
    return (total >> 24) * m + (((total & 0xFFFFFF) * m) >> 24)


def want(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """Row by row, as include/dsv4_speculative.h has it."""
    tokens, logprobs = [], []
    for n in range(logits.shape[0]):
        l = logits[n].float()
        l = torch.where(torch.isnan(l), -INF, l)
        top = l.max()
        if top == -INF:
            tokens.append(-1)
            logprobs.append(-INF)
            continue
        t = torch.ones((), device="cuda") if temperature is None else temperature[n]
        if not t > 0:
            tokens.append(int((l == top).nonzero()[0]))
            logprobs.append(0.0)
            continue
        x = torch.where(l == top, 0.0, (l - top) * (1 / t))
        e = torch.exp(x)
        w = (e * 2.0 ** 40).long()
        order = torch.sort(l, descending=True, stable=True).indices
        s, es = w[order].clone(), e[order]
        if top_k is not None and 0 < int(top_k[n]) < l.numel():
            s[int(top_k[n]):] = 0
        if top_p is not None and float(top_p[n]) < 1:
            upto = s.cumsum(0)
            most = max(1, int(share(upto[-1], int(max(float(top_p[n]), 0.0) * 2 ** 24))))
            s[upto - s >= most] = 0
        if min_p is not None and float(min_p[n]) > 0:
            s[es < min(float(min_p[n]), 1.0)] = 0
        kept = torch.zeros_like(w)
        kept[order] = s
        upto = kept.cumsum(0)
        total = int(upto[-1])
        m = min(max(int(float(u[n]) * 2 ** 24), 0), 2 ** 24 - 1) if u[n] == u[n] else 0
        target = ((total >> 24) * m) + (((total & 0xFFFFFF) * m) >> 24)
        tok = int((upto > target).nonzero()[0])
        tokens.append(tok)
        logprobs.append(float((l[tok].double() - top.double()) / t.double() if l[tok] != top else 0.0) - math.log(total / 2 ** 40))
    return torch.tensor(tokens, dtype=torch.int32, device="cuda"), torch.tensor(logprobs, dtype=torch.float64, device="cuda")


def check(got, exp):
    assert torch.equal(got[0], exp[0]), (got[0] != exp[0]).nonzero()[:4]
    fin = torch.isfinite(exp[1])
    assert torch.equal(torch.isneginf(got[1]), torch.isneginf(exp[1]))
    # (each logit is an exact FP32 number: only the two roundings of (l - l_max) * (1 / t), up to 28 in size, and the logarithm's count)
    assert (got[1][fin] - exp[1][fin]).abs().max().item() <= 6e-6 if fin.any() else True


def rows(seed, N, V, dtype, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(N, V, device="cuda", generator=g) * spread).to(dtype), torch.rand(N, device="cuda", generator=g), g


SIZES = [1, 2, 7, 255, 1000, 4097, 32000, 50257, 131072, 262144]


@pytest.mark.parametrize("V", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("filters", ["none", "top_k", "top_p", "min_p", "all"])
def test_against_the_definition(lib, V, dtype, filters):
    N = 9
    logits, u, g = rows(V, N, V, dtype)
    s = dict(temperature=0.4 + torch.rand(N, device="cuda", generator=g))
    if filters in ("top_k", "all"):
        s["top_k"] = torch.tensor([0, 1, 2, 40, 50, 1000, V, V - 1, 3000], device="cuda", dtype=torch.int32)
    if filters in ("top_p", "all"):
        s["top_p"] = torch.tensor([0.0, 0.1, 0.5, 0.9, 0.95, 0.999, 1.0, 2.0, 0.8], device="cuda")
    if filters in ("min_p", "all"):
        s["min_p"] = torch.tensor([0.0, 1e-9, 0.01, 0.05, 0.2, 0.9, 1.0, 5.0, -1.0], device="cuda")
    check(lib.sample(logits, u, **s), want(logits, u, **s))


def test_a_row_does_not_depend_on_its_batch(lib):
    """One row, small batches and large ones take clusters of different sizes: the same token for the same row."""
    logits, u, g = rows(3, 300, 40000, torch.float32)
    s = dict(top_k=torch.full((300,), 0, device="cuda", dtype=torch.int32), top_p=torch.full((300,), 0.97, device="cuda"))
    s["top_k"][::3] = 60
    token, logprob = lib.sample(logits, u, **s)
    for n in (0, 1, 2, 151, 299):
        one = lib.sample(logits[n:n + 1], u[n:n + 1], **{k: v[n:n + 1] for k, v in s.items()})
        assert one[0].item() == token[n].item() and one[1].item() == logprob[n].item()


@pytest.mark.parametrize("filters", [dict(), dict(top_k=12), dict(top_p=0.8), dict(min_p=0.05)])
def test_distribution(lib, filters):
    """65,536 evenly spread random numbers on one row: every token comes up as often as its probability in FP64 says, to within one."""
    N, V = 1 << 16, 300
    logits, _, _ = rows(4, 1, V, torch.float32, 1.5)
    u = (torch.arange(N, device="cuda", dtype=torch.float64) + 0.5) / N
    s = {k: torch.full((N,), v, device="cuda", dtype=torch.int32 if k == "top_k" else torch.float32) for k, v in filters.items()}
    token, logprob = lib.sample(logits.expand(N, V).contiguous(), u.float(), temperature=torch.full((N,), 0.7, device="cuda"), **s)
    p = torch.softmax(logits[0].double() / 0.7, 0)
    ranked, order = p.sort(descending=True)
    keep = torch.ones_like(p, dtype=torch.bool)
    if "top_k" in filters:
        keep[order[12:]] = False
    if "top_p" in filters:
        keep[order] = ranked.cumsum(0) - ranked < 0.8
    if "min_p" in filters:
        keep = p >= 0.05 * p.max()
    p = p * keep / (p * keep).sum()
    count = torch.bincount(token.long(), minlength=V)
    assert (count - N * p).abs().max().item() <= 1.01
    assert (logprob.double() - torch.log(p)[token.long()]).abs().max().item() <= 6e-6


@pytest.mark.parametrize("V", [5, 3000, 70000])
def test_ties(lib, V):
    """Equal logits: the lower index comes first, at a top-k and a top-p cut in the middle of thousands of them."""
    N = 40
    logits = torch.zeros(N, V, device="cuda")
    logits[:, V // 2] = 0.5
    logits[:, ::7] = -0.0
    u = torch.linspace(0, 0.999, N, device="cuda")
    for s in (dict(top_k=torch.full((N,), V // 2, device="cuda", dtype=torch.int32)), dict(top_p=torch.full((N,), 0.3, device="cuda")), dict(),
              dict(top_k=torch.full((N,), V // 2, device="cuda", dtype=torch.int32), top_p=torch.full((N,), 0.4, device="cuda")), dict(temperature=torch.zeros(N, device="cuda"))):
        check(lib.sample(logits, u, **s), want(logits, u, **s))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,V", [(1, 40000), (5, 200001), (20, 262144), (150, 60000)])
@pytest.mark.parametrize("spread", [0.02, 0.5, 1.0])
def test_many_tokens_near_the_cut(lib, N, V, dtype, spread):
    """Flat rows, whose cuts lie among thousands of nearly equal logits (in 16 bits, of equal ones); a third of the 32-bit rows are such of 16 bits."""
    logits, u, g = rows(N + V, N, V, dtype, spread)
    if dtype == torch.float32:
        logits[::3] = logits[::3].bfloat16().float()
    s = dict(temperature=0.5 + torch.rand(N, device="cuda", generator=g), top_p=0.2 + 0.79 * torch.rand(N, device="cuda", generator=g),
             top_k=torch.randint(3000, 30000, (N,), device="cuda", generator=g, dtype=torch.int32))
    s["top_k"][::2] = 0
    check(lib.sample(logits, u, **s), want(logits, u, **s))
    s.pop("top_p")
    check(lib.sample(logits, u, **s), want(logits, u, **s))


@pytest.mark.parametrize("N,V", [(64, 3000), (64, 70000)])
def test_min_p_on_both_sides_of_the_cut(lib, N, V):
    """min-p thresholds that are far above the cut of top-p, far below it, and within parts in a thousand of it."""
    logits, u, g = rows(V, N, V, torch.float32, 1.5)
    top_p = 0.3 + 0.65 * torch.rand(N, device="cuda", generator=g)
    e = torch.exp((logits - logits.amax(1, keepdim=True)).double()).sort(1, descending=True).values
    at_cut = e.gather(1, ((e.cumsum(1) < top_p[:, None] * e.sum(1, keepdim=True)).sum(1, keepdim=True)).clamp(max=V - 1))[:, 0]
    factor = torch.tensor([0.01, 0.5, 0.97, 0.999, 0.9999, 1.0, 1.0001, 1.001, 1.03, 2.0, 1e-30, 30.0, 0.99, 1.01, 1.02, 0.98], device="cuda").repeat(N // 16)
    min_p = (at_cut * factor).float()
    for t in (None, torch.ones(N, device="cuda")):
        check(lib.sample(logits, u, temperature=t, top_p=top_p, min_p=min_p), want(logits, u, t, None, top_p, min_p))


@pytest.mark.parametrize("t", [1e-30, 1e-6, 1e-4, 1e4, 1e30])
def test_temperatures_far_from_one(lib, t):
    N, V = 6, 30000
    logits, u, g = rows(11, N, V, torch.float32)
    logits += torch.tensor([0.0, 1e4, -1e4, 1.0, 100.0, -100.0], device="cuda")[:, None]
    s = dict(temperature=torch.full((N,), t, device="cuda"), top_p=torch.tensor([0.5, 0.9, 0.99, 0.9, 0.9, 0.1], device="cuda"))
    check(lib.sample(logits, u, **s), want(logits, u, **s))
    s["min_p"] = torch.tensor([0.1, 0.9, 1e-3, 0.5, 0.999, 0.01], device="cuda")
    check(lib.sample(logits, u, **s), want(logits, u, **s))


def test_masked_infinite_and_nan_logits(lib):
    V = 9000
    logits, u, _ = rows(5, 12, V, torch.float32)
    logits[0] = -INF
    logits[1] = float("nan")
    logits[2, 1:] = -INF
    logits[3, :V - 1] = torch.finfo(torch.float32).min          # a mask of the type's lowest value
    logits[4] = torch.finfo(torch.float32).min                  # ... everywhere: all alike
    logits[5, ::3] = float("nan")
    logits[6, [10, 20]] = INF
    logits[7, V - 1] = 3e38
    logits[7, 0] = -3e38
    logits[8, ::2] = -INF
    for s in (dict(), dict(top_k=torch.full((12,), 50, device="cuda", dtype=torch.int32)), dict(top_p=torch.full((12,), 0.9, device="cuda")),
              dict(temperature=torch.zeros(12, device="cuda"), min_p=torch.full((12,), 0.1, device="cuda"))):
        got = lib.sample(logits, u, **s)
        check(got, want(logits, u, **s))
        assert got[0][0].item() == -1 and got[0][1].item() == -1 and got[0][2].item() == 0


def test_settings_out_of_range(lib):
    """Temperatures of 0, below 0 and NaN are greedy; the filters' odd values leave them out; u is clamped."""
    N, V = 12, 5000
    logits, u, _ = rows(6, N, V, torch.float32)
    logits[3, [7, 9]] = 50.0
    t = torch.tensor([0.0, -1.0, float("nan"), 0.0, 1e-30, 1e-42, 1e30, INF, 1.0, 1.0, 1.0, 1.0], device="cuda")
    k = torch.tensor([5, 5, 5, 5, 0, 3, -1, 2 ** 31 - 1, 7, 7, 7, 7], device="cuda", dtype=torch.int32)
    p = torch.tensor([0.5, 0.5, 0.5, 0.5, 0.5, -3.0, float("nan"), 0.5, INF, 0.9, 0.9, 0.9], device="cuda")
    m = torch.tensor([0.5, 0.5, 0.5, 0.5, float("nan"), 0.1, -INF, 0.0, 0.0, 0.0, 0.0, 0.0], device="cuda")
    u[8:12] = torch.tensor([0.0, 1.0, -2.0, 5.0], device="cuda")
    got = lib.sample(logits, u, temperature=t, top_k=k, top_p=p, min_p=m)
    exp = want(logits, u, temperature=t, top_k=k, top_p=p, min_p=m)
    assert torch.equal(got[0], exp[0])
    assert got[0][3].item() == 7 and got[1][:4].tolist() == [0.0] * 4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("offset,pad", [(0, 1), (1, 0), (3, 5), (5, 1000)])
def test_strides_and_alignment(lib, dtype, offset, pad):
    """Rows that start anywhere in a buffer whose other values would win if they were read."""
    N, V = 5, 1001
    logits, u, _ = rows(7, N, V, dtype)
    buffer = torch.full((N * (V + pad) + offset + 64,), 1000.0, device="cuda", dtype=dtype)
    view = buffer[offset:offset + N * (V + pad)].view(N, V + pad)[:, :V]
    view.copy_(logits)
    got, dense = lib.sample(view, u), lib.sample(logits, u)
    assert torch.equal(got[0], dense[0]) and torch.equal(got[1], dense[1])


def test_the_longest_rows(lib):
    """Rows that do not fit the shared memory of a cluster are read again where they are needed."""
    for V in (400_001, 1 << 22):
        logits, u, _ = rows(8, 3, V, torch.float16)
        s = dict(top_k=torch.tensor([0, 100, 0], device="cuda", dtype=torch.int32), top_p=torch.tensor([1.0, 0.9, 0.6], device="cuda"))
        check(lib.sample(logits, u, **s), want(logits, u, **s))


def test_sums_at_their_limit(lib):
    """A thread's sum of weights takes 4,095 terms: rows of equal logits, of the length from which two blocks share one and just below."""
    for V in (8176 * 256, 8180 * 256, 8192 * 256):
        logits = torch.full((2, V), 0.25, device="cuda", dtype=torch.bfloat16)
        u = torch.tensor([0.0, 0.999], device="cuda")
        for s in (dict(), dict(top_p=torch.full((2,), 0.75, device="cuda"))):
            check(lib.sample(logits, u, **s), want(logits, u, **s))


def test_no_rows_outputs_and_graph(lib):
    empty = lib.sample(torch.empty(0, 100, device="cuda"), torch.empty(0, device="cuda"))
    assert empty[0].shape == (0,)
    logits, u, _ = rows(9, 4, 33000, torch.bfloat16)
    out, lp = torch.empty(4, dtype=torch.int32, device="cuda"), torch.empty(4, device="cuda")
    r = lib.sample(logits, u, out=out, logprob=lp)
    assert r[0] is out and r[1] is lp
    base = (out.clone(), lp.clone())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        lib.sample(logits, u, out=out, logprob=lp)
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, base[0]) and torch.equal(lp, base[1])


def test_refusals(lib):
    logits, u, _ = rows(10, 4, 100, torch.float32)
    for args, kw in (((logits.double(), u), {}), ((logits[0], u), {}), ((logits.t(), u[:1].expand(100)), {}), ((logits, u[:3]), {}), ((logits, u.double()), {}), ((logits.cpu(), u), {}),
                     ((logits, u), dict(temperature=u.double())), ((logits, u), dict(top_k=u)), ((logits, u), dict(top_p=u[:2])), ((logits, u), dict(min_p=u.cpu())),
                     ((logits, u), dict(out=torch.empty(4, dtype=torch.int64, device="cuda"))), ((logits[:, :0], u), {}), ((logits[:1].expand(4, 100), u), {})):
        with pytest.raises(ValueError):
            lib.sample(*args, **kw)
