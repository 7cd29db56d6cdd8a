"""Sampling where a call's size decides how rows are dealt to blocks: the order of rows that take longest, clusters of two and four, and the longest sums a
thread may take.  Run with `-m gpu` on a B200."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_sample import check, rows, share, want  # noqa: E402


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import dsv4_attn_b200 as d
    return d


@pytest.mark.parametrize("N", [297, 1023, 1024, 1025, 4097, 8191, 8192, 8193])
@pytest.mark.parametrize("heavy", ["all", "none", "alternating", "front", "back", "random", "one"])
def test_every_row_is_drawn_whatever_the_order(lib, N, heavy):
    """Rows with top-p alone are begun first where there are many rows: each row's answer is the one it has in a batch too small for that."""
    V = 700
    logits, u, g = rows(N, N, V, torch.bfloat16)
    at = torch.arange(N, device="cuda")
    is_heavy = dict(all=at >= 0, none=at < 0, alternating=at % 2 == 0, front=at < N // 3, back=at >= N - N // 5, random=torch.rand(N, device="cuda", generator=g) < 0.2, one=at == N - 1)[heavy]
    s = dict(temperature=0.5 + torch.rand(N, device="cuda", generator=g), top_k=torch.where(is_heavy, 0, 20).int(), top_p=torch.full((N,), 0.9, device="cuda"))
    s["temperature"][3::7] = 0.0                   # (greedy rows take no time, with top-p or without)
    out, logprob = torch.full((N,), -7, dtype=torch.int32, device="cuda"), torch.full((N,), math.nan, device="cuda")
    lib.sample(logits, u, out=out, logprob=logprob, **s)
    for n in range(0, N, 250):
        part = slice(n, min(n + 250, N))
        token, lp = lib.sample(logits[part], u[part], **{k: v[part].contiguous() for k, v in s.items()})
        assert torch.equal(out[part], token) and torch.equal(logprob[part], lp)
    some = torch.randperm(N, device="cuda", generator=g)[:40]
    check((out[some], logprob[some]), want(logits[some], u[some], **{k: v[some] for k, v in s.items()}))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("filters", ["none", "top_k", "top_p", "min_p", "all"])
def test_clusters_of_two(lib, dtype, filters):
    """Rows of more than 32,768 logits, fewer of them than SMs, but more than half as many."""
    N, V = 120, 40_001
    logits, u, g = rows(V, N, V, dtype)
    s = dict(temperature=0.4 + torch.rand(N, device="cuda", generator=g))
    if filters in ("top_k", "all"):
        s["top_k"] = torch.tensor([0, 1, 2, 40, 50, 1000, 1025, 2048, 3000, V - 1], device="cuda", dtype=torch.int32).repeat(N // 10)
    if filters in ("top_p", "all"):
        s["top_p"] = torch.tensor([0.0, 0.1, 0.5, 0.9, 0.95, 0.999, 1.0, 2.0, 0.8, 0.3, 0.7, 0.99], device="cuda").repeat(N // 12)
    if filters in ("min_p", "all"):
        s["min_p"] = torch.tensor([0.0, 1e-9, 0.01, 0.05, 0.2, -1.0], device="cuda").repeat(N // 6)
    check(lib.sample(logits, u, **s), want(logits, u, **s))


# the longest rows of which one and two blocks take all (511 steps of 256 logits a warp, with the up to seven elements before a row that its alignment adds), one
# logit more, and the longest rows there are
LIMITS = [8176 * 256 - 7, 8176 * 256 - 6, 16352 * 256 - 7, 16352 * 256 - 6, 1 << 22]


@pytest.mark.parametrize("V", LIMITS)
def test_the_longest_sums(lib, V):
    """Rows of equal logits, more of them than SMs, so that nothing but a thread's sum of at most 4,095 weights asks for another block; they start at every
    alignment.  A token is then known from the definition: all weigh 2^40."""
    N = 150
    buffer = torch.full((N * (V + 1) + 8,), 0.25, device="cuda", dtype=torch.bfloat16)
    logits = buffer[3:3 + N * (V + 1)].view(N, V + 1)[:, :V]
    g = torch.Generator(device="cuda").manual_seed(V)
    u = torch.rand(N, device="cuda", generator=g)
    u[:4] = torch.tensor([0.0, 0.99999994, 0.5, 1e-7], device="cuda")
    for top_p in (None, 0.75):
        kept = V if top_p is None else -(-share(V << 40, int(top_p * 2 ** 24)) // (1 << 40))
        token = torch.tensor([share(kept << 40, int(x * 2 ** 24)) >> 40 for x in u.double().tolist()], dtype=torch.int32, device="cuda")
        got = lib.sample(logits, u, top_p=None if top_p is None else torch.full((N,), top_p, device="cuda"))
        assert torch.equal(got[0], token), (got[0] != token).nonzero()[:4]
        assert (got[1] + math.log(kept)).abs().max().item() <= 6e-6
