"""Cuts of top-p that lie at the edge of what the histogram's sums tell apart: right, and found about as fast as any other.  Run with `-m gpu` on a B200.

A cut takes a few passes over a row (a histogram, an exact sum, a list or a table; now and then the sum again).  Where the histogram names no place for it, it is sought
all over the bins and then digit by digit, ten to twenty times as long: that is what the factors of 3 and 5 look for."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_sample import check, rows, want  # noqa: E402


def per_call(f, calls=10):
    for _ in range(3):
        f()
    times = []
    for _ in range(5):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(calls):
            f()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) / calls)
    return sorted(times)[2]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("top_k", [0, 3000])
def test_top_p_zero(dtype, top_k):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import dsv4_attn_b200 as d
    N, V = 300, 100_000
    logits, u, _ = rows(1, N, V, dtype)
    logits[5, [70, 90_000]] = 40.0                  # a tie: the lower index is kept
    s = dict(top_k=torch.full((N,), top_k, device="cuda", dtype=torch.int32))
    for p in (0.0, -1.0, 1e-9):
        got = d.sample(logits, u, top_p=torch.full((N,), p, device="cuda"), **s)
        check(got, want(logits, u, top_p=torch.full((N,), p, device="cuda"), **s))
        assert torch.equal(got[0].long(), logits.float().argmax(1)) and (got[1] == 0).all()
    zero, half = (per_call(lambda: d.sample(logits, u, top_p=p, **s)) for p in (torch.zeros(N, device="cuda"), torch.full((N,), 0.5, device="cuda")))
    assert zero <= 3 * half, (zero, half)


@pytest.mark.parametrize("dtype,spread,p", [(torch.bfloat16, 5.0, 0.999), (torch.float16, 5.0, 0.999), (torch.float32, 5.0, 0.9999), (torch.float16, 8.0, 0.9999)])
def test_cuts_among_bins_of_little_weight(dtype, spread, p):
    """Bins around the cut weigh about as much as the rounding of the sums up to them."""
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import dsv4_attn_b200 as d
    N, V = 1200, 100_000
    logits, u, _ = rows(2, N, V, dtype, spread)
    far, half = (torch.full((N,), x, device="cuda") for x in (p, 0.5))
    got = d.sample(logits, u, top_p=far)
    check((got[0][::40], got[1][::40]), want(logits[::40], u[::40], top_p=far[::40]))
    assert per_call(lambda: d.sample(logits, u, top_p=far)) <= 5 * per_call(lambda: d.sample(logits, u, top_p=half))
