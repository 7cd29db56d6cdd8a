"""Sums of very many small weights behind a large one: the denominators of long caches.  Run with `-m gpu` on a B200."""
import math

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


# whole requests in a share, many rows, prompts
@pytest.mark.parametrize("B,T,G,packed", [(400, 1, 4, False), (200, 5, 8, False), (2, 700, 8, True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
@pytest.mark.parametrize("small", [0.55, 1.45, 10.45])                       # of 2^-24 of the first weight
def test_the_denominator_of_a_long_cache(lib, B, T, G, packed, dtype, small):
    D, n = 64, 30_000
    pages = (n + PAGE - 1) // PAGE
    # all requests hold the same pages: the first entry's score is the large one, the others' are 0
    k, v = torch.zeros(pages, PAGE, 1, D, device="cuda"), torch.ones(pages, PAGE, 1, D, device="cuda")
    k[0, 0, :, 0] = 14.0
    k, v = k.to(dtype), v.to(dtype)
    one = torch.ones(1, device="cuda")
    scales = dict(k_scale=one, v_scale=one) if dtype == torch.float8_e4m3fn else {}
    q = torch.zeros(B * T, G, D, device="cuda", dtype=torch.bfloat16 if dtype == torch.bfloat16 else torch.float16)
    q[..., 0] = 1.0
    table = torch.arange(pages, device="cuda", dtype=torch.int32).expand(B, -1).contiguous()
    kv_len = torch.full((B,), n, device="cuda", dtype=torch.int32)
    scale = float(torch.tensor(math.log(2.0 ** 24 / small) / 14.0, dtype=torch.float32))
    if packed:
        _, lse = lib.gqa_prefill(q, torch.arange(0, B * T + 1, T, device="cuda", dtype=torch.int32), k, v, table, kv_len, scale, **scales)
    else:
        _, lse = lib.gqa_decode(q.unflatten(0, (B, T)), k, v, table, kv_len, scale, **scales)
    want = torch.log(math.exp(14.0 * scale) + torch.arange(n - T, n, device="cuda", dtype=torch.float64))[None, :, None]
    # a sum goes up in steps of 16 entries at least, 1,875 of them, or 469 of 64 entries, and each of the additions, the steps' own included, is off by 2^-24 of it at most; the score is
    # 24 log2 units in 32 bits (a product of three rounded factors: 3 * 2^-24 of it), and so are logarithm and result (2 * 2^-24 of 17, 2^-22)
    tol = (1875 + 24 * 3 + 2 * 17) * 2.0 ** -24 * math.log(2) + 2.0 ** -22 + 16 * 2.0 ** -24 * n * small * 2.0 ** -24
    err = (lse.reshape(B, T, G).double() - want).abs()
    assert (err <= tol).all(), f"off by up to {float(err.max()):.3e}, {float(err.max() / tol):.2f} of the tolerance"
