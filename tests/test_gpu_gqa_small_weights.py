"""Many small weights beside one entry that outweighs them all and whose value is 0: what the others leave is the whole output.  Run with `-m gpu` on a B200."""
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


# one token (in shares, each of some units), many rows, prompts, few packed tokens
@pytest.mark.parametrize("T,G,packed", [(1, 4, False), (1, 16, False), (5, 8, False), (1, 100, False), (700, 2, True), (5, 4, True)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float8_e4m3fn])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("small", [10.45, 2.49, 0.3])                        # of 2^-24 of the largest weight
def test_what_many_small_weights_leave(lib, T, G, packed, dtype, D, small):
    B, Hkv, n = 24, 8, 3000
    if packed:
        B = 3
    pages = (n + PAGE - 1) // PAGE
    g = torch.Generator(device="cuda").manual_seed(D)
    score = math.log(2.0 ** 24 / small)
    table = torch.randperm(B * pages, device="cuda", generator=g).int().reshape(B, pages)
    k = torch.zeros(B * pages, PAGE, Hkv, D, device="cuda")
    v = 1 + torch.rand(B * pages, PAGE, Hkv, D, device="cuda", generator=g)
    k[table[:, 0].long(), 0, :, 0] = 14.0
    v[table[:, 0].long(), 0] = 0.0
    eight = dtype == torch.float8_e4m3fn
    k, v = k.to(dtype), v.to(dtype)
    scales = dict(k_scale=torch.ones(Hkv, device="cuda"), v_scale=torch.ones(Hkv, device="cuda")) if eight else {}
    q = torch.randn(B * T, Hkv * G, D, device="cuda", generator=g).half()
    q[..., 0] = 1.0
    kv_len = torch.full((B,), n, device="cuda", dtype=torch.int32)
    scale = score / 14.0
    if packed:
        start = torch.arange(0, B * T + 1, T, device="cuda", dtype=torch.int32)
        out, _ = lib.gqa_prefill(q, start, k, v, table, kv_len, scale, **scales)
    else:
        out, _ = lib.gqa_decode(q.unflatten(0, (B, T)), k, v, table, kv_len, scale, **scales)
    out = out.reshape(B, T, Hkv, G, D).double()
    # every entry but the first has score 0; sums of their values up to the tokens' places
    rows = v.view(torch.uint8)[table.long()].view(dtype).double().flatten(1, 2)[:, :n]
    upto = rows.cumsum(1)[:, n - T:]                                          # [B, T, Hkv, D]
    places = torch.arange(n - T, n, device="cuda", dtype=torch.float64)      # of the tokens: as many others
    total = places + math.exp(float(torch.tensor(scale, dtype=torch.float32)) * 14.0)
    want = (upto / total[:, None, None])[:, :, :, None]
    # half a step of FP16 for the weights and one for the output (2^-24 where that is below its normal numbers), exponentials of scores to 24 log2 units in 32 bits (8 roundings
    # of 2^-24 of that, and 2^-22); weights below 2^-21 of the largest are off by up to 2^-32 of it
    tol = (2.0 ** -11 * 2.01 + 24 * 8 * 2.0 ** -24) * want + 2.0 ** -32 * (upto / (total / total.max())[:, None, None])[:, :, :, None] * 1.01 * (math.exp(score) / total.max()) + 2.0 ** -25
    err = (out - want).abs()
    assert (err <= tol).all(), f"off by up to {float((err / want).max()):.4f} of the output, {float((err / tol).max()):.2f} of the tolerance"
