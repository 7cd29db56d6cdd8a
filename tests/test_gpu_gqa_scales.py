"""Scales of an 8-bit cache's heads that are 0 or negative, and factors of a row's scores that are too small for 32 bits, in every kernel.  Run with `-m gpu` on a B200."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.gqa_util import Case, PAGE  # noqa: E402


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import dsv4_attn_b200 as d
    return d


# up to 16 rows of a head in clusters and in shares, more rows, prompts, a few packed tokens
CALLS = [dict(kv_len=[200, 65, 3], new=1, G=4), dict(kv_len=[200, 65, 3], new=1, G=4, width=300), dict(kv_len=[700, 65, 5], new=5, G=8), dict(kv_len=[300, 1000], new=1, G=100),
         dict(kv_len=[900, 400], new=[700, 400], G=4, packed=True), dict(kv_len=[900, 30], new=[5, 30], G=3, packed=True)]


@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("q_dtype,D", [("bf16", 128), ("f16", 64), ("bf16", 256)])
@pytest.mark.parametrize("call", CALLS)
def test_scales_of_any_sign(lib, call, q_dtype, D, window):
    c = Case(Hkv=4, D=D, dtype="e4m3", q_dtype=q_dtype, window=window, sink=True, **call)
    c.scales = [torch.tensor(s, device="cuda") for s in ([0.0, -0.04, 0.05, -0.0], [0.03, -0.04, 0.0, 0.05])]
    c.check(*c.call(lib))


@pytest.mark.parametrize("call", CALLS[:4])
def test_weights_over_scales_of_any_sign(lib, call):
    c = Case(Hkv=2, D=64, dtype="e4m3", **call)
    c.scales = [torch.tensor(s, device="cuda") for s in ([0.0, -0.04], [0.03, 0.0])]
    before = torch.rand(c.B, c.table.shape[1] * PAGE, device="cuda")
    w = before.clone()
    out, lse = c.call(lib, weights=w)
    c.check(out, lse, w, before)


@pytest.mark.parametrize("call", CALLS)
def test_a_row_of_zeros_beside_rows_far_outside_fp16(lib, call):
    """The factor that such a row's scores are scaled by is below the smallest number of 32 bits."""
    c = Case(Hkv=2, D=128, dtype="e4m3", by=1e30, **call)
    c.q[0].zero_()
    c.scale = 1e-31
    c.check(*c.call(lib))
