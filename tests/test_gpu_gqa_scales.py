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


def test_zeros_over_a_scale_of_zero(lib):
    for src in (torch.bfloat16, torch.float16):
        k = torch.zeros(2, 3, 3, 64, device="cuda", dtype=src)
        k[:, :, 1] = torch.randn(2, 3, 64, device="cuda").to(src)
        k[0, 0, 2, 5], k[0, 0, 2, 6], k[0, 0, 2, 7] = 3.0, -3.0, -0.0
        pools = [torch.full((2, PAGE, 3, 64), 7.0, device="cuda").to(torch.float8_e4m3fn) for _ in "kv"]
        scale = torch.tensor([0.0, 0.05, 0.0], device="cuda")
        table, at = torch.tensor([[1], [0]], device="cuda", dtype=torch.int32), torch.tensor([0, 5], device="cuda", dtype=torch.int32)
        lib.gqa_insert(k, k, *pools, table, at, k_scale=scale, v_scale=scale)
        for p in pools:
            got = torch.stack([p[1, :3], p[0, 5:8]]).float()
            want = (k.float() / scale[:, None]).nan_to_num(0.0, 1e9, -1e9).clamp(-448, 448).to(torch.float8_e4m3fn).float()
            assert torch.equal(got, want) and (got[..., 0, :] == 0).all()
            assert (got * scale[:, None])[:, :, [0, 2]].abs().max() == 0
        # and such a cache is read as zeros
        q = torch.randn(2, 1, 6, 64, device="cuda").to(src)
        out, lse = lib.gqa_decode(q, *pools, table[:, :1], at + 3, 0.125, k_scale=scale, v_scale=scale, window=3)
        assert out.isfinite().all() and (out[:, :, [0, 1, 4, 5]] == 0).all()
        assert torch.allclose(lse[:, 0, [0, 1]], torch.full((2, 2), 3.0, device="cuda").log())
