"""Sinks of any size: infinite ones, and those whose exponent of two 32 bits do not hold.  Run with `-m gpu` on a B200."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.gqa_util import Case, PAGE  # noqa: E402

CALLS = [dict(kv_len=[200, 65, 0], new=1, G=4), dict(kv_len=[200, 65, 3], new=1, G=4, width=300), dict(kv_len=[700, 65, 5], new=5, G=8), dict(kv_len=[900, 400], new=[700, 400], G=4, packed=True),
         dict(kv_len=[900, 30], new=[5, 30], G=4, packed=True)]


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import dsv4_attn_b200 as d
    return d


@pytest.mark.parametrize("dtype", ["bf16", "f16", "e4m3"])
@pytest.mark.parametrize("call", CALLS)
def test_sinks(lib, call, dtype):
    c = Case(Hkv=2, D=64, dtype=dtype, **call)
    plain = Case(Hkv=2, D=64, dtype=dtype, **call)
    top = torch.finfo(torch.float32).max
    c.sink = torch.zeros(c.H, device="cuda")
    c.sink[1:8] = torch.tensor([math.inf, -math.inf, top, -top, 1e4, -1e4, 3e38], device="cuda")
    more = {}
    if not c.packed:
        more = dict(weights=torch.zeros(c.B, c.table.shape[1] * PAGE, device="cuda"))
    out, lse = c.call(lib, **more)
    want, want_lse = plain.call(lib)
    assert torch.equal(lse, want_lse)                                        # without the sink
    assert (out[..., [1, 3, 5, 7], :] == 0).all()                            # nothing is left to the entries
    assert torch.equal(out[..., [2, 4, 6], :], want[..., [2, 4, 6], :])      # nothing is taken from them
    if more:
        for b, n in enumerate(c.kv_len):
            # a row's weights add up to 1 for the three heads whose sinks take nothing, to 0 for four, and with a sink of 0 to e^lse / (e^lse + 1), between 0 and 1, for H - 7
            total = float(more["weights"][b].sum()) / c.new[b]
            assert (total == 0) if n == 0 else 3 - 1e-3 < total <= 3 + c.H - 7 + 1e-3
