"""Weights of entries in wide tables, with the longest length given: right for all entries up to it, nothing for those behind it.  Run with `-m gpu` on a B200."""
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


@pytest.mark.parametrize("T,G,dtype", [(1, 4, "bf16"), (3, 4, "f16"), (1, 4, "e4m3"), (5, 8, "bf16"), (5, 16, "e4m3")])
@pytest.mark.parametrize("width", [0, 300])
def test_weights_up_to_max_len(lib, T, G, dtype, width):
    lens = [900, 64, 333, 5, 700]
    c = Case(lens, T, Hkv=2, G=G, D=64, dtype=dtype, width=width, seed=G + T)
    before = torch.rand(c.B, c.table.shape[1] * PAGE, device="cuda")
    for longest in (900, 901, 960, 5000, c.table.shape[1] * PAGE, (1 << 31) - 1):
        w = before.clone()
        st = lib.new_status("cuda")
        out, lse = c.call(lib, weights=w, max_len=longest, status=st)
        c.check(out, lse, w, before)
        assert st.tolist() == [0, 0, 0, 0]
    # a length that is not what it says: entries behind it get nothing, all else is as it was
    whole = before.clone()
    c.call(lib, weights=whole)
    for longest in (1, 63, 64, 65, 300, 700, 899):
        w = before.clone()
        out, lse = c.call(lib, weights=w, max_len=longest)
        c.check(out, lse)
        want = before.clone()
        want[:, :longest] = whole[:, :longest]
        assert torch.equal(w[:, longest:], before[:, longest:])
        assert torch.allclose(w, want, atol=1e-5, rtol=1e-5)
