"""Lengths beyond the block table, with a window that has left it behind: nothing is looked up, nothing is seen, other requests stay as they are.  Run with `-m gpu` on a B200."""
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


@pytest.mark.parametrize("width", [0, 300])                                 # clusters, shares
@pytest.mark.parametrize("G,dtype", [(4, "bf16"), (4, "e4m3"), (40, "bf16"), (40, "e4m3")])
@pytest.mark.parametrize("window,first", [(1, 0), (70, 0), (70, 3)])
def test_new_tokens(lib, G, dtype, width, window, first):
    for longer in (0, 2):                                                    # the request in front of the others, and the last one, behind whose row the table ends
        lens = [300, 200, 300]
        c = Case(lens, 2, Hkv=2, G=G, D=64, dtype=dtype, window=window, first=first, width=width, seed=G)
        room = c.table.shape[1] * PAGE
        for n in (room + window + 1, room + window + 64, 10_000_000, (1 << 31) - 1):
            st = lib.new_status("cuda")
            length = c.len_t.clone()
            length[longer] = n
            a, kw = c.args()
            before = torch.rand(3, room, device="cuda")
            w = before.clone()
            out, lse = lib.gqa_decode(c.q, *a[:3], length, a[4], **kw, weights=w, status=st)
            assert st[0] == 7
            others = [b for b in range(3) if b != longer]
            plain = before.clone()
            want, want_lse = c.call(lib, weights=plain)
            assert torch.equal(out[others], want[others]) and torch.equal(lse[others], want_lse[others]) and torch.equal(w[others], plain[others])
            if first == 0:
                assert (out[longer] == 0).all() and torch.isneginf(lse[longer]).all() and torch.equal(w[longer], before[longer])
            else:
                assert out[longer].isfinite().all() and torch.equal(w[longer, first:], before[longer, first:])


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_prompts(lib, dtype):
    for T in (700, 5):                                                       # either kernel
        c = Case([900, 800], [T, T], Hkv=2, G=4, D=64, dtype=dtype, window=70, packed=True)
        a, kw = c.args()
        want, want_lse = c.call(lib)
        for n in (c.table.shape[1] * PAGE + 70 + T, 10_000_000):
            st = lib.new_status("cuda")
            length = torch.tensor([900, n], device="cuda", dtype=torch.int32)
            out, lse = lib.gqa_prefill(c.q, c.start_t, *a[:3], length, a[4], **kw, status=st)
            assert st[0] == 7
            assert torch.equal(out[:T], want[:T]) and torch.equal(lse[:T], want_lse[:T])
            assert (out[T:] == 0).all() and torch.isneginf(lse[T:]).all()
