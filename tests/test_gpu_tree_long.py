"""hca_tree_decode over a cache and a workspace whose offsets pass 32 bits.  Run with `-m gpu` on a B200."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_tree import LSE_ABS, SCALE, entries, values  # noqa: E402


@pytest.mark.parametrize("rows,splits", [(False, None), (True, None), (True, 7), (False, 64)])
def test_offsets_beyond_32_bits(rows, splits):
    """Two requests over a pool of 4.6 GB (rows of 4.9 GB), all of its entries 0 but those of the first pages, pages in the middle and the last ones: an entry of 0 has a
    logit of 0 and no value, so that the formula is a sum over the others and a count."""
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import dsv4_attn_b200 as d
    from dsv4_attn_b200 import layout
    P, B, T, H, W = 110_000, 2, 2, 64, 5
    g = torch.Generator(device="cuda").manual_seed(1)
    pool = torch.zeros(P, 64, 656, dtype=torch.uint8, device="cuda")
    filled = torch.tensor([0, 1, P // 3, P // 2, P - 2, P - 1], device="cuda")
    pool[filled] = entries(g, 6, 64)
    each = 33_000
    # a request's last pages are the pool's last, and the other way round
    table = torch.stack([torch.arange(P - each, P, device="cuda"), torch.arange(each, device="cuda").flip(0)]).int()
    kv_len = torch.tensor([each * 64 - 10, each * 64], dtype=torch.int32, device="cuda")
    sees = torch.rand(B, T, W, device="cuda", generator=g) < 0.5
    q, win = torch.randn(B, T, H, 576, device="cuda", generator=g).bfloat16(), entries(g, B, W)
    q *= 3.0                                       # (entries that are not 0 stand out)
    st = d.new_status("cuda")
    out, lse = d.hca_tree_decode(q, pool, table, kv_len, win, torch.full((B,), W, dtype=torch.int32, device="cuda"), layout.pack_tree_mask(sees), SCALE, share_rows=rows,
                                 num_splits=splits, status=st)
    assert st.tolist() == [0, 0, 0, 0]
    for b in range(B):
        mine = [p for p in filled.tolist() if p in set(table[b].tolist())]
        assert len(mine) >= 2
        k = values(torch.cat([pool[p][:54] if b == 0 and p == P - 1 else pool[p] for p in mine] + [win[b]]))
        cache = k.shape[0] - W
        x = q[b].double() @ k.T * SCALE
        x[..., cache:] = x[..., cache:].masked_fill(~sees[b][:, None], float("-inf"))
        zeros = int(kv_len[b]) - cache
        want = torch.logaddexp(torch.logsumexp(x, -1), torch.tensor(float(zeros), device="cuda", dtype=torch.float64).log())
        o = torch.exp(x - want[..., None]) @ k[:, :512]
        # (q is three times that of the tolerances' derivation)
        assert (lse[b] - want).abs().max().item() <= 3 * LSE_ABS
        assert ((out[b].double() - o).abs() - (2 ** -8 * o.abs() + 3 * 3e-3)).max().item() <= 0
