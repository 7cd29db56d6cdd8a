"""hca_tree_decode behind block tables that are wider than the requests need.  Run with `-m gpu` on a B200."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,T,H", [(1, 2, 16), (3, 16, 128), (100, 2, 128)])
@pytest.mark.parametrize("fill", [-1, 2 ** 31 - 1])
def test_a_table_wider_than_the_requests_need(B, T, H, fill):
    """Slots behind a request's last page hold anything; with and without `max_len`, by every route, the answer is that of a table of the right width (on the
    same route with the same split, bit for bit)."""
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import dsv4_attn_b200 as d
    from dsv4_attn_b200 import layout
    g = torch.Generator(device="cuda").manual_seed(B)
    pages, wide, W = 3, 40, 33
    x = torch.randn(B * pages + 1, 64, 576, device="cuda", generator=g)
    pool = layout.pack_entries(x[..., :512], x[..., 512:])
    kv_len = torch.randint(0, pages * 64 + 1, (B,), device="cuda", generator=g).int()
    kv_len[-1] = pages * 64
    table = torch.randperm(B * pages + 1, device="cuda", generator=g)[:B * pages].int().reshape(B, pages)
    wider = torch.full((B, wide), fill, dtype=torch.int32, device="cuda")
    for b in range(B):
        held = (int(kv_len[b]) + 63) // 64
        wider[b, :held] = table[b, :held]
    mask = torch.randint(-2 ** 31, 2 ** 31, (B, T, 2), device="cuda", generator=g).int()
    w = torch.randn(B, W, 576, device="cuda", generator=g)
    args = dict(q=torch.randn(B, T, H, 576, device="cuda", generator=g).bfloat16(), kv_pool=pool, kv_len=kv_len, win_pool=layout.pack_entries(w[..., :512], w[..., 512:]),
                win_len=torch.full((B,), W, dtype=torch.int32, device="cuda"), tree_mask=mask, sm_scale=576 ** -0.5)
    for rows in (False, True):
        for splits in (1, 2):
            want = d.hca_tree_decode(**args, block_table=table, share_rows=rows, num_splits=splits)
            st = d.new_status("cuda")
            got = d.hca_tree_decode(**args, block_table=wider, share_rows=rows, num_splits=splits, status=st)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and st.tolist() == [0, 0, 0, 0]
    for max_len in (None, pages * 64 + W, 1):
        st = d.new_status("cuda")
        out, lse = d.hca_tree_decode(**args, block_table=wider, max_len=max_len, status=st)
        assert st.tolist() == [0, 0, 0, 0]
        # (other splits: 16-bit partials; the lse of a row comes from the same FP16 logits in another order of sums)
        assert (lse - want[1]).abs().max().item() <= 1e-4 and (out.float() - want[0].float()).abs().max().item() <= 2e-2
