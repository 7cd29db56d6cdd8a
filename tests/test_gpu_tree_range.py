"""hca_tree_decode's check of the FP16 operands' range, as the other decode calls have it.  Run with `-m gpu` on a B200."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [False, True])
def test_operands_out_of_range_are_refused_on_request(rows):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import dsv4_attn_b200 as d
    from dsv4_attn_b200 import layout
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(3, 64, 576, device="cuda", generator=g)
    entries = layout.pack_entries(x[..., :512], x[..., 512:])
    args = dict(q=torch.randn(1, 2, 16, 576, device="cuda", generator=g).bfloat16(), kv_pool=entries[:2].contiguous(), block_table=torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"),
                kv_len=torch.tensor([100], dtype=torch.int32, device="cuda"), win_pool=entries[2:, :40].contiguous(), win_len=torch.tensor([40], dtype=torch.int32, device="cuda"),
                tree_mask=torch.full((1, 2, 2), -1, dtype=torch.int32, device="cuda"), sm_scale=576 ** -0.5, share_rows=rows)
    plain = d.hca_tree_decode(**args)
    checked = d.hca_tree_decode(**args, check_fp16_range=True)
    assert torch.equal(plain[0], checked[0]) and torch.equal(plain[1], checked[1])

    def scaled(pool, value):
        pool = pool.clone()
        pool.view(-1, 656)[7, 516:520] = torch.tensor([value], device="cuda").view(torch.uint8)
        return pool

    far = args["q"].clone()
    far[0, 1, 3, 5] = -65536.0
    for bad in (dict(q=far), dict(kv_pool=scaled(args["kv_pool"], 147.0)), dict(win_pool=scaled(args["win_pool"], 147.0)), dict(win_pool=scaled(args["win_pool"], float("nan")))):
        with pytest.raises(ValueError):
            d.hca_tree_decode(**{**args, **bad}, check_fp16_range=True)
    d.hca_tree_decode(**{**args, "kv_pool": scaled(args["kv_pool"], 146.0)}, check_fp16_range=True)
    # what the check is given is looked at like any other argument
    for bad in (dict(q=args["q"].float()), dict(kv_pool=args["kv_pool"].cpu()), dict(win_pool=args["win_pool"][..., :600].contiguous())):
        with pytest.raises(ValueError):
            d.hca_tree_decode(**{**args, **bad}, check_fp16_range=True)
