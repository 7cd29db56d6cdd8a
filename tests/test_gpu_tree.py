"""Tree decode (hca_tree_decode) against the formula in 64 bits.  Run with `-m gpu` on a B200.

Tolerances.  Inputs are N(0, 1), the softmax scale 1/24.  K and V pass through FP16 (relative error at most 2^-11, uniform: 2.8e-4 rms), so a logit,
a sum of 576 products over 24, is off by 2.8e-4 rms and, over the 1e6 logits of a case, by less than 1.4e-3.  That moves an output by at
most 1.4e-3 times the mean |v| of 0.8; P and V in FP16 add 2^-11 of it each, and BF16 rounds the result by 2^-9 of itself: 2^-8 |out| + 3e-3 holds
twice that.  lse moves by no more than a logit: 1.4e-3."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

LSE_ABS = 1.4e-3


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import dsv4_attn_b200 as d
    return d


def entries(g, *lead):
    from dsv4_attn_b200 import layout
    x = torch.randn(*lead, 576, device="cuda", generator=g)
    return layout.pack_entries(x[..., :512], x[..., 512:])


def values(e):
    lat = e[..., :512].contiguous().view(torch.float8_e4m3fn).double().reshape(*e.shape[:-1], 4, 128)
    scale = e[..., 512:528].contiguous().view(torch.float32).double()
    return torch.cat([(lat * scale[..., None]).reshape(*e.shape[:-1], 512), e[..., 528:].contiguous().view(torch.bfloat16).double()], -1)


def make(seed, B, T, H, kv_len, W, win_len=None, density=0.6):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = max(1, (max(kv_len) + 63) // 64)
    spare = 3
    sees = torch.rand(B, T, W, device="cuda", generator=g) < density
    return dict(q=torch.randn(B, T, H, 576, device="cuda", generator=g).bfloat16(), kv_pool=entries(g, B * pages + spare, 64),
                block_table=torch.randperm(B * pages + spare, device="cuda", generator=g)[:B * pages].int().reshape(B, pages),
                kv_len=torch.tensor(kv_len, device="cuda", dtype=torch.int32), win_pool=entries(g, B, W) if W else torch.empty(B, 0, 656, device="cuda", dtype=torch.uint8),
                win_len=torch.tensor(win_len or [W] * B, device="cuda", dtype=torch.int32), sees=sees)


def want(c, scale, sink=None):
    B, T, H, _ = c["q"].shape
    out, lse = [], []
    for b in range(B):
        n, m = int(c["kv_len"][b]), int(c["win_len"][b])
        k = values(torch.cat([c["kv_pool"][c["block_table"][b].long()].reshape(-1, 656)[:n], c["win_pool"][b, :m]]))
        seen = torch.cat([torch.ones(T, n, dtype=torch.bool, device="cuda"), c["sees"][b, :, :m]], 1)
        x = (c["q"][b].double() @ k.T * scale).masked_fill(~seen[:, None], -math.inf)
        l = torch.logsumexp(x, -1) if n + m else torch.full((T, H), -math.inf, device="cuda", dtype=torch.float64)
        below = l if sink is None else torch.logaddexp(l, sink.double())
        p = torch.exp(x - torch.where(below == -math.inf, 0.0, below)[..., None])
        out.append(torch.where((l == -math.inf)[..., None], 0.0, p @ k[:, :512]))
        lse.append(l)
    return torch.stack(out), torch.stack(lse)


def call(lib, c, scale, mask=None, **kw):
    from dsv4_attn_b200 import layout
    st = lib.new_status("cuda")
    out, lse = lib.hca_tree_decode(c["q"], c["kv_pool"], c["block_table"], c["kv_len"], c["win_pool"], c["win_len"],
                                   layout.pack_tree_mask(c["sees"]) if mask is None else mask, scale, status=st, **kw)
    torch.cuda.synchronize()
    assert st.tolist() == [0, 0, 0, 0]
    return out, lse


def check(got, exp):
    (out, lse), (o, l) = got, exp
    assert torch.equal(torch.isneginf(lse), torch.isneginf(l))
    fin = ~torch.isneginf(l)
    assert (lse[fin] - l[fin]).abs().max().item() <= LSE_ABS if fin.any() else True
    err = (out.double() - o).abs() - (2 ** -8 * o.abs() + 3e-3)
    assert err.max().item() <= 0, err.max().item()
    assert (out[~fin] == 0).all()


SCALE = 576 ** -0.5
CASES = [
    # B, T, H, kv_len, W, win_len
    (1, 1, 1, [0], 1, None),                     # one token, one entry
    (1, 1, 128, [65], 5, None),                  # a plain step; the window begins inside the cache's last tile
    (2, 3, 16, [63, 64], 33, None),              # several nodes share a row group; a mask of two words, the second nearly empty
    (3, 11, 40, [0, 130, 1], 101, [101, 77, 0]), # odd counts; a request without cache, one without window
    (2, 64, 20, [200, 31], 192, None),           # wide trees
    (1, 5, 128, [1000], 0, None),                # no window at all
    (5, 16, 128, [300, 0, 782, 64, 5], 144, None),   # more row groups than pairs of SMs
]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("route", ["auto", "one", "three", "plan", "rows", "rows_three", "rows_plan"])
def test_against_the_formula(lib, case, route):
    B, T, H, kv_len, W, win_len = CASES[case]
    c = make(100 + case, B, T, H, kv_len, W, win_len)
    sink = torch.randn(H, device="cuda") if case % 2 else None
    kw = dict(auto={}, one=dict(num_splits=1), three=dict(num_splits=3), plan={}, rows=dict(num_splits=1), rows_three=dict(num_splits=3), rows_plan={})[route]
    if route != "auto":
        kw["share_rows"] = route.startswith("rows")
    if route.endswith("plan"):
        kw |= dict(plan=lib.plan_hca(B, 1, T * H, c["kv_len"][:, None].contiguous(), c["win_len"][:, None].contiguous()))
    check(call(lib, c, SCALE, attn_sink=sink, **kw), want(c, SCALE, sink))


@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("H", [8, 100, 128])
def test_nodes_that_see_nothing(lib, H, rows):
    """No cache, and masks that leave every second node empty: 0 and -inf there, also next to nodes that see something."""
    c = make(7, 2, 6, H, [0, 0], 70)
    c["sees"][:, ::2] = False
    got = call(lib, c, SCALE, share_rows=rows)
    check(got, want(c, SCALE))
    assert torch.isneginf(got[1][:, ::2]).all() and torch.isfinite(got[1][:, 1::2]).all()


@pytest.mark.parametrize("rows", [False, True])
def test_mask_shorter_and_longer_than_the_window(lib, rows):
    from dsv4_attn_b200 import layout
    c = make(8, 2, 4, 64, [100, 3], 96)
    short = layout.pack_tree_mask(c["sees"])[..., :2].contiguous()
    c["sees"][..., 64:] = False                  # rows beyond the mask's words are seen by no node
    check(call(lib, c, SCALE, mask=short, share_rows=rows), want(c, SCALE))
    longer = torch.nn.functional.pad(layout.pack_tree_mask(c["sees"]), (0, 2), value=-1)
    check(call(lib, c, SCALE, mask=longer, share_rows=rows), want(c, SCALE))


@pytest.mark.parametrize("rows", [False, True])
def test_what_masked_rows_hold_does_not_matter(lib, rows):
    """Rows that no node sees hold NaN and infinities in every field; a row that some nodes see has a NaN RoPE tail: only they are NaN."""
    c = make(9, 2, 4, 32, [70, 0], 80)
    c["sees"][:, :, 10] = False
    c["sees"][:, :, 79] = False
    c["win_pool"][:, 10] = 0xFF
    c["win_pool"][:, 79, :528] = 0x7F
    exp = want({**c, "win_pool": torch.where(torch.arange(80, device="cuda")[None, :, None] % 69 == 10, torch.zeros_like(c["win_pool"]), c["win_pool"])}, SCALE)
    check(call(lib, c, SCALE, share_rows=rows), exp)
    c["sees"][:, :, 20] = False
    c["sees"][:, 1, 20] = True
    c["win_pool"][:, 20, 528:] = 0xFF
    out, lse = call(lib, c, SCALE, share_rows=rows)
    c["win_pool"][:, 10] = c["win_pool"][:, 79] = c["win_pool"][:, 20] = 0
    o, l = want(c, SCALE)
    nan = torch.zeros_like(l, dtype=torch.bool)
    nan[:, 1] = True
    assert torch.isnan(lse[nan]).all() and torch.isnan(out[nan]).all()
    check((out[:, [0, 2, 3]], lse[:, [0, 2, 3]]), (o[:, [0, 2, 3]], l[:, [0, 2, 3]]))


def test_a_chain_is_the_plain_decode(lib):
    """One node that sees the whole window gives bit for bit what hca_dense_decode gives."""
    c = make(10, 3, 1, 128, [782, 64, 0], 128, [128, 100, 3])
    c["sees"][:] = True
    out, lse = call(lib, c, SCALE, num_splits=1)
    o, l = lib.hca_dense_decode(c["q"], c["kv_pool"], c["block_table"], c["kv_len"][:, None].contiguous(), c["win_pool"], c["win_len"][:, None].contiguous(), SCALE, num_splits=1)
    assert torch.equal(out, o) and torch.equal(lse, l)


@pytest.mark.parametrize("rows", [False, True])
def test_outputs_of_any_alignment(lib, rows):
    """`out` at 16 bytes from a sector's start, and many items of one and two tiles a pair of blocks."""
    from dsv4_attn_b200 import layout
    B, T, H = 40, 10, 128
    c = make(15, B, T, H, [(7 * b) % 90 for b in range(B)], 40)
    buffer = torch.zeros(B * T * H * 512 + 8, device="cuda", dtype=torch.bfloat16)
    out = buffer[8:].view(B, T, H, 512)
    got = call(lib, c, SCALE, out=out, share_rows=rows)
    assert got[0] is out and buffer[:8].eq(0).all()
    check(got, want(c, SCALE))


@pytest.mark.parametrize("B,T,H", [(20, 9, 128), (40, 33, 20), (7, 32, 128), (257, 1, 128)])
def test_row_groups_dealt_to_pairs(lib, B, T, H):
    """Several rounds of row groups for every pair, the last one partly filled, over requests of equal, very different and no lengths; and more
    requests than are put in order."""
    kv_len = [(37 * b * b) % 700 if b % 4 else (0, 640)[b % 8 == 0] for b in range(B)]
    win_len = [0 if b % 5 == 3 else 33 - b % 3 for b in range(B)]
    c = make(B, B, T, H, kv_len, 33, win_len)
    sink = torch.randn(H, device="cuda")
    check(call(lib, c, SCALE, attn_sink=sink, num_splits=1, share_rows=True), want(c, SCALE, sink))


def test_a_workspace_off_its_boundary_is_refused(lib):
    c = make(2, 2, 16, 64, [100, 200], 8)
    room = torch.empty(lib.tree_rows_bytes(2, c["block_table"].shape[1], 8) + 32, device="cuda", dtype=torch.uint8)
    with pytest.raises(lib.Dsv4Error):
        call(lib, c, SCALE, share_rows=room[16:])
    check(call(lib, c, SCALE, share_rows=room[32:]), want(c, SCALE))


def test_tree_sees():
    """Ancestors, the node itself, and the committed tokens that have not slid out."""
    from dsv4_attn_b200 import layout
    got = layout.tree_sees(torch.tensor([[-1, 0, 0, 2]]), 3)[0].int().tolist()
    assert got == [[0, 1, 1, 1, 0, 0, 0], [0, 0, 1, 1, 1, 0, 0], [0, 0, 1, 1, 0, 1, 0], [0, 0, 0, 1, 0, 1, 1]]


@pytest.mark.parametrize("rows", [False, True])
def test_entries_out_of_range_are_reported(lib, rows):
    from dsv4_attn_b200 import layout
    c = make(11, 1, 2, 16, [100], 40)
    c["sees"][:] = True
    mask = layout.pack_tree_mask(c["sees"])
    for change in (dict(kv_len=torch.tensor([129], device="cuda", dtype=torch.int32)), dict(win_len=torch.tensor([41], device="cuda", dtype=torch.int32)),
                   dict(block_table=torch.tensor([[0, 99]], device="cuda", dtype=torch.int32))):
        d = {**c, **change}
        st = lib.new_status("cuda")
        longer = torch.nn.functional.pad(mask, (0, 1), value=-1)
        lib.hca_tree_decode(d["q"], d["kv_pool"], d["block_table"], d["kv_len"], d["win_pool"], d["win_len"], longer, SCALE, status=st, share_rows=rows)
        torch.cuda.synchronize()
        assert st[0].item() == 7, change


def test_graph_replay_and_another_stream(lib):
    from dsv4_attn_b200 import layout
    c = make(12, 6, 16, 128, [300, 0, 782, 64, 5, 90], 144)
    mask = layout.pack_tree_mask(c["sees"])
    args = (c["q"], c["kv_pool"], c["block_table"], c["kv_len"], c["win_pool"], c["win_len"], mask, SCALE)
    base = lib.hca_tree_decode(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = lib.hca_tree_decode(*args)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kept = lib.hca_tree_decode(*args)
    c["q"].copy_(c["q"].flip(0))
    c["q"].copy_(c["q"].flip(0))
    g.replay()
    torch.cuda.synchronize()
    for r in (other, kept):
        assert torch.equal(r[0], base[0]) and torch.equal(r[1], base[1])


def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_unaffected(lib):
    """The hand-over of a tile is withheld in every pair: the kernel returns with a status, and the next launch is right."""
    from dsv4_attn_b200 import layout
    c = make(14, 2, 8, 128, [300, 100], 40)
    args = (c["q"], c["kv_pool"], c["block_table"], c["kv_len"], c["win_pool"], c["win_len"], layout.pack_tree_mask(c["sees"]), SCALE)
    for rows in (False, True):
        st = lib.new_status("cuda")
        lib.LIB.dsv4_debug_set_wait(20_000_000, 1)
        try:
            lib.hca_tree_decode(*args, status=st, share_rows=rows)
            torch.cuda.synchronize()
        finally:
            lib.LIB.dsv4_debug_set_wait(0, -1)
        assert st[0].item() in (1, 2, 3, 4, 5, 6, 9)
        check(call(lib, c, SCALE, share_rows=rows), want(c, SCALE))


def test_refusals(lib):
    from dsv4_attn_b200 import layout
    c = make(13, 2, 3, 16, [64, 10], 40)
    mask = layout.pack_tree_mask(c["sees"])
    good = dict(q=c["q"], kv_pool=c["kv_pool"], block_table=c["block_table"], kv_len=c["kv_len"], win_pool=c["win_pool"], win_len=c["win_len"], tree_mask=mask, sm_scale=SCALE)
    lib.hca_tree_decode(**good)
    for bad in (dict(q=c["q"].float()), dict(q=c["q"][..., :512].contiguous()), dict(q=c["q"].transpose(1, 2)), dict(kv_len=c["kv_len"].long()), dict(kv_len=c["kv_len"][:1]),
                dict(win_len=c["win_len"][:, None].contiguous()), dict(win_pool=c["win_pool"][:1]), dict(tree_mask=mask[:, :2].contiguous()), dict(tree_mask=mask.long()),
                dict(attn_sink=torch.zeros(4, device="cuda")), dict(num_splits=0), dict(num_splits=65), dict(out=torch.empty(2, 3, 16, 576, device="cuda", dtype=torch.bfloat16)),
                dict(lse=torch.empty(2, 3, device="cuda")), dict(share_rows=torch.empty(100, device="cuda", dtype=torch.uint8)), dict(share_rows=3), dict(block_table=c["block_table"].cpu()),
                dict(plan=lib.plan_hca(2, 3, 16, torch.zeros(2, 3, device="cuda", dtype=torch.int32), torch.zeros(2, 3, device="cuda", dtype=torch.int32)))):
        with pytest.raises(ValueError):
            lib.hca_tree_decode(**{**good, **bad})
    for scale in (0.0, float("nan"), -1.0):
        with pytest.raises(lib.Dsv4Error):
            lib.hca_tree_decode(**{**good, "sm_scale": scale})
