"""Attention of new tokens over K and V pages against its definition in 64 bits: types, head layouts, lengths around the tiles' ends, windows, rows that see nothing,
pages out of range, strides, graphs and streams.  Run with `-m gpu` on a B200."""
import itertools

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


@pytest.mark.parametrize("dtype", ["bf16", "f16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_lengths_around_tiles(lib, dtype, D):
    st = lib.new_status("cuda")
    c = Case([1, 2, 63, 64, 65, 127, 128, 129, 200, 0, 1000], 1, Hkv=2, G=4, D=D, dtype=dtype, seed=D)
    c.check(*c.call(lib, status=st))
    assert st.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("B", [1, 20, 50, 150])
@pytest.mark.parametrize("D,G,dtype", [(64, 8, "f16"), (128, 8, "bf16"), (128, 24, "e4m3"), (256, 8, "e4m3")])
def test_parts_joined_by_any_number_of_warps(lib, B, D, G, dtype):
    """Few rows in many parts to many rows in few: a row of the merge has eight warps, four, two or one."""
    c = Case([6000 // B + i * 97 % 700 for i in range(B)], 1, Hkv=4, G=G, D=D, dtype=dtype, seed=B, width=400, sink=True)
    c.check(*c.call(lib))


@pytest.mark.parametrize("G,T", [(4, 1), (5, 4), (32, 1)])
@pytest.mark.parametrize("dtype,D", [("bf16", 64), ("bf16", 128), ("e4m3", 128), ("f16", 256)])
def test_weights_after_clusters_shares_and_many_rows(lib, G, T, dtype, D):
    for width, B in ((0, 2), (300, 2), (0, 60)):
        c = Case([1500 // B + i * 71 % 300 + T for i in range(B)], T, Hkv=3, G=G, D=D, dtype=dtype, seed=B, width=width)
        w = torch.zeros(B, c.table.shape[1] * PAGE, device="cuda")
        before = w.clone()
        c.check(*c.call(lib, weights=w), w, before)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_lengths_in_wide_tables(lib, dtype, D):
    """Tables with room for far more than the lengths: the cache is shared out over resident blocks instead of clusters."""
    for kw in (dict(G=4), dict(G=20), dict(G=3, window=70, first=2)):
        c = Case([1, 64, 65, 129, 0, 1000, 63], 1, Hkv=2, D=D, dtype=dtype, seed=D, width=200, **kw)
        c.check(*c.call(lib))
    st = lib.new_status("cuda")
    c = Case([700, 2], 1, Hkv=1, G=1, D=D, dtype=dtype, width=300)
    c.check(*c.call(lib, max_len=700, status=st))        # (steers the launch)
    w = torch.zeros(2, 300 * PAGE, device="cuda")
    c.check(*c.call(lib, weights=w, status=st), w, torch.zeros_like(w))
    assert st.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("B,Hkv", [(1, 1), (4, 8), (9, 8), (30, 4), (70, 2), (148, 1), (300, 1)])
def test_clusters_of_all_widths(lib, B, Hkv):
    """Eight, four and two blocks a unit, and none; units with fewer tiles than blocks."""
    for D in (64, 256):
        c = Case([(37 * b) % 600 for b in range(B)], 1, Hkv=Hkv, G=2, D=D, dtype="f16", seed=B)
        c.check(*c.call(lib))


@pytest.mark.parametrize("Hkv,G,T", [(1, 1, 1), (1, 16, 1), (3, 5, 1), (8, 1, 1), (2, 7, 3), (1, 17, 1), (2, 8, 4), (1, 33, 1), (1, 64, 1), (2, 16, 5), (1, 8, 40), (1, 100, 1)])
@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_heads_and_tokens(lib, Hkv, G, T, dtype):
    c = Case([T, T + 1, 70 + T, 500, 3], T, Hkv=Hkv, G=G, D=128, dtype=dtype, seed=Hkv * G + T, sink=True)
    c.check(*c.call(lib))


@pytest.mark.parametrize("window,first", [(1, 0), (1, 1), (10, 0), (10, 3), (64, 64), (100, 65), (130, 500), (1 << 30, 4), ((1 << 31) - 1, 4), (7, (1 << 31) - 1)])
@pytest.mark.parametrize("T", [1, 5, 70])
def test_windows(lib, window, first, T):
    for dtype, D in (("f16", 64), ("e4m3", 128)):
        c = Case([1, 5, 64, 129, 300, 777], T, Hkv=2, G=3, D=D, dtype=dtype, window=window, first=first, seed=T, sink=T == 5)
        c.check(*c.call(lib))


def test_one_request_and_long_ones_are_shared_out(lib):
    for kv in ([9000], [20000, 1, 300], [64 * 37]):
        for dtype in ("bf16", "e4m3"):
            c = Case(kv, 1, Hkv=4, G=4, D=128, dtype=dtype, seed=len(kv))
            c.check(*c.call(lib))


def test_many_requests(lib):
    lens = [(i * 37) % 400 for i in range(1500)]
    c = Case(lens, 1, Hkv=1, G=2, D=64, dtype="f16", seed=3)
    c.check(*c.call(lib))


@pytest.mark.parametrize("dtype,T,G,window", [("bf16", 1, 4, 0), ("f16", 3, 4, 0), ("e4m3", 2, 16, 0), ("bf16", 4, 2, 50), ("e4m3", 5, 16, 100), ("f16", 1, 1, 1)])
def test_weights(lib, dtype, T, G, window):
    st = lib.new_status("cuda")
    c = Case([3, 64, 65, 700, 5, 0], T, Hkv=3, G=G, D=64, dtype=dtype, window=window, first=2 if window else 0, sink=True, seed=T)
    before = torch.rand(c.B, c.table.shape[1] * PAGE + 5, device="cuda")
    w = before.clone()
    out, lse = c.call(lib, weights=w, status=st)
    c.check(out, lse, w, before)
    assert st.tolist() == [0, 0, 0, 0]
    again = before.clone()
    c.call(lib, weights=again)
    assert torch.equal(again, w)                        # one order of sums


def test_rows_of_a_fused_projection_and_given_outputs(lib):
    c = Case([100, 300], 2, Hkv=2, G=4, D=128, dtype="bf16", fused=True)
    assert not c.q.is_contiguous()
    out = torch.full((2, 2, 8, 128), 7.0, device="cuda", dtype=torch.bfloat16)
    lse = torch.full((2, 2, 8), 7.0, device="cuda")
    o, s = c.call(lib, out=out, lse=lse)
    assert o is out and s is lse
    c.check(out, lse)
    # heads before tokens
    c.q = c.q.transpose(1, 2).contiguous().transpose(1, 2)
    c.check(*c.call(lib))


def test_queries_of_both_types_over_8_bits_and_their_range(lib):
    for q_dtype in ("bf16", "f16"):
        c = Case([200, 65], 1, Hkv=2, G=4, D=128, dtype="e4m3", q_dtype=q_dtype)
        c.check(*c.call(lib))
    # rows far outside FP16's range, with a scale that brings the scores back
    for by in (1e30, 1e-30):
        c = Case([200, 65], 1, Hkv=2, G=4, D=128, dtype="e4m3", by=by)
        c.scale = 1.0 / (by * 128 ** 0.5)
        c.check(*c.call(lib))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_many_rows_of_a_head(lib, dtype, D):
    """Drafted tokens x query heads beyond what a few warps hold: one group and several, streams without a page, units that are cut."""
    for Hkv, G, T, kv in ((2, 8, 5, [64, 5, 65, 128, 129, 700, 0, 3000]), (1, 40, 1, [1, 63, 200, 1000]), (4, 16, 9, [9, 100, 777]), (1, 3, 50, [50, 64, 500]), (1, 128, 2, [300, 2]),
                          (8, 17, 1, [40, 4000])):
        c = Case(kv, T, Hkv=Hkv, G=G, D=D, dtype=dtype, seed=G, sink=G == 8)
        c.check(*c.call(lib))


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_many_rows_with_windows_and_weights(lib, dtype):
    for window, first in ((1, 0), (60, 3), (64, 64), (129, 200), (1 << 30, 0)):
        c = Case([5, 64, 300, 1000, 12], 5, Hkv=2, G=12, D=128, dtype=dtype, window=window, first=first, seed=first)
        before = torch.rand(c.B, c.table.shape[1] * PAGE, device="cuda")
        w = before.clone()
        out, lse = c.call(lib, weights=w)
        c.check(out, lse, w, before)


def test_scores_that_grow_with_many_rows(lib):
    for dtype in ("f16", "e4m3"):
        c = Case([2000], 4, Hkv=2, G=16, D=64, dtype=dtype)
        n = torch.arange(2000, device="cuda")
        c.q.fill_(0)
        c.q[..., 0] = 1.0
        c.q[..., 1:] = torch.randn(1, 4, 32, 63, device="cuda").to(c.q.dtype)
        c.pools[0].view(torch.uint8 if dtype == "e4m3" else torch.int16)[c.table[0, n // 64].long(), n % 64, :, 0] = \
            (n.float() / 2000 * 60).to(c.pools[0].dtype).view(torch.uint8 if dtype == "e4m3" else torch.int16)[:, None]
        c.scale = 1.0
        c.check(*c.call(lib))


def test_queries_that_share_their_rows(lib):
    """Expanded queries: axes with a stride of 0."""
    for G, T in ((4, 1), (48, 1), (8, 5)):
        c = Case([100, 300], T, Hkv=2, G=G, D=128, dtype="bf16")
        c.q = c.q[:1].expand(2, -1, -1, -1)
        a, kw = c.args()
        out, lse = lib.gqa_decode(c.q, *a, **kw)
        c.q = c.q.contiguous()
        c.check(out, lse)


def test_equal_and_extreme_scores(lib):
    """Scores that are all alike, and one that outweighs the others by far."""
    c = Case([130, 64], 1, Hkv=1, G=2, D=64, dtype="bf16")
    c.q.zero_()
    c.check(*c.call(lib))
    c = Case([1000], 1, Hkv=1, G=2, D=64, dtype="bf16", by=100.0)
    c.check(*c.call(lib))


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_a_nan_query_spoils_its_own_row_only(lib, dtype):
    c = Case([500, 30], 1, Hkv=2, G=4, D=128, dtype=dtype)
    for d in (c, Case([500, 30], 3, Hkv=2, G=20, D=128, dtype=dtype)):
        nan_query(lib, d)


def nan_query(lib, c):
    want, want_lse = c.call(lib)
    c.q[0, 0, 2, 5] = float("nan")
    out, lse = c.call(lib)
    assert out[0, 0, 2].isnan().all() and lse[0, 0, 2].isnan()
    keep = torch.ones_like(lse, dtype=torch.bool)
    keep[0, 0, 2] = False
    assert torch.equal(out[keep], want[keep]) and torch.equal(lse[keep], want_lse[keep])


def test_pages_out_of_range_are_left_out_and_reported(lib):
    c = Case([300, 200], 1, Hkv=2, G=4, D=64, dtype="f16")
    P = c.pools[0].shape[0]
    for bad in (P, -1, (1 << 31) - 1, -(1 << 31)):
        st = lib.new_status("cuda")
        table = c.table.clone()
        table[0, 2] = bad
        w = torch.zeros(2, table.shape[1] * PAGE, device="cuda")
        out, lse = lib.gqa_decode(c.q, *c.pools, table, c.len_t, c.scale, status=st, weights=w)
        assert st[0] == 7
        # as if the entries of that page were not there
        k = torch.cat([c.entries(0, 0)[:128], c.entries(0, 0)[192:]])
        x = torch.einsum("hd,nhd->hn", c.q[0, 0].double(), k.repeat_interleave(4, 1)) * c.scale
        assert torch.allclose(lse[0, 0].double(), torch.logsumexp(x, -1), atol=1e-5)
        assert (w[0, 128:192] == 0).all() and torch.allclose(w[0].sum(), torch.tensor(8.0, device="cuda"), atol=1e-4)
    # a length beyond the table
    st = lib.new_status("cuda")
    longer = c.len_t + torch.tensor([0, 10_000_000], device="cuda", dtype=torch.int32)
    out, lse = lib.gqa_decode(c.q, *c.pools, c.table, longer, c.scale, status=st)
    assert st[0] == 7
    st.zero_()
    out, lse = lib.gqa_decode(c.q, *c.pools, c.table, torch.tensor([-5, 200], device="cuda", dtype=torch.int32), c.scale, status=st)
    assert st[0] == 0 and (out[0] == 0).all() and torch.isneginf(lse[0]).all()


@pytest.mark.parametrize("width", [0, 400])
@pytest.mark.parametrize("G,dtype", [(4, "f16"), (4, "e4m3"), (40, "f16"), (40, "e4m3")])
def test_a_wait_that_runs_out(lib, G, dtype, width):
    c = Case([3000, 200], 1, Hkv=2, G=G, D=64, dtype=dtype, width=width)
    st = lib.new_status("cuda")
    lib.LIB.dsv4_debug_set_wait(200_000, 1)
    try:
        c.call(lib, status=st)
        torch.cuda.synchronize()
    finally:
        lib.LIB.dsv4_debug_set_wait(0, -1)
    assert st[0] == 1
    st.zero_()
    c.check(*c.call(lib, status=st))
    assert st[0] == 0


def test_captured_and_replayed_with_other_lengths(lib):
    for G in (4, 48):
        captured(lib, G)


def captured(lib, G):
    c = Case([100, 900, 64, 0], 1, Hkv=2, G=G, D=128, dtype="bf16", width=20)
    c.call(lib)
    w = torch.zeros(4, c.table.shape[1] * PAGE, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = c.call(lib, weights=w)
    w.zero_()
    graph.replay()
    first = w.clone()
    c.check(out, lse, w, torch.zeros_like(w))
    d = Case([333, 1, 1280, 77], 1, Hkv=2, G=G, D=128, dtype="bf16", seed=9, width=20)
    assert d.table.shape == c.table.shape
    for to, of in ((c.q, d.q), (c.len_t, d.len_t), (c.table, d.table), (c.pools[0].view(torch.int16), d.pools[0].view(torch.int16)), (c.pools[1].view(torch.int16), d.pools[1].view(torch.int16))):
        to.copy_(of)
    w.zero_()
    graph.replay()
    d.check(out, lse, w, torch.zeros_like(w))
    assert not torch.equal(first, w)


def test_two_streams_at_once(lib):
    cases = [Case([5000, 3], 1, Hkv=4, G=4, D=128, dtype="bf16", seed=i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _, (c, s) in itertools.product(range(5), zip(cases, streams)):
        with torch.cuda.stream(s):
            got.append((c, c.call(lib)))
    torch.cuda.synchronize()
    for c, r in got:
        c.check(*r)


def test_offsets_beyond_32_bits(lib):
    """A pool of more than 2^32 bytes each for K and V, read at its end."""
    P, Hkv, D = 70_000, 8, 64                        # 4.6 GB a pool
    pools = [torch.zeros(P, PAGE, Hkv, D, device="cuda", dtype=torch.bfloat16) for _ in "kv"]
    c = Case([100, 640], 1, Hkv=Hkv, G=2, D=D, dtype="bf16")
    n = c.pools[0].shape[0]
    for big, small in zip(pools, c.pools):
        big[P - n:] = small
    c.pools = pools
    c.table = torch.where(c.table >= 0, c.table + (P - n), c.table)
    c.check(*c.call(lib))


def test_prefill_small(lib):
    for dtype, D in (("bf16", 128), ("f16", 64), ("e4m3", 128), ("bf16", 256)):
        for window, first in ((0, 0), (40, 3)):
            c = Case([5, 70, 200, 1, 300], [5, 6, 150, 1, 0], Hkv=2, G=3, D=D, dtype=dtype, packed=True, window=window, first=first, sink=True)
            c.check(*c.call(lib))


def test_refusals(lib):
    """What is not a call says so, and launches nothing."""
    c = Case([100, 65], 1, Hkv=2, G=4, D=128, dtype="bf16")
    q, k, v, table, n = c.q, *c.pools, c.table, c.len_t
    w = torch.zeros(2, table.shape[1] * PAGE, device="cuda")
    ok = dict(q=q, k_pool=k, v_pool=v, block_table=table, kv_len=n, sm_scale=0.1)

    def refused(what, **kw):
        with pytest.raises((ValueError, lib.Dsv4Error), match=what):
            lib.gqa_decode(**dict(ok, **kw))
    refused("q must be \\[B, T", q=q[0])
    refused("bf16 or f16", q=q.float())
    refused("strides of q", q=torch.zeros(2, 1, 8, 132, device="cuda", dtype=torch.bfloat16)[..., :128])
    refused("16-byte", q=torch.zeros(2 * 1024 + 1, device="cuda", dtype=torch.bfloat16)[1:].reshape(2, 1, 8, 128))
    refused("head_dim", q=q[..., :64])
    refused("multiple of the pools'", q=q[:, :, :7])
    refused("kv_len must be", kv_len=n[:1])
    refused("int32", kv_len=n.long())
    refused("block_table", block_table=table[:1])
    refused("one shape", v_pool=v[:1])
    refused("contiguous", k_pool=k.transpose(1, 2))
    refused("pools must be", k_pool=k.half(), v_pool=v.half())
    refused("k_scale goes with", k_scale=torch.ones(2, device="cuda"))
    refused("k_scale goes with", k_pool=k.to(torch.float8_e4m3fn), v_pool=v.to(torch.float8_e4m3fn))
    refused("sm_scale", sm_scale=0.0)
    refused("sm_scale", sm_scale=float("inf"))
    refused("sm_scale", sm_scale=float("nan"))
    refused("window", window=-1)
    refused("first", first=1 << 31)
    refused("max_len", max_len=-1)
    refused("attn_sink", attn_sink=torch.zeros(7, device="cuda"))
    refused("weights", weights=w[:, :-1])
    refused("out must", out=torch.empty(2, 1, 8, 64, device="cuda", dtype=torch.bfloat16))
    refused("lse must", lse=torch.empty(2, 8, device="cuda"))
    refused("status", status=torch.zeros(2, device="cuda", dtype=torch.int32))
    x = torch.zeros(2, PAGE, 2, 96, device="cuda", dtype=torch.bfloat16)
    refused("64, 128 or 256", q=q[..., :96].contiguous(), k_pool=x, v_pool=x)
    with pytest.raises(ValueError, match="q_start must be"):
        lib.gqa_prefill(q[:, 0], torch.zeros(2, device="cuda", dtype=torch.int32), k, v, table, n, 0.1)
    with pytest.raises(ValueError, match="n_rows goes with"):
        lib.gqa_insert(k[:2, 0], v[:2, 0], k, v, table, n, q_start=torch.zeros(3, device="cuda", dtype=torch.int32), n_rows=n)
    with pytest.raises(ValueError, match="heads and head_dim"):
        lib.gqa_insert(q[:, :, :1], q[:, :, :1], k, v, table, n)
    refs = torch.ones(k.shape[0], device="cuda", dtype=torch.int32)
    for match, kw in (("keep must be", dict(keep=-1)), ("first must be", dict(first=-1)), ("weights must be", dict(weights=w[:, 1:])), ("pools must be", dict(pools=())),
                      ("16 bytes", dict(pools=torch.zeros(1, k.shape[0], PAGE, 7, device="cuda", dtype=torch.bfloat16))), ("page_refs", dict(page_refs=refs.long())),
                      ("a pool must be|pools must be", dict(pools=(k, v))), ("new_len", dict(new_len=n.long()))):
        a = dict(dict(pools=(k[None], v[None]), block_table=table, kv_len=n, page_refs=refs, weights=w, keep=10), **kw)
        with pytest.raises(ValueError, match=match):
            lib.kv_evict(**a)
    c.check(*c.call(lib))
