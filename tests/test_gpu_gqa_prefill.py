"""Attention of prompts over K and V pages against its definition in 64 bits, at sizes that the tensor-core kernel takes.  Run with `-m gpu` on a B200."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.gqa_util import Case  # noqa: E402


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import dsv4_attn_b200 as d
    return d


def run(lib, *a, **kw):
    st = lib.new_status("cuda")
    c = Case(*a, packed=True, **kw)
    c.check(*c.call(lib, status=st))
    assert st.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_whole_prompts(lib, dtype, D):
    run(lib, [700], [700], Hkv=4, G=2, D=D, dtype=dtype, seed=D)


@pytest.mark.parametrize("Hkv,G", [(8, 1), (3, 3), (2, 5), (2, 7), (4, 8), (1, 16), (8, 32), (2, 100), (1, 128)])
def test_head_layouts(lib, Hkv, G):
    T = max(1200 // G, 70)
    run(lib, [T + 130, T], [T, T], Hkv=Hkv, G=G, D=64, dtype="f16", seed=G, sink=True)


@pytest.mark.parametrize("window,first", [(1, 0), (1, 1), (50, 3), (64, 64), (128, 200), (129, 1), (1000, 70), (1 << 30, 4), ((1 << 31) - 1, 0)])
@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("e4m3", 64), ("f16", 256)])
def test_windows(lib, window, first, dtype, D):
    run(lib, [900, 2000, 300], [900, 300, 150], Hkv=2, G=4, D=D, dtype=dtype, window=window, first=first, seed=window % 97)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_ragged_and_empty_requests(lib, D):
    run(lib, [1, 0, 64, 500, 129, 1000, 3, 65, 400], [1, 0, 64, 333, 0, 1000, 2, 65, 127], Hkv=2, G=8, D=D, dtype="bf16", seed=D)


def test_tokens_that_stand_before_the_first_entry(lib):
    """More new tokens than entries: the first of them see nothing."""
    run(lib, [100, 700], [300, 700], Hkv=4, G=2, D=64, dtype="bf16")


def test_many_short_prompts(lib):
    lens = [(i * 53) % 90 + 60 for i in range(300)]
    run(lib, [n + i % 7 * 30 for i, n in enumerate(lens)], lens, Hkv=1, G=4, D=64, dtype="f16", window=40, first=2)


def test_a_long_cache(lib):
    run(lib, [20_000], [600], Hkv=2, G=8, D=128, dtype="bf16")
    run(lib, [20_000], [600], Hkv=2, G=8, D=128, dtype="e4m3", window=5000, first=3)


def test_scores_that_grow_along_the_cache(lib):
    """Every step's maximum passes the one before by far, so that the outputs so far are rescaled again and again; and falls."""
    for down in (False, True):
        for D in (64, 128, 256):
            c = Case([1500], [1500], Hkv=2, G=2, D=D, dtype="f16", packed=True)
            n = torch.arange(1500, device="cuda")
            up = (1499 - n if down else n).half() / 1500 * 60
            c.q.fill_(0)
            c.q[:, :, 0] = 1.0
            c.q[:, :, 1:] = torch.randn(1500, 4, D - 1, device="cuda").half()
            c.pools[0][c.table[0, n // 64].long(), n % 64, :, 0] = up[:, None]
            c.scale = 1.0
            c.check(*c.call(lib))


def test_rows_of_no_request_and_bad_offsets(lib):
    c = Case([700, 300], [700, 300], Hkv=2, G=4, D=128, dtype="bf16", packed=True)
    q = torch.cat([torch.full((3, 8, 128), float("nan"), device="cuda", dtype=torch.bfloat16), c.q, torch.full((300, 8, 128), float("nan"), device="cuda", dtype=torch.bfloat16)])
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    a, kw = c.args()
    st = lib.new_status("cuda")
    lib.gqa_prefill(q, c.start_t + 3, *a, **kw, out=out, lse=lse, status=st)
    c.check(out[3:1003], lse[3:1003])
    assert st[0] == 0
    for x in (out, lse):
        assert (x[:3] == 7).all() and (x[1003:] == 7).all()
    # offsets outside the rows, that fall, that overlap: nothing outside is written, and it is reported
    for start in ([-5, 700, 2000], [0, 700, 600], [5000, 0, 700], [700, 0, 1303]):
        st.zero_()
        lib.gqa_prefill(q, torch.tensor(start, device="cuda", dtype=torch.int32), *a, **kw, out=out, lse=lse, status=st)
        assert st[0] == 7, start


def test_overlapping_offsets_of_many_requests(lib):
    c = Case([300] * 40, [300] * 40, Hkv=1, G=4, D=64, dtype="bf16", packed=True)
    start = torch.tensor([0, 12000] * 20 + [0], device="cuda", dtype=torch.int32)
    a, kw = c.args()
    st = lib.new_status("cuda")
    lib.gqa_prefill(c.q, start, *a, **kw, status=st)
    assert st[0] == 7
    st.zero_()
    c.check(*c.call(lib, status=st))
    assert st[0] == 0


def test_pages_out_of_range(lib):
    for dtype in ("bf16", "e4m3"):
        c = Case([1000], [700], Hkv=2, G=4, D=64, dtype=dtype, packed=True)
        st = lib.new_status("cuda")
        a, kw = c.args()
        table = c.table.clone()
        for bad in (-1, c.pools[0].shape[0], (1 << 31) - 1):
            st.zero_()
            table[0, 3] = bad
            out, lse = lib.gqa_prefill(c.q, c.start_t, a[0], a[1], table, *a[3:], **kw, status=st)
            assert st[0] == 7
            k = torch.cat([c.entries(0, 0)[:192], c.entries(0, 0)[256:]])
            x = torch.einsum("hd,nhd->hn", c.q[-1].double(), k.repeat_interleave(4, 1)) * c.scale
            assert torch.allclose(lse[-1].double(), torch.logsumexp(x, -1), atol=1e-5) and out.isfinite().all()
    # between the first entries and the window pages may be gone
    c = Case([5000], [700], Hkv=2, G=4, D=64, dtype="bf16", packed=True, window=100, first=5)
    c.table[0, 2:40] = -1
    st = lib.new_status("cuda")
    want = c.expected
    out, lse = c.call(lib, status=st)
    assert st[0] == 0
    c.table[0, 2:40] = 0
    c.check(out, lse)
    del want


@pytest.mark.parametrize("D", [128, 256])
def test_a_wait_that_runs_out(lib, D):
    c = Case([1500], [1500], Hkv=4, G=2, D=D, dtype="f16", packed=True)
    st = lib.new_status("cuda")
    for drop in (0, 2):
        lib.LIB.dsv4_debug_set_wait(200_000, drop)
        try:
            c.call(lib, status=st)
            torch.cuda.synchronize()
        finally:
            lib.LIB.dsv4_debug_set_wait(0, -1)
        assert st[0] == 1
        st.zero_()
        c.check(*c.call(lib, status=st))
        assert st[0] == 0


def test_fused_rows_and_heads_before_tokens(lib):
    c = Case([700, 100], [700, 100], Hkv=2, G=4, D=128, dtype="bf16", packed=True, fused=True)
    assert not c.q.is_contiguous()
    c.check(*c.call(lib))
    c.q = c.q.transpose(0, 1).contiguous().transpose(0, 1)
    c.check(*c.call(lib))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_nan_queries_and_infinite_ones(lib, dtype):
    c = Case([700], [700], Hkv=2, G=4, D=128, dtype=dtype, packed=True)
    want, want_lse = c.call(lib)
    c.q[300, 2, 5] = float("nan")
    c.q[301, 7] = float("inf")
    out, lse = c.call(lib)
    keep = torch.ones_like(lse, dtype=torch.bool)
    keep[300, 2] = keep[301, 7] = False
    assert out[300, 2].isnan().all() and lse[300, 2].isnan() and out[301, 7].isnan().all()
    assert torch.equal(out[keep], want[keep]) and torch.equal(lse[keep], want_lse[keep])


def test_captured_and_replayed(lib):
    c = Case([700, 300], [700, 300], Hkv=2, G=4, D=128, dtype="e4m3", packed=True)
    c.call(lib)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = c.call(lib)
    out.zero_()
    for _ in range(2):
        graph.replay()
    c.check(out, lse)
    d = Case([500, 640], [100, 590], Hkv=2, G=4, D=128, dtype="e4m3", packed=True, seed=5)
    # other lengths and offsets in the same buffers
    d_q = torch.zeros_like(c.q)
    d_q[:690] = d.q
    c.q.copy_(d_q)
    c.start_t.copy_(d.start_t)
    c.len_t.copy_(d.len_t)
    c.table.fill_(-1)
    c.table[:, :d.table.shape[1]] = d.table[:, :c.table.shape[1]]
    for to, of in zip(c.pools, d.pools):
        to.view(torch.uint8)[:of.shape[0]] = of.view(torch.uint8)
    for to, of in zip(c.scales, d.scales):
        to.copy_(of)
    graph.replay()
    d.check(out[:690], lse[:690])
