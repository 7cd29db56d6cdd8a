"""Prompts over an 8-bit cache whose tables have room for far more than the requests hold: the same results as over narrow ones, in rounds of requests and of heads, and with max_len.
Run with `-m gpu` on a B200."""
import ctypes

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


def widened(c, width):
    wide = torch.full((c.B, width), -1, device="cuda", dtype=torch.int32)
    wide[:, :c.table.shape[1]] = c.table
    c.table = wide


def copies(lib, c):
    """The call, over a wide table, has 16-bit copies of pages in its workspace: the prompts' kernel runs, which rounds weights to the queries' type; the other one, which few tokens in many rounds take, to FP16."""
    p = lib._lib.GqaParams(B=c.B, Hkv=c.Hkv, G=c.G, D=c.D, max_pages=c.table.shape[1], window=c.window, first=c.first, q_dtype=1, kv_dtype=3, sm_scale=1.0, rows=c.start[-1], num_pages=1,
                           q_stride_t=c.H * c.D, q_stride_h=c.D, q_start=4096)
    return lib.LIB.dsv4_gqa_workspace_bytes(ctypes.byref(p)) > 64 << 20          # (the other's parts: 40 MB with heads of 256)


# of 4 GiB a request takes 0.24, 0.49, 1.2 or 2.4 times as much with heads of 256, half of that with heads of 128
@pytest.mark.parametrize("width", [2000, 4000, 10_000, 20_000])
@pytest.mark.parametrize("D,window", [(256, 0), (256, 90), (128, 0)])
def test_wide_tables(lib, width, D, window):
    st = lib.new_status("cuda")
    c = Case([700, 5, 640, 300, 900], [700, 5, 333, 300, 70], Hkv=8, G=2, D=D, dtype="e4m3", packed=True, window=window, first=3 if window else 0, sink=True, seed=width)
    want, want_lse = c.call(lib, status=st)
    c.check(want, want_lse)
    widened(c, width)
    out, lse = c.call(lib, status=st)
    c.check(out, lse)
    if copies(lib, c):
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    out, lse = c.call(lib, status=st, max_len=901)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    assert st.tolist() == [0, 0, 0, 0]
    # a request of a later round is reported by its own number
    right = c.len_t.clone()
    c.len_t[4] += 64 * width
    out, lse = c.call(lib, status=st)
    assert st[0] == 7 and st[3] == 4
    c.len_t.copy_(right)
    out[1338:], lse[1338:] = want[1338:], want_lse[1338:]
    c.check(out, lse)


@pytest.mark.parametrize("width,D,Hkv,window", [(20_000, 128, 8, 0), (9000, 256, 8, 700), (3000, 64, 100, 0), (300_000, 64, 5, 0)])
def test_rounds_of_heads(lib, width, D, Hkv, window):
    """A request whose table alone has room for more than 4 GiB of copies; where a head's alone has (300,000 pages x 64 entries x 64 elements x 4 bytes: 4.9 GB), the other kernel runs."""
    c = Case([1500, 1400], [1500, 1300], Hkv=Hkv, G=16 if Hkv < 20 else 4, D=D, dtype="e4m3", packed=True, window=window, seed=D)
    want, want_lse = c.call(lib)
    assert width * 64 * Hkv * D * 4 > 1 << 32
    widened(c, width)
    ours = width * 64 * D * 4 <= 1 << 32
    assert copies(lib, c) == ours
    st = lib.new_status("cuda")
    out, lse = c.call(lib, status=st)
    assert st.tolist() == [0, 0, 0, 0]
    assert not ours or (torch.equal(out, want) and torch.equal(lse, want_lse))
    c.check(out, lse)


def test_lengths_beyond_max_len(lib):
    c = Case([700, 640], [600, 600], Hkv=8, G=2, D=64, dtype="e4m3", packed=True)
    want, want_lse = c.call(lib)
    st = lib.new_status("cuda")
    out, lse = c.call(lib, status=st, max_len=640)
    assert st[0] == 7 and out.isfinite().all()
    assert torch.equal(out[600:], want[600:]) and torch.equal(out[:540], want[:540]) and torch.equal(lse[600:], want_lse[600:])      # tokens whose entries lie below it


def test_captured_in_rounds(lib):
    c = Case([700, 640, 300], [700, 333, 300], Hkv=8, G=2, D=256, dtype="e4m3", packed=True)
    want, want_lse = c.call(lib)
    widened(c, 6000)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = c.call(lib)
    for _ in range(2):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_not_over_16_bits(lib):
    """max_len steers nothing that a 16-bit cache's prompts are right by."""
    c = Case([700, 640], [600, 600], Hkv=4, G=2, D=128, dtype="bf16", packed=True)
    st = lib.new_status("cuda")
    c.check(*c.call(lib, status=st, max_len=700))
    assert st[0] == 0
