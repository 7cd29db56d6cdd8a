"""Moves whose lists overlap (kv_entries_move: all entries are read before any is written), and copies whose lists do (kv_pages_copy: reported).  Run with
`-m gpu` on a B200.  Bytes: everything has to be equal."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import dsv4_attn_b200 as d
    return d


def filled(*shape, seed=0):
    return torch.randint(0, 256, (*shape, 656), dtype=torch.uint8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def i32(x):
    return torch.as_tensor(x, device="cuda").to(torch.int32).contiguous()


def moved(items, src, dst):
    """items [layers, count, ...]: gathered, then scattered."""
    take = (src >= 0) & (dst >= 0)
    out = items.clone()
    out[:, dst[take].long()] = items[:, src[take].long()]
    return out


@pytest.mark.parametrize("layers", [1, 3])
def test_accepted_rows_close_up(lib, layers):
    """Nodes 0, 2 and 3 of six drafts behind five committed rows go to the places of nodes 0, 1 and 2."""
    B, W = 7, 11
    win = filled(layers, B, W)
    first = torch.arange(B, device="cuda")[:, None] * W + 5
    src, dst = i32((first + torch.tensor([0, 2, 3], device="cuda")).reshape(-1)), i32((first + torch.tensor([0, 1, 2], device="cuda")).reshape(-1))
    want = moved(win.view(layers, B * W, 656), src, dst)
    lib.kv_entries_move(win, src, dst)
    assert torch.equal(win.view(layers, B * W, 656), want)


# the number of items at which one way of copying takes over from another, on both sides
@pytest.mark.parametrize("B,W,by", [(1, 2, 1), (4, 128, 3), (4, 129, 1), (5, 133, 7), (64, 136, 5), (112, 129, 1)])
def test_windows_slide(lib, B, W, by):
    """Every window moves `by` rows towards its front: all rows but the last are in both lists, in any order of the items."""
    layers = 2
    win = filled(layers, B, W, seed=B)
    rows = torch.arange(B * W, device="cuda").view(B, W)
    order = torch.randperm(B * (W - by), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    src, dst = i32(rows[:, by:].reshape(-1)[order]), i32(rows[:, :W - by].reshape(-1)[order])
    st = lib.new_status("cuda")
    want = moved(win.view(layers, B * W, 656), src, dst)
    lib.kv_entries_move(win, src, dst, status=st)
    assert torch.equal(win.view(layers, B * W, 656), want) and st.tolist() == [0, 0, 0, 0]
    back = moved(want, dst, src)
    lib.kv_entries_move(win, dst, src)
    assert torch.equal(win.view(layers, B * W, 656), back)


@pytest.mark.parametrize("n", [1, 2, 31, 513, 2048, 2049, 4096, 4097, 16384])
def test_entries_change_places(lib, n):
    """A permutation (cycles of every length, entries that stay where they are), with items left out between."""
    g = torch.Generator(device="cuda").manual_seed(n)
    items = filled(2, n + 5, seed=n)
    src, dst = i32(torch.randperm(n, device="cuda", generator=g)), i32(torch.randperm(n, device="cuda", generator=g))
    src[n // 2] = -1
    want = moved(items, src, dst)
    lib.kv_entries_move(items[:, None], src, dst)
    assert torch.equal(items, want)


@pytest.mark.parametrize("P,n", [(3, 1), (7000, 2), (7000, 2049), (132_000, 2048), (132_000, 2049)])
def test_a_page_in_both_lists_is_reported(lib, P, n):
    """Found by a table for few pages of a large pool, else by bits of 131,072 pages at a time.  (The page that is in both goes to itself.)"""
    pool = torch.zeros(1, P, 64, 656, dtype=torch.uint8, device="cuda")
    order = torch.randperm(P, device="cuda", generator=torch.Generator(device="cuda").manual_seed(n))
    pool[0, order[:n], 5] = filled(n, seed=n)
    src, dst = order[:n].clone(), order[n:2 * n].clone()
    for at in (None, 0, P - 1, 131_071, 131_072):
        s, d = src.clone(), dst.clone()
        if at is not None:
            if at >= P:
                continue
            s[s == at], d[d == at] = -1, -1
            s[n // 2] = d[n // 2] = at
        st = lib.new_status("cuda")
        take = (s >= 0) & (d >= 0)
        want = pool[0, :, 5].clone()
        want[d[take]] = want[s[take]]
        lib.kv_pages_copy(pool, i32(s), i32(d), status=st)
        assert st[0].item() == (0 if at is None else 11) and torch.equal(pool[0, :, 5], want)


def test_a_list_too_long_to_overlap(lib):
    """Beyond 16,384 items lists that overlap are reported and left alone, others are copied."""
    n = 16385
    items = filled(1, 2 * n)
    before = items.clone()
    st = lib.new_status("cuda")
    a, b = torch.arange(n, device="cuda"), torch.arange(n, device="cuda") + n
    lib.kv_entries_move(items[:, None], i32(a), i32(b - 1), status=st)
    assert st[0].item() == 11 and torch.equal(items, before)
    st = lib.new_status("cuda")
    lib.kv_entries_move(items[:, None], i32(a), i32(b), status=st)
    assert st.tolist() == [0, 0, 0, 0] and torch.equal(items, moved(before, a, b))


@pytest.mark.parametrize("n", [600, 2100])
def test_overlaps_far_apart(lib, n):
    """A pool of more entries than a block has bits for: the one entry in both lists lies in any round of them, or is found by a table."""
    E = 1_900_000
    g = torch.Generator(device="cuda").manual_seed(5)
    for at in ((1 << 19) - 1, 1 << 19, (3 << 19) - 1, 3 << 19, E - 1):
        items = torch.zeros(1, E, 656, dtype=torch.uint8, device="cuda")
        src = torch.randperm(900_000, device="cuda", generator=g)[:n]
        dst = 900_000 + torch.randperm(900_000, device="cuda", generator=g)[:n + 1]
        src, dst = src[src != at][:n - 1], dst[dst != at][:n - 1]
        src[3], dst[-1] = at, at
        items[0, src] = filled(src.numel(), seed=6)
        want = moved(items, src, dst)
        lib.kv_entries_move(items[:, None], i32(src), i32(dst))
        assert torch.equal(items, want)
        del items, want


@pytest.mark.parametrize("n", [2, 700])
@pytest.mark.parametrize("what", ["pages", "entries"])
def test_numbers_out_of_range_next_to_others(lib, what, n):
    """Reported and left out; the others are copied (entries: in lists that overlap)."""
    step = 2 if what == "pages" else 1
    count = step * n + 4
    items = filled(1, count, 64) if what == "pages" else filled(1, 1, count)
    src, dst = torch.arange(n, device="cuda") * step, torch.arange(n, device="cuda") * step + 1
    src[n - 1], dst[0] = count, count
    flat = items.view(1, count, -1, 656)
    want = moved(flat, torch.where((src < count) & (dst < count), src, -1), dst)
    st = lib.new_status("cuda")
    (lib.kv_pages_copy if what == "pages" else lib.kv_entries_move)(items, i32(src), i32(dst), status=st)
    assert st[0].item() == 7 and torch.equal(flat, want)


@pytest.mark.parametrize("layers,n", [(1, 1), (7, 5), (16, 321), (40, 1024), (61, 2049), (9, 16385)])
def test_lists_that_do_not_overlap(lib, layers, n):
    """As many entries as a warp takes at once, and several rounds of them for every warp, the last one a part of one; some left out."""
    g = torch.Generator(device="cuda").manual_seed(n)
    items = filled(layers, 1, 2 * n + 3, seed=n)
    order = torch.randperm(2 * n + 3, device="cuda", generator=g)
    src, dst = order[:n].clone(), order[n:2 * n].clone()
    src[1::5], dst[4::7] = -1, -1
    want = moved(items[:, 0], src, dst)
    st = lib.new_status("cuda")
    lib.kv_entries_move(items, i32(src), i32(dst), status=st)
    assert torch.equal(items[:, 0], want) and st.tolist() == [0, 0, 0, 0]
