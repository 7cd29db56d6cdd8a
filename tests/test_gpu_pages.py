"""Pages of the cache (kv_pages_copy / fork / free / compact, kv_entries_move) against a restatement with loops on the host.  Run with `-m gpu` on
a B200.  Bytes and counts: everything has to be equal."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import dsv4_attn_b200 as d
    return d


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Cache:
    """A cache on the device and the same on the host."""

    def __init__(self, seed, L, P, B, width, lengths):
        rng = np.random.default_rng(seed)
        self.pool = rng.integers(0, 256, (L, P, 64, 656), dtype=np.uint8)
        self.table = np.full((B, width), -1, np.int32)
        self.lens = np.array(lengths, np.int32)
        self.refs = np.zeros(P, np.int32)
        order = rng.permutation(P)
        at = 0
        for b, n in enumerate(lengths):
            for i in range((n + 63) // 64):
                self.table[b, i] = order[at]
                self.refs[order[at]] = 1
                at += 1
        self.d = [torch.from_numpy(x.copy()).cuda() for x in (self.pool, self.table, self.lens, self.refs)]

    def free(self, requests):
        for r in requests:
            if r < 0:
                continue
            for i in range((self.lens[r] + 63) // 64):
                if self.table[r, i] >= 0:
                    self.refs[self.table[r, i]] -= 1
            self.table[r] = -1
            self.lens[r] = 0

    def fork(self, parents, children):
        took, short = [], False
        free = [p for p in range(len(self.refs)) if self.refs[p] <= 0]
        for p, c in zip(parents, children):
            if p < 0 or c < 0:
                continue
            n = int(self.lens[p])
            full, rest = n // 64, n % 64
            self.table[c] = -1
            self.table[c, :full] = self.table[p, :full]
            for q in self.table[p, :full]:
                self.refs[q] += 1
            if rest and free:
                q = free.pop(0)
                took.append(q)
                self.refs[q] = 1
                self.table[c, full] = q
                self.pool[:, q, :rest] = self.pool[:, self.table[p, full], :rest]
            elif rest:
                short, n = True, full * 64
            self.lens[c] = n
        return short

    def compact(self):
        live = int((self.refs > 0).sum())
        movers = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        holes = [p for p in range(live) if self.refs[p] <= 0]
        to = np.arange(len(self.refs))
        for s, d in zip(movers, holes):
            to[s] = d
            self.pool[:, d] = self.pool[:, s]
            self.refs[d], self.refs[s] = self.refs[s], 0
        self.table = np.where(self.table >= 0, to[np.maximum(self.table, 0)], self.table).astype(np.int32)
        return live

    def check(self, got=None):
        torch.cuda.synchronize()
        for want, have in zip((self.pool, self.table, self.lens, self.refs), got or self.d):
            assert np.array_equal(want, have.cpu().numpy())


# lengths with pages that end inside, exactly at, and one past a page; none; one entry
LENGTHS = [130, 64, 0, 1, 65, 63, 128, 200]


@pytest.mark.parametrize("L", [1, 3])
def test_free_and_fork(lib, L):
    c = Cache(1, L, 40, 8, 4, LENGTHS)
    pool, table, lens, refs = c.d
    st = lib.new_status("cuda")
    lib.kv_pages_free(table, lens, refs, i32([3, -1, 6, 4]), status=st)
    c.free([3, 6, 4])
    c.check()
    # one parent of two children, an empty parent, a parent of full pages only, items left out
    lib.kv_pages_fork(pool if L > 1 else pool[0], table, lens, refs, i32([0, 2, 0, -1, 1]), i32([3, 4, 6, 5, -1]), status=st)
    assert not c.fork([0, 2, 0, -1, 1], [3, 4, 6, 5, -1])
    c.check()
    # freeing a parent leaves the children's shared pages alive, whose forks fork again
    lib.kv_pages_free(table, lens, refs, i32([0, 4]))
    c.free([0, 4])
    lib.kv_pages_fork(pool, table, lens, refs, i32([3, 7]), i32([0, 4]), status=st)
    c.fork([3, 7], [0, 4])
    c.check()
    assert st.tolist() == [0, 0, 0, 0]


def test_many_children_and_pages(lib):
    """More children than the planner's block has threads, and free pages all over a pool of several rounds of it."""
    B = 2500
    c = Cache(2, 1, 9000, B, 2, [70] * 1200 + [0] * (B - 1200))
    parents = [i % 1200 for i in range(B - 1200)]
    children = list(range(1200, B))
    pool, table, lens, refs = c.d
    lib.kv_pages_fork(pool, table, lens, refs, i32(parents), i32(children))
    c.fork(parents, children)
    c.check()


def test_no_free_page(lib):
    c = Cache(3, 2, 4, 4, 3, [130, 0, 0, 0])            # three pages in use, one free
    pool, table, lens, refs = c.d
    st = lib.new_status("cuda")
    lib.kv_pages_fork(pool, table, lens, refs, i32([0, 0, 0]), i32([1, 2, 3]), status=st)
    assert c.fork([0, 0, 0], [1, 2, 3])
    c.check()
    assert st[0].item() == 10 and c.lens.tolist() == [130, 130, 128, 128]


@pytest.mark.parametrize("L,P,seed", [(1, 1, 0), (2, 37, 1), (1, 4100, 2), (3, 64, 3)])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(lib, L, P, seed, in_place):
    rng = np.random.default_rng(seed)
    B, width = 12, 5
    lengths, left = [], P
    for b in range(B):
        n = int(rng.integers(0, min(left, width) * 64 + 1))
        lengths.append(n)
        left -= (n + 63) // 64
    c = Cache(10 + seed, L, P, B, width, lengths)
    pool, table, lens, refs = c.d
    lib.kv_pages_free(table, lens, refs, i32([1, 5, 7]))
    c.free([1, 5, 7])
    before = [t.clone() for t in (table, refs)]
    if in_place:
        new_table, new_refs, count = lib.kv_pages_compact(pool, table, refs, new_table=table, new_refs=refs)
        assert new_table is table and new_refs is refs
    else:
        new_table, new_refs, count = lib.kv_pages_compact(pool, table, refs)
        assert torch.equal(table, before[0]) and torch.equal(refs, before[1])
    assert count.tolist() == [c.compact()]
    c.check([pool, new_table, lens, new_refs])
    # nothing is left to move
    again = lib.kv_pages_compact(pool, new_table, new_refs)
    c.check([pool, again[0], lens, again[1]])


def test_copy_and_move(lib):
    c = Cache(4, 3, 20, 1, 1, [0])
    pool = c.d[0]
    lib.kv_pages_copy(pool, i32([3, -1, 19, 0]), i32([4, 5, 1, -1]))
    c.pool[:, 4], c.pool[:, 1] = c.pool[:, 3], c.pool[:, 19]
    c.check()
    lib.kv_entries_move(pool, i32([0, 63, -1, 1279]), i32([64, 130, 7, 2]))
    flat = c.pool.reshape(3, -1, 656)
    flat[:, [64, 130, 2]] = flat[:, [0, 63, 1279]]
    c.check()
    lib.kv_entries_move(pool[1], i32([5]), i32([6]))
    flat[1, 6] = flat[1, 5]
    c.check()
    for f in (lib.kv_pages_copy, lib.kv_entries_move):
        f(pool, i32([]), i32([]))
    c.check()


def test_offsets_beyond_32_bits(lib):
    """A pool of more than 4 GiB: its last page is copied to, and moved from, places before and behind that border."""
    P = 103_000                                          # 4.3 GB
    pool = torch.zeros(1, P, 64, 656, dtype=torch.uint8, device="cuda")
    pool[0, P - 1] = torch.arange(64, device="cuda", dtype=torch.uint8)[:, None]
    pool[0, 0] = 200
    lib.kv_pages_copy(pool, i32([P - 1, 0]), i32([7, P - 2]))
    lib.kv_entries_move(pool, i32([P * 64 - 1]), i32([9 * 64 + 5]))
    assert torch.equal(pool[0, 7], pool[0, P - 1]) and (pool[0, P - 2] == 200).all() and (pool[0, 9, 5] == 63).all()
    assert int(pool.sum(dtype=torch.int64)) == 64 * 656 * 400 + 2 * 656 * 2016 + 656 * 63


def test_numbers_out_of_range_are_reported(lib):
    c = Cache(5, 2, 10, 3, 2, [100, 64, 0])
    pool, table, lens, refs = c.d
    for call in (lambda st: lib.kv_pages_copy(pool, i32([10]), i32([0]), status=st), lambda st: lib.kv_pages_copy(pool, i32([0]), i32([10]), status=st),
                 lambda st: lib.kv_entries_move(pool, i32([640]), i32([0]), status=st), lambda st: lib.kv_pages_free(table, lens, refs, i32([3]), status=st),
                 lambda st: lib.kv_pages_fork(pool, table, lens, refs, i32([0]), i32([3]), status=st)):
        st = lib.new_status("cuda")
        call(st)
        c.check()
        assert st[0].item() == 7


def test_fork_and_free_replay_from_a_graph(lib):
    c = Cache(6, 2, 40, 8, 4, LENGTHS)
    pool, table, lens, refs = c.d
    parents, children = i32([0, 7, 1]), i32([4, 5, 6])
    lib.kv_pages_free(table, lens, refs, children)
    torch.cuda.synchronize()
    c.free([4, 5, 6])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        lib.kv_pages_free(table, lens, refs, children)
        lib.kv_pages_fork(pool, table, lens, refs, parents, children)
    for _ in range(3):
        g.replay()
        c.free([4, 5, 6])
        c.fork([0, 7, 1], [4, 5, 6])
    c.check()


def test_refusals(lib):
    c = Cache(7, 1, 10, 3, 2, [100, 64, 0])
    pool, table, lens, refs = c.d
    one = i32([0])
    for call in (lambda: lib.kv_pages_copy(pool[..., :640].contiguous(), one, one), lambda: lib.kv_pages_copy(pool, one, i32([0, 1])),
                 lambda: lib.kv_pages_copy(pool, one.long(), one), lambda: lib.kv_pages_copy(pool.cpu(), one, one), lambda: lib.kv_pages_copy(pool[:, ::2], one, one),
                 lambda: lib.kv_entries_move(pool.float(), one, one), lambda: lib.kv_pages_free(table, lens[:2], refs, one), lambda: lib.kv_pages_free(table.long(), lens, refs, one),
                 lambda: lib.kv_pages_fork(pool, table, lens, refs[:9], one, one), lambda: lib.kv_pages_fork(pool, table.t(), lens, refs, one, one),
                 lambda: lib.kv_pages_fork(pool, table, lens, refs, one, one, status=torch.zeros(3, dtype=torch.int32, device="cuda")),
                 lambda: lib.kv_pages_compact(pool, table, refs[:9]), lambda: lib.kv_pages_compact(pool, table, refs, new_table=table[:2]),
                 lambda: lib.kv_pages_compact(pool, table, refs, workspace=one)):
        with pytest.raises(ValueError):
            call()
    c.check()
