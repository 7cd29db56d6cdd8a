"""Forks and compactions of pools that their planning block goes through in several chunks, against a restatement with tensors and loops.  Run with `-m gpu` on a
B200.  Bytes and counts: everything has to be equal."""
import re
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

SOURCE = (Path(__file__).resolve().parents[1] / "dsv4_attn_b200" / "csrc" / "kv_pages.cuh").read_text()
THREADS = int(re.search(r"constexpr int kPagesPlanThreads = (\d+);", SOURCE)[1])
CHUNK = THREADS * int(re.search(r"constexpr int kPlanPages = (\d+),", SOURCE)[1])            # pages that the planner looks at together


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import dsv4_attn_b200 as d
    return d


def i32(x):
    return torch.as_tensor(x, device="cuda").to(torch.int32).contiguous()


def marked_pool(P):
    """A pool whose pages all differ, in every byte from their neighbours and in the first four from all."""
    pool = torch.empty(1, P, 64, 656, dtype=torch.uint8, device="cuda")
    pool[0] = (torch.arange(P, device="cuda") % 251).to(torch.uint8)[:, None, None]
    pool[0, :, 0, :4] = torch.arange(P, dtype=torch.int32, device="cuda").view(torch.uint8).view(P, 4)
    return pool


def live_pages(P, pattern, gen):
    at = torch.arange(P, device="cuda")
    return dict(half=lambda: torch.rand(P, device="cuda", generator=gen) < 0.5, few=lambda: torch.rand(P, device="cuda", generator=gen) < 0.01,
                most=lambda: torch.rand(P, device="cuda", generator=gen) < 0.99,
                ends=lambda: (at >= CHUNK // 2) & (at < CHUNK) | (at >= P - CHUNK),              # holes in the first chunk, pages that move in the last ones
                border=lambda: (at >= 5) & (at < CHUNK) | (at >= P - 5),                         # as many as a chunk has
                none=lambda: at < 0, all=lambda: at >= 0)[pattern]()


@pytest.mark.parametrize("pattern", ["half", "few", "most", "ends", "border", "none", "all"])
@pytest.mark.parametrize("P", [CHUNK, CHUNK + 1, 2 * CHUNK + CHUNK // 2 + 1])
@pytest.mark.parametrize("in_place,offset", [(False, 0), (True, 0), (True, 1)])
def test_compaction_over_chunks(lib, P, pattern, in_place, offset):
    """offset: the counts begin off a 16-byte boundary."""
    gen = torch.Generator(device="cuda").manual_seed(P)
    live = live_pages(P, pattern, gen)
    refs = torch.zeros(P + offset, dtype=torch.int32, device="cuda")[offset:]
    refs.copy_(torch.where(live, torch.randint(1, 9, (P,), device="cuda", generator=gen), -torch.randint(0, 2, (P,), device="cuda", generator=gen)))
    at = torch.arange(P, device="cuda")
    count = int(live.sum())
    src, dst = torch.nonzero(live & (at >= count))[:, 0], torch.nonzero(~live & (at < count))[:, 0]
    to = at.clone()
    to[src] = dst
    table = i32(torch.where(torch.rand(P, device="cuda", generator=gen) < 0.9, torch.randperm(P, device="cuda", generator=gen), -1)).view(1, P)
    pool = marked_pool(P)
    want_pool, want_refs = pool.clone(), refs.clone()
    want_pool[0, dst] = pool[0, src]
    want_refs[dst] = refs[src]
    want_refs[src] = 0
    want_table = torch.where(table >= 0, to[table.clamp(min=0).long()].int(), table)
    got = lib.kv_pages_compact(pool, table, refs, new_table=table, new_refs=refs) if in_place else lib.kv_pages_compact(pool, table, refs)
    assert got[2].tolist() == [count]
    assert torch.equal(got[0], want_table) and torch.equal(got[1], want_refs) and torch.equal(pool, want_pool)


@pytest.mark.parametrize("free", [(1100, 700, 900), (0, 0, 2700), (2600, 0, 50), (1024, 1024, 1024), (1100, 700, 500), (3, 0, 0)])
@pytest.mark.parametrize("offset", [0, 1])
def test_forks_over_chunks(lib, free, offset):
    """More children than the planner has threads, with so many free pages in each of three chunks: enough, and too few (the last children get none)."""
    P, parents, children = 2 * CHUNK + CHUNK // 2 + 1, 900, 2 * THREADS + 452
    gen = torch.Generator(device="cuda").manual_seed(sum(free))
    is_free = torch.zeros(P, dtype=torch.bool, device="cuda")
    for c, n in enumerate(free):
        size = min(CHUNK, P - c * CHUNK)
        is_free[c * CHUNK + torch.randperm(size, device="cuda", generator=gen)[:n]] = True
    refs = torch.zeros(P + offset, dtype=torch.int32, device="cuda")[offset:]
    refs.copy_((~is_free).int())
    held = torch.nonzero(~is_free)[:, 0]
    held = held[torch.randperm(held.numel(), device="cuda", generator=gen)[:2 * parents]].view(parents, 2)
    table = torch.full((parents + children, 3), -1, dtype=torch.int32, device="cuda")
    table[:parents, :2] = held
    kv_len = torch.zeros(parents + children, dtype=torch.int32, device="cuda")
    kv_len[:parents] = torch.tensor([70, 64, 127, 3, 128], device="cuda", dtype=torch.int32).repeat(parents // 5)
    parent, child = torch.randint(0, parents, (children,), device="cuda", generator=gen), parents + torch.randperm(children, device="cuda", generator=gen)
    pool = marked_pool(P)
    want_pool, want_table, want_len, want_refs = pool.clone(), table.tolist(), kv_len.tolist(), refs.tolist()
    left, short, moves = torch.nonzero(is_free)[:, 0].tolist()[::-1], False, []
    for p, c in zip(parent.tolist(), child.tolist()):
        full, rest = want_len[p] // 64, want_len[p] % 64
        row = want_table[p][:full]
        for q in row:
            want_refs[q] += 1
        want_len[c] = want_len[p]
        if rest and left:
            q = left.pop()
            want_refs[q] = 1
            moves.append((want_table[p][full], q, rest))
            row = row + [q]
        elif rest:
            short, want_len[c] = True, full * 64
        want_table[c] = row + [-1] * (3 - len(row))
    for rest in {r for _, _, r in moves}:
        s, q = i32([m[0] for m in moves if m[2] == rest]).long(), i32([m[1] for m in moves if m[2] == rest]).long()
        want_pool[0, q, :rest] = pool[0, s, :rest]
    st = lib.new_status("cuda")
    lib.kv_pages_fork(pool, table, kv_len, refs, i32(parent), i32(child), status=st)
    assert st[0].item() == (10 if short else 0)
    assert table.tolist() == want_table and kv_len.tolist() == want_len and refs.tolist() == want_refs and torch.equal(pool, want_pool)
