"""Eviction refuses pools that overlap: without a GPU, before anything is launched."""
import ctypes

import pytest

torch = pytest.importorskip("torch")
INVALID = 1
SIZE = 2 * 8 * 64 * 256                                                     # of a pool: two layers of eight pages


@pytest.fixture(scope="module")
def lib():
    from dsv4_attn_b200 import _lib, build
    build.build(quiet=True)
    return _lib


@pytest.mark.parametrize("at", [[0, 0], [0, SIZE - 256], [SIZE - 16, 0], [0, SIZE, 2 * SIZE, SIZE + 16], [0, 2 * SIZE, SIZE, 0]])
def test_pools_that_overlap(lib, at):
    p = lib.KvEvictParams(B=2, max_pages=4, pools=len(at), keep=10, num_pages=8, layers=2, block_table=4096, kv_len=4096, refs=4096, weights=4096, weight_stride=256, new_table=4096,
                          new_len=4096, new_refs=4096, new_weights=4096, kept=4096, scratch=4096)
    for i, x in enumerate(at):
        p.pool[i], p.entry_bytes[i] = (1 << 40) + x, 256
    assert lib.LIB.dsv4_kv_evict(ctypes.byref(p), None) == INVALID


@pytest.mark.gpu
def test_the_python_call_says_so_and_takes_neighbours():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import dsv4_attn_b200 as d
    both = torch.randn(2, 1, 3, 64, 16, device="cuda").half()
    table, n, refs = torch.tensor([[0, 2]], device="cuda", dtype=torch.int32), torch.tensor([100], device="cuda", dtype=torch.int32), torch.ones(3, device="cuda", dtype=torch.int32)
    w = torch.rand(1, 128, device="cuda")
    before = both.clone()
    for pools in ((both[0], both[0]), (both[0], both[1], both[0])):
        with pytest.raises(ValueError, match="must not overlap"):
            d.kv_evict(pools, table, n, refs, w, 50)
    assert torch.equal(both, before)
    *_, kept = d.kv_evict((both[1], both[0]), table, n, refs, w, 50)
    j = kept[0, :50].long()
    for x, y in zip(both, before):
        assert torch.equal(x[0, 0, :50], y[0][table[0, j // 64].long(), j % 64])
