"""examples/draft_step.py runs and leaves its cache consistent; its calls together give what plain attention over the same entries gives.  Run with `-m gpu` on a B200."""
import importlib.util
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    path = Path(__file__).resolve().parents[1] / "examples" / "draft_step.py"
    spec = importlib.util.spec_from_file_location("draft_step", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_the_draft_example(example, dtype):
    cache, drafted, held, status = example.run(requests=5, steps=40, dtype=dtype)
    assert status.tolist() == [0, 0, 0, 0]
    assert (drafted >= 0).all() and held[-1].max() <= example.BUDGET + example.SLACK + 8 and held.max() > example.BUDGET + example.SLACK
    # every page is counted as often as the tables name it, and no request has more pages than its entries need
    named = cache.table[cache.table >= 0].long()
    assert torch.equal(torch.bincount(named, minlength=cache.refs.numel()), cache.refs.long())
    assert torch.equal((cache.table >= 0).sum(1), (cache.kv_len + 63) // 64)
    place = torch.arange(cache.weights.shape[1], device="cuda")
    there = place < cache.kv_len[:, None]
    assert (cache.weights[~there] == 0).all() and (cache.weights[there] >= 0).all()
    # entries are in the order of the text, the first and the last ones among them
    for b, n in enumerate(cache.kv_len.tolist()):
        t = cache.tokens[b, :n]
        assert (t[1:] > t[:-1]).all() and t[:example.FIRST].tolist() == list(range(example.FIRST)) and torch.equal(t[-example.RECENT:], t[-1] - example.RECENT + 1 + torch.arange(example.RECENT, device="cuda"))


def test_steps_against_plain_attention(example):
    """Insert, decode with weights and evict, step by step, beside lists of the rows that were inserted."""
    import dsv4_attn_b200 as d
    gen = torch.Generator(device="cuda").manual_seed(3)
    B, Hkv, H, D, cap = 3, 2, 8, 64, 5
    k_pool, v_pool = (torch.full((1, B * cap, 64, Hkv, D), float("nan"), device="cuda", dtype=torch.bfloat16) for _ in "kv")
    table = torch.randperm(B * cap, device="cuda", generator=gen).int().reshape(B, cap)
    refs, kv_len, weights = torch.ones(B * cap, device="cuda", dtype=torch.int32), torch.zeros(B, device="cuda", dtype=torch.int32), torch.zeros(B, cap * 64, device="cuda")
    rows, got = [[] for _ in range(B)], [[] for _ in range(B)]
    for step in range(220):
        q, k, v = (torch.randn(B, 1, n, D, device="cuda", generator=gen).bfloat16() for n in (H, Hkv, Hkv))
        d.gqa_insert(k, v, k_pool[0], v_pool[0], table, kv_len)
        kv_len = kv_len + 1
        out, lse = d.gqa_decode(2 * q, k_pool[0], v_pool[0], table, kv_len, D ** -0.5, weights=weights)
        for b in range(B):
            rows[b].append((k[b, 0], v[b, 0]))
            got[b].append(0.0)
            kk, vv = (torch.stack([r[i] for r in rows[b]]).double().repeat_interleave(H // Hkv, 1) for i in range(2))
            x = torch.einsum("hd,nhd->hn", 2 * q[b, 0].double(), kk) * D ** -0.5
            p = torch.softmax(x, -1)
            want = torch.einsum("hn,nhd->hd", p, vv)
            # weights rounded by 2^-8 of themselves, and so the output
            tol = 2.0 ** -8 * 1.02 * (torch.einsum("hn,nhd->hd", p, vv.abs()) + want.abs()) + 1e-6
            assert ((out[b, 0].double() - want).abs() <= tol).all() and torch.allclose(lse[b, 0].double(), torch.logsumexp(x, -1), atol=2e-5)
            got[b] = [g + w for g, w in zip(got[b], p.sum(0).tolist())]
        if step % 50 == 49:
            assert all(torch.allclose(weights[b, :len(got[b])].double(), torch.tensor(got[b], device="cuda", dtype=torch.float64), rtol=2e-4, atol=2e-4) for b in range(B))
            old = [w[:n].clone() for w, n in zip(weights, kv_len.tolist())]
            table, kv_len, refs, weights, kept = d.kv_evict((k_pool, v_pool), table, kv_len, refs, weights, 40, first=2, recent=10)
            for b in range(B):
                stay = kept[b, :40].tolist()
                n = len(rows[b])
                best = sorted(range(2, n - 10), key=lambda j: (-float(old[b][j]), j))[:28]
                assert stay == sorted([0, 1, *best, *range(n - 10, n)])
                rows[b], got[b] = [rows[b][j] for j in stay], [got[b][j] for j in stay]
            held = table >= 0
            assert kv_len.tolist() == [40] * B and held.sum().item() >= B
            # (the table's later slots, held from the start, stay; those of the entries that went are given back: pages for the next steps)
            free = (refs == 0).nonzero()[:, 0].int()
            need = ~held
            table[need] = free[:int(need.sum())]
            refs[table[need].long()] += 1
