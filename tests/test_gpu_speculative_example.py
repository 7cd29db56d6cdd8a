"""examples/speculative_step.py runs and leaves its cache consistent.  Run with `-m gpu` on a B200."""
import importlib.util
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_the_speculative_example():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    path = Path(__file__).resolve().parents[1] / "examples" / "speculative_step.py"
    spec = importlib.util.spec_from_file_location("speculative_step", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    cache, taken, status = m.run(requests=6, steps=8)
    assert status.tolist() == [0, 0, 0, 0]
    assert taken.min().item() >= 1 and taken.max().item() > 1          # some drafts are accepted
    # every page is counted as often as the tables name it, and the pages in use are the first ones
    held = torch.arange(cache.table.shape[1], device="cuda") < ((cache.kv_len + 63) // 64)[:, None]
    named = cache.table[held].long()
    assert (named >= 0).all() and torch.equal(torch.bincount(named, minlength=cache.refs.numel()), cache.refs.long())
    live = int((cache.refs > 0).sum())
    assert (cache.refs[:live] > 0).all() and (cache.table[~held] == -1).all()
