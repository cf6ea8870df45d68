"""The example's step when the pages run out: nothing is appended."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


def _stack(**kw):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_serving.py")
    spec = importlib.util.spec_from_file_location("paged_serving", path)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    return ex.Stack(n_layers=2, hidden=256, n_q=4, n_kv=2, head_dim=64, max_seqs=4, max_len=256, **kw)


def test_a_step_without_pages_leaves_the_cache_alone(torch, m27b):
    s = _stack(n_pages=6)
    x = torch.randn(64, 256, device="cuda")
    s.step([0], [64], x)    # four whole pages
    s.fork(0, [1, 2])       # shared by all three
    state = [s.pages.table, s.pages.ref, s.pages.lens, s.pages.pools[0]]
    before = [t.clone() for t in state]
    with pytest.raises(m27b.M27BError, match="too few free pages"):
        s.step([0, 1, 2], [1, 1, 1], x[:3])
    assert all(torch.equal(a, b) for a, b in zip(state, before))
    s.step([0, 1], [1, 1], x[:2])  # two pages are left
    with pytest.raises(m27b.M27BError, match="too few free pages"):
        s.step([2], [1], x[:1])
    s.step([0, 1], [10, 3], x[:13])  # within their pages
    with pytest.raises(m27b.M27BError, match="bad request"):
        s.fork(0, [1])
    assert m27b.device_status() == 0
