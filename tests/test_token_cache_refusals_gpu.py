"""Refusals of the token cache's calls that need tensors on a GPU."""
import pytest
import torch

from hnsw_amd import HNSW, TokenCache, TokenMemory
from tests.test_token_cache_gpu import F32, Setup, _gpu, _queries

pytestmark = pytest.mark.gpu


def test_scales_that_require_a_gradient():
    """Refused when the cache is made, and by its calls where the gradient is asked for later; no graph is needed within no_grad."""
    s = Setup([30, 4], 2, 16, 64, torch.int8)
    c, q, ids = s.cache, _queries(2, 4, 64, F32), _gpu([[[0, 3]] * 2] * 2)
    rows, slots = _queries(1, 2, 64, F32), _gpu([0], torch.int64)
    for name in ("k_scale", "v_scale"):
        leaf = getattr(c, name).clone().requires_grad_()
        scales = dict(k_scale=c.k_scale, v_scale=c.v_scale)
        with pytest.raises(ValueError, match="gradient"):
            TokenCache(c.k_codes, c.v_codes, **dict(scales, **{name: leaf}))
        getattr(c, name).requires_grad_()
        for call in (lambda: c.attend(q, s.d_table, s.d_lens), lambda: c.attend_found(q, s.d_table, s.d_lens, ids), lambda: c.read(slots), lambda: c.append(rows, rows, slots)):
            with pytest.raises(ValueError, match=name):
                call()
        with torch.no_grad():
            want = TokenCache(c.k_codes, c.v_codes, c.k_scale.detach(), c.v_scale.detach()).attend(q, s.d_table, s.d_lens)
            assert all(torch.equal(a, b) for a, b in zip(c.attend(q, s.d_table, s.d_lens), want))
        getattr(c, name).requires_grad_(False)


def test_recall_refuses_before_it_searches(monkeypatch):
    m = TokenMemory(2, 8, 2, 16, block_tokens=16, max_len=64)
    rows = _queries(40, 2, 16, F32)
    m.remember([30, 10], rows, rows)
    m.index(0)
    searches = []
    monkeypatch.setattr(HNSW, "search_batch_device_begin", lambda *a, **k: searches.append(a))
    for q in (_queries(1, 2, 16, F32), _queries(2, 3, 16, F32), _queries(2, 1, 16, F32), _queries(2, 2, 1, F32), _queries(2, 2, 32, F32), _queries(2, 2, 16, F32)[0], _queries(2, 2, 16, F32)[:, :0]):
        with pytest.raises(ValueError, match="recall"):
            m.recall(q, 3)
    with pytest.raises(ValueError, match="positive"):
        m.recall(_queries(2, 2, 16, F32), 0)
    assert not searches


def test_recall_of_more_than_an_index_holds():
    """Lists end where the index does, and attention is over what there is."""
    m = TokenMemory(2, 8, 1, 16, block_tokens=16, max_len=64)
    rows = _queries(13, 1, 16, F32)
    m.remember([5, 8], rows, rows)
    m.index(0)
    m.index(1)
    m.remember([1, 0], rows[:1], rows[:1])
    q = _queries(2, 3, 16, F32)
    out, lse, ids = m.recall(q, 32)
    for b, n in ((0, 6), (1, 8)):
        for h in range(3):
            assert sorted(i for i in ids[b, h].tolist() if 0 <= i < n) == list(range(n))
    want, want_lse = m.attend(q)
    assert torch.allclose(out, want, rtol=1e-4, atol=1e-5) and torch.allclose(lse, want_lse, rtol=1e-5, atol=1e-5)
