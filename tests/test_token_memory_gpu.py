"""The token memory: remembering, indexing and recalling together, as a decoding loop uses them, against plain attention in 64 bits."""
import numpy as np
import pytest
import torch

from hnsw_amd import capi
from hnsw_amd.memory import TokenMemory
from tests import cache_reference as ref

pytestmark = pytest.mark.gpu


def _stored(m, b):
    """Request b's keys and values as the cache holds them, [tokens, heads, dim] in 64 bits."""
    c, n = m.cache, m.host_lens[b]
    pos = torch.arange(n, device=m.device)
    return [x.double().cpu() for x in c.read(m.table[b][pos // c.block_tokens].long() * c.block_tokens + pos % c.block_tokens)]


def _check(m, q, out, lse, seen, scale):
    """seen(b, h): positions that query head h of request b attends over."""
    group = q.shape[1] // m.cache.n_heads
    largest = float(m.cache.v_scale.max()) * 448
    for b in range(q.shape[0]):
        keys, values = _stored(m, b)
        for h in range(q.shape[1]):
            at = torch.as_tensor(seen(b, h), dtype=torch.long)
            want, want_lse, spread, qk, peak = ref.attend_row(q[b, h].double().cpu(), keys[at, h // group], values[at, h // group], scale)
            tol = ref.tolerance(want, spread, qk, peak, len(at), m.cache.dim, q.dtype, largest)
            assert bool(((out[b, h].double().cpu() - want).abs() <= tol).all()), (b, h)
            if len(at):
                assert abs(float(lse[b, h]) - want_lse) <= ref.lse_tolerance(want_lse, qk, peak, len(at), m.cache.dim)


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
def test_a_decoding_loop(codes):
    """Prompts, an index over one of them, decoding steps with and without the search, a request that ends and one that starts in its blocks."""
    gen = torch.Generator().manual_seed(7)
    heads, q_heads, dim, scale = 2, 4, 64, 64 ** -0.5
    m = TokenMemory(3, 80, heads, dim, block_tokens=16, max_len=900, codes=codes)
    rows = lambda n, h=heads: torch.randn((n, h, dim), generator=gen).bfloat16().cuda()  # noqa: E731
    m.remember([700, 300, 0], rows(1000), rows(1000))
    m.index(0)
    m.index(2)                                                       # nothing to index
    for step in range(3):
        m.remember([1, 1, 1], rows(3), rows(3))
        q = rows(3, q_heads) * 2
        out, lse = m.attend(q)
        _check(m, q, out, lse, lambda b, h: range(m.host_lens[b]), scale)
        out, lse, ids = m.recall(q, 32, 64)
        listed = ids.cpu().numpy()
        # request 0: 32 found and what came after; the others: everything, as nothing of them is indexed
        assert all(len(set(listed[0, h, :32])) == 32 and 0 <= listed[0, h, :32].min() and listed[0, h, :32].max() < 700 for h in range(q_heads))
        assert [m.host_lens[b] for b in range(3)] == [701 + step, 301 + step, 1 + step]
        for b in range(3):
            extra = sorted(int(i) for i in listed[b, 0, 32:] if i >= 0)
            assert extra == list(range(700 if b == 0 else 0, m.host_lens[b]))
        _check(m, q, out, lse, lambda b, h: [int(i) for i in listed[b, h] if 0 <= i < m.host_lens[b]], scale)
        # the search finds most of the largest inner products of each query head
        keys = _stored(m, 0)[0]
        hits = 0
        for h in range(q_heads):
            best = torch.topk(keys[:700, h // 2] @ q[0, h].double().cpu(), 32).indices
            hits += len(set(best.tolist()) & set(listed[0, h, :32].tolist()))
        assert hits >= 0.8 * 32 * q_heads, hits
    m.remember([-1, 0, 0], rows(0), rows(0))
    assert m.host_lens == [0, 303, 3] and m.indexes[0] is None
    m.remember([600, 0, 0], rows(600), rows(600))                    # into blocks that were given back, with no index of the request that ended
    q = rows(3, q_heads)
    out, lse, ids = m.recall(q, 5)
    _check(m, q, out, lse, lambda b, h: range(m.host_lens[b]), scale)
    out2, lse2 = m.attend(q)
    assert torch.allclose(out.float(), out2.float(), atol=2e-2, rtol=2e-2) and torch.allclose(lse, lse2, atol=1e-4, rtol=1e-5)
    # negative scales look for the smallest products
    m.index(0)
    out, lse, ids = m.recall(q, 600, 1200, scale=-0.2)
    _check(m, q, out, lse, lambda b, h: [int(i) for i in ids[b, h].tolist() if 0 <= i < m.host_lens[b]], -0.2)


def test_what_does_not_fit_is_refused_and_changes_nothing():
    m = TokenMemory(2, 4, 1, 16, block_tokens=16, max_len=48)
    rows = torch.ones((60, 1, 16), device="cuda")
    m.remember([20, 0], rows[:20], rows[:20])
    for grow, n in (([29, 0], 29), ([20, 30], 50)):                  # beyond max_len; beyond the blocks
        with pytest.raises(capi.HnswAmdError) as e:
            m.remember(grow, rows[:n], rows[:n])
        assert e.value.code == capi.E_FULL
        assert m.host_lens == [20, 0] and m.lens.tolist() == [20, 0] and m.state.tolist() == [2, 4]
    with pytest.raises(ValueError):
        m.remember([1, 1], rows[:1], rows[:1])
    with pytest.raises(ValueError):
        m.recall(rows[:1], 3)
    m.remember([28, 0], rows[:28], rows[:28])
    assert np.isclose(m.attend(rows[:2, :, :])[0][0].cpu().numpy(), 1.0).all()
