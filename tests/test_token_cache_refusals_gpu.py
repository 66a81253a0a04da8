"""Refusals of the token cache's calls that need tensors on a GPU."""
import pytest
import torch

from hnsw_amd import TokenCache
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
