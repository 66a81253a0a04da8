"""What the token cache's calls refuse (no GPU needed: they refuse before any device call), and the test oracle against small cases
that are worked out by hand."""
import ctypes

import pytest
import torch

from hnsw_amd import capi
from tests import cache_reference as ref


def _cache(**kw):
    v = dict(k_codes=4096, v_codes=8192, k_scale=64, v_scale=128, n_blocks=4, n_heads=2, block_tokens=16, dim=64, codes=0)
    v.update(kw)
    return capi.TokenCacheC(*[v[n] for n, _ in capi.TokenCacheC._fields_])


def _attend(cache, found=False, q=1, rows=2, heads=4, row_type=0, table=1, width=4, lens=1, requests=2, cu=None, ids=1, id_heads=2, n_ids=3, scale=1.0, out=16,
            work=None, nbytes=0):
    L, c = capi.lib(), ctypes.addressof(cache) if cache is not None else None
    if found:
        return L.hnsw_amd_cache_attend_found_device(c, q, rows, heads, 256, 64, row_type, table, width, lens, requests, cu, 1, ids, id_heads, n_ids, scale, out,
                                                    None, work, nbytes, 0, None)
    return L.hnsw_amd_cache_attend_device(c, q, rows, heads, 256, 64, row_type, table, width, lens, requests, cu, 1, scale, 0, out, None, work, nbytes, 0, None)


@pytest.mark.parametrize("field,value", [("k_codes", 0), ("v_scale", 0), ("k_codes", 4100), ("block_tokens", 8), ("block_tokens", 48), ("block_tokens", 512),
                                         ("dim", 0), ("dim", 72), ("dim", 272), ("codes", 2), ("n_heads", 0), ("n_blocks", 0), ("n_blocks", 0x80000000)])
def test_a_cache_that_cannot_be_is_refused_by_every_call(field, value):
    c = _cache(**{field: value})
    L, at = capi.lib(), ctypes.addressof(c)
    assert _attend(c) == capi.E_ARG and _attend(c, found=True) == capi.E_ARG
    assert L.hnsw_amd_cache_append_device(at, 16, 16, 1, 0, 128, 64, 128, 64, 1, 0, None) == capi.E_ARG
    assert L.hnsw_amd_cache_read_device(at, 16, 1, 0, 16, 16, 0, None) == capi.E_ARG
    assert L.hnsw_amd_last_error()


def test_rows_beyond_32_bits_are_refused():
    assert _attend(_cache(n_blocks=1 << 24, n_heads=16)) == capi.E_ARG       # 2^24 blocks x 16 heads x 16 tokens = 2^32 rows


@pytest.mark.parametrize("bad", [dict(heads=3), dict(heads=0), dict(requests=0), dict(width=0), dict(width=1 << 27), dict(rows=3), dict(row_type=3),
                                 dict(scale=float("nan")), dict(scale=float("inf")), dict(q=None), dict(out=None), dict(out=24), dict(table=None), dict(lens=None),
                                 dict(rows=1 << 31, cu=1), dict(rows=1 << 30, cu=1)])
def test_attend_refuses(bad):
    assert _attend(_cache(), **bad) == capi.E_ARG
    assert _attend(None) == capi.E_ARG


@pytest.mark.parametrize("bad", [dict(id_heads=1), dict(id_heads=3), dict(id_heads=8), dict(id_heads=0), dict(ids=None)])
def test_attend_found_refuses(bad):
    assert _attend(_cache(), found=True, **bad) == capi.E_ARG


def test_nothing_to_do_is_no_error():
    assert _attend(_cache(), rows=0, cu=1) == capi.OK
    L, c = capi.lib(), _cache()
    assert L.hnsw_amd_cache_append_device(ctypes.addressof(c), None, None, 0, 0, 0, 0, 0, 0, None, 0, None) == capi.OK
    assert L.hnsw_amd_cache_read_device(ctypes.addressof(c), None, 0, 0, 16, 16, 0, None) == capi.OK


def test_append_and_read_refuse():
    L, c = capi.lib(), _cache()
    at = ctypes.addressof(c)
    assert L.hnsw_amd_cache_append_device(at, 16, 16, 1, 3, 128, 64, 128, 64, 16, 0, None) == capi.E_ARG          # type
    assert L.hnsw_amd_cache_append_device(at, None, 16, 1, 0, 128, 64, 128, 64, 16, 0, None) == capi.E_ARG
    assert L.hnsw_amd_cache_append_device(at, 16, 16, 1 << 31, 0, 128, 64, 128, 64, 16, 0, None) == capi.E_ARG
    assert L.hnsw_amd_cache_read_device(at, 16, 1, 3, 16, 16, 0, None) == capi.E_ARG
    assert L.hnsw_amd_cache_read_device(at, 16, 1, 0, 20, 16, 0, None) == capi.E_ARG                              # alignment
    assert L.hnsw_amd_cache_read_device(at, None, 1, 0, 16, 16, 0, None) == capi.E_ARG


def _plan(requests=2, width=4, n_blocks=8, block=16, n_slots=4, lens=16, lens_out=32, state=48, state_out=64, status=80, slots=96):
    return capi.lib().hnsw_amd_cache_plan_device(lens, 112, requests, 128, width, 144, n_blocks, state, block, n_slots, slots, 160, lens_out, state_out, status, 0, None)


@pytest.mark.parametrize("bad", [dict(requests=0), dict(requests=8193), dict(width=0), dict(width=1 << 27), dict(n_blocks=0), dict(n_blocks=1 << 31), dict(block=24),
                                 dict(n_slots=1 << 31), dict(lens=None), dict(lens_out=16), dict(state_out=48), dict(status=None), dict(slots=None)])
def test_plan_refuses(bad):
    assert _plan(**bad) == capi.E_ARG


def test_python_refuses_before_the_library_is_asked():
    from hnsw_amd import TokenCache, cache_plan
    z = torch.zeros
    with pytest.raises(ValueError, match="GPU"):
        TokenCache(z(2, 1, 16, 64, dtype=torch.int8), z(2, 1, 16, 64, dtype=torch.int8), z(2, 1), z(2, 1))
    with pytest.raises(ValueError, match="GPU"):
        cache_plan(z(2, dtype=torch.int32), z(2, dtype=torch.int32), z(2, 4, dtype=torch.int32), z(8, dtype=torch.int32), z(2, dtype=torch.int64), block_tokens=16, n_slots=2)


def test_the_oracle_by_hand():
    # two requests of 15 and 0 tokens grow by 2 and 1, a third ends: blocks 7 and 3 are taken, 5 goes back
    got = ref.plan([15, 0, 16], [2, 1, -1], [[4, -1], [-1, -1], [5, -1]], [9, 7, 3, 2, 0, 0, 0, 0, 0, 0], [1, 4], 16, 5)
    assert got[:5] == ([4 * 16 + 15, 7 * 16, 3 * 16, -1, -1], [0, 2, 3, 3], [17, 1, 0], [3, 5], 0)
    assert got[5] == [[4, 7], [3, -1], [5, -1]] and got[6][4] == 5
    assert ref.plan([15], [2], [[4]], [9], [0, 1], 16, 2)[4] == 2                                      # the table is too narrow
    # e4m3 around 1: steps of 1/8, ties to even; the smallest step is 2^-9
    x = torch.tensor([1.0, 1.0625, 1.1875, 2.0 ** -10, 3 * 2.0 ** -10, 500.0, float("nan"), -float("inf")], dtype=torch.float64)
    assert ref.nearest(x, torch.float8_e4m3fn).tolist() == [1.0, 1.0, 1.25, 0.0, 2.0 ** -8, 448.0, 0.0, -448.0]
    assert ref.nearest(torch.tensor([0.5, 1.5, -2.5, 130.0], dtype=torch.float64), torch.int8).tolist() == [0.0, 2.0, -2.0, 127.0]
    # a block of int8 whose largest value is 127 has scale 1; a token of 128 moves it to 2
    v, s = torch.zeros(1, 1, 16, 1, dtype=torch.float64), torch.zeros(1, 1, dtype=torch.float64)
    ref.append(v, s, torch.tensor([[[127.0]], [[3.0]]], dtype=torch.float64), [0, 1], 16, torch.int8)
    assert s.item() == 1 and v[0, 0, :2, 0].tolist() == [127, 3]
    ref.append(v, s, torch.tensor([[[128.0]]], dtype=torch.float64), [2], 16, torch.int8)
    assert s.item() == 2 and v[0, 0, :3, 0].tolist() == [64, 2, 64]                                    # 63.5 and 1.5: ties to even
