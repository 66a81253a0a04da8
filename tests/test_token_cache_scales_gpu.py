"""Attention over blocks whose value scales are far apart: what a row gives depends on the tokens it sees and on what they weigh in it, not on
the largest scale that lies next to them.  Against plain attention in 64 bits.

How far an output may be off is tests/cache_reference.py's `tolerance` with the row's OWN largest weight: the operands that meet the values are
16-bit floats of p_t S_t (probability times value scale) in units of 2^-11 of the row's largest p_t S_t, so that their smallest step costs
2^-36 of that largest product, whatever other scales there are."""
import math

import numpy as np
import pytest
import torch

from tests import cache_reference as ref
from tests.test_token_cache_gpu import BF16, E4, F32, I8, Setup, _gpu, _queries

pytestmark = pytest.mark.gpu


def _set(s, v_scale=None, first=None):
    """New value scales ([n_blocks, heads]), and new codes of the keys' first dim ([n_blocks, heads, block])."""
    c = s.cache
    if v_scale is not None:
        c.v_scale.copy_(v_scale)
        s.v64 = c.v_codes.cpu().double() * v_scale.double()[:, :, None, None]
    if first is not None:
        k = c.k_codes.cpu().double()
        k[..., 0] = first
        c.k_codes.copy_(k.to(c.k_codes.dtype))
        s.k64 = k * c.k_scale.cpu().double()[:, :, None, None]


def _check(s, q, out, lse, see, scale, rows):
    """see(row, head): (request, positions)."""
    group = q.shape[1] // s.heads
    q64, out, lse, vs = q.double().cpu(), out.double().cpu(), lse.double().cpu(), s.cache.v_scale.cpu().double()
    for row in rows:
        for h in range(q.shape[1]):
            b, positions = see(row, h)
            positions = np.asarray(positions, dtype=np.int64)
            keys, values = s.tokens(b, h // group, positions)
            want, want_lse, spread, qk, peak = ref.attend_row(q64[row, h], keys, values, scale)
            if len(positions) == 0:
                assert not out[row, h].any() and lse[row, h] == -math.inf
                continue
            x = keys @ q64[row, h] * scale
            own = float((torch.exp(x - x.max()) * vs[s.table[b].long()[positions // s.block], h // group]).max())
            tol = ref.tolerance(want, spread, qk, peak, len(positions), s.dim, q.dtype, own * 448)
            off = (out[row, h] - want).abs()
            assert bool((off <= tol).all()), (row, h, len(positions), float((off / tol).max()), float(want.abs().max()))
            assert abs(lse[row, h] - want_lse) <= ref.lse_tolerance(want_lse, qk, peak, len(positions), s.dim), (row, h)


# rows of one request, query heads of a key head, dims: single tokens and a few in registers (16 or 32 rows at a time), many through LDS tiles (two
# halves of the wavefronts, both numbers of rows, one buffer)
FORMS = [(1, 1, 64), (9, 1, 128), (30, 2, 64), (40, 1, 128), (40, 1, 192), (200, 1, 64), (300, 8, 128), (300, 1, 112), (200, 1, 192), (200, 1, 256)]


@pytest.mark.parametrize("codes,dtype", [(I8, F32), (E4, BF16)])
@pytest.mark.parametrize("rows,group,dim", FORMS)
@pytest.mark.parametrize("far", [30, 60, 100])
def test_rows_before_tokens_of_large_values(rows, group, dim, codes, dtype, far):
    """The last block's values are 2^far times the others'; rows before it see none of them."""
    length, block = 430, 16
    s = Setup([length], 1, block, dim, codes)
    vs = s.cache.v_scale.cpu()
    vs[s.table[0, (length - 1) // block].long()] *= 2.0 ** far
    _set(s, vs)
    q = _queries(rows, group, dim, dtype)
    cu = _gpu([0, rows])
    for max_len in (0, 1, 100000):
        out, lse = s.cache.attend(q, s.d_table, s.d_lens, cu_q=cu, max_len=max_len)
        pick = range(rows) if rows < 50 else [0, 1, rows // 2, rows - 30, rows - 16, rows - 15, rows - 14, rows - 1]
        _check(s, q, out, lse, lambda r, h: (0, np.arange(length - rows + r + 1)), dim ** -0.5, pick)


@pytest.mark.parametrize("codes,dtype", [(I8, F32), (E4, BF16)])
@pytest.mark.parametrize("rows,group,dim", FORMS)
@pytest.mark.parametrize("far,apart", [(40, 50.0), (36, 25.0), (90, 62.5), (-40, 50.0)])
def test_tokens_of_large_values_and_small_probability(rows, group, dim, codes, dtype, far, apart):
    """Every third block's values are 2^far times the others', and their scores lie `apart` (in base e) under the others': 2^-72 for 2^40 leaves nothing of
    them, 2^-36 for 2^36 as much as of the others, 2^-90 for 2^90 likewise."""
    length, block = 700, 32
    s = Setup([length], 1, block, dim, codes)
    gen = torch.Generator().manual_seed(rows)
    large = torch.zeros(s.cache.n_blocks, 1)
    large[s.table[0, 1::3].long()] = 1.0
    vs = torch.exp2(torch.randint(-8, -4, large.shape, generator=gen).float()) * torch.where(large > 0, 2.0 ** far, 1.0)
    _set(s, vs, torch.where(large > 0, -96.0, 96.0)[:, :, None].expand(-1, -1, block))
    s.cache.k_scale.fill_(apart / 192)
    s.k64 = s.cache.k_codes.cpu().double() * (s.cache.k_scale.cpu().double()[:, :, None, None])
    q = _queries(rows, group, dim, dtype) / 64
    q[..., 0] = 1.0
    for causal in (True, False):
        out, lse = s.cache.attend(q, s.d_table, s.d_lens, cu_q=_gpu([0, rows]), causal=causal, scale=1.0)
        pick = range(rows) if rows < 10 else [0, 1, rows // 2, rows - 1]
        _check(s, q, out, lse, lambda r, h: (0, np.arange(length - rows + r + 1 if causal else length)), 1.0, pick)  # noqa: B023
    if rows == 1:
        ids = np.random.default_rng(0).permutation(length)[:300].astype(np.int32)
        for some in (ids, np.sort(ids), ids[:40]):
            out, lse = s.cache.attend_found(q, s.d_table, s.d_lens, _gpu(some.reshape(1, 1, -1)), scale=1.0)
            _check(s, q, out, lse, lambda r, h: (0, some), 1.0, [0])  # noqa: B023


@pytest.mark.parametrize("codes,dtype", [(I8, BF16), (E4, F32)])
@pytest.mark.parametrize("rows,dim", [(1, 64), (40, 128), (300, 64), (300, 128), (300, 192)])
@pytest.mark.parametrize("first,second,third", [(0.0, 1.0, 2.0 ** -4), (2.0 ** 60, 1.0, 2.0 ** -70), (2.0 ** -60, 2.0 ** 70, 1.0), (1.0, 0.0, 0.0), (0.0, 0.0, 0.0), (2.0 ** 6, 2.0 ** -6, 2.0 ** 11)])
def test_scales_that_change_from_table_to_table(rows, dim, codes, dtype, first, second, third):
    """A workgroup takes 4096 tokens' blocks at a time: what the first of these leave in its sums does not show through, nor does what comes
    later reach rows that do not see it.  A scale of 0 makes any codes zeros."""
    length, block = 2 * 4096 + 150, 32
    s = Setup([length], 1, block, dim, codes)
    vs = s.cache.v_scale.cpu()
    for i, by in enumerate((first, second, third)):
        vs[s.table[0, 128 * i:128 * (i + 1)].long()] = (torch.exp2(torch.randint(-2, 2, (len(s.table[0, 128 * i:128 * (i + 1)]), 1),
                                                                                  generator=torch.Generator().manual_seed(i)).float()) * by)
    _set(s, vs)
    q = _queries(rows, 1, dim, dtype)
    for max_len in (1, length):                                  # (a hint of one token: nothing is cut)
        out, lse = s.cache.attend(q, s.d_table, s.d_lens, cu_q=_gpu([0, rows]), max_len=max_len)
        _check(s, q, out, lse, lambda r, h: (0, np.arange(length - rows + r + 1)), dim ** -0.5, sorted({0, rows // 2, rows - 1}))
    if rows == 300:
        # rows that end in the first table, next to others that see the second
        out, lse = s.cache.attend(q, s.d_table, _gpu([4096 + 200]), cu_q=_gpu([0, rows]), max_len=1)
        _check(s, q, out, lse, lambda r, h: (0, np.arange(4096 + 200 - rows + r + 1)), dim ** -0.5, [0, 99, 100, 101, 299])


def test_a_large_scale_that_is_listed_behind_the_row():
    """Listed positions that a row does not see leave no mark, whatever their scale."""
    lens, new, dim = [200], [150], 64
    s = Setup(lens, 1, 16, dim, I8)
    vs = s.cache.v_scale.cpu()
    vs[s.table[0, 8:].long()] = 2.0 ** 90
    _set(s, vs)
    ids = np.random.default_rng(3).permutation(200)[:120].astype(np.int32)
    q = _queries(150, 2, dim, F32)
    out, lse = s.cache.attend_found(q, s.d_table, s.d_lens, _gpu(np.broadcast_to(ids, (150, 1, 120)).copy()), cu_q=_gpu([0, 150]))
    _check(s, q, out, lse, lambda r, h: (0, ref.visible(ids, 50 + r + 1)), dim ** -0.5, range(0, 150, 7))


@pytest.mark.parametrize("none", [float("inf"), float("nan"), -1.0])
@pytest.mark.parametrize("rows,dim", [(9, 128), (40, 64), (200, 64), (300, 128), (200, 192)])
def test_rows_before_a_block_whose_scales_are_none(rows, dim, none):
    """What rows that see such a block give is not defined; the others in the same tiles give what they give without it."""
    length, block = 430, 16
    s = Setup([length], 1, block, dim, I8)
    q, cu = _queries(rows, 1, dim, F32), _gpu([0, rows])
    last = s.table[0, (length - 1) // block].long()
    s.cache.k_scale[last], s.cache.v_scale[last] = none, none
    out, lse = s.cache.attend(q, s.d_table, s.d_lens, cu_q=cu)
    _check(s, q, out, lse, lambda r, h: (0, np.arange(length - rows + r + 1)), dim ** -0.5, range(0, rows - 14, 1 if rows < 50 else 17))


@pytest.mark.parametrize("rows,dim", [(1, 64), (40, 128), (200, 64), (300, 128)])
def test_scales_that_are_minus_zero(rows, dim):
    """-0 is a scale of 0: scores of 0 for a key scale, values of zeros for a value scale."""
    length = 430
    s = Setup([length], 1, 16, dim, I8)
    q, cu = _queries(rows, 1, dim, F32), _gpu([0, rows])
    some = s.table[0, 2::3].long()
    s.cache.k_scale[some], s.cache.v_scale[s.table[0, 1::3].long()] = -0.0, -0.0
    s.k64, s.v64 = (c.cpu().double() * x.cpu().double()[:, :, None, None] for c, x in ((s.cache.k_codes, s.cache.k_scale), (s.cache.v_codes, s.cache.v_scale)))
    out, lse = s.cache.attend(q, s.d_table, s.d_lens, cu_q=cu)
    _check(s, q, out, lse, lambda r, h: (0, np.arange(length - rows + r + 1)), dim ** -0.5, sorted({0, rows // 2, rows - 1}))


@pytest.mark.parametrize("codes,dtype", [(I8, F32), (E4, BF16)])
@pytest.mark.parametrize("rows,group,dim", FORMS)
@pytest.mark.parametrize("at", [0, 70, 150, 215, 280, 330, 400, 470])
def test_one_block_of_large_values_anywhere(rows, group, dim, codes, dtype, at):
    """Wavefronts take the tokens' tiles in turn: any one of them, and no other, meets the block, and their sums become one."""
    length, block = 500, 16
    s = Setup([length], 1, block, dim, codes)
    vs = s.cache.v_scale.cpu()
    vs[s.table[0, at // block].long()] *= 2.0 ** 60
    _set(s, vs)
    q, cu = _queries(rows, group, dim, dtype), _gpu([0, rows])
    out, lse = s.cache.attend(q, s.d_table, s.d_lens, cu_q=cu)
    _check(s, q, out, lse, lambda r, h: (0, np.arange(length - rows + r + 1)), dim ** -0.5, sorted({0, rows // 3, rows // 2, rows - 1}))


@pytest.mark.parametrize("rows,dim", [(1, 64), (40, 128), (200, 64), (300, 128)])
def test_values_of_zeros_and_scores_far_below_zero(rows, dim):
    """Scores around -600 (in base e), and nothing but scales of 0 among the values."""
    length = 430
    s = Setup([length], 1, 16, dim, I8)
    _set(s, torch.zeros_like(s.cache.v_scale.cpu()), torch.full((s.cache.n_blocks, 1, 16), -96.0))
    s.cache.k_scale.fill_(600 / 96)
    s.k64 = s.cache.k_codes.cpu().double() * s.cache.k_scale.cpu().double()[:, :, None, None]
    q = _queries(rows, 1, dim, F32) / 4096
    q[..., 0] = 1.0
    out, lse = s.cache.attend(q, s.d_table, s.d_lens, cu_q=_gpu([0, rows]), scale=1.0)
    _check(s, q, out, lse, lambda r, h: (0, np.arange(length - rows + r + 1)), 1.0, sorted({0, rows // 2, rows - 1}))
    ids = _gpu(np.broadcast_to(np.arange(0, length, 3, dtype=np.int32), (rows, 1, 144)).copy())
    out, lse = s.cache.attend_found(q, s.d_table, s.d_lens, ids, cu_q=_gpu([0, rows]), causal=False, scale=1.0)
    _check(s, q, out, lse, lambda r, h: (0, np.arange(0, length, 3)), 1.0, sorted({0, rows // 2, rows - 1}))
