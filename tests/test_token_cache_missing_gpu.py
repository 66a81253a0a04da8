"""Attention over tables whose first blocks do not exist, one to more than a wavefront's lanes of them: tokens of no block read a live token's
codes, whose place comes from the first entry that exists, whichever lane has it.  Against plain attention in 64 bits."""
import numpy as np
import pytest
import torch

from tests.test_token_cache_gpu import BF16, E4, F16, F32, I8, Setup, _compare, _gpu, _queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("missing", [1, 37, 63, 64, 65, 130])
@pytest.mark.parametrize("dim,codes,dtype", [(64, I8, F32), (64, E4, BF16), (128, E4, F32), (128, I8, F16), (192, E4, BF16)])
@pytest.mark.parametrize("new", [1, 30, 200])
def test_first_blocks_that_are_none(missing, dim, codes, dtype, new):
    length = 16 * missing + 53                                       # (the request's last block ends behind its last token)
    s = Setup([length], 2, 16, dim, codes)
    s.table[0, :missing] = torch.where(torch.arange(missing) % 2 == 0, -1, 10 ** 6).int()
    s.d_table = s.table.cuda()
    q = _queries(new, 4, dim, dtype)
    out, lse = s.cache.attend(q, s.d_table, s.d_lens, cu_q=None if new == 1 else _gpu([0, new]))
    _compare(s, q, out, lse, lambda r, h: (0, np.arange(max(0, length - new + r + 1))), dim ** -0.5, pick=sorted({0, new // 2, new - 1}))
