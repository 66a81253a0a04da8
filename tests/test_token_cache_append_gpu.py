"""Appends whose slots leave out others of the same block: rows behind a gap are written as by a further call.  Against the plain statement in
64 bits, which takes runs of slots that follow one another in order; codes and scales are exact."""
import random

import pytest
import torch

from hnsw_amd import TokenCache
from tests import cache_reference as ref
from tests.test_token_cache_gpu import BF16, E4, F16, F32, I8, _gpu, _values

pytestmark = pytest.mark.gpu


def _append(codes, dtype, heads, block, dim, slots, n_blocks, seed):
    """The call, and what it has to leave; later rows of a block are louder, so that scales rise from run to run."""
    gen = torch.Generator().manual_seed(seed)
    k0, v0 = (_values(n_blocks, heads, block, dim, codes, gen) for _ in range(2))
    scale0 = torch.exp2(torch.randint(-9, 1, (2, n_blocks, heads), generator=gen).float())
    loud = torch.tensor([2.0 ** min(s % block // 4 - 3, 9) if s >= 0 else 1.0 for s in slots]).view(-1, 1, 1)
    new = [(torch.randn((len(slots), heads, dim), generator=gen) * loud).to(dtype) for _ in range(2)]
    cache = TokenCache(k0.cuda(), v0.cuda(), scale0[0].cuda(), scale0[1].cuda())
    cache.append(new[0].cuda(), new[1].cuda(), _gpu(slots, torch.int64))
    for got, scale, before, s0, x in ((cache.k_codes, cache.k_scale, k0, scale0[0], new[0]), (cache.v_codes, cache.v_scale, v0, scale0[1], new[1])):
        want, want_scale = before.double(), s0.double()
        ref.append(want, want_scale, x.double(), slots, block, codes)
        assert torch.equal(scale.double().cpu(), want_scale)
        assert torch.equal(got.cpu().double(), want)


@pytest.mark.parametrize("codes", [I8, E4])
@pytest.mark.parametrize("slots", [[3, 5], [0, 2, 4, 6, 8], [0, 1, 2, 3, 8, 9, 10, 15], [15, 16, 18, 31, 32], [20, 22, -1, 40, 41, 43], [1, 3, 17, 19, 33, 35]])
def test_slots_that_are_left_out(codes, slots):
    _append(codes, BF16, 2, 16, 64, slots, 4, 3)


@pytest.mark.parametrize("codes,dtype,dim,block,rows", [(I8, BF16, 128, 64, 300), (E4, F32, 48, 256, 900), (I8, F16, 256, 128, 2500), (E4, BF16, 16, 16, 6000), (I8, F32, 80, 32, 5000), (E4, BF16, 128, 256, 9000)])
def test_runs_and_gaps_of_all_lengths(codes, dtype, dim, block, rows):
    """In calls of all sizes, so that a block's runs begin and go on anywhere in what a wavefront or workgroup looks at."""
    rng, heads = random.Random(rows), 4
    slots, blk = [], 0
    while len(slots) < rows:
        chance = rng.choice([0.02, 0.3, 0.9, 1.0])                   # of a slot of this block to be named
        slots += [blk * block + i for i in range(block) if rng.random() < chance]
        slots += [-1] * rng.choice([0, 0, 0, 2])
        blk += 1
    slots = slots[:rows]
    order = rng.sample(range(blk + 1), blk + 1)
    slots = [order[x // block] * block + x % block if x >= 0 else x for x in slots]
    _append(codes, dtype, heads, block, dim, slots, blk + 1, rows)
