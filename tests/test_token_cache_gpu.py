"""The token cache's kernels against plain statements of the same operators in 64 bits (tests/cache_reference.py)."""
import ctypes
import random

import numpy as np
import pytest
import torch

from hnsw_amd import HNSW, TokenCache, cache_plan, capi
from tests import cache_reference as ref

pytestmark = pytest.mark.gpu
I8, E4 = torch.int8, torch.float8_e4m3fn
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _gpu(x, dtype=torch.int32):
    return torch.as_tensor(x, dtype=dtype).cuda()


# ------------------------------------------------------------------------------------------------------------ plan

def _stock(rng, lens, block, width, n_blocks):
    """A table for these lengths and a ring with what is left, gone round a few times."""
    order = rng.sample(range(n_blocks), n_blocks)
    table, used = [], 0
    for a in lens:
        held = ref.blocks_of(max(a, 0), block)
        table.append(order[used:used + held] + [-1] * (width - held))
        used += held
    start = rng.randrange(3 * n_blocks)
    ring = [0] * n_blocks
    for i, blk in enumerate(order[used:]):
        ring[(start + i) % n_blocks] = blk
    return table, ring, [start, start + n_blocks - used]


def _check_plan(lens, grow, table, ring, state, block, n_slots):
    dev = [_gpu(lens), _gpu(grow), _gpu(table), _gpu(ring), _gpu(state, torch.int64)]
    want = ref.plan(lens, grow, table, ring, state, block, n_slots)
    for _ in range(2):                                  # a repeated call gives the same
        p = cache_plan(*dev, block_tokens=block, n_slots=n_slots)
        got = [t.tolist() for t in (p.slots, p.cu_new, p.lens, p.state)] + [p.status.item(), dev[2].tolist(), dev[3].tolist()]
        for g, w, name in zip(got, want, ("slots", "cu", "lens", "state", "status", "table", "ring")):
            assert g == w, name
    return want[4]


@pytest.mark.parametrize("n,block,longest,most", [(1, 16, 0, 1), (1, 64, 100, 300), (3, 16, 40, 0), (64, 32, 5000, 1), (65, 16, 70, 40), (257, 128, 900, 5), (1000, 16, 200, 60),
                                                  (4097, 16, 50, 3), (8192, 256, 600, 20)])
def test_plan(n, block, longest, most):
    rng = random.Random(n * block)
    lens = [rng.randint(0, longest) for _ in range(n)]
    grow = [rng.randint(0, most) if rng.random() < 0.9 else -1 for _ in range(n)]
    width = ref.blocks_of(longest + most, block) + 1
    total = sum(max(g, 0) for g in grow)
    n_blocks = sum(ref.blocks_of(a + max(g, 0), block) for a, g in zip(lens, grow)) + 2
    table, ring, state = _stock(rng, lens, block, width, n_blocks)
    assert _check_plan(lens, grow, table, ring, state, block, total) == 0
    assert _check_plan(lens, grow, table, ring, state, block, total + 13) == 0


def test_plan_takes_the_last_free_block_and_refuses_one_more():
    rng = random.Random(1)
    table, ring, state = _stock(rng, [16, 5], 16, 4, 5)          # 2 held, 3 free
    assert _check_plan([16, 5], [32, 12], table, ring, state, 16, 44) == 0
    assert _check_plan([16, 5], [33, 12], table, ring, state, 16, 45) == capi.PLAN_NO_BLOCKS
    assert _check_plan([16, 5], [-1, 44], table, ring, state, 16, 44) == 0             # what is given back is not there for this call
    assert _check_plan([16, 5], [-1, 60], table, ring, state, 16, 60) == capi.PLAN_TABLE_FULL


@pytest.mark.parametrize("lens,grow,n_slots,state,status", [
    ([16, 5], [1, 1], 1, None, capi.PLAN_SLOTS_FULL), ([-1, 5], [1, 1], 2, None, capi.PLAN_BAD_LENGTH), ([16, 5], [-2, 1], 2, None, capi.PLAN_BAD_LENGTH),
    ([16, 5], [1, 1], 2, [3, 2], capi.PLAN_BAD_LENGTH), ([16, 5], [1, 1], 2, [0, 9], capi.PLAN_BAD_LENGTH), ([16, 5], [1, 1], 2, [-1, 1], capi.PLAN_BAD_LENGTH),
    ([16, 5], [2 ** 31 - 1, 2 ** 31 - 1], 2, None, capi.PLAN_TABLE_FULL | capi.PLAN_SLOTS_FULL), ([16, 2 ** 31 - 1], [0, 0], 2, None, capi.PLAN_TABLE_FULL),
    ([64, 64], [-1, -1], 2, [0, 6], capi.PLAN_BAD_LENGTH)])
def test_plan_that_cannot_be_done_changes_nothing(lens, grow, n_slots, state, status):
    table, ring, good = _stock(random.Random(2), [16, 5], 16, 4, 8)
    table = [[2, 3, 4, 5], [1, 0, 6, 7]] if lens == [64, 64] else table
    assert _check_plan(lens, grow, table, ring, state or good, 16, n_slots) == status


def test_plan_with_block_numbers_that_are_none():
    assert _check_plan([17], [3], [[5, -7, 0]], [1, 2, 900, 900], [0, 2], 16, 3) == 0              # the held block is outside: no slots
    assert _check_plan([16], [3], [[0, 0, 0]], [900, 2, 3, 1], [4, 6], 16, 3) == 0                 # the taken one is


# ---------------------------------------------------------------------------------------------------- append, read

def _values(n_blocks, heads, block, dim, dtype, gen):
    if dtype is I8:
        return torch.randint(-127, 128, (n_blocks, heads, block, dim), generator=gen).to(I8)
    return (torch.randn((n_blocks, heads, block, dim), generator=gen) * 60).clamp(-448, 448).to(E4)


@pytest.mark.parametrize("codes", [I8, E4])
@pytest.mark.parametrize("rows,dim,heads,block,runs", [
    (BF16, 128, 2, 32, [(0, 1), (37, 1), (95, 1)]), (F16, 64, 1, 16, [(3, 13), (16, 16), (32, 5)]), (F32, 16, 3, 16, [(15, 1), (48, 20)]),
    (BF16, 80, 2, 64, [(10, 54), (64, 64), (130, 1)]), (F32, 256, 2, 128, [(0, 128), (129, 100)]), (F16, 208, 1, 256, [(200, 56), (256, 256), (513, 3)]),
    (BF16, 96, 8, 16, [(0, 700)])])
def test_append_and_read(codes, rows, dim, heads, block, runs):
    """Codes and scales are exact: scaling by a power of two loses nothing, and one rounding has one answer."""
    gen = torch.Generator().manual_seed(dim + block)
    n_blocks = max(ref.blocks_of(a + n, block) for a, n in runs) + 2
    k0, v0 = (_values(n_blocks, heads, block, dim, codes, gen) for _ in range(2))
    scale0 = torch.exp2(torch.randint(-8, 3, (2, n_blocks, heads), generator=gen).float())
    scale0[0, 0] = 0.0                                               # a block that was never written
    scale0[1, -1] = 0.3                                              # a scale from elsewhere
    perm = torch.randperm(n_blocks, generator=gen)
    slots = torch.cat([perm[torch.arange(a, a + n) // block] * block + torch.arange(a, a + n) % block for a, n in runs] + [torch.tensor([-1, n_blocks * block, -2 ** 40])])
    new = torch.randn((2, len(slots), heads, dim), generator=gen) * torch.exp2(torch.randint(-3, 4, (2, len(slots), heads, 1), generator=gen).float())
    new[0, 0, 0, :3] = torch.tensor([float("inf"), float("nan"), -float("inf")])
    new[1, -4] = 0.0
    new = new.to(rows)
    cache = TokenCache(k0.cuda(), v0.cuda(), scale0[0].cuda(), scale0[1].cuda())
    cache.append(new[0].cuda(), new[1].cuda(), slots.cuda())
    back = torch.cat([torch.randperm(n_blocks * block, generator=gen)[:500], torch.tensor([-5, n_blocks * block])])
    got = cache.read(back.cuda())
    got16 = cache.read(back.cuda(), BF16)
    for part, (name, before, have, scale) in enumerate((("k", k0, cache.k_codes, cache.k_scale), ("v", v0, cache.v_codes, cache.v_scale))):
        want, s = before.double(), scale0[part].double().clone()
        ref.append(want, s, new[part].double(), slots.tolist(), block, codes)
        assert torch.equal(scale.cpu().double(), s), name
        assert torch.equal(have.cpu().double(), want), name
        value = (want * s[:, :, None, None]).permute(0, 2, 1, 3).reshape(n_blocks * block, heads, dim)
        inside = (back >= 0) & (back < n_blocks * block)
        value = torch.where(inside[:, None, None], value[back.clamp(0, n_blocks * block - 1)], 0.0)
        assert torch.equal(got[part].cpu(), value.float())
        assert torch.equal(got16[part].cpu(), value.float().to(BF16))


@pytest.mark.parametrize("codes", [I8, E4])
def test_append_many_rows(codes):
    """So many rows that a wavefront looks at more than one: runs that begin anywhere, and rows that are skipped between them."""
    gen = torch.Generator().manual_seed(5)
    heads, block, dim, n_blocks = 8, 16, 16, 400
    rng = random.Random(5)
    slots = []
    for blk in rng.sample(range(n_blocks), n_blocks):
        a = rng.randrange(16)
        slots += [blk * block + i for i in range(a, rng.randint(a, 15) + 1)] + [-1] * rng.choice([0, 0, 1, 70])
    n = len(slots)
    assert n * heads > 16384
    new = torch.randn((2, n, heads, dim), generator=gen)
    k0 = _values(n_blocks, heads, block, dim, codes, gen)
    scale0 = torch.exp2(torch.randint(-9, -3, (n_blocks, heads), generator=gen).float())
    cache = TokenCache(k0.cuda(), k0.cuda().clone(), scale0.cuda(), scale0.cuda().clone())
    cache.append(new[0].cuda(), new[1].cuda(), _gpu(slots, torch.int64))
    for rows, have, scale in ((new[0], cache.k_codes, cache.k_scale), (new[1], cache.v_codes, cache.v_scale)):
        want, s = k0.double(), scale0.double().clone()
        ref.append(want, s, rows.double(), slots, block, codes)
        assert torch.equal(scale.cpu().double(), s) and torch.equal(have.cpu().double(), want)


@pytest.mark.parametrize("rows,dim,codes,dtype", [(300, 128, I8, BF16), (1100, 128, E4, BF16), (2500, 48, I8, F32), (4500, 128, I8, F16), (9000, 16, E4, BF16), (9000, 256, I8, BF16)])
def test_append_runs_of_all_lengths(rows, dim, codes, dtype):
    """Single rows, short runs, whole blocks and rows without a slot, mixed, in calls of all sizes: exact, as the rows of a block lie together."""
    heads, block, rng, gen = 4, 64, random.Random(rows + dim), torch.Generator().manual_seed(rows)
    slots, blk = [], 0
    while len(slots) < rows:
        kind = rng.randrange(6)
        n = [1, 1, rng.randint(2, 9), rng.randint(10, 63), block, 0][kind]
        if n == 0:
            slots += [rng.choice([-1, 2 ** 40])] * rng.randint(1, 3)
            continue
        off = rng.choice([0, rng.randint(0, block - n)])
        slots += range(blk * block + off, blk * block + off + n)
        blk += 1
    slots = slots[:rows]
    order = rng.sample(range(blk + 1), blk + 1)
    slots = [order[x // block] * block + x % block if 0 <= x < blk * block else x for x in slots]
    k0, v0 = (_values(blk + 1, heads, block, dim, codes, gen) for _ in range(2))
    scale0 = torch.exp2(torch.randint(-9, 1, (2, blk + 1, heads), generator=gen).float())
    new = [(torch.randn((rows, heads, dim), generator=gen) * torch.exp2(torch.randint(-4, 5, (rows, 1, 1), generator=gen).float())).to(dtype) for _ in range(2)]
    cache = TokenCache(k0.cuda(), v0.cuda(), scale0[0].cuda(), scale0[1].cuda())
    cache.append(new[0].cuda(), new[1].cuda(), _gpu(slots, torch.int64))
    for got, scale, before, s0, x in ((cache.k_codes, cache.k_scale, k0, scale0[0], new[0]), (cache.v_codes, cache.v_scale, v0, scale0[1], new[1])):
        want, want_scale = before.double(), s0.double()
        ref.append(want, want_scale, x.double(), slots, block, codes)
        assert torch.equal(scale.double().cpu(), want_scale)
        assert torch.equal(got.cpu().double(), want)


@pytest.mark.parametrize("peak", [0.0, 2.0 ** -140, 2.0 ** -100 * 127, 127.0, 127.00001, 448.0, 3.0e38, torch.finfo(F32).max])
@pytest.mark.parametrize("codes", [I8, E4])
def test_scale_at_the_borders(peak, codes):
    cache = TokenCache.empty(1, 1, 16, 16, codes)
    rows = torch.zeros((1, 1, 16))
    rows[0, 0, 3] = -peak
    cache.append(rows.cuda(), rows.cuda(), _gpu([0], torch.int64))
    want, s = torch.zeros(1, 1, 16, 16, dtype=torch.float64), torch.zeros(1, 1, dtype=torch.float64)
    ref.append(want, s, rows.double(), [0], 16, codes)
    assert cache.k_scale.item() == s.item() and torch.equal(cache.k_codes.cpu().double(), want)


def test_append_strided_rows():
    """Rows cut out of a wider tensor, aligned to 16 bytes and not."""
    wide = torch.randn((40, 3, 4, 70), generator=torch.Generator().manual_seed(0)).cuda().to(BF16)
    slots = torch.arange(40).cuda()
    for k, v in ((wide[:, 0, :, :64], wide[:, 2, :, 3:67]), (wide[:, 1, :, 1:65].transpose(0, 0), wide[:, 1, :, :64])):
        a, b = TokenCache.empty(3, 4, 16, 64), TokenCache.empty(3, 4, 16, 64)
        a.append(k, v, slots)
        b.append(k.contiguous(), v.contiguous(), slots)
        for x, y in ((a.k_codes, b.k_codes), (a.v_codes, b.v_codes), (a.k_scale, b.k_scale), (a.v_scale, b.v_scale)):
            assert torch.equal(x, y)
        assert a.k_codes.any()


# ------------------------------------------------------------------------------------------------------- attention

class Setup:
    """A cache of random codes, a table of shuffled blocks, and the tokens' values in 64 bits."""

    def __init__(self, lens, heads, block, dim, codes, seed=0, width=None, spare=2):
        gen = torch.Generator().manual_seed(seed)
        held = [ref.blocks_of(a, block) for a in lens]
        self.lens, self.heads, self.block, self.dim = lens, heads, block, dim
        n_blocks = sum(held) + spare
        k, v = (_values(n_blocks, heads, block, dim, codes, gen) for _ in range(2))
        ks, vs = (torch.exp2(torch.randint(-8, -4, (n_blocks, heads), generator=gen).float()) * (1.37 if i else 1.0) for i in range(2))
        order = torch.randperm(n_blocks, generator=gen)
        width = width or max(1, max(held))
        table = torch.full((len(lens), width), -1, dtype=torch.int32)
        at = 0
        for b, h in enumerate(held):
            table[b, :h] = order[at:at + h].int()
            at += h
        # what no token owns is as bad as it can be: codes that are NaN, scales that are infinite
        if codes is E4:
            for b, a in enumerate(lens):
                if a % block:
                    for t in (k, v):
                        t.view(torch.int8)[int(table[b, a // block]), :, a % block:] = 0x7f
        for blk in order[at:]:
            ks[blk], vs[blk] = float("nan"), float("inf")
            if codes is E4:
                k.view(torch.int8)[blk], v.view(torch.int8)[blk] = 0x7f, 0x7f
        self.table = table
        self.k64, self.v64 = k.double() * ks.double()[:, :, None, None], v.double() * vs.double()[:, :, None, None]
        self.cache = TokenCache(k.cuda(), v.cuda(), ks.cuda(), vs.cuda())
        self.d_table, self.d_lens = table.cuda(), _gpu(lens)
        self.largest = float(vs[torch.isfinite(vs)].max()) * ref.QMAX[codes]

    def tokens(self, b, head, positions):
        """(keys, values) of these positions of request b, those of blocks that are none left out."""
        positions = np.asarray(positions, dtype=np.int64)
        blk = self.table[b].numpy()[positions // self.block] if len(positions) else np.zeros(0, np.int64)
        fine = (blk >= 0) & (blk < self.k64.shape[0])
        blk, off = torch.from_numpy(blk[fine].astype(np.int64)), torch.from_numpy(positions[fine] % self.block)
        return self.k64[blk, head, off], self.v64[blk, head, off]


def _compare(s, q, out, lse, see, scale, pick=None):
    """see(row) -> (request, positions by head) ; rows of which `pick` says so."""
    group = q.shape[1] // s.heads
    q64, out, lse = q.double().cpu(), out.double().cpu(), lse.double().cpu()
    for row in range(q.shape[0]) if pick is None else pick:
        for h in range(q.shape[1]):
            b, positions = see(row, h)
            keys, values = s.tokens(b, h // group, positions)
            want, want_lse, spread, qk, peak = ref.attend_row(q64[row, h], keys, values, scale)
            n = keys.shape[0]
            tol = ref.tolerance(want, spread, qk, peak, n, s.dim, q.dtype, s.largest)
            off = (out[row, h] - want).abs()
            assert bool((off <= tol).all()), (row, h, n, float((off / tol).max()))
            if n == 0:
                assert lse[row, h] == -np.inf
            else:
                assert abs(lse[row, h] - want_lse) <= ref.lse_tolerance(want_lse, qk, peak, n, s.dim), (row, h, float(lse[row, h]), want_lse)


def _queries(rows, heads, dim, dtype, seed=1):
    return torch.randn((rows, heads, dim), generator=torch.Generator().manual_seed(seed)).mul(1.5).to(dtype).cuda()


ONE = [
    # lens, kv heads, group, block, dim, codes, type
    ([1], 1, 1, 16, 16, I8, F32), ([0, 1, 2], 1, 1, 16, 64, E4, F16), ([17, 0, 400], 2, 4, 16, 128, I8, BF16), ([31, 32, 33, 127, 128, 129], 1, 3, 32, 128, E4, BF16),
    ([1000, 5], 2, 5, 64, 80, I8, F16), ([700], 3, 8, 128, 96, E4, F32), ([300, 257], 1, 16, 256, 64, I8, F32), ([513, 2], 1, 17, 16, 128, E4, F16),
    ([2049], 2, 2, 32, 256, I8, BF16), ([65, 90], 1, 33, 16, 192, E4, BF16), ([260], 2, 1, 64, 112, I8, F32), ([1500, 3], 1, 40, 64, 208, I8, F16), ([333], 1, 6, 16, 144, E4, F32),
    ([90, 5000], 1, 2, 16, 32, I8, BF16), ([2300], 1, 1, 128, 48, E4, F16)]


# requests in such numbers, and so short or long, that a call is cut in other ways: one wavefront each, eight, chunks of tokens
ONE += [([(7 * i) % 251 for i in range(300)], 4, 1, 16, 64, E4, BF16), ([1000 - i for i in range(3)], 2, 1, 32, 192, I8, F16), ([1024, 1025], 1, 2, 256, 256, E4, F32),
        ([256 - (i % 3) for i in range(520)], 2, 2, 256, 128, I8, F32), ([9000, 10, 4000], 1, 1, 32, 96, E4, BF16)]


@pytest.mark.parametrize("lens,heads,group,block,dim,codes,dtype", ONE)
def test_attend_one_token(lens, heads, group, block, dim, codes, dtype):
    s = Setup(lens, heads, block, dim, codes)
    q = _queries(len(lens), heads * group, dim, dtype)
    for max_len in (0, max(lens), 1, 10 ** 6):
        out, lse = s.cache.attend(q, s.d_table, s.d_lens, max_len=max_len)
        _compare(s, q, out, lse, lambda r, h: (r, np.arange(lens[r])), dim ** -0.5, pick=None if len(lens) < 100 else [0, 1, 36, 40, 255, 299])


MANY = [
    # lens, new rows, kv heads, group, block, dim, codes, type, causal
    ([40, 3, 0, 200], [5, 3, 0, 1], 2, 2, 16, 64, I8, BF16, True), ([20, 3], [7, 9], 1, 1, 16, 128, E4, F32, True), ([300, 64], [130, 64], 1, 4, 32, 128, I8, BF16, True),
    ([257, 90], [100, 30], 2, 1, 64, 80, E4, F16, False), ([70, 500, 1], [70, 33, 1], 1, 8, 128, 96, I8, F16, True), ([150], [200], 1, 2, 16, 256, E4, BF16, True),
    ([600, 0], [20, 4], 1, 3, 16, 192, I8, F32, False), ([129, 130], [129, 2], 3, 2, 256, 64, E4, BF16, True), ([1000], [300], 1, 1, 64, 112, I8, F32, True),
    ([333, 40], [64, 40], 1, 16, 32, 48, I8, BF16, False), ([90], [90], 1, 5, 16, 144, E4, F16, True)]


@pytest.mark.parametrize("lens,new,heads,group,block,dim,codes,dtype,causal", MANY)
def test_attend_many_tokens(lens, new, heads, group, block, dim, codes, dtype, causal):
    """Rows of several requests, some without rows and some with more rows than tokens (the first see nothing), and rows behind the
    last request, which stay as they are."""
    s = Setup(lens, heads, block, dim, codes)
    cu = np.concatenate([[0], np.cumsum(new)])
    rows, behind = int(cu[-1]), 3
    q = _queries(rows + behind, heads * group, dim, dtype)
    owner = np.repeat(np.arange(len(lens)), new)

    def see(r, h):
        b = owner[r]
        return b, np.arange(max(0, lens[b] - new[b] + (r - cu[b]) + 1) if causal else lens[b])

    L, cache = capi.lib(), s.cache
    c = capi.TokenCacheC(cache.k_codes.data_ptr(), cache.v_codes.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), *cache.k_codes.shape, int(codes is E4))
    c_at = ctypes.addressof(c)
    nbytes = L.hnsw_amd_cache_attend_workspace(c_at, rows + behind, heads * group, len(lens), s.table.shape[1], max(lens))
    work = torch.full((max(nbytes, 1),), 0xff, dtype=torch.uint8, device="cuda")
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    d_cu = _gpu(cu)
    capi.check(L.hnsw_amd_cache_attend_device(c_at, q.data_ptr(), rows + behind, heads * group, q.stride(0), q.stride(1), {F32: 0, F16: 1, BF16: 2}[dtype],
                                              s.d_table.data_ptr(), s.table.shape[1], s.d_lens.data_ptr(), len(lens), d_cu.data_ptr(), int(causal), dim ** -0.5, max(lens),
                                              out.data_ptr(), lse.data_ptr(), work.data_ptr(), nbytes, 0, torch.cuda.current_stream().cuda_stream))
    assert bool((out[rows:] == 7.0).all()) and bool((lse[rows:] == 7.0).all())
    _compare(s, q, out, lse, see, dim ** -0.5, pick=range(rows) if rows <= 150 else sorted(random.Random(0).sample(range(rows), 60)) + [rows - 1])
    out2, lse2 = cache.attend(q, s.d_table, s.d_lens, cu_q=d_cu, causal=causal)
    assert torch.equal(out2[:0], out[:0]) and torch.allclose(out2[:rows].float(), out[:rows].float(), rtol=2 ** -6, atol=1e-3)


FOUND = [
    # lens, kv heads, lists per kv head, group, block, dim, codes, type, ids
    ([1], 1, 1, 1, 16, 64, I8, F32, 5), ([100, 0, 9], 2, 1, 4, 16, 128, I8, BF16, 10), ([3000, 700], 2, 4, 4, 32, 128, E4, BF16, 100), ([900], 1, 2, 8, 64, 96, I8, F16, 257),
    ([5000, 1], 1, 1, 16, 128, 80, E4, F32, 1100), ([400], 1, 3, 3, 16, 256, I8, F16, 33), ([800, 60], 1, 1, 40, 32, 192, E4, BF16, 64), ([4000], 2, 1, 8, 16, 128, E4, F16, 4000),
    ([70], 3, 1, 1, 16, 48, I8, BF16, 1), ([i for i in range(600)], 2, 2, 4, 16, 128, E4, F16, 200), ([3 * i for i in range(300)], 4, 1, 1, 32, 256, I8, F32, 257),
    ([2000] * 3, 1, 2, 2, 64, 192, E4, BF16, 1000)]


@pytest.mark.parametrize("lens,heads,share,group,block,dim,codes,dtype,k", FOUND)
def test_attend_found(lens, heads, share, group, block, dim, codes, dtype, k):
    s = Setup(lens, heads, block, dim, codes)
    rng = np.random.default_rng(k)
    ids = np.full((len(lens), heads * share, k), -1, np.int32)
    for b, a in enumerate(lens):
        for h in range(heads * share):
            some = rng.permutation(a)[:k]
            ids[b, h, rng.permutation(k)[:len(some)]] = some                    # the padding lies anywhere
    if k >= 5:
        ids[0, 0, :3] = [lens[0], 2 ** 31 - 1, -2]                              # positions that are none
        ids[0, -1, 3] = ids[0, -1, 4] = 0                                       # one that is listed twice counts twice
    ids[-1, 0] = -1                                                             # a list that holds nothing
    q = _queries(len(lens), heads * group, dim, dtype)
    out, lse = s.cache.attend_found(q, s.d_table, s.d_lens, _gpu(ids))
    each = heads * group // (heads * share)
    _compare(s, q, out, lse, lambda r, h: (r, ref.visible(ids[r, h // each], lens[r])), dim ** -0.5, pick=None if len(lens) < 100 else [0, 1, 2, 150, 256, len(lens) - 1])


def test_work_that_needs_no_splitting_and_more_than_one_table():
    """So many rows that no chunk is cut, over more tokens (entries of a list) than a workgroup's table of blocks (tokens) holds; scales differ
    between the tables."""
    s = Setup([4500, 64], 8, 16, 64, E4)
    v = s.cache.v_scale.cpu()
    v[s.table[0, :256].long()] *= 2.0 ** -3
    s.cache.v_scale.copy_(v)
    s.v64 = s.cache.v_codes.cpu().double() * v.double()[:, :, None, None]
    new, cu = [600, 40], [0, 600, 640]
    q = _queries(640, 8 * 16, 64, BF16)
    out, lse = s.cache.attend(q, s.d_table, s.d_lens, cu_q=_gpu(cu))
    _compare(s, q[:, :], out, lse, lambda r, h: (int(r >= 600), np.arange([4500, 64][r >= 600] - [600, 40][r >= 600] + r - cu[int(r >= 600)] + 1)), 64 ** -0.5, pick=[0, 599, 600, 639])
    lens = [3000] * 64
    s = Setup(lens, 4, 64, 32, I8)
    ids = np.stack([np.random.default_rng(i).permutation(3000)[:1500] for i in range(64 * 16)]).reshape(64, 16, 1500).astype(np.int32)
    q = _queries(64, 16, 32, BF16)
    out, lse = s.cache.attend_found(q, s.d_table, s.d_lens, _gpu(ids))
    _compare(s, q, out, lse, lambda r, h: (r, ref.visible(ids[r, h], 3000)), 32 ** -0.5, pick=[0, 31, 63])


def test_attend_found_of_many_rows_sees_no_later_token():
    lens, new = [50, 9], [6, 12]
    s = Setup(lens, 1, 16, 64, I8)
    cu = np.concatenate([[0], np.cumsum(new)])
    owner = np.repeat(np.arange(2), new)
    ids = np.random.default_rng(0).integers(-1, 55, (18, 2, 40)).astype(np.int32)
    q = _queries(18, 4, 64, BF16)
    for causal in (True, False):
        out, lse = s.cache.attend_found(q, s.d_table, s.d_lens, _gpu(ids), cu_q=_gpu(cu), causal=causal)
        seen = lambda r: max(0, lens[owner[r]] - new[owner[r]] + r - cu[owner[r]] + 1) if causal else lens[owner[r]]  # noqa: E731, B023
        _compare(s, q, out, lse, lambda r, h: (owner[r], ref.visible(ids[r, h // 2], seen(r))), 64 ** -0.5)


def test_no_ids_and_no_rows():
    s = Setup([30, 4], 1, 16, 64, I8)
    q = _queries(2, 2, 64, F16)
    out, lse = s.cache.attend_found(q, s.d_table, s.d_lens, torch.empty((2, 1, 0), dtype=torch.int32, device="cuda"))
    assert not out.any() and bool((lse == -np.inf).all())
    out, lse = s.cache.attend(q[:0], s.d_table, s.d_lens, cu_q=_gpu([0, 0, 0]))
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)


@pytest.mark.parametrize("codes", [I8, E4])
def test_blocks_that_are_none(codes):
    """Block numbers outside the cache (tables of a request that has ended, a plan that was refused): their tokens do not exist."""
    lens = [100, 40, 70]
    s = Setup(lens, 2, 16, 64, codes)
    s.table[0, 1], s.table[0, 4], s.table[1] = -1, 10 ** 6, -5
    s.table[2, 4] = 2 ** 31 - 1
    s.d_table = s.table.cuda()
    q = _queries(3, 4, 64, BF16)
    out, lse = s.cache.attend(q, s.d_table, s.d_lens)
    _compare(s, q, out, lse, lambda r, h: (r, np.arange(lens[r])), 64 ** -0.5)
    assert not out[1].any()
    ids = np.stack([np.random.default_rng(i).permutation(100)[:64] for i in range(6)]).reshape(3, 2, 64).astype(np.int32)
    out, lse = s.cache.attend_found(q, s.d_table, s.d_lens, _gpu(ids))
    _compare(s, q, out, lse, lambda r, h: (r, ref.visible(ids[r, h // 2], lens[r])), 64 ** -0.5)
    rows = _queries(90, 4, 64, BF16)
    out, lse = s.cache.attend(rows, s.d_table, s.d_lens, cu_q=_gpu([0, 60, 60, 90]))
    cu, new = [0, 60, 60, 90], [60, 0, 30]
    owner = np.repeat(np.arange(3), new)
    _compare(s, rows, out, lse, lambda r, h: (owner[r], np.arange(lens[owner[r]] - new[owner[r]] + r - cu[owner[r]] + 1)), 64 ** -0.5)


@pytest.mark.parametrize("dim,codes,dtype,causal", [(16, I8, F32, True), (64, E4, BF16, True), (80, I8, F16, True), (128, I8, BF16, True), (128, E4, F32, False), (112, E4, F16, False), (96, I8, BF16, True)])
def test_many_rows_cut_for_longer_requests_than_there_are(dim, codes, dtype, causal):
    """The table is for 20000 tokens and the host knows no lengths: 128 rows a workgroup and chunks that most requests do not reach."""
    lens, new = [130, 1500, 64, 0, 601], [40, 200, 64, 3, 1]
    s = Setup(lens, 2, 16, dim, codes, width=1250)
    cu = np.concatenate([[0], np.cumsum(new)])
    owner = np.repeat(np.arange(5), new)
    q = _queries(int(cu[-1]), 6, dim, dtype)
    see = lambda r: max(0, lens[owner[r]] - new[owner[r]] + r - cu[owner[r]] + 1) if causal else lens[owner[r]]  # noqa: E731
    out, lse = s.cache.attend(q, s.d_table, s.d_lens, cu_q=_gpu(cu), causal=causal)
    _compare(s, q, out, lse, lambda r, h: (owner[r], np.arange(see(r))), dim ** -0.5)


@pytest.mark.parametrize("dim", [64, 128, 192])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_blocks_that_are_none_before_one_that_is_begun(dim, dtype):
    """The only block that exists holds few tokens; what lies behind those (codes that are NaN) does not reach the outputs, though tokens of
    no block read something."""
    lens, block = [2 * 128 + 5, 70], 128
    s = Setup(lens, 2, block, dim, E4)
    s.table[0, :2] = torch.tensor([-1, 10 ** 6])
    s.d_table = s.table.cuda()
    q = _queries(2, 4, dim, dtype)
    out, lse = s.cache.attend(q, s.d_table, s.d_lens)
    _compare(s, q, out, lse, lambda r, h: (r, np.arange(lens[r])), dim ** -0.5)
    for new in ([30, 0], [100, 60]):                                 # in registers, and through LDS
        rows, cu = _queries(sum(new), 4, dim, dtype), np.concatenate([[0], np.cumsum(new)])
        out, lse = s.cache.attend(rows, s.d_table, s.d_lens, cu_q=_gpu(cu))
        owner = np.repeat(np.arange(2), new)
        _compare(s, rows, out, lse, lambda r, h: (owner[r], np.arange(lens[owner[r]] - new[owner[r]] + r - cu[owner[r]] + 1)), dim ** -0.5)  # noqa: B023


@pytest.mark.parametrize("codes", [I8, E4])
def test_tables_whose_values_are_zeros(codes):
    """Blocks of zeros have the least scale there is, 2^-100; behind thousands of other tokens they fill a table of their own."""
    lens, dim = [14000], 64
    s = Setup(lens, 1, 16, dim, codes)
    vs = s.cache.v_scale.cpu() * 2.0 ** 20
    s.largest *= 2.0 ** 20
    zeros = s.table[0, 256:256 * 3].long()
    s.cache.v_codes.view(torch.int8)[zeros.cuda()] = 0
    vs[zeros] = 2.0 ** -100
    s.cache.v_scale.copy_(vs)
    s.v64 = s.cache.v_codes.cpu().double() * vs.double()[:, :, None, None]
    for rows in (1, 300):                                            # (a hint of one token: nothing is cut)
        q = _queries(rows, 8, dim, BF16)
        cu = None if rows == 1 else _gpu([0, rows])
        out, lse = s.cache.attend(q, s.d_table, s.d_lens, cu_q=cu, max_len=1)
        _compare(s, q, out, lse, lambda r, h: (0, np.arange(lens[0] - rows + r + 1)), dim ** -0.5, pick=[0, rows - 1])  # noqa: B023
    # lists of 1024 entries and more: first the others, then zeros, and the other way
    some = np.random.default_rng(0)
    full, none = some.permutation(4096)[:1024], 4096 + some.permutation(8000)[:1024]
    ids = np.stack([np.concatenate([full, none]), np.concatenate([none, full])])[None].repeat(800, 0).astype(np.int32)
    q = _queries(800, 2, dim, BF16)
    s1 = s.cache.attend_found(q, s.d_table, s.d_lens, _gpu(ids), cu_q=_gpu([0, 800]), causal=False)
    _compare(s, q, *s1, lambda r, h: (0, ids[r, h]), dim ** -0.5, pick=[0, 17, 799])


def test_every_row_in_one_of_as_many_requests():
    """As many rows as requests, but not one each."""
    lens = [40, 90, 7, 1, 0]
    s = Setup(lens, 1, 16, 64, I8)
    q = _queries(5, 20, 64, BF16)
    for cu in ([0, 0, 5, 5, 5, 5], [0, 2, 2, 2, 5, 5], [0, 0, 0, 0, 0, 5]):
        owner = np.searchsorted(cu, np.arange(5), side="right") - 1
        out, lse = s.cache.attend(q, s.d_table, s.d_lens, cu_q=_gpu(cu))
        see = lambda r: max(0, lens[owner[r]] - (cu[owner[r] + 1] - cu[owner[r]]) + r - cu[owner[r]] + 1)  # noqa: E731, B023
        _compare(s, q, out, lse, lambda r, h: (owner[r], np.arange(see(r))), 64 ** -0.5)


def test_queries_that_are_not_numbers_stay_alone():
    """A row with a NaN or an infinity gives no number, and its neighbours in the same tile what they give without it."""
    s = Setup([300], 1, 16, 64, I8)
    for rows in (16, 200):
        q = _queries(rows, 2, 64, BF16)
        want, want_lse = s.cache.attend(q, s.d_table, s.d_lens, cu_q=_gpu([0, rows]))
        bad = q.clone()
        bad[3, 1, 5], bad[9, 0, 0] = float("nan"), float("inf")
        out, lse = s.cache.attend(bad, s.d_table, s.d_lens, cu_q=_gpu([0, rows]))
        for r, h in ((3, 1), (9, 0)):
            assert bool(out[r, h].isnan().all()) and bool(lse[r, h].isnan())
            out[r, h], lse[r, h] = want[r, h], want_lse[r, h]
        assert torch.allclose(out.float(), want.float(), rtol=2.0 ** -7, atol=1e-3) and torch.allclose(lse, want_lse, rtol=1e-5, atol=1e-5)


def test_a_table_of_a_hundred_million_tokens():
    """The lengths are not known to the host, and the table is as wide as it may be."""
    s = Setup([700, 20], 1, 256, 64, I8, width=(2 ** 31 - 1) // 256)
    q = _queries(2, 2, 64, BF16)
    out, lse = s.cache.attend(q, s.d_table, s.d_lens)
    _compare(s, q, out, lse, lambda r, h: (r, np.arange(s.lens[r])), 64 ** -0.5)


def test_rows_behind_the_last_request_are_left_as_they_are():
    s = Setup([300, 20], 2, 16, 64, I8)
    for new, total in (([3, 2], 9), ([200, 10], 260)):
        q, cu = _queries(total, 4, 64, BF16), _gpu(np.concatenate([[0], np.cumsum(new)]))
        ids = _gpu(np.random.default_rng(1).integers(0, 300, (total, 2, 1500)).astype(np.int32))
        for found in (False, True):
            out, lse = torch.full((total, 4, 64), 7.0, dtype=BF16, device="cuda"), torch.full((total, 4), 7.0, device="cuda")
            c = s.cache
            desc = capi.TokenCacheC(c.k_codes.data_ptr(), c.v_codes.data_ptr(), c.k_scale.data_ptr(), c.v_scale.data_ptr(), c.n_blocks, c.n_heads, c.block_tokens, c.dim, capi.CODES_I8)
            L, at = capi.lib(), ctypes.byref(desc)
            front = (at, q.data_ptr(), total, 4, q.stride(0), q.stride(1), capi.TYPE_BF16, s.d_table.data_ptr(), s.d_table.shape[1], s.d_lens.data_ptr(), 2, cu.data_ptr(), 1)
            if found:
                bytes_ = L.hnsw_amd_cache_attend_found_workspace(at, total, 4, 2, 1500)
                work = torch.empty(max(bytes_, 16), dtype=torch.uint8, device="cuda")
                rc = L.hnsw_amd_cache_attend_found_device(*front, ids.data_ptr(), 2, 1500, 0.125, out.data_ptr(), lse.data_ptr(), work.data_ptr(), bytes_, 0, torch.cuda.current_stream().cuda_stream)
            else:
                bytes_ = L.hnsw_amd_cache_attend_workspace(at, total, 4, 2, s.d_table.shape[1], 0)
                work = torch.empty(max(bytes_, 16), dtype=torch.uint8, device="cuda")
                rc = L.hnsw_amd_cache_attend_device(*front, 0.125, 0, out.data_ptr(), lse.data_ptr(), work.data_ptr(), bytes_, 0, torch.cuda.current_stream().cuda_stream)
            capi.check(rc)
            n = sum(new)
            assert bool((out[n:] == 7.0).all()) and bool((lse[n:] == 7.0).all()) and not bool((lse[:n] == 7.0).any())


def test_lengths_that_are_none():
    """A negative length counts as 0, one beyond the table as the table's end."""
    s = Setup([64, 64, 64], 1, 16, 64, I8)
    q = _queries(3, 2, 64, F32)
    out, lse = s.cache.attend(q, s.d_table, _gpu([-3, 10 ** 9, 64]))
    want, want_lse = s.cache.attend(q, s.d_table, _gpu([0, 64, 64]))
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_offsets_past_32_bits():
    """Codes that lie more than 2^32 bytes into the buffers."""
    block, dim, heads = 256, 256, 1
    n_blocks = (1 << 32) // (block * dim) + 4
    cache = TokenCache.empty(n_blocks, heads, block, dim, I8)
    gen = torch.Generator().manual_seed(3)
    k = torch.randn((2 * block, heads, dim), generator=gen)
    slots = torch.arange((n_blocks - 2) * block, n_blocks * block)
    cache.append(k.cuda(), (-k).cuda(), slots.cuda())
    small = TokenCache.empty(2, heads, block, dim, I8)
    small.append(k.cuda(), (-k).cuda(), torch.arange(2 * block).cuda())
    assert torch.equal(cache.k_codes[-2:], small.k_codes) and small.k_codes.any()
    assert torch.equal(cache.read(slots.cuda())[1], small.read(torch.arange(2 * block).cuda())[1])
    ids = torch.arange(0, 500, 3, dtype=torch.int32, device="cuda").view(1, 1, -1)
    far, near, lens = _gpu([[n_blocks - 2, n_blocks - 1]]), _gpu([[0, 1]]), _gpu([500])
    for rows in (1, 80):
        q = _queries(rows, 2, dim, BF16)
        cu = _gpu([0, rows])
        assert all(torch.equal(a, b) for a, b in zip(cache.attend(q, far, lens, cu_q=cu), small.attend(q, near, lens, cu_q=cu)))
    q = _queries(1, 2, dim, BF16)
    assert all(torch.equal(a, b) for a, b in zip(cache.attend_found(q, far, lens, ids), small.attend_found(q, near, lens, ids)))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_strided_queries(dtype):
    """Queries cut out of a wider tensor, aligned to 16 bytes and not, and shared by the heads (a stride of 0)."""
    s = Setup([100, 37], 2, 16, 64, E4)
    wide = _queries(2, 7, 200, dtype)
    for q in (wide[:, 1:5, 8:72], wide[:, :4, 3:67], wide[:, 2:3, :64].expand(2, 4, 64), wide.transpose(0, 1)[:2, :2, 64:128].repeat(1, 2, 1)):
        a = s.cache.attend(q, s.d_table, s.d_lens)
        b = s.cache.attend(q.contiguous(), s.d_table, s.d_lens)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    big = _queries(60, 7, 200, dtype)
    cu = _gpu([0, 50, 60])
    for q in (big[:, 1:5, 8:72], big[:, :4, 3:67], big[:, 2:3, :64].expand(60, 4, 64)):
        a = s.cache.attend(q, s.d_table, s.d_lens, cu_q=cu)
        b = s.cache.attend(q.contiguous(), s.d_table, s.d_lens, cu_q=cu)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0, 1e-30, 300.0])
def test_scales_of_the_scores(scale):
    """Flat scores, turned ones, and scores so far apart that one token takes all."""
    lens = [200, 3]
    s = Setup(lens, 1, 32, 64, I8)
    q = _queries(2, 3, 64, F32)
    out, lse = s.cache.attend(q, s.d_table, s.d_lens, scale=scale)
    assert torch.isfinite(out).all()
    if abs(scale) <= 4.0:
        _compare(s, q, out, lse, lambda r, h: (r, np.arange(lens[r])), scale)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_queries_that_are_very_large_or_small(dtype):
    s = Setup([100, 50, 70, 20], 1, 16, 64, I8)
    q = _queries(4, 1, 64, dtype)
    size = {F32: 1e25, F16: 6e3, BF16: 1e25}[dtype]
    q[0] *= size
    q[1] /= size
    q[2] = 0
    q[3, :, 1:] = 0
    scales = [1 / size, 0.125, 0.125, 0.125]
    for r, scale in enumerate(scales):
        out, lse = s.cache.attend(q, s.d_table, s.d_lens, scale=scale)
        _compare(s, q, out, lse, lambda r, h: (r, np.arange(s.lens[r])), scale, pick=[r])


def test_values_whose_scales_differ_by_much():
    """Scales of neighbouring blocks that differ by 2^40: what weighs little by its probability must not vanish with it."""
    lens = [200]
    s = Setup(lens, 1, 16, 64, I8)
    vs = torch.exp2(torch.tensor([-20.0, 20.0, 0.0, 10.0, -20.0, 3.0, -7.0, 20.0, -20.0, -20.0, 5.0, 0.0, 1.0, 20.0, 0.0]))[:s.cache.n_blocks]
    s.v64 = s.cache.v_codes.cpu().double() * vs.double()[:, None, None, None]
    s.cache.v_scale.copy_(vs[:, None])
    s.largest = float(vs.max()) * 128
    q = _queries(1, 4, 64, F32)
    out, lse = s.cache.attend(q, s.d_table, s.d_lens)
    _compare(s, q, out, lse, lambda r, h: (r, np.arange(200)), 64 ** -0.5)


# --------------------------------------------------------------------------------------- streams, graphs, refusals

def test_on_another_stream_and_two_calls_at_once():
    s = Setup([3000, 500], 2, 32, 128, I8)
    q = [_queries(2, 8, 128, BF16, seed=i) for i in range(6)]
    ids = _gpu(np.random.default_rng(0).integers(0, 400, (2, 2, 90)).astype(np.int32))
    want = [s.cache.attend(x, s.d_table, s.d_lens) + s.cache.attend_found(x, s.d_table, s.d_lens, ids) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [None] * 6
    for i, x in enumerate(q):
        with torch.cuda.stream(streams[i % 3]):
            got[i] = s.cache.attend(x, s.d_table, s.d_lens) + s.cache.attend_found(x, s.d_table, s.d_lens, ids)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_decoding_step_captured_and_replayed():
    """plan, append, attend and attend_found in one graph, replayed as the lengths grow, against the same calls made eagerly on a
    second cache."""
    heads, block, dim, width, n_blocks = 2, 16, 64, 8, 24
    gen = torch.Generator().manual_seed(9)

    def fresh():
        return dict(cache=TokenCache.empty(n_blocks, heads, block, dim, E4), lens=_gpu([0, 14, 31]), table=_gpu([[-1] * width] * 3), ring=torch.arange(n_blocks, dtype=torch.int32).cuda(),
                    state=_gpu([0, n_blocks], torch.int64), grow=_gpu([1, 1, 1]), k=torch.zeros((3, heads, dim), dtype=BF16, device="cuda"),
                    v=torch.zeros((3, heads, dim), dtype=BF16, device="cuda"), q=torch.zeros((3, 4, dim), dtype=BF16, device="cuda"),
                    ids=torch.zeros((3, heads, 20), dtype=torch.int32, device="cuda"))

    def step(w):
        p = cache_plan(w["lens"], w["grow"], w["table"], w["ring"], w["state"], block_tokens=block, n_slots=3)
        w["cache"].append(w["k"], w["v"], p.slots)
        a = w["cache"].attend(w["q"], w["table"], p.lens, max_len=128)
        f = w["cache"].attend_found(w["q"], w["table"], p.lens, w["ids"])
        w["lens"].copy_(p.lens)
        w["state"].copy_(p.state)
        return a + f

    eager, caught = fresh(), fresh()
    for w in (eager, caught):                       # requests that hold tokens already: their blocks, and rows in them
        first = cache_plan(_gpu([0, 0, 0]), w["lens"], w["table"], w["ring"], w["state"], block_tokens=block, n_slots=45)
        assert first.status.item() == 0
        rows = torch.randn((45, heads, dim), generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
        w["cache"].append(rows, -rows, first.slots)
        w["state"].copy_(first.state)
    warm = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(warm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(caught)
    for i in range(40):
        for name in ("k", "v", "q"):
            x = torch.randn(eager[name].shape, generator=gen).to(BF16).cuda() * (1 + i % 5)
            eager[name].copy_(x)
            caught[name].copy_(x)
        x = torch.randint(-1, 60, eager["ids"].shape, generator=gen).int().cuda()
        eager["ids"].copy_(x)
        caught["ids"].copy_(x)
        want = step(eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), i
        assert torch.equal(caught["lens"], eager["lens"]) and torch.equal(caught["table"], eager["table"])
        assert torch.isfinite(want[0]).all() and want[0].abs().sum() > 0


def test_a_plan_of_many_requests_captured():
    """The largest call there is, in a graph that is replayed with other lengths."""
    n, block, rng = 8192, 16, random.Random(5)
    lens = [rng.randint(0, 40) for _ in range(n)]
    d = dict(lens=_gpu(lens), grow=_gpu([0] * n), table=torch.full((n, 6), -1, dtype=torch.int32, device="cuda"), ring=torch.arange(4 * n, dtype=torch.int32).cuda(),
             state=_gpu([0, 4 * n], torch.int64))
    plan_ = lambda: cache_plan(d["lens"], d["grow"], d["table"], d["ring"], d["state"], block_tokens=block, n_slots=3 * n)  # noqa: E731
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p = plan_()
    table, ring, state = [[-1] * 6 for _ in range(n)], list(range(4 * n)), [0, 4 * n]
    lens = [0] * n
    for step in range(4):
        grow = [rng.randint(0, 3) if rng.random() < 0.9 or not step else -1 for _ in range(n)]
        d["lens"].copy_(_gpu(lens))
        d["grow"].copy_(_gpu(grow))
        d["state"].copy_(_gpu(state, torch.int64))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        slots, cu, lens, state, status, table, ring = ref.plan(lens, grow, table, ring, state, block, 3 * n)
        assert p.status.item() == status == 0 and p.slots.tolist() == slots and p.cu_new.tolist() == cu and p.lens.tolist() == lens
        assert p.state.tolist() == state and d["table"].tolist() == table and d["ring"].tolist() == ring


def test_two_graphs_of_split_work_at_once():
    """Each graph has a workspace of its own, so that their replays may overlap."""
    s = Setup([5000, 3000], 2, 32, 128, I8)
    q = [_queries(2, 4, 128, BF16, seed=i) for i in range(2)]
    want = [s.cache.attend(x, s.d_table, s.d_lens, max_len=20000) for x in q]
    graphs, outs = [], []
    for x in q:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(s.cache.attend(x, s.d_table, s.d_lens, max_len=20000))
    streams = [torch.cuda.Stream() for _ in q]
    for _ in range(5):
        for o in outs:
            o[0].zero_()
            o[1].zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1])


def test_python_refuses():
    s = Setup([30, 4], 2, 16, 64, I8)
    c, t, n = s.cache, s.d_table, s.d_lens
    q = _queries(2, 4, 64, BF16)
    for bad in (lambda: c.attend(q[:, :3], t, n), lambda: c.attend(q[..., :48], t, n), lambda: c.attend(q.double(), t, n), lambda: c.attend(q.cpu(), t, n),
                lambda: c.attend(q, t.long(), n), lambda: c.attend(q, t[:1], n), lambda: c.attend(q, t, n, cu_q=_gpu([0, 1])), lambda: c.attend(q.transpose(1, 2), t, n),
                lambda: c.attend(q.float().requires_grad_(), t, n), lambda: c.attend_found(q, t, n, _gpu(np.zeros((2, 2)))), lambda: c.attend_found(q, t, n, _gpu(np.zeros((1, 2, 3)))),
                lambda: c.append(q, q, _gpu([0, 1], torch.int64)), lambda: c.append(q[:, :2], q[:1, :2], _gpu([0, 1], torch.int64)), lambda: c.append(q[:, :2], q[:, :2], _gpu([0, 1])),
                lambda: c.read(_gpu([0, 1])), lambda: c.read(_gpu([0], torch.int64), torch.float64), lambda: TokenCache(c.k_codes, c.v_codes[1:], c.k_scale, c.v_scale),
                lambda: TokenCache(c.k_codes.float(), c.v_codes.float(), c.k_scale, c.v_scale), lambda: TokenCache(c.k_codes, c.v_codes, c.k_scale.half(), c.v_scale),
                lambda: cache_plan(n, n.long(), t, t[0], _gpu([0, 0], torch.int64), block_tokens=16, n_slots=2)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: c.attend(q[:1], t, n), lambda: c.attend(q, t, n, scale=float("nan")), lambda: c.attend_found(q, t, n, _gpu(np.zeros((2, 3, 4))))):
        with pytest.raises(capi.HnswAmdError) as e:
            bad()
        assert e.value.code == capi.E_ARG
    with torch.no_grad():
        c.attend(q.float().requires_grad_(), t, n)


# ---------------------------------------------------------------------------------------------- the index and the cache

def test_attention_over_what_the_index_finds():
    """A request's stored keys are read back and indexed; a search lists tokens for each query head, and attention over the listed tokens
    that hold nearly all of the softmax's weight is near attention over all tokens, and equal to it when the list holds all."""
    heads, group, dim, block, n = 2, 2, 64, 32, 1500
    gen = torch.Generator().manual_seed(4)
    k = torch.nn.functional.normalize(torch.randn((n, heads, dim), generator=gen), dim=-1)
    v = torch.randn((n, heads, dim), generator=gen)
    width = ref.blocks_of(n, block)
    cache = TokenCache.empty(width + 1, heads, block, dim, I8)
    table, ring, state = torch.full((1, width), -1, dtype=torch.int32, device="cuda"), torch.arange(width + 1, dtype=torch.int32).cuda(), _gpu([0, width + 1], torch.int64)
    p = cache_plan(_gpu([0]), _gpu([n]), table, ring, state, block_tokens=block, n_slots=n)
    cache.append(k.cuda(), v.cuda(), p.slots)
    stored = cache.read(p.slots)[0].cpu().numpy()
    q = (k[torch.randperm(n, generator=gen)[:heads * group]][:, 0] + 0.2 * torch.randn((heads * group, dim), generator=gen))
    for h in range(heads):
        q[h * group:(h + 1) * group] = k[torch.randperm(n, generator=gen)[:group], h] * 1.0
    q = q.view(1, heads * group, dim)
    ids = torch.empty((1, heads * group, 64), dtype=torch.int32, device="cuda")
    for h in range(heads):
        index = HNSW(16, 32, 100)
        index.init(dim, n)
        index.insert_batch(np.ascontiguousarray(stored[:, h]))
        index.sync_device(0)
        dist = torch.empty((group, 64), dtype=torch.float32, device="cuda")
        d_q = torch.nn.functional.normalize(q[0, h * group:(h + 1) * group], dim=-1).cuda().contiguous()
        index.search_batch_device(d_q.data_ptr(), group, 100, 64, ids[0, h * group].data_ptr(), dist.data_ptr(), stream=torch.cuda.current_stream().cuda_stream,
                                  flags=capi.KEYS_FLOAT)
    qd = q.cuda()
    scale = 40.0                                        # sharp: the listed tokens hold nearly all the weight
    some, some_lse = cache.attend_found(qd, table, p.lens, ids, scale=scale)
    full, full_lse = cache.attend(qd, table, p.lens, scale=scale)
    # the weight outside the list, computed: what it can move the output by is twice that times the largest value
    s64 = torch.einsum("hgd,nhd->hgn", q.view(heads, group, dim).double(), torch.from_numpy(stored).double()) * scale
    w = torch.softmax(s64, -1).view(heads * group, n)
    missed = 1 - w.gather(1, ids[0].cpu().long()).sum(-1)
    assert float(missed.max()) < 0.05
    most = float(cache.read(p.slots)[1].abs().max())
    assert bool(((some - full).abs().cpu()[0].amax(-1) <= 2 * missed * most + 1e-3).all())
    assert bool((some_lse <= full_lse + 1e-4).all())
    every = torch.arange(n, dtype=torch.int32, device="cuda").flip(0).expand(1, heads, n).contiguous()
    out, lse = cache.attend_found(qd, table, p.lens, every, scale=scale)
    assert torch.allclose(out, full, rtol=1e-4, atol=1e-4) and torch.allclose(lse, full_lse, rtol=1e-5, atol=1e-4)
