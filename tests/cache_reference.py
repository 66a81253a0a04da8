"""Plain statements of the token cache's operators, on the host and in 64 bits, for the tests."""
import math

import numpy as np
import torch

QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def blocks_of(n, block):
    return -(-n // block)


def plan(lens, grow, table, ring, state, block, n_slots):
    """What hnsw_amd_cache_plan_device documents, step by step, on lists: (slots, cu, lens, state, status, table, ring)."""
    lens, grow, ring, table = list(lens), list(grow), list(ring), [list(r) for r in table]
    head, tail = state
    n, width = len(ring), len(table[0])
    status = 0
    if any(a < 0 for a in lens) or any(g < -1 for g in grow) or head < 0 or not 0 <= tail - head <= n:
        status |= 8
    if any(blocks_of(max(a, 0) + max(g, 0), block) > width for a, g in zip(lens, grow)):
        status |= 2
    if sum(max(g, 0) for g in grow) > n_slots:
        status |= 4
    need = [blocks_of(max(a, 0) + max(g, 0), block) - blocks_of(max(a, 0), block) for a, g in zip(lens, grow)]
    back = [blocks_of(a, block) if g == -1 else 0 for a, g in zip(lens, grow)]
    if not status and sum(need) > tail - head:
        status |= 1
    if not status and sum(back) > n - (tail - head):
        status |= 8
    if status:
        return [-1] * n_slots, [0] * (len(lens) + 1), lens, [head, tail], status, table, ring
    before, slots, cu, given, taken = list(ring), [], [0], 0, 0
    for b, (a, g) in enumerate(zip(lens, grow)):
        held = blocks_of(a, block)
        if g == -1:
            for j in range(held):
                ring[(tail + given) % n] = table[b][j]
                given += 1
        for j in range(need[b]):
            table[b][held + j] = before[(head + taken) % n]
            taken += 1
        for p in range(a, a + max(g, 0)):
            blk = table[b][p // block]
            slots.append(blk * block + p % block if 0 <= blk < n else -1)
        cu.append(cu[-1] + max(g, 0))
    after = [0 if g == -1 else a + g for a, g in zip(lens, grow)]
    return slots + [-1] * (n_slots - len(slots)), cu, after, [head + taken, tail + given], 0, table, ring


def nearest(x, dtype):
    """Codes of 64-bit values that are divided by their scale, as 64-bit values."""
    most = QMAX[dtype]
    x = torch.nan_to_num(x, nan=0.0, posinf=most, neginf=-most).clamp(-most, most)
    if dtype is torch.int8:
        return x.round()                                                  # ties to even
    a = x.abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)      # e4m3: 3 bits behind the leading one, smallest normal 2^-6
    return torch.copysign((a / step).round() * step, x)


def append(values, scale, rows, slots, block, dtype):
    """values: 64-bit codes [n_blocks, heads, block, dim], scale [n_blocks, heads] (both changed in place); rows 64-bit [n, heads, dim]."""
    most = QMAX[dtype]
    n_slots = values.shape[0] * block
    t = 0
    while t < len(slots):
        s = slots[t]
        if not 0 <= s < n_slots:
            t += 1
            continue
        n = 1
        while t + n < len(slots) and slots[t + n] == s + n and s % block + n < block:
            n += 1
        blk, off = s // block, s % block
        for h in range(values.shape[1]):
            x = rows[t:t + n, h]
            fine = x.abs()[torch.isfinite(x)]
            peak = float(fine.max()) if fine.numel() else 0.0
            e = -100
            while e < 121 and peak > most * 2.0 ** e:
                e += 1
            before = float(scale[blk, h])
            if off > 0 and 0 < before < math.inf:
                e = max(e, max(-100, min(121, math.ceil(math.log2(before)))))
                if 2.0 ** e != before:
                    kept = torch.ones(block, dtype=torch.bool)
                    kept[off:off + n] = False
                    values[blk, h, kept] = nearest(values[blk, h, kept] * (before / 2.0 ** e), dtype)
            scale[blk, h] = 2.0 ** e
            values[blk, h, off:off + n] = nearest(x / 2.0 ** e, dtype)
        t += n


def attend_row(q, keys, values, scale):
    """One query [dim] over the tokens it sees [n, dim], in 64 bits: (out, lse, sum p |v| / sum p, largest sum |q k| * scale, largest |score|)."""
    if keys.shape[0] == 0:
        z = torch.zeros_like(q)
        return z, -math.inf, z, 0.0, 0.0
    s = keys @ q * scale
    top = s.max()
    p = torch.exp(s - top)
    total = p.sum()
    return (p @ values) / total, float(top + torch.log(total)), (p @ values.abs()) / total, float((keys.abs() @ q.abs()).max() * abs(scale)), float(s.abs().max())


def tolerance(out, spread, qk, peak, n, dim, dtype, largest=0.0):
    """How far an output may be from `out`.  The result is rounded once to `dtype`: half a step of the value.  Inside, scores are sums of
    dim products in 32 bits (each step off by half a step of a partial sum, at most qk: (dim + 8) 2^-24 qk with the query's
    split into halves, the scale and the base-2 logarithm's factor), the exponential adds its argument's rounding and its own, probabilities that meet
    the values as 16-bit floats are off by 2^-11 of themselves, and sums over n tokens by n 2^-24.
    Those 16-bit floats have a smallest step: a token's weight, its probability (1 at the softmax's reference, which is one of the row's
    scores) times its value scale over the largest scale S, is held in units of 2^-11, where the step is never under 2^-24, so it is off
    by up to half of that, 2^-25 2^-11 = 2^-36, whatever its size.  That meets a code of at most C and the unit S: n tokens move the
    sum by n 2^-36 S C at most (`largest` is S C), and the sum of the probabilities that it is divided by is at least 1."""
    half = torch.finfo(dtype).eps / 2
    score = (dim + 8) * 2.0 ** -24 * qk
    p = 2 * (score + 2.0 ** -22 * (1 + peak)) + 2 * n * 2.0 ** -24 + 2.0 ** -22
    if dtype is not torch.float32:
        p += 2.0 ** -11
    least = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps       # values under the smallest normal round by a fixed step
    return half * out.abs() + (spread * p + n * 2.0 ** -36 * largest) * (1 + half) + least


def lse_tolerance(lse, qk, peak, n, dim):
    return (dim + 8) * 2.0 ** -24 * qk + 2.0 ** -22 * (1 + peak) + n * 2.0 ** -24 + 2.0 ** -22 * abs(lse)


def visible(ids, seen):
    """Listed positions that count, in order (an unsigned view: -1 is behind everything)."""
    u = np.asarray(ids).astype(np.uint32).astype(np.int64)
    return u[u < seen]
