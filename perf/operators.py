"""The token cache's operators as they are measured: cases, inputs, plain forms and the framework's calls.

The cache holds the keys and values of a language model's tokens in 8 bits, in blocks of `block` tokens, with one scale
for each block and head:

  codes  [n_blocks, kv_heads, block, dim]  int8 or float8_e4m3fn        value = code * scale
  scale  [n_blocks, kv_heads]              float32, a power of two where this framework wrote it

Requests own blocks through a table [batch, width]; free blocks wait in a ring (`ring`, and [head, tail] in `state`).

  plan    grows (or, at -1, ends) requests: takes blocks off the ring, fills the table, maps every new token to its slot
  append  quantises new rows into their slots, and reads back every token of the blocks it touched (as a caller does that
          indexes the stored keys for searching)
  attend  softmax attention of queries over all cached tokens of their request
  found   the same over the tokens that a search listed for each query token and head
"""
import math
import random

import torch

own = False

QMAX = {"int8": 127.0, "e4m3": 448.0}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
ROWS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one decoding step of 64 requests: one new token each
        {"name": "plan_step", "kind": "plan", "batch": 64, "len_lo": 1, "len_hi": 8192, "grow_lo": 1, "grow_hi": 1, "ended": 0.0, "block": 32, "pattern": 1},
        # a scheduler's step with prompts among the running requests, some of them ending
        {"name": "plan_prompts", "kind": "plan", "batch": 1000, "len_lo": 0, "len_hi": 3000, "grow_lo": 0, "grow_hi": 700, "ended": 0.1, "block": 16, "pattern": 2},
        # the same decoding step's 64 new rows
        {"name": "append_step", "kind": "append", "batch": 64, "len_lo": 0, "len_hi": 2000, "grow_lo": 1, "grow_hi": 1, "kv_heads": 8, "dim": 128, "block": 32, "codes": "int8", "rows": "bf16", "pattern": 3},
        # three prompts written at once, one of them behind an earlier part
        {"name": "append_prompts", "kind": "append", "batch": 3, "len_lo": 0, "len_hi": 100, "grow_lo": 5000, "grow_hi": 8001, "kv_heads": 8, "dim": 128, "block": 64, "codes": "e4m3", "rows": "f16", "pattern": 4},
        # the smallest call: one short request
        {"name": "attend_single", "kind": "attend", "batch": 1, "len_lo": 777, "len_hi": 777, "new_lo": 0, "new_hi": 0, "q_heads": 8, "kv_heads": 8, "dim": 64, "block": 16, "codes": "int8", "rows": "f16", "causal": True, "pattern": 5},
        # an ordinary decoding step: 64 requests of all lengths up to 8k, four query heads to a key head
        {"name": "attend_step", "kind": "attend", "batch": 64, "len_lo": 1, "len_hi": 8192, "new_lo": 0, "new_hi": 0, "q_heads": 32, "kv_heads": 8, "dim": 128, "block": 32, "codes": "e4m3", "rows": "bf16", "causal": True, "pattern": 6},
        # two long contexts
        {"name": "attend_long", "kind": "attend", "batch": 2, "len_lo": 150001, "len_hi": 200000, "new_lo": 0, "new_hi": 0, "q_heads": 64, "kv_heads": 8, "dim": 128, "block": 128, "codes": "int8", "rows": "bf16", "causal": True, "pattern": 7},
        # 32-bit queries (the type this framework's searches take), 96 dims
        {"name": "attend_f32", "kind": "attend", "batch": 17, "len_lo": 100, "len_hi": 3000, "new_lo": 0, "new_hi": 0, "q_heads": 12, "kv_heads": 4, "dim": 96, "block": 64, "codes": "int8", "rows": "f32", "causal": True, "pattern": 8},
        # parts of three prompts, each behind what is cached of it
        {"name": "attend_prompts", "kind": "attend", "batch": 3, "len_lo": 2000, "len_hi": 6000, "new_lo": 700, "new_hi": 1500, "q_heads": 32, "kv_heads": 8, "dim": 128, "block": 64, "codes": "int8", "rows": "bf16", "causal": True, "pattern": 9},
        # a decoder's tokens over an encoder's stored states (no mask)
        {"name": "attend_states", "kind": "attend", "batch": 8, "len_lo": 500, "len_hi": 1500, "new_lo": 100, "new_hi": 227, "q_heads": 16, "kv_heads": 16, "dim": 64, "block": 32, "codes": "e4m3", "rows": "f16", "causal": False, "pattern": 10},
        # a decoding step over what a search found for every query head
        {"name": "found_heads", "kind": "found", "batch": 64, "len_lo": 1000, "len_hi": 30000, "listed": 100, "list_heads": 32, "q_heads": 32, "kv_heads": 8, "dim": 128, "block": 32, "codes": "int8", "rows": "bf16", "pattern": 11},
        # few requests, long contexts, long lists shared by the query heads of a key head
        {"name": "found_shared", "kind": "found", "batch": 6, "len_lo": 100000, "len_hi": 262144, "listed": 4001, "list_heads": 8, "q_heads": 64, "kv_heads": 8, "dim": 128, "block": 64, "codes": "e4m3", "rows": "f16", "pattern": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "append", "attend", "attend", "attend", "found"])
    block, pattern = rng.choice([16, 32, 64, 128]), rng.randrange(1 << 20)
    codes, rows = rng.choice(["int8", "e4m3"]), rng.choice(["bf16", "bf16", "f16", "f32"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8, 16])
    dim = rng.choice([64, 80, 96, 112, 128, 128, 192, 256])
    if kind == "plan":
        batch = _log(rng, 1, 2000)
        few = rng.random() < 0.5
        return {"kind": kind, "batch": batch, "len_lo": 0, "len_hi": _log(rng, 1, 9000), "grow_lo": 0, "grow_hi": 1 if few else max(1, _log(rng, 1, 600000) // batch),
                "ended": rng.choice([0.0, 0.1]), "block": block, "pattern": pattern}
    if kind == "append":
        batch = _log(rng, 1, 200)
        return {"kind": kind, "batch": batch, "len_lo": 0, "len_hi": _log(rng, 1, 2000), "grow_lo": 1, "grow_hi": 1 if rng.random() < 0.5 else max(1, _log(rng, 1, 20000) // batch),
                "kv_heads": kv_heads, "dim": dim, "block": block, "codes": codes, "rows": rows, "pattern": pattern}
    if kind == "found":
        batch = _log(rng, 1, 64)
        lists = kv_heads * rng.choice([g for g in range(1, group + 1) if group % g == 0])
        return {"kind": kind, "batch": batch, "len_lo": 1, "len_hi": max(1, _log(rng, 100, 1000000) // batch), "listed": max(1, min(4001, _log(rng, 10, 400000) // (batch * lists))),
                "list_heads": lists, "q_heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "block": block, "codes": codes, "rows": rows, "pattern": pattern}
    batch = _log(rng, 1, 64)
    new = rng.choice([0, 0, 4, 300])
    if new:
        batch = min(batch, 8)
    tokens = _log(rng, 200, 300000 if not new else 12000 if new > 4 else 60000)
    case = {"kind": kind, "batch": batch, "len_lo": 0 if rng.random() < 0.3 else 1, "len_hi": max(1, tokens // batch), "new_lo": 1 if new else 0, "new_hi": new,
            "q_heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "block": block, "codes": codes, "rows": rows, "causal": rng.random() < 0.7, "pattern": pattern}
    while work(case)["bytes"] > 6e8 or work(case)["flops"] > 1.5e11:                  # no dearer than the listed ones
        case["len_hi"] = case["len_hi"] * 2 // 3
    return case


def _lengths(case):
    """Lengths before the call and tokens that come with it, one of each for every request: part of the case, not of the seed."""
    rng = random.Random(case["pattern"])
    lens = [rng.randint(case["len_lo"], case["len_hi"]) for _ in range(case["batch"])]
    lo, hi = (case["grow_lo"], case["grow_hi"]) if "grow_lo" in case else (case.get("new_lo", 0), case.get("new_hi", 0))
    new = [rng.randint(lo, hi) for _ in lens]
    if case["kind"] == "plan":
        new = [-1 if rng.random() < case["ended"] else n for n in new]
    return lens, new


def _blocks(n, block):
    return -(-n // block)


def work(case):
    lens, new = _lengths(case)
    block, batch = case["block"], case["batch"]
    if case["kind"] == "plan":
        grown = sum(max(n, 0) for n in new)
        taken = sum(_blocks(a + max(n, 0), block) - _blocks(a, block) for a, n in zip(lens, new))
        given = sum(_blocks(a, block) for a, n in zip(lens, new) if n < 0)
        return {"bytes": 16 * batch + 8 * (taken + given) + 8 * grown + 40, "flops": 0}
    kv, dim = case["kv_heads"], case["dim"]
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["rows"]]
    if case["kind"] == "append":
        grown = sum(new)
        back = sum(a + n - (a // block) * block for a, n in zip(lens, new))      # tokens of the blocks that are touched
        touched = sum(_blocks(a + n, block) - a // block for a, n in zip(lens, new))
        # new rows read and their codes written; every code and scale of the touched blocks read again, values written in 32 bits
        return {"bytes": 2 * kv * dim * (grown * (size + 1) + back * (1 + 4)) + 16 * kv * touched + 8 * (grown + back), "flops": 0}
    q_heads = case["q_heads"]
    if case["kind"] == "found":
        pairs = sum(min(case["listed"], a) for a in lens)
        rows = pairs * case["list_heads"]
        return {"bytes": rows * (2 * dim + 4 + 8) + 2 * batch * q_heads * dim * size + 4 * batch * q_heads, "flops": 4 * dim * q_heads * pairs}
    if not case["new_hi"]:
        tokens, pairs = batch, sum(lens)
    else:
        tokens = sum(new)
        pairs = sum(sum(max(0, a - n + i + 1) for i in range(n)) if case["causal"] else a * n for a, n in zip(lens, new))
    cached = sum(lens)
    return {"bytes": 2 * kv * (cached * dim + 4 * sum(_blocks(a, block) for a in lens)) + 2 * tokens * q_heads * dim * size + 4 * tokens * q_heads, "flops": 4 * dim * q_heads * pairs}


# --------------------------------------------------------------------------------------------------------- inputs

def _fill(n_blocks, case, gen, dev):
    """Codes and scales as quantising normal values gives them: codes fill the upper half of their range, scales differ by block."""
    shape = (n_blocks, case["kv_heads"], case["block"], case["dim"])
    x = torch.randn(shape, generator=gen, device=dev, dtype=torch.float16)
    if case["codes"] == "int8":
        codes, base = (x * 28).round().clamp(-127, 127).to(torch.int8), -5
    else:
        codes, base = (x * 70).clamp(-448, 448).to(torch.float8_e4m3fn), -6
    scale = torch.exp2(torch.randint(base, base + 2, shape[:2], generator=gen, device=dev).float())
    return codes, scale


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    cpu = torch.Generator().manual_seed(int(seed))
    lens, new = _lengths(case)
    block, batch, kind = case["block"], case["batch"], case["kind"]
    grown = [max(n, 0) for n in new]
    total = [a + n if kind in ("plan", "append") else a for a, n in zip(lens, grown)]
    width = max(1, max(_blocks(a, block) for a in total))
    held = [_blocks(a, block) for a in (lens if kind == "plan" else total)]
    n_blocks = sum(held) + (sum(_blocks(a, block) - h for a, h in zip(total, held)) if kind == "plan" else 0) + 3
    order = torch.randperm(n_blocks, generator=cpu, dtype=torch.int64).to(torch.int32)
    ends = torch.tensor(held).cumsum(0)
    at = torch.arange(width)[None, :]
    own_of = at < torch.tensor(held)[:, None]
    table = torch.where(own_of, order[(at + (ends - torch.tensor(held))[:, None]).clamp(max=n_blocks - 1)], -1).to(torch.int32)
    s = {"kind": kind, "block": block, "case": dict(case), "lens": torch.tensor(lens, dtype=torch.int32, device=dev)}
    if kind == "plan":
        used = sum(held)
        start = int(torch.randint(0, 5 * n_blocks, (1,), generator=cpu))           # the ring has gone round before
        ring = torch.empty(n_blocks, dtype=torch.int32)
        ring[(torch.arange(n_blocks) + start) % n_blocks] = torch.cat([order[used:], order[:used].flip(0)])
        s.update(grow=torch.tensor(new, dtype=torch.int32, device=dev), table=table.to(dev), ring=ring.to(dev),
                 state=torch.tensor([start, start + n_blocks - used], dtype=torch.int64, device=dev), n_slots=max(1, sum(grown)))
        return s
    s["table"] = table.to(dev)
    s["k"], s["k_scale"] = _fill(n_blocks, case, gen, dev)
    s["v"], s["v_scale"] = _fill(n_blocks, case, gen, dev)
    dtype = ROWS[case["rows"]]
    if kind == "append":
        slots, back = [], []
        for b in range(batch):
            for out, lo in ((slots, lens[b]), (back, lens[b] // block * block)):
                p = torch.arange(lo, lens[b] + new[b])
                out.append(table[b][p // block].long() * block + p % block)
        s["slots"], s["back"] = torch.cat(slots).to(dev), torch.cat(back).to(dev)
        n = s["slots"].numel()
        for name in ("new_k", "new_v"):
            x = torch.randn((n, case["kv_heads"], case["dim"]), generator=gen, device=dev)
            s[name] = (x * torch.exp(0.3 * torch.randn((n, 1, 1), generator=gen, device=dev))).to(dtype)     # some tokens are louder
        return s
    tokens = sum(new) if case.get("new_hi") else batch
    s["q"] = (1.5 * torch.randn((tokens, case["q_heads"], case["dim"]), generator=gen, device=dev)).to(dtype)
    s["cu"] = torch.tensor([0] + new, dtype=torch.int32).cumsum(0).to(torch.int32).to(dev) if case.get("new_hi") else None
    s["max_new"] = max(new) if case.get("new_hi") else 1
    s["max_len"] = max(lens)
    if kind == "found":
        # distinct tokens in no order, as a search leaves them; short requests' lists end early, padded with -1
        k = case["listed"]
        stride = torch.randint(0, 1 << 30, (batch, case["list_heads"], 1), generator=gen, device=dev)
        first = torch.randint(0, 1 << 30, (batch, case["list_heads"], 1), generator=gen, device=dev)
        n = s["lens"].long().view(-1, 1, 1)
        step = torch.clamp(n // max(k, 1), min=1)
        j = torch.arange(k, device=dev).view(1, 1, -1)
        rot = (j * 7919 + stride) % k if math.gcd(7919, k) == 1 else (j + stride) % k
        ids = torch.where(n >= k, (rot * step + first) % n.clamp(min=1), torch.where(j < n, (j + first) % n.clamp(min=1), -1))
        s["ids"] = ids.to(torch.int32)
    return s


# ---------------------------------------------------------------------------------------------------- plain forms

def _plan(s):
    lens, grow, table, ring, state, block = s["lens"].long(), s["grow"].long(), s["table"], s["ring"], s["state"], s["block"]
    batch, width = table.shape
    n = ring.numel()
    live = grow >= 0
    g = grow.clamp(min=0)
    have = (lens + block - 1) // block
    want = torch.where(live, (lens + g + block - 1) // block, have)
    need = want - have
    back = torch.where(live, 0, have)
    cu = torch.cat([g.new_zeros(1), g.cumsum(0)])
    taken, given = need.sum(), back.sum()
    ok = (taken <= state[1] - state[0]) & (want.max() <= width) & (cu[-1] <= s["n_slots"])
    j = torch.arange(width, device=ring.device)[None, :]
    fresh = ok & (j >= have[:, None]) & (j < want[:, None])
    src = (state[0] + (need.cumsum(0) - need)[:, None] + j - have[:, None]) % n
    new_table = torch.where(fresh, ring[src], table)
    freed = ok & (j < back[:, None])
    dst = (state[1] + (back.cumsum(0) - back)[:, None] + j) % n
    ring[dst[freed]] = table[freed]
    table.copy_(new_table)
    t = torch.arange(s["n_slots"], device=ring.device)
    b = torch.searchsorted(cu[1:], t, right=True).clamp(max=batch - 1)
    pos = lens[b] + t - cu[b]
    slots = torch.where(ok & (t < cu[-1]), table[b, (pos // block).clamp(max=width - 1)].long() * block + pos % block, -1)
    lens_out = torch.where(ok, torch.where(live, lens + g, 0), lens)
    return (slots, torch.where(ok, cu, 0).to(torch.int32), lens_out.to(torch.int32), state + torch.where(ok, torch.stack([taken, given]), 0),
            (~ok).to(torch.int32).view(1), table, ring)


def _quantise(codes, scale, rows, slots, qmax):
    """One of the two halves of an append: the scale of a block is the smallest power of two that its largest value fits under,
    and never shrinks while the block holds earlier tokens, which move to the new scale with it."""
    n_blocks, heads, block, dim = codes.shape
    x = rows.float()
    blk, off = slots // block, slots % block
    peak = torch.zeros((n_blocks, heads), device=x.device).index_reduce_(0, blk, x.abs().amax(-1), "amax")
    start = torch.zeros(n_blocks, dtype=torch.bool, device=x.device).index_fill_(0, blk[off == 0], True)
    touched = torch.unique(blk)
    peak, start, before = peak[touched], start[touched, None], scale[touched]
    # smallest e with peak <= qmax * 2^e
    e = torch.ceil(torch.log2(peak.double() / qmax))
    e = torch.where(peak.double() <= qmax * torch.exp2(e - 1), e - 1, e)
    e = torch.where(peak.double() > qmax * torch.exp2(e), e + 1, e).clamp(-100, 121)
    now = torch.exp2(e).float()
    now = torch.where(start, now, torch.maximum(now, before))
    ratio = torch.where(start, 1.0, before / now)
    moved = codes[touched].float() * ratio[:, :, None, None]
    codes[touched] = (moved.round() if qmax == 127.0 else moved).to(codes.dtype)
    scale[touched] = now
    y = x / scale[blk][:, :, None]
    codes[blk, :, off] = (y.round() if qmax == 127.0 else y).to(codes.dtype)


def _append(s):
    qmax = QMAX[s["case"]["codes"]]
    _quantise(s["k"], s["k_scale"], s["new_k"], s["slots"], qmax)
    _quantise(s["v"], s["v_scale"], s["new_v"], s["slots"], qmax)
    blk, off = s["back"] // s["block"], s["back"] % s["block"]
    k = s["k"][blk, :, off].float() * s["k_scale"][blk][:, :, None]
    v = s["v"][blk, :, off].float() * s["v_scale"][blk][:, :, None]
    return k, v, s["k"], s["v"], s["k_scale"], s["v_scale"]


def _softmax_over(score, seen, value):
    """score, seen [..., r, n], value [..., n, d]: rows that see nothing give zeros and -inf."""
    score = torch.where(seen, score, -torch.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -torch.inf, 0.0, top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, value) / torch.where(total == 0, 1.0, total)
    return out, (top + torch.log(total)).squeeze(-1)


def _attend(s):
    case, q, table, lens, block = s["case"], s["q"].float(), s["table"], s["lens"].long(), s["block"]
    batch, width = table.shape
    heads, dim = case["kv_heads"], case["dim"]
    group = case["q_heads"] // heads
    at = table.clamp(min=0).long()
    take = lambda codes, scale: (codes[at].float() * scale[at][..., None, None]).permute(0, 2, 1, 3, 4).reshape(batch, heads, width * block, dim)  # noqa: E731
    key, value = take(s["k"], s["k_scale"]), take(s["v"], s["v_scale"])
    n = s["max_new"]
    i = torch.arange(n, device=q.device)
    if s["cu"] is None:
        count, first = torch.ones_like(lens), torch.arange(batch, device=q.device)
    else:
        first, count = s["cu"][:-1].long(), s["cu"][1:].long() - s["cu"][:-1].long()
    there = i[None, :] < count[:, None]                                              # [batch, n]
    row = (first[:, None] + i[None, :]).clamp(max=q.shape[0] - 1)
    x = q[row].reshape(batch, n, heads, group, dim).permute(0, 2, 1, 3, 4).reshape(batch, heads, n * group, dim)
    score = torch.matmul(x, key.transpose(-1, -2)) / math.sqrt(dim)
    t = torch.arange(width * block, device=q.device)
    last = (lens - count)[:, None] + i[None, :] if case["causal"] else (lens - 1)[:, None].expand(batch, n)
    seen = (t[None, None, :] <= last[:, :, None]) & (t[None, None, :] < lens[:, None, None])
    seen = seen[:, None, :, None, :].expand(batch, 1, n, group, width * block).reshape(batch, 1, n * group, -1)
    out, lse = _softmax_over(score, seen, torch.where((t[None, :] < lens[:, None])[:, None, :, None], value, 0.0))
    out = out.reshape(batch, heads, n, group, dim).permute(0, 2, 1, 3, 4).reshape(batch, n, heads * group, dim)
    lse = lse.reshape(batch, heads, n, group).permute(0, 2, 1, 3).reshape(batch, n, heads * group)
    return out[there].to(s["q"].dtype), lse[there]


def _found(s):
    case, q, lens, ids, block = s["case"], s["q"].float(), s["lens"].long(), s["ids"].long(), s["block"]
    tokens, lists, k = ids.shape
    heads, dim = case["kv_heads"], case["dim"]
    seen = (ids >= 0) & (ids < lens[:, None, None])
    at = torch.where(seen, ids, 0)
    blk = s["table"].long()[torch.arange(tokens, device=q.device)[:, None, None], at // block].clamp(min=0)
    head = (torch.arange(lists, device=q.device) // (lists // heads))[None, :, None]
    take = lambda codes, scale: codes[blk, head, at % block].float() * scale[blk, head][..., None]  # noqa: E731
    key, value = take(s["k"], s["k_scale"]), take(s["v"], s["v_scale"])
    x = q.reshape(tokens, lists, -1, dim)
    score = torch.matmul(x, key.transpose(-1, -2)) / math.sqrt(dim)
    out, lse = _softmax_over(score, seen[:, :, None, :], torch.where(seen[..., None], value, 0.0))
    return out.reshape(s["q"].shape).to(s["q"].dtype), lse.reshape(tokens, -1)


# ------------------------------------------------------------------------------------------------------- one pass

def _own(s):
    import hnsw_amd
    kind = s["kind"]
    if kind == "plan":
        p = hnsw_amd.cache_plan(s["lens"], s["grow"], s["table"], s["ring"], s["state"], block_tokens=s["block"], n_slots=s["n_slots"])
        return p.slots, p.cu_new, p.lens, p.state, p.status, s["table"], s["ring"]
    cache = hnsw_amd.TokenCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if kind == "append":
        cache.append(s["new_k"], s["new_v"], s["slots"])
        k, v = cache.read(s["back"], torch.float32)
        return k, v, s["k"], s["v"], s["k_scale"], s["v_scale"]
    if kind == "attend":
        return cache.attend(s["q"], s["table"], s["lens"], cu_q=s["cu"], causal=s["case"]["causal"], max_len=s["max_len"])
    return cache.attend_found(s["q"], s["table"], s["lens"], s["ids"])


def run(state):
    if own:
        return _own(state)
    return {"plan": _plan, "append": _append, "attend": _attend, "found": _found}[state["kind"]](state)


# --------------------------------------------------------------------------------------------- the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    lens, new = _lengths(case)
    block, batch = case["block"], case["batch"]
    if case["kind"] == "plan":
        table, ring, (head, tail) = s["table"].tolist(), s["ring"].tolist(), s["state"].tolist()
        taken, given, cu, slots, after = 0, 0, [0], [], []
        for b in range(batch):
            held = _blocks(lens[b], block)
            for j in range(held, _blocks(lens[b] + max(new[b], 0), block)):
                table[b][j] = ring[(head + taken) % len(ring)]
                taken += 1
            slots += [table[b][p // block] * block + p % block for p in range(lens[b], lens[b] + max(new[b], 0))]
            cu.append(cu[-1] + max(new[b], 0))
            after.append(0 if new[b] < 0 else lens[b] + new[b])
        for b in range(batch):
            if new[b] < 0:
                for j in range(_blocks(lens[b], block)):
                    ring[(tail + given) % len(ring)] = table[b][j]
                    given += 1
        slots += [-1] * (s["n_slots"] - len(slots))
        whole = lambda v, t: torch.tensor(v, dtype=t)  # noqa: E731
        return (whole(slots, torch.int64), whole(cu, torch.int32), whole(after, torch.int32), whole([head + taken, tail + given], torch.int64),
                whole([0], torch.int32), whole(table, torch.int32), whole(ring, torch.int32))
    heads, dim = case["kv_heads"], case["dim"]
    if case["kind"] == "append":
        qmax = QMAX[case["codes"]]
        nearest = lambda y: y.round() if qmax == 127.0 else y.float().to(torch.float8_e4m3fn).double()  # noqa: E731
        values = {}
        for name in ("k", "v"):
            codes, scale, rows = s[name].double(), s[name + "_scale"].double(), s["new_" + name].double()
            t = 0
            for b in range(batch):
                p = lens[b]
                while p < lens[b] + new[b]:
                    n = min(block - p % block, lens[b] + new[b] - p)
                    i, o = int(s["slots"][t]) // block, p % block
                    x = rows[t:t + n].transpose(0, 1)                                 # heads, n, dim
                    e = torch.full((heads,), -100.0, dtype=torch.float64, device=x.device)
                    peak = x.abs().amax((1, 2))
                    for _ in range(222):
                        e = torch.where(peak > qmax * torch.exp2(e), e + 1, e) if bool((peak > qmax * torch.exp2(e)).any()) else e
                    now = torch.exp2(e)
                    if o:
                        now = torch.maximum(now, scale[i])
                        codes[i] = nearest(codes[i] * (scale[i] / now)[:, None, None])
                    scale[i] = now
                    codes[i][:, o:o + n] = nearest(x / now[:, None, None])
                    t, p = t + n, p + n
            values[name] = codes, scale
        blk, off = s["back"] // block, s["back"] % block
        k, v = (values[n][0][blk, :, off] * values[n][1][blk][:, :, None] for n in ("k", "v"))
        codes = [values[n][0] if qmax != 127.0 else None for n in ("k", "v")]
        return k, v, codes[0], codes[1], values["k"][1], values["v"][1]
    outs, lses = [], []
    group = case["q_heads"] // heads
    q = s["q"].double()
    first = 0
    for b in range(batch):
        count = new[b] if case.get("new_hi") else 1
        x = q[first:first + count].reshape(count, heads, group, dim)
        first += count
        blocks = s["table"][b][: _blocks(lens[b], block)].long()
        rows = lambda codes, scale: (codes[blocks].double() * scale[blocks].double()[..., None, None]).transpose(0, 1).reshape(heads, -1, dim)[:, : lens[b]]  # noqa: E731, B023
        key, value = rows(s["k"], s["k_scale"]), rows(s["v"], s["v_scale"])
        out = torch.zeros((count, heads, group, dim), dtype=torch.float64, device=q.device)
        lse = torch.full((count, heads, group), -torch.inf, dtype=torch.float64, device=q.device)
        if case["kind"] == "found":
            share = case["list_heads"] // heads
            for h in range(case["list_heads"]):
                ids = s["ids"][b, h]
                ids = ids[(ids >= 0) & (ids < lens[b])].long()
                if ids.numel():
                    g = slice(h % share * (group // share), (h % share + 1) * (group // share))
                    y = key[h // share][ids] @ x[0, h // share, g].T / math.sqrt(dim)
                    out[0, h // share, g] = torch.softmax(y, 0).T @ value[h // share][ids]
                    lse[0, h // share, g] = torch.logsumexp(y, 0)
        else:
            for lo in range(0, count, 128):
                part = x[lo:lo + 128]
                y = torch.einsum("chgd,hnd->chgn", part, key) / math.sqrt(dim)
                last = torch.arange(lo, lo + part.shape[0], device=q.device) + (lens[b] - count) if case["causal"] else torch.full((part.shape[0],), lens[b] - 1, device=q.device)
                y = y.masked_fill((torch.arange(lens[b], device=q.device)[None, :] > last[:, None])[:, None, None, :], -torch.inf)
                some = last >= 0
                if lens[b]:
                    out[lo:lo + 128] = torch.where(some[:, None, None, None], torch.einsum("chgn,hnd->chgd", torch.softmax(y, -1), value).nan_to_num(0.0), 0.0)
                    lse[lo:lo + 128] = torch.logsumexp(y, -1)
        outs.append(out.reshape(count, -1, dim))
        lses.append(lse.reshape(count, -1))
    return torch.cat(outs), torch.cat(lses)
