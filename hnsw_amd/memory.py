"""A language model's memory over one attention layer: the keys and values of several requests in a TokenCache, and HNSW indexes
over their keys.

    remember    new tokens' keys and values (blocks, slots, quantising writes)
    attend      attention over all remembered tokens
    index       builds (again) the indexes over a request's stored keys, one for each key head
    recall      searches the indexes with each query head and attends over the tokens found, and over those that came after the
                index was built

The reference (RadimBaca/HNSW) is the index alone and has no counterpart.
"""
from __future__ import annotations

import numpy as np

from . import capi
from .cache import TokenCache, cache_plan
from .index import HNSW


class TokenMemory:
    def __init__(self, n_requests: int, n_blocks: int, n_heads: int, dim: int, *, block_tokens: int = 32, max_len: int, codes=None, device: int = 0,
                 ctor=(16, 16, 200)):
        import torch
        self._torch, self.device, self.ctor = torch, torch.device("cuda", device), ctor
        self.cache = TokenCache.empty(n_blocks, n_heads, block_tokens, dim, codes, self.device)
        z = lambda *shape, dtype=torch.int32: torch.zeros(shape, dtype=dtype, device=self.device)  # noqa: E731
        self.lens, self.table = z(n_requests), z(n_requests, -(-max_len // block_tokens)) - 1
        self.ring, self.state = torch.arange(n_blocks, dtype=torch.int32, device=self.device), z(2, dtype=torch.int64)
        self.state[1] = n_blocks
        self.host_lens = [0] * n_requests                   # (what `lens` holds on the GPU)
        self.indexes: list = [None] * n_requests            # a request's indexes by head, and how many of its tokens they hold

    def remember(self, grow, k, v) -> None:
        """grow[b] new tokens of request b, -1: the request ends.  k, v: [sum of the new tokens, heads, dim], request after request.
        Raises capi.HnswAmdError and remembers nothing where blocks or table rows run out (this waits for the GPU to say so)."""
        torch = self._torch
        grow = [int(g) for g in grow]
        if len(grow) != len(self.host_lens) or sum(max(g, 0) for g in grow) != k.shape[0]:
            raise ValueError("remember: grow names every request, and k and v hold their new tokens")
        p = cache_plan(self.lens, torch.tensor(grow, dtype=torch.int32, device=self.device), self.table, self.ring, self.state,
                       block_tokens=self.cache.block_tokens, n_slots=k.shape[0])
        status = p.status.item()
        if status:
            raise capi.HnswAmdError(capi.E_FULL, "token memory: " + ", ".join(
                text for bit, text in ((capi.PLAN_NO_BLOCKS, "no free blocks"), (capi.PLAN_TABLE_FULL, "a request is longer than max_len"),
                                       (capi.PLAN_SLOTS_FULL, "more tokens than slots"), (capi.PLAN_BAD_LENGTH, "a length that cannot be")) if status & bit))
        self.cache.append(k, v, p.slots)
        self.lens, self.state = p.lens, p.state
        for b, g in enumerate(grow):
            self.host_lens[b] = 0 if g < 0 else self.host_lens[b] + g
            if g < 0:
                self.indexes[b] = None

    def attend(self, q, *, cu_q=None, scale=None):
        """(out, lse) of q [rows, heads, dim] over all remembered tokens (TokenCache.attend)."""
        return self.cache.attend(q, self.table, self.lens, cu_q=cu_q, scale=scale, max_len=max(self.host_lens))

    def index(self, b: int, threads: int = 16) -> None:
        """Indexes request b's stored keys, as the cache's codes give them.  The index ranks by squared L2 distance; the inner
        product ranks the same when a coordinate sqrt(M^2 - |x|^2) is added to the keys (M: the longest key's length) and 0 to the queries."""
        n, c = self.host_lens[b], self.cache
        if n == 0:
            self.indexes[b] = None
            return
        pos = self._torch.arange(n, device=self.device)
        keys = c.read(self.table[b][pos // c.block_tokens].long() * c.block_tokens + pos % c.block_tokens)[0].cpu().numpy()
        heads = []
        for h in range(c.n_heads):
            rows = np.zeros((n, c.dim + 16), np.float32)                # (distances use whole groups of 16 dims)
            rows[:, :c.dim] = keys[:, h]
            length = (rows.astype(np.float64) ** 2).sum(1)
            rows[:, c.dim] = np.sqrt(np.maximum(length.max() - length, 0.0))
            x = HNSW(*self.ctor, device=self.device.index)
            x.init(c.dim + 16, n)
            x.set_build_float_keys(True)
            x.insert_batch(rows, threads=threads)
            x.sync_device(self.device.index)
            heads.append(x)
        self.indexes[b] = (heads, n)

    def recall(self, q, k: int, ef: int | None = None, *, scale=None):
        """(out, lse, ids) of one query row for each request, q [requests, heads, dim], over the k tokens that the indexes find for each
        query head (scores with the sign of `scale`; ef: the search's breadth, 2 k unless given) and over the tokens that are not indexed."""
        torch, c = self._torch, self.cache
        if q.dim() != 3 or q.shape[0] != len(self.host_lens) or q.shape[1] < 1 or q.shape[1] % c.n_heads or q.shape[2] != c.dim:
            raise ValueError(f"recall: one row for each request, [{len(self.host_lens)}, a multiple of {c.n_heads} heads, {c.dim}]")
        if k < 1:
            raise ValueError("recall: k must be positive")
        n, heads = q.shape[0], q.shape[1]
        ef, group = max(k, ef or 2 * k), heads // c.n_heads
        known = [x[1] if x else 0 for x in self.indexes]
        tail = max(a - i for a, i in zip(self.host_lens, known))
        ids = torch.full((n, heads, k + tail), -1, dtype=torch.int32, device=self.device)
        if tail:
            at = torch.arange(tail, dtype=torch.int32, device=self.device) + torch.tensor(known, dtype=torch.int32, device=self.device)[:, None]
            ids[:, :, k:] = torch.where(at < self.lens[:, None], at, -1)[:, None]
        asked = torch.zeros((n, heads, c.dim + 16), dtype=torch.float32, device=self.device)
        asked[:, :, :c.dim] = q if scale is None or scale >= 0 else -q
        found = torch.full((n, heads, k), -1, dtype=torch.int32, device=self.device)
        dist = torch.empty((n, heads, k), dtype=torch.float32, device=self.device)
        stream = torch.cuda.current_stream(self.device).cuda_stream
        calls = []
        try:
            for b, known_b in enumerate(self.indexes):                  # all searches are under way before the first is waited for
                for h in range(c.n_heads if known_b else 0):
                    calls.append((known_b[0][h], known_b[0][h].search_batch_device_begin(
                        asked[b, h * group].data_ptr(), group, ef, k, found[b, h * group].data_ptr(), dist[b, h * group].data_ptr(), stream=stream,
                        flags=capi.DIST_SSE | capi.KEYS_FLOAT)))
        finally:
            errors = []
            for x, call in calls:                                       # every search is waited for, also when one of them fails
                try:
                    x.search_batch_device_finish(call)
                except capi.HnswAmdError as e:
                    errors.append(e)
        if errors:
            raise errors[0]
        ids[:, :, :k] = found
        out, lse = c.attend_found(q, self.table, self.lens, ids, scale=scale)
        return out, lse, ids
