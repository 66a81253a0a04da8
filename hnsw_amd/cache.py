"""The token cache: keys and values of a language model's tokens in 8 bits, on the GPU, and attention over them.

An index over a request's keys says which earlier tokens a query needs (HNSW.search_batch_device); the cache holds what the
model then reads from them.  `attend` reads all tokens of a request, as the brute-force scan reads all rows; `attend_found`
reads the tokens that a search listed.  include/hnsw_amd.h has the formats and what each call does with values out of range.
The reference (RadimBaca/HNSW) indexes vectors and has no counterpart.

All tensors live on one GPU; calls run on that GPU's current torch stream, wait for nothing and can be captured into a
graph.  Nothing here has a gradient.  Arguments that do not fit raise ValueError (tensors) or capi.HnswAmdError (the library).
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

from . import capi

_BINDING = None         # hnsw_amd/_tensors.so, loaded (with torch) when a cache is first used


def _binding():
    global _BINDING
    if _BINDING is None:
        import torch  # noqa: F401  (its libraries and its HIP runtime come first)
        L = capi.lib()
        try:
            from . import _tensors
        except ImportError as e:
            raise ImportError(f"hnsw_amd/_tensors.so cannot be loaded ({e}): build it with `python -m hnsw_amd.build`") from e
        _tensors.bind(*(C.cast(getattr(L, "hnsw_amd_cache_" + name), C.c_void_p).value for name in
                        ("plan_device", "append_device", "read_device", "attend_workspace", "attend_found_workspace", "attend_device",
                         "attend_found_device")), capi.check)
        _BINDING = _tensors
    return _BINDING


class Plan(NamedTuple):
    """What cache_plan returns: the new tokens' slots [n_slots] (-1 behind the last), cu_new [n + 1], the new lengths [n], the
    ring's new [head, tail], and a status [1] that is 0 unless nothing was done (capi.PLAN_* bits).  The five lie in one allocation."""
    slots: object
    cu_new: object
    lens: object
    state: object
    status: object


def cache_plan(lens, grow, table, ring, state, *, block_tokens: int, n_slots: int) -> Plan:
    """Grows requests by grow[b] tokens, or ends them (-1): takes blocks off the ring and enters them into `table`, gives blocks
    of ended requests back to `ring` (both in place), and maps every new token to its slot.  lens, grow: [n] int32; table:
    [n, width] int32; ring: [n_blocks] int32; state: [2] int64.  Lengths and state come back as new tensors."""
    return Plan._make((_BINDING or _binding()).plan(lens, grow, table, ring, state, block_tokens, n_slots))


class TokenCache:
    """A view of the cache's buffers: codes [n_blocks, n_heads, block_tokens, dim] (int8 or float8_e4m3fn), scales [n_blocks,
    n_heads] float32.  `TokenCache.empty` allocates them."""

    def __init__(self, k_codes, v_codes, k_scale, v_scale):
        self._b = _BINDING or _binding()
        self._c = self._b.cache(k_codes, v_codes, k_scale, v_scale)
        self.k_codes, self.v_codes, self.k_scale, self.v_scale = k_codes, v_codes, k_scale, v_scale
        self.n_blocks, self.n_heads, self.block_tokens, self.dim = k_codes.shape

    @classmethod
    def empty(cls, n_blocks: int, n_heads: int, block_tokens: int, dim: int, codes=None, device="cuda") -> "TokenCache":
        """New buffers (codes: torch.int8, the default, or torch.float8_e4m3fn)."""
        import torch
        shape = (n_blocks, n_heads, block_tokens, dim)
        k, v = (torch.zeros(shape, dtype=torch.int8, device=device).view(codes or torch.int8) for _ in range(2))
        return cls(k, v, torch.zeros(shape[:2], device=device), torch.zeros(shape[:2], device=device))

    def append(self, k, v, slots) -> None:
        """Quantises the rows k, v [rows, n_heads, dim] into their slots [rows] int64 (as cache_plan lays them out: a block's rows next to each
        other, their slots ascending; -1 is skipped)."""
        self._b.append(self._c, k, v, slots)

    def read(self, slots, dtype=None):
        """(keys, values) of the slots [rows] int64: two [rows, n_heads, dim] tensors, float32 unless `dtype` says otherwise."""
        return self._b.read(self._c, slots, dtype)

    def attend(self, q, table, lens, *, cu_q=None, causal: bool = True, scale: float | None = None, max_len: int = 0):
        """(out, lse) of the queries q [rows, heads, dim] over all tokens of their requests; table [n, width], lens [n] int32.  Without
        cu_q each request has one row; with it ([n + 1] int32) request b has the rows cu_q[b] .. cu_q[b + 1], its last tokens; what the
        result holds in rows behind the last request is not defined.  (Single tokens of long requests are faster in a call of their own
        than next to prompts.)  scale: 1 / sqrt(dim) unless given.  max_len: the longest length, if the caller knows it (a hint for splitting
        the work; without it the workspace is for requests as long as the table is wide)."""
        return self._b.attend(self._c, q, table, lens, cu_q, causal, scale, max_len, None)

    def attend_found(self, q, table, lens, ids, *, cu_q=None, causal: bool = True, scale: float | None = None):
        """(out, lse) over the listed tokens: ids [rows, list_heads, n_ids] int32 (the 32-bit words a search writes), positions in the
        row's request; -1 and positions the row does not see are skipped.  list_heads is a multiple of the cache's heads and
        divides q's: query heads that follow one another share a list."""
        return self._b.attend(self._c, q, table, lens, cu_q, causal, scale, 0, ids)
