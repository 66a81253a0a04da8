"""The token cache: keys and values of a language model's tokens in 8 bits, on the GPU, and attention over them.

An index over a request's keys says which earlier tokens a query needs (HNSW.search_batch_device); the cache holds what the
model then reads from them.  `attend` reads all tokens of a request, as the brute-force scan reads all rows; `attend_found`
reads the tokens that a search listed.  include/hnsw_amd.h has the formats and what each call does with values out of range.
The reference (RadimBaca/HNSW) indexes vectors and has no counterpart.

All tensors live on one GPU; calls run on that GPU's current torch stream, wait for nothing and can be captured into a
graph.  Nothing here has a gradient.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

from . import capi

_TYPES: dict = {}       # torch dtype -> TYPE_*
_CODES: dict = {}       # torch dtype -> CODES_*
_T = None               # torch, which is only imported when a cache is used


def _torch():
    global _T
    if _T is None:
        import torch
        _CODES.update({torch.int8: capi.CODES_I8, torch.float8_e4m3fn: capi.CODES_E4M3})
        _TYPES.update({torch.float32: capi.TYPE_F32, torch.float16: capi.TYPE_F16, torch.bfloat16: capi.TYPE_BF16})
        _T = torch
    return _T


def _stream(device) -> int:
    """The hipStream_t of the device's current torch stream (torch.cuda.current_stream builds an object first, which costs as much
    as a launch)."""
    raw = getattr(_T._C, "_cuda_getCurrentRawStream", None)
    return raw(device.index) if raw is not None else _T.cuda.current_stream(device).cuda_stream


def _need(t, name, dtype, shape, device):
    """`t` is a contiguous tensor of this type and shape (None: any extent) on `device`."""
    if t.dtype is dtype and t.shape == shape and t.is_contiguous() and t.device == device:
        return
    if t.dtype is not dtype or t.device != device or t.dim() != len(shape) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {len(shape)}-dimensional {dtype} tensor on {device}")
    for have, want in zip(t.shape, shape):
        if want is not None and have != want:
            raise ValueError(f"{name} must have the shape {tuple('any' if s is None else s for s in shape)}, not {tuple(t.shape)}")


class Plan(NamedTuple):
    """What cache_plan returns: the new tokens' slots [n_slots] (-1 behind the last), cu_new [n + 1], the new lengths [n], the
    ring's new [head, tail], and a status [1] that is 0 unless nothing was done (capi.PLAN_* bits)."""
    slots: object
    cu_new: object
    lens: object
    state: object
    status: object


def cache_plan(lens, grow, table, ring, state, *, block_tokens: int, n_slots: int) -> Plan:
    """Grows requests by grow[b] tokens, or ends them (-1): takes blocks off the ring and enters them into `table`, gives blocks
    of ended requests back to `ring` (both in place), and maps every new token to its slot.  lens, grow: [n] int32; table:
    [n, width] int32; ring: [n_blocks] int32; state: [2] int64.  Lengths and state come back as new tensors."""
    torch = _torch()
    dev = lens.device
    if dev.type != "cuda":
        raise ValueError("cache_plan: the tensors must be on a GPU")
    i32 = torch.int32
    _need(lens, "lens", i32, (None,), dev)
    n = lens.shape[0]
    _need(grow, "grow", i32, (n,), dev)
    _need(table, "table", i32, (n, None), dev)
    _need(ring, "ring", i32, (None,), dev)
    _need(state, "state", torch.int64, (2,), dev)
    if not 0 <= n_slots < 1 << 31:
        raise ValueError("cache_plan: n_slots must be 0..2^31 - 1")
    longs, words = state.new_empty(n_slots + 2), lens.new_empty(2 * n + 2)
    slots, state_out = longs.split_with_sizes((n_slots, 2))
    cu_new, lens_out, status = words.split_with_sizes((n + 1, n, 1))
    at, word = longs.data_ptr(), words.data_ptr()
    capi.check(capi.lib().hnsw_amd_cache_plan_device(lens.data_ptr(), grow.data_ptr(), n, table.data_ptr(), table.shape[1], ring.data_ptr(), ring.shape[0],
                                                     state.data_ptr(), block_tokens, n_slots, at, word, word + 4 * (n + 1), at + 8 * n_slots,
                                                     word + 4 * (2 * n + 1), dev.index, _stream(dev)))
    return Plan(slots, cu_new, lens_out, state_out, status)


class TokenCache:
    """A view of the cache's buffers: codes [n_blocks, n_heads, block_tokens, dim] (int8 or float8_e4m3fn), scales [n_blocks,
    n_heads] float32.  `TokenCache.empty` allocates them."""

    def __init__(self, k_codes, v_codes, k_scale, v_scale):
        torch = _torch()
        self.k_codes, self.v_codes, self.k_scale, self.v_scale = k_codes, v_codes, k_scale, v_scale
        self.device = dev = k_codes.device
        if dev.type != "cuda":
            raise ValueError("TokenCache: the buffers must be on a GPU")
        if k_codes.dtype not in _CODES:
            raise ValueError("TokenCache: codes must be int8 or float8_e4m3fn")
        shape = k_codes.shape
        _need(k_codes, "k_codes", k_codes.dtype, (None,) * 4, dev)
        _need(v_codes, "v_codes", k_codes.dtype, shape, dev)
        _need(k_scale, "k_scale", torch.float32, shape[:2], dev)
        _need(v_scale, "v_scale", torch.float32, shape[:2], dev)
        self.n_blocks, self.n_heads, self.block_tokens, self.dim = shape
        self._c = capi.TokenCacheC(k_codes.data_ptr(), v_codes.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), *shape, _CODES[k_codes.dtype])
        self._at = C.addressof(self._c)

    @classmethod
    def empty(cls, n_blocks: int, n_heads: int, block_tokens: int, dim: int, codes=None, device="cuda") -> "TokenCache":
        """New buffers (codes: torch.int8, the default, or torch.float8_e4m3fn)."""
        torch = _torch()
        shape = (n_blocks, n_heads, block_tokens, dim)
        make = lambda: torch.zeros(shape, dtype=torch.int8, device=device).view(codes or torch.int8)  # noqa: E731
        return cls(make(), make(), torch.zeros(shape[:2], device=device), torch.zeros(shape[:2], device=device))

    def _rows(self, t, name, heads):
        if t.dtype not in _TYPES or t.device != self.device or t.dim() != 3 or t.shape[1] != heads or t.shape[2] != self.dim:
            raise ValueError(f"{name} must be a [rows, {heads}, {self.dim}] tensor of float32, float16 or bfloat16 on {self.device}")
        if t.requires_grad and _torch().is_grad_enabled():
            raise ValueError(f"{name} requires a gradient: the token cache has none")
        s = t.stride()
        if s[2] != 1:
            raise ValueError(f"{name}: the last dimension must be contiguous")
        return s

    def append(self, k, v, slots) -> None:
        """Quantises the rows k, v [rows, n_heads, dim] into their slots [rows] int64 (as cache_plan lays them out; -1 is skipped)."""
        torch = _torch()
        ks, vs = self._rows(k, "k", self.n_heads), self._rows(v, "v", self.n_heads)
        if v.shape != k.shape or v.dtype is not k.dtype:
            raise ValueError("append: k and v must have the same shape and type")
        _need(slots, "slots", torch.int64, (k.shape[0],), self.device)
        capi.check(capi.lib().hnsw_amd_cache_append_device(self._at, k.data_ptr(), v.data_ptr(), k.shape[0], _TYPES[k.dtype], ks[0], ks[1], vs[0], vs[1],
                                                           slots.data_ptr(), self.device.index, _stream(self.device)))

    def read(self, slots, dtype=None):
        """(keys, values) of the slots [rows] int64: two [rows, n_heads, dim] tensors (float32 unless `dtype` says otherwise)."""
        torch = _torch()
        dtype = dtype or torch.float32
        if dtype not in _TYPES:
            raise ValueError("read: float32, float16 or bfloat16")
        _need(slots, "slots", torch.int64, (None,), self.device)
        n = slots.shape[0]
        k = torch.empty((n, self.n_heads, self.dim), dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        capi.check(capi.lib().hnsw_amd_cache_read_device(self._at, slots.data_ptr(), n, _TYPES[dtype], k.data_ptr(), v.data_ptr(), self.device.index,
                                                         _stream(self.device)))
        return k, v

    def _asked(self, q, table, lens, cu_q):
        torch = _torch()
        dev = self.device
        if q.dim() != 3 or q.shape[1] % self.n_heads:
            raise ValueError("q must be [rows, heads, dim], its heads a multiple of the cache's")
        s = self._rows(q, "q", q.shape[1])
        n = lens.shape[0] if lens.dim() == 1 else -1
        _need(lens, "lens", torch.int32, (None,), dev)
        _need(table, "table", torch.int32, (n, None), dev)
        if cu_q is not None:
            _need(cu_q, "cu_q", torch.int32, (n + 1,), dev)
        return s, n, q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)

    def attend(self, q, table, lens, *, cu_q=None, causal: bool = True, scale: float | None = None, max_len: int = 0):
        """(out, lse) of the queries q [rows, heads, dim] over all tokens of their requests; table [n, width], lens [n] int32.  Without
        cu_q each request has one row; with it ([n + 1] int32) request b has the rows cu_q[b] .. cu_q[b + 1], its last tokens.
        scale: 1 / sqrt(dim) unless given.  max_len: the longest length, if the caller knows it (a hint for splitting the work)."""
        torch = _torch()
        s, n, out, lse = self._asked(q, table, lens, cu_q)
        L, rows, heads, width = capi.lib(), q.shape[0], q.shape[1], table.shape[1]
        nbytes = L.hnsw_amd_cache_attend_workspace(self._at, rows, heads, n, width, max_len)
        work = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        capi.check(L.hnsw_amd_cache_attend_device(self._at, q.data_ptr(), rows, heads, s[0], s[1], _TYPES[q.dtype], table.data_ptr(), width, lens.data_ptr(), n,
                                                  cu_q.data_ptr() if cu_q is not None else None, 1 if causal else 0,
                                                  self.dim ** -0.5 if scale is None else scale, max_len, out.data_ptr(), lse.data_ptr(),
                                                  work.data_ptr() if nbytes else None, nbytes, self.device.index, _stream(self.device)))
        return out, lse

    def attend_found(self, q, table, lens, ids, *, cu_q=None, causal: bool = True, scale: float | None = None):
        """(out, lse) over the listed tokens: ids [rows, list_heads, n_ids] int32 (the 32-bit words a search writes), positions in the
        row's request; -1 and positions the row does not see are skipped.  list_heads is a multiple of the cache's heads and
        divides q's: query heads that follow one another share a list."""
        torch = _torch()
        s, n, out, lse = self._asked(q, table, lens, cu_q)
        L, rows, heads = capi.lib(), q.shape[0], q.shape[1]
        _need(ids, "ids", torch.int32, (rows, None, None), self.device)
        lists, n_ids = ids.shape[1], ids.shape[2]
        nbytes = L.hnsw_amd_cache_attend_found_workspace(self._at, rows, heads, lists, n_ids)
        work = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        capi.check(L.hnsw_amd_cache_attend_found_device(self._at, q.data_ptr(), rows, heads, s[0], s[1], _TYPES[q.dtype], table.data_ptr(), table.shape[1],
                                                        lens.data_ptr(), n, cu_q.data_ptr() if cu_q is not None else None, 1 if causal else 0,
                                                        ids.data_ptr(), lists, n_ids, self.dim ** -0.5 if scale is None else scale,
                                                        out.data_ptr(), lse.data_ptr(), work.data_ptr() if nbytes else None, nbytes,
                                                        self.device.index, _stream(self.device)))
        return out, lse
