"""A paged key-value cache: one pool of pages per layer, handed out to sequences of any length.

The pool of a layer is ``[pages, kv_heads, page_size, head_dim]`` for K and for V, so the positions of one head in one
page are one contiguous block.  Cached values are fp16 / bf16, or int8 / e4m3 codes with one fp32 scale per (token,
head).  The operators that write, read and attend over it are in ``ops`` (``rope_paged_kv``, ``paged_kv_read``,
``paged_attention``); this class owns the memory and the host-side page accounting."""
from __future__ import annotations

import ctypes

import torch

from ._lib import KairosError, KvLayer

KV_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.int8: 3, torch.float8_e4m3fn: 4}
_NAMES = {'float16': torch.float16, 'bfloat16': torch.bfloat16, 'int8': torch.int8, 'fp8_e4m3': torch.float8_e4m3fn}


class PagedKVCache:
    """`layers` pools of `num_pages` pages of `page_size` (16, 32, 64, 128 or 256) positions.

    kv_dtype: torch.float16, bfloat16, int8 or float8_e4m3fn, or 'float16', 'bfloat16', 'int8', 'fp8_e4m3'.
    Sequences are named by any hashable key: ``reserve(key, tokens)`` hands pages out, ``release(key)`` takes them
    back.  Page tables, slots and positions are built on the host and copied; a captured decode step keeps its own
    device copies and needs none of this while the pages suffice."""

    def __init__(self, layers, num_pages, kv_heads, head_dim, page_size=64, kv_dtype=torch.float16, device='cuda'):
        kv_dtype = _NAMES.get(kv_dtype, kv_dtype)
        shape = (layers, num_pages, kv_heads, page_size, head_dim)
        self._check(shape, kv_dtype)
        k = torch.zeros(shape, dtype=kv_dtype, device=device)
        v = torch.zeros(shape, dtype=kv_dtype, device=device)
        scales = [None, None]
        if kv_dtype in (torch.int8, torch.float8_e4m3fn):
            scales = [torch.zeros(shape[:-1], dtype=torch.float32, device=device) for _ in range(2)]
        self._adopt(k, v, *scales)

    @classmethod
    def from_tensors(cls, k, v, k_scale=None, v_scale=None):
        """A cache over pools that exist already: k, v [layers, pages, kv_heads, page_size, head_dim], the scales
        [layers, pages, kv_heads, page_size] fp32 for int8 / e4m3 pools.  The tensors are used, not copied."""
        if k.dim() != 5 or v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError('k and v: expected two tensors [layers, pages, kv_heads, page_size, head_dim] of one type')
        cls._check(tuple(k.shape), k.dtype)
        scaled = k.dtype in (torch.int8, torch.float8_e4m3fn)
        for s in (k_scale, v_scale):
            if scaled != (s is not None) or (s is not None and (s.shape != k.shape[:-1] or s.dtype != torch.float32)):
                raise ValueError('k_scale and v_scale: float32 [layers, pages, kv_heads, page_size] for int8 and e4m3 '
                                 'pools, none otherwise')
        for t in (k, v, k_scale, v_scale):
            if t is not None and (not t.is_contiguous() or t.device != k.device or t.data_ptr() % 16):
                raise ValueError('the pools and their scales: contiguous, 16-byte aligned, on one device')
        self = cls.__new__(cls)
        self._adopt(k, v, k_scale, v_scale)
        return self

    @staticmethod
    def _check(shape, kv_dtype):
        if kv_dtype not in KV_DTYPES:
            raise ValueError(f'kv_dtype must be one of {sorted(_NAMES)}, got {kv_dtype}')
        layers, pages, heads, page_size, dim = shape
        if min(layers, pages, heads) < 1 or page_size not in (16, 32, 64, 128, 256) or dim not in (64, 128, 256):
            raise ValueError('a paged cache has layers, pages and kv_heads > 0, page_size 16, 32, 64, 128 or 256 and '
                             f'head_dim 64, 128 or 256; got {shape}')

    def _adopt(self, k, v, k_scale, v_scale):
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.layers, self.num_pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.kv_dtype, self.device = k.dtype, k.device
        self._structs = [KvLayer(k[i].data_ptr(), v[i].data_ptr(),
                                 k_scale[i].data_ptr() if k_scale is not None else None,
                                 v_scale[i].data_ptr() if v_scale is not None else None,
                                 self.num_pages, self.kv_heads, self.page_size, self.head_dim, KV_DTYPES[k.dtype])
                         for i in range(self.layers)]
        self.layer_ptrs = [ctypes.addressof(s) for s in self._structs]
        # as the operators ask for it on every call
        self.index = self.device.index if self.device.index is not None else -1
        self.workspace_bytes = {}               # (batch, heads, table width) -> bytes of an attention call's scratch
        self._next, self._returned = 0, []      # pages never handed out start at _next
        self._pages = {}

    @property
    def nbytes(self):
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale) if t is not None)

    # ---- page accounting (host) ---------------------------------------------------------------
    @property
    def free_pages(self):
        return self.num_pages - self._next + len(self._returned)

    def _take(self):
        if self._returned:
            return self._returned.pop()
        self._next += 1
        return self._next - 1

    def reserve(self, key, tokens):
        """Pages for the first `tokens` positions of sequence `key` (no-op where it has them)."""
        if tokens < 0:
            raise ValueError(f'tokens must not be negative, got {tokens}')
        pages = self._pages.get(key, [])
        more = -(-tokens // self.page_size) - len(pages)
        if more > self.free_pages:
            raise KairosError(f'paged cache: sequence {key!r} needs {more} more pages, {self.free_pages} are free')
        self._pages[key] = pages + [self._take() for _ in range(more)]
        return self._pages[key]

    def pages(self, key):
        """The pages of sequence `key` in the order of its positions, none where it is unknown."""
        return list(self._pages.get(key, ()))

    def release(self, key):
        """Takes the pages of sequence `key` back.  Work that still reads them has to be ordered before their next use,
        which it is on one stream."""
        self._returned.extend(reversed(self._pages.pop(key)))

    def page_table(self, keys, width=None):
        """int32 [len(keys), width] on the device: the pages of each sequence in order, -1 behind its last one."""
        rows = [self._pages[key] for key in keys]
        need = max((len(r) for r in rows), default=0)
        width = need if width is None else width
        if need > width:
            raise ValueError(f'a sequence has {need} pages, the table is {width} wide')
        table = torch.full((len(rows), width), -1, dtype=torch.int32)
        for i, r in enumerate(rows):
            table[i, :len(r)] = torch.tensor(r, dtype=torch.int32)
        return table.to(self.device)

    def slots(self, keys, counts, starts=None):
        """Slots and positions (int64, device) of `counts[i]` tokens of each sequence from position `starts[i]` (0) on,
        one sequence after the other."""
        starts = [0] * len(keys) if starts is None else starts
        slots, positions = [torch.empty(0, dtype=torch.int64)], [torch.empty(0, dtype=torch.int64)]
        for key, n, first in zip(keys, counts, starts, strict=True):
            pages = torch.tensor(self._pages[key], dtype=torch.int64)
            if first < 0 or n < 0 or first + n > len(pages) * self.page_size:
                raise ValueError(f'sequence {key!r}: positions {first}..{first + n} are not reserved')
            at = torch.arange(first, first + n)
            slots.append(pages[at // self.page_size] * self.page_size + at % self.page_size)
            positions.append(at)
        return torch.cat(slots).to(self.device), torch.cat(positions).to(self.device)
