"""A paged KV cache: one pool of pages for many sequences (tkh_paged_*).

``PagedKv`` owns the pool, the page tables and the pages' reference counts.
Sequences are opened, forked (sharing pages), extended (with a copy of a shared,
partly filled last page), truncated and closed; ``compact`` moves the pages in use
to the pool's front.  ``batch`` describes new tokens of open sequences for the
operators, ``append`` and ``attend`` call them for one layer:

    kv.extend(seqs, new)                      # room for the new tokens
    b = kv.batch(seqs, new)
    for layer in range(layers):
        kv.append(layer, b, rotary, q_proj, k_proj, v_proj, q)
        kv.attend(layer, b, q, context, scale=scale)

``PagedKv(None, ...)`` keeps the books alone, without a device.
"""

from __future__ import annotations

import ctypes
from typing import List, Optional, Sequence

import torch

from . import _lib, ops
from .kv import _CODE, _DeviceView, device_tensor
from .ops import Context, TkhError, _check


class PagedKv:
    def __init__(self, ctx: Optional[Context], layers: int, kv_heads: int, head_dim: int, page_tokens: int,
                 pages: int, sequences: int, sequence_pages: int, storage: torch.dtype):
        self.ctx, self.storage = ctx, storage
        handle, err = ctypes.c_void_p(), _lib.Error()
        o = _lib.PagedOptions(layers, kv_heads, head_dim, page_tokens, pages, sequences, sequence_pages,
                              _CODE[storage])
        _check(_lib.load().tkh_paged_create(ctx.handle if ctx is not None else None, ctypes.byref(o),
                                            ctypes.byref(handle), ctypes.byref(err)), err)
        self.handle = handle
        _lib.track(self, _lib.KV_OWNER)
        self.layers, self.page_tokens, self.sequence_pages = layers, page_tokens, sequence_pages
        if ctx is not None:
            i = self.info()
            self.pool = device_tensor(i.pool, (layers, 2, pages, kv_heads, page_tokens, head_dim), storage, ctx.device)
            self.page_table = self._words(i.page_table, (sequences, sequence_pages))
            self.key_lens = self._words(i.key_lens, (sequences,))

    def _words(self, ptr, shape):
        view = _DeviceView(ptr, shape, torch.float32)
        view.__cuda_array_interface__["typestr"] = "<i4"
        return torch.as_tensor(view, device=f"cuda:{self.ctx.device}")

    def info(self) -> _lib.PagedInfo:
        i = _lib.PagedInfo()
        if _lib.load().tkh_paged_info_get(self.handle, ctypes.byref(i)) != _lib.OK:
            raise ValueError("the paged cache is closed")
        return i

    @property
    def free_pages(self) -> int:
        return int(self.info().free_pages)

    def _sequence(self, f, *args) -> int:
        out, err = ctypes.c_uint64(), _lib.Error()
        _check(f(self.handle, *args, ctypes.byref(out), ctypes.byref(err)), err)
        return int(out.value)

    def open(self) -> int:
        """An empty sequence's number (its slot in the device tables)."""
        return self._sequence(_lib.load().tkh_paged_open)

    def fork(self, sequence: int) -> int:
        """A new sequence with the keys of `sequence`, sharing its pages."""
        return self._sequence(_lib.load().tkh_paged_fork, sequence)

    def compact(self) -> int:
        """Moves the pages in use to the pool's lowest numbers; how many moved."""
        return self._sequence(_lib.load().tkh_paged_compact)

    def extend(self, sequences: Sequence[int], tokens: Sequence[int]):
        """Room for tokens[i] more keys of sequences[i]: all of it, or CAPACITY and nothing."""
        if len(sequences) != len(tokens):
            raise ValueError("one token count per sequence")
        err = _lib.Error()
        _check(_lib.load().tkh_paged_extend(self.handle, ops._u64s(sequences), ops._u64s(tokens), len(sequences),
                                            ctypes.byref(err)), err)

    def truncate(self, sequence: int, length: int):
        err = _lib.Error()
        _check(_lib.load().tkh_paged_truncate(self.handle, sequence, length, ctypes.byref(err)), err)

    def close_sequence(self, sequence: int):
        err = _lib.Error()
        _check(_lib.load().tkh_paged_close(self.handle, sequence, ctypes.byref(err)), err)

    def length(self, sequence: int) -> int:
        n = ctypes.c_uint64()
        if _lib.load().tkh_paged_sequence_get(self.handle, sequence, ctypes.byref(n), None, 0) != _lib.OK:
            raise ValueError(f"sequence {sequence} is not open")
        return int(n.value)

    def pages(self, sequence: int) -> List[int]:
        """The sequence's page numbers, in key order."""
        n = -(-self.length(sequence) // self.page_tokens)
        out = (ctypes.c_uint64 * max(1, n))()
        _lib.load().tkh_paged_sequence_get(self.handle, sequence, None, out, n)
        return [int(x) for x in out[:n]]

    def batch(self, sequences: Sequence[int], tokens: Sequence[int], max_keys: int = 0) -> ops.PagedBatch:
        """The batch of the last tokens[i] keys of sequences[i].  max_keys bounds the
        lengths (0: what they are now); a captured batch that grows takes a larger one."""
        if len(sequences) != len(tokens) or not len(sequences):
            raise ValueError("one token count per sequence")
        start = [0]
        for n in tokens:
            start.append(start[-1] + int(n))
        dev = self.key_lens.device
        return ops.PagedBatch(page_table=self.page_table, key_lens=self.key_lens, total_queries=start[-1],
                              max_queries=max(1, max(int(n) for n in tokens)),
                              max_keys=max_keys or max(1, max(self.length(s) for s in sequences)),
                              query_start=torch.tensor(start, dtype=torch.int32, device=dev),
                              slots=torch.tensor([int(s) for s in sequences], dtype=torch.int32, device=dev))

    def append(self, layer: int, batch: ops.PagedBatch, rotary: ops.RotaryPositions, q_proj, k_proj, v_proj, q_out,
               q_norm=None, k_norm=None, norm_epsilon: float = 1e-6):
        """The producer of one layer: new rows normalised, rotated and rounded, K and V into their pages."""
        ops.paged_produce(self.ctx, batch, rotary, q_proj, k_proj, v_proj, q_norm, k_norm, q_out,
                          self.pool[layer, 0], self.pool[layer, 1], norm_epsilon)

    def attend(self, layer: int, batch: ops.PagedBatch, q, context, *, scale: float, window: Optional[int] = None,
               softcap: float = 0.0):
        """Attention of one layer's new tokens over their sequences' pages."""
        ops.paged_attention(self.ctx, batch, q, self.pool[layer, 0], self.pool[layer, 1], context, scale=scale,
                            window=window, softcap=softcap)

    def close(self):
        if getattr(self, "handle", None):
            self.pool = self.page_table = self.key_lens = None
            _lib.load().tkh_paged_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


__all__ = ["PagedKv", "TkhError"]
