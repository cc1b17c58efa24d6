"""The token mixer of the port block's full-attention layers over libdismoen_hip.so.

  KVCache         keys and values of many sequences in pages, held in 4 bits: rows are
                  quantised as they are written and can be read back
  CacheAttention  causal attention of rows over the cache
  AttentionMixer  both, as a layer runs them between its projections
A mixer.SeqBatch says which rows are which sequence's and which slot of the cache it
has.  The caller norms and rotates queries and keys before they get here.

Arrays are torch tensors on the block's device or numpy arrays, as in mixer.py.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from ._lib import (DMH_F_CHECK, DMH_F_DEVICE, DmhAttention, DmhKvCache, DmhKvRows, check)
from .mixer import SeqBatch, _bad, _Operator, _packed, _strides, _type


class _Heads(_Operator):
    """An operator on rows of heads, which may lie apart."""

    def _heads(self, a, heads, dim, dtype, device, what, written=False):
        """(rows, address, stride, stride of heads) of a row array [rows][heads][dim]."""
        if device is None:
            if not isinstance(a, np.ndarray) or a.ndim != 3:
                raise _bad(f"{what} must be a numpy array as the others, [rows][{heads}][{dim}]")
            if written and not a.flags.writeable:
                raise _bad(f"{what} is written, and the array is read-only")
            (n, h, d), (s, sh, sd), p = a.shape, _strides(a), a.ctypes.data
        else:
            try:
                n, h, d = a.shape
                s, sh, sd = a.stride()
                if a.get_device() != device:
                    raise ValueError
            except (ValueError, AttributeError, TypeError):
                raise _bad(f"{what} must be a tensor on cuda:{device}, [rows][{heads}][{dim}]") \
                    from None
            p = a.data_ptr()
        if h != heads or d != dim or a.dtype != dtype or sd != 1:
            raise _bad(f"{what} must be rows of {heads} heads of {dim} elements of the call's type")
        if h == 1:
            sh = d
        return n, p, s if n > 1 else max(s, (h - 1) * sh + d), sh


class KVCache(_Heads):
    """The caller's arrays of a cache:
      codes   uint8 [num_pages][2][kv_heads][page_size][dim / 2]
      scales  uint8 [num_pages][2][kv_heads][page_size][dim / 32]
      pages   int32 [num_slots][max_pages]: the pages of each slot's positions, in order
      past    int32 [num_slots]: the tokens that each slot held before the step's rows
    A page's page_size is a power of two from 16 on.  Within a page the order of codes and
    scales is the library's.  pages and past are read by each call and never changed; past
    is the caller's to bring up to date when all layers have had a step's rows.  Several
    layers' caches may share them."""

    def __init__(self, blk, codes, scales, pages, past):
        super().__init__(blk)
        if len(codes.shape) != 5 or codes.shape[1] != 2:
            raise _bad("codes must be [num_pages][2][kv_heads][page_size][dim / 2]")
        n, _, h, page, half = codes.shape
        host = self.host = isinstance(codes, np.ndarray)
        self.kv_heads, self.dim, self.num_slots = h, 2 * half, past.shape[0]
        self.device = None if host else blk.device
        for a, shape, kind, what in (
                (codes, (n, 2, h, page, half), "uint8", "codes"),
                (scales, (n, 2, h, page, half // 16), "uint8", "scales"),
                (pages, (self.num_slots, pages.shape[-1]), "int32", "pages"),
                (past, (self.num_slots,), "int32", "past")):
            if isinstance(a, np.ndarray) is not host or tuple(a.shape) != shape \
                    or str(a.dtype).split(".")[-1] != kind or not _packed(a.shape, _strides(a)):
                raise _bad(f"{what} must be a contiguous {kind} array of shape {list(shape)} on the"
                           " side of codes")
            if not host and (not a.is_cuda or a.get_device() != blk.device):
                raise _bad(f"{what} must be on the block's device, cuda:{blk.device}")
        if host and not (codes.flags.writeable and scales.flags.writeable):
            raise _bad("codes and scales are written, and an array is read-only")
        self.arrays = (codes, scales, pages, past)
        ptrs = [a.ctypes.data if host else a.data_ptr() for a in self.arrays]
        self._c = DmhKvCache(h, self.dim, page, n, pages.shape[1], *ptrs)
        self._cref = C.addressof(self._c)
        self._r = DmhKvRows()
        self._rref = C.addressof(self._r)

    @staticmethod
    def shapes(num_pages: int, kv_heads: int, page_size: int, dim: int):
        """The shapes of codes and scales."""
        return ((num_pages, 2, kv_heads, page_size, dim // 2),
                (num_pages, 2, kv_heads, page_size, dim // 32))

    def _for(self, batch):
        """The batch's flags, checked to fit the cache."""
        if batch.device != self.device:
            raise _bad("the batch's arrays are not where the cache's are")
        if batch.num_slots != self.num_slots:
            raise _bad(f"the batch has {batch.num_slots} slots, and the cache {self.num_slots}")
        return 0 if self.device is None else DMH_F_DEVICE

    def _set(self, k, v, batch, written):
        flags, r, t = self._for(batch), self._r, k.dtype
        r.dtype = _type(k)
        nk, r.k, r.k_stride, r.k_head_stride = self._heads(k, self.kv_heads, self.dim, t,
                                                           self.device, "k", written)
        nv, r.v, r.v_stride, r.v_head_stride = self._heads(v, self.kv_heads, self.dim, t,
                                                           self.device, "v", written)
        if min(nk, nv) < batch.total_tokens:
            raise _bad("k or v has fewer rows than total_tokens")
        return flags

    def _go(self, call, batch, flags):
        e = self._err
        rc = call(self._blk.handle, self._cref, self._rref, batch._ref, flags, e, 2048)
        if rc:
            check(rc, e)

    def write(self, k, v, batch: SeqBatch) -> None:
        """Rows k, v [rows][kv_heads][dim] into the cache, at the positions behind past."""
        self._go(self._blk._lib.dmh_kv_write, batch, self._set(k, v, batch, False))

    def read(self, k, v, batch: SeqBatch) -> None:
        """What the cache holds at the positions of the batch's rows into k and v
        [rows][kv_heads][dim]; of sequences marked in fresh, from position 0 on."""
        self._go(self._blk._lib.dmh_kv_read, batch, self._set(k, v, batch, True))


class CacheAttention(_Heads):
    """Causal attention of q_heads query heads over a cache; q_heads / kv_heads of them
    share a key head.  scale: None is dim ** -0.5."""

    def __init__(self, blk, q_heads: int, scale: float | None = None):
        super().__init__(blk)
        a = self._c = DmhAttention()
        a.q_heads, self._scale = q_heads, scale
        self._ref = C.addressof(a)

    def __call__(self, q, cache: KVCache, batch: SeqBatch, out, gate=None):
        """out[t] for rows q [rows][q_heads][dim], whose own keys and values the cache
        holds already; times sigmoid(gate) where that is given."""
        self._go(cache, batch, self._set(q, cache, batch, out, gate))
        return out

    def _set(self, q, cache, batch, out, gate):
        c, t, h, d = self._c, q.dtype, self._c.q_heads, cache.dim
        flags, dev = cache._for(batch), cache.device
        if cache._blk is not self._blk:
            raise _bad("the cache is another block's")
        c.dtype = _type(q)
        c.scale = d ** -0.5 if self._scale is None else self._scale
        n, c.q, c.q_stride, c.q_head_stride = self._heads(q, h, d, t, dev, "q")
        m, c.o, c.o_stride, c.o_head_stride = self._heads(out, h, d, t, dev, "out", True)
        if gate is None:
            c.gate = None
        else:
            g, c.gate, c.gate_stride, c.gate_head_stride = self._heads(gate, h, d, t, dev, "gate")
            n = min(n, g)
        if min(n, m) < batch.total_tokens:
            raise _bad("a row array has fewer rows than total_tokens")
        return flags

    def _go(self, cache, batch, flags):
        blk, e = self._blk, self._err
        rc = blk._lib.dmh_attention_forward(blk.handle, self._ref, cache._cref, batch._ref, flags, e,
                                            2048)
        if rc:
            check(rc, e)


class AttentionMixer:
    """One full-attention layer between its projections: the step's keys and values
    into the cache, then attention over it, gated where `gate` is given."""

    def __init__(self, blk, q_heads: int, scale: float | None = None):
        self.attention = CacheAttention(blk, q_heads, scale)

    def __call__(self, q, k, v, cache: KVCache, batch: SeqBatch, out, gate=None):
        """out [rows][q_heads][dim] for rows q [rows][q_heads][dim] and k, v [rows]
        [kv_heads][dim].  A call that is refused leaves the cache as it was."""
        flags = cache._set(k, v, batch, False)
        self.attention._set(q, cache, batch, out, gate)
        # (all that the library can refuse, before the first of them runs)
        self.attention._go(cache, batch, flags | DMH_F_CHECK)
        cache._go(cache._blk._lib.dmh_kv_write, batch, flags)
        self.attention._go(cache, batch, flags)
        return out
