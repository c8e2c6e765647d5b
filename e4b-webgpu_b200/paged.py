"""Paged KV cache of sequences of unequal length, in f16 or 4 bits (host side).

`PagedKV` is the descriptor (e4b_paged_kv, include/e4b_b200.h) that
`ops.headprep_paged`, `ops.attn_paged`, `ops.kvread_paged` and
`ops.paged_advance` take.  It holds device addresses: buffers that the caller
owns, or ones that it allocates on the device when they are not given.  Which
page belongs to which sequence is the caller's to decide (`set_tables` uploads
a page table).
"""
from __future__ import annotations

import ctypes

import numpy as np

from ._lib import lib
from .device import Buffer


class PagedStruct(ctypes.Structure):
    """e4b_paged_kv (include/e4b_b200.h)"""
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "pages", "lens", "rows")] + \
        [(n, ctypes.c_int) for n in ("bits", "page", "n_pages", "max_pages", "nseq", "kv_heads", "head_dim")]


class PagedKV:
    """A paged cache of one layer; `ref` is what the C entry points take."""

    def __init__(self, dev, *, BITS, PAGE, PAGES, MAX_PAGES, SEQS, KV_HEADS, HEAD_DIM, k=None, v=None, pages=None,
                 lens=None, rows=None):
        pool = lib().e4b_paged_pool_bytes(BITS, PAGE, PAGES, KV_HEADS, HEAD_DIM)
        if pool == 0:
            raise ValueError(f"paged cache: bad sizes bits={BITS} page={PAGE} pages={PAGES} kv_heads={KV_HEADS} "
                             f"head_dim={HEAD_DIM}")
        self.dev, self.pool_bytes, self.owned = dev, pool, []
        self.nseq, self.max_pages = SEQS, MAX_PAGES

        self.struct = PagedStruct(None, None, None, None, None if rows is None else int(rows), BITS, PAGE, PAGES,
                                  MAX_PAGES, SEQS, KV_HEADS, HEAD_DIM)
        self.ref = ctypes.addressof(self.struct)
        parts = (("k", k, pool, "paged k"), ("v", v, pool, "paged v"),
                 ("pages", pages, SEQS * MAX_PAGES * 4, "page table"), ("lens", lens, SEQS * 4, "lengths"))
        try:
            for field, given, nbytes, name in parts:
                if given is None:
                    given = dev.alloc(nbytes, name)
                    self.owned.append((field, given))
                elif isinstance(given, Buffer) and given.nbytes < nbytes:
                    raise ValueError(f"paged cache: {name} has {given.nbytes} bytes, needs {nbytes}")
                setattr(self.struct, field, int(given.ptr if hasattr(given, "ptr") else given))
        except Exception:
            self.free()                                  # a pool that could not be had leaves none behind
            raise

    def set_tables(self, pages=None, lens=None, rows=None):
        """Upload the page table [SEQS][MAX_PAGES] and / or the lengths; `rows`: device address of the rows table
        (0: one row per sequence)."""
        if pages is not None:
            a = np.ascontiguousarray(pages, np.uint32)
            if a.shape != (self.nseq, self.max_pages):
                raise ValueError(f"paged cache: page table {a.shape}, expected {(self.nseq, self.max_pages)}")
            self._write(self.struct.pages, a)
        if lens is not None:
            a = np.ascontiguousarray(lens, np.uint32)
            if a.shape != (self.nseq,):
                raise ValueError(f"paged cache: lengths {a.shape}, expected {(self.nseq,)}")
            self._write(self.struct.lens, a)
        if rows is not None:
            self.struct.rows = int(rows) or None

    def _write(self, ptr, a):
        if not ptr:
            raise ValueError("paged cache: freed")
        self.dev.write(ptr, a)

    def free(self):
        """Free what the cache allocated; calls on it are refused from then on (a recorded plan of such calls is to be
        destroyed before)."""
        owned, self.owned = self.owned, []
        for field, b in owned:
            setattr(self.struct, field, None)
            self.dev.free(b)
