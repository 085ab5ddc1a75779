"""Pages of the paged caches: copy, fork, extend, free and compact (no reference counterpart: the reference keeps
one contiguous cache per batch and grows it by torch.cat, ffa-fp8fp8/e2e/fp8fp8_cache.py:84-89).

`PagePool` counts, for the caches of one or several layers that share page ids, the block-table rows that hold each
page.  Forked sequences share whole pages and own a copy of the last partial one, so appends never write to a page
that another sequence holds:

    pool = PagePool([layer0_cache, layer1_cache, ...])
    pool.extend(table, lens, 900)            # pages for prompts; append(..., ragged=True) fills every layer's
    children = pool.fork(table, lens, parents)   # samples, beams
    pool.free(table, lens)
    pool.extend(children, child_lens, 64)
    plan = SharedPrefix(children, child_lens)    # the shared pages, read once by attend(..., shared=plan)

Everything runs on the current stream without synchronising, except for `check=True` (the default), which reads the
call's error word and raises; `check=False` serves captured graphs and loops that look at `errors` now and then.
Calls of one pool read and change its counts: they belong on one stream, or ordered.
"""
from __future__ import annotations

import ctypes

import torch

from . import _native as N
from .attend import _on

PAGE = 64
_ERRORS = {1: "not enough free pages", 2: "a row that cannot be served (its parent, length or partial page)",
           4: "a page outside the pool, or one that was free"}


class PagePool:
    """Reference counts of the pages of caches that share page ids (PagedQ2Cache / PagedKfmtCache, one per layer).

    refs [P] int32: block-table rows that hold each page (0: free).  errors [1] int32: error bits of all calls so far."""

    def __init__(self, caches):
        self.caches = list(caches)
        if not self.caches:
            raise ValueError("no caches")
        self.P, self.device = self.caches[0].P, self.caches[0].v.device
        if any(c.P != self.P or c.v.device != self.device for c in self.caches):
            raise ValueError("the caches must have the same number of pages and device")
        if self.device.type != "cuda":
            raise ValueError("the caches must be on a GPU")
        pools = [t for c in self.caches for t in c.pools()]
        if any(not t.is_contiguous() or t.data_ptr() % 16 for t in pools):
            raise ValueError("the pools must be contiguous and multiples of 16 bytes")
        self.refs = torch.zeros(self.P, dtype=torch.int32, device=self.device)
        self.errors = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._tensors = pools
        self._ptrs = (ctypes.c_void_p * len(pools))(*[t.data_ptr() for t in pools])
        self._bytes = (ctypes.c_size_t * len(pools))(*[t.stride(0) * t.element_size() for t in pools])
        self._pg = N.Pages(ctypes.addressof(self._ptrs), ctypes.addressof(self._bytes), len(pools), self.P,
                           self.refs.data_ptr())

    # ------------------------------------------------------------------ arguments
    def _ints(self, t: torch.Tensor, what: str) -> torch.Tensor:
        if t.ndim != 1:
            raise ValueError(f"{what} must be one-dimensional")
        return t.to(device=self.device, dtype=torch.int32).contiguous()

    def _table(self, t: torch.Tensor, writable: bool) -> torch.Tensor:
        if t.ndim != 2 or 0 in t.shape:
            raise ValueError("a block table must be [rows, columns]")
        if writable:
            if t.dtype != torch.int32 or t.device != self.device or not t.is_contiguous():
                raise ValueError("a block table that is changed must be contiguous int32 on the caches' device")
            return t
        return t.to(device=self.device, dtype=torch.int32).contiguous()

    def _rows(self, block_table, seq_lens, writable=False):
        table, lens = self._table(block_table, writable), self._ints(seq_lens, "seq_lens")
        if lens.shape[0] != table.shape[0]:
            raise ValueError("seq_lens must have one length per row of the block table")
        return table, lens

    def _scratch(self, words: int) -> torch.Tensor:
        return torch.empty(words, dtype=torch.int32, device=self.device)

    def _stream(self) -> int:
        return N.stream_of(self.device)

    @staticmethod
    def _raise(bits: int, what: str) -> None:
        if bits:
            text = "; ".join(m for b, m in _ERRORS.items() if bits & b)
            raise (RuntimeError if bits == 1 else ValueError)(f"{what}: {text}")

    # ------------------------------------------------------------------ calls
    def num_free(self) -> int:
        """Free pages (reads the counts)."""
        return int((self.refs == 0).sum().item())

    def copy(self, src: torch.Tensor, dst: torch.Tensor, check: bool = True) -> None:
        """Contents of page src[i] to page dst[i] in every cache.  The destinations must be distinct and none of them
        a source (check: read and refused; unchecked, pairs outside the pool are left out)."""
        src, dst = self._ints(src, "src"), self._ints(dst, "dst")
        if src.shape != dst.shape:
            raise ValueError("src and dst must have the same length")
        if check and src.numel():
            s, d = src.cpu(), dst.cpu()
            if min(int(s.min()), int(d.min())) < 0 or max(int(s.max()), int(d.max())) >= self.P:
                raise ValueError("pages outside the pool")
            if d.unique().numel() != d.numel() or torch.isin(d, s).any():
                raise ValueError("destinations must be distinct and no sources")
        with _on(self.device):
            rc = N.lib().ffa_pages_copy(ctypes.byref(self._pg), src.data_ptr(), dst.data_ptr(), src.shape[0], self._stream())
        N.check(rc, "ffa_pages_copy")

    def fork(self, block_table: torch.Tensor, seq_lens: torch.Tensor, parents: torch.Tensor, check: bool = True) -> torch.Tensor:
        """Block table [len(parents), columns] of children that continue sequences parents[c]: the parent's whole
        pages, held once more, and a copy of its last partial page; -1 past them.  The children's lengths are
        seq_lens[parents].  All children or, on an error, none (rows of -1)."""
        table, lens = self._rows(block_table, seq_lens)
        parents = self._ints(parents, "parents")
        C = parents.shape[0]
        child = torch.empty((C, table.shape[1]), dtype=torch.int32, device=self.device)
        if C == 0:
            return child
        lib = N.lib()
        scratch = self._scratch(lib.ffa_pages_alloc_scratch(C, 0))
        with _on(self.device):
            rc = lib.ffa_pages_fork(ctypes.byref(self._pg), table.data_ptr(), table.shape[1], table.shape[0],
                                    lens.data_ptr(), parents.data_ptr(), C, child.data_ptr(), scratch.data_ptr(),
                                    self.errors.data_ptr(), self._stream())
        N.check(rc, "ffa_pages_fork")
        if check:
            self._raise(int(scratch[0].item()), "fork")
        return child

    def extend(self, block_table: torch.Tensor, seq_lens: torch.Tensor, tokens: int, check: bool = True) -> None:
        """New pages in block_table (changed in place) for the next `tokens` tokens of every sequence; all rows or,
        on an error, none.  A partial last page is the sequence's own (fork copies it) and is filled first."""
        table, lens = self._rows(block_table, seq_lens, writable=True)
        tokens = int(tokens)
        if tokens < 0 or tokens > table.shape[1] * PAGE:
            raise ValueError("tokens must be within the block table")
        lib = N.lib()
        scratch = self._scratch(lib.ffa_pages_alloc_scratch(table.shape[0], tokens))
        with _on(self.device):
            rc = lib.ffa_pages_extend(ctypes.byref(self._pg), table.data_ptr(), table.shape[1], table.shape[0],
                                      lens.data_ptr(), tokens, scratch.data_ptr(), self.errors.data_ptr(), self._stream())
        N.check(rc, "ffa_pages_extend")
        if check:
            self._raise(int(scratch[0].item()), "extend")

    def _count(self, block_table, seq_lens, step, check, what):
        table, lens = self._rows(block_table, seq_lens)
        call = torch.zeros(1, dtype=torch.int32, device=self.device) if check else self.errors
        with _on(self.device):
            rc = N.lib().ffa_pages_count(ctypes.byref(self._pg), table.data_ptr(), table.shape[1], table.shape[0],
                                         lens.data_ptr(), step, call.data_ptr(), self.errors.data_ptr(), self._stream())
        N.check(rc, "ffa_pages_count")
        if check:
            self._raise(int(call.item()), what)

    def hold(self, block_table: torch.Tensor, seq_lens: torch.Tensor, check: bool = True) -> None:
        """Count the pages of rows that were filled without this pool (or are held once more)."""
        self._count(block_table, seq_lens, 1, check, "hold")

    def free(self, block_table: torch.Tensor, seq_lens: torch.Tensor, check: bool = True) -> None:
        """Let the rows' pages go; pages that no row holds any more are free.  (A count of 0 stays 0, an error.)"""
        self._count(block_table, seq_lens, -1, check, "free")

    def compact(self, *block_tables: torch.Tensor, check: bool = True) -> int | None:
        """Move the held pages to the lowest ids (contents, counts and the given tables' entries, in place).  Every
        table that holds pages has to be given: others go on naming the old ids.  Returns the number of pages held
        (ids from there on are free), or None with check=False."""
        tables = [self._table(t, True) for t in block_tables]
        lib = N.lib()
        scratch = self._scratch(lib.ffa_pages_compact_scratch(self.P))
        ptrs = (ctypes.c_void_p * max(len(tables), 1))(*[t.data_ptr() for t in tables])
        sizes = (ctypes.c_size_t * max(len(tables), 1))(*[t.numel() for t in tables])
        with _on(self.device):
            rc = lib.ffa_pages_compact(ctypes.byref(self._pg), ctypes.addressof(ptrs), ctypes.addressof(sizes),
                                       len(tables), scratch.data_ptr(), self._stream())
        N.check(rc, "ffa_pages_compact")
        return int(scratch[1].item()) if check else None
