"""Block tables of the paged cache on the device: requests come, grow, fork and go without a look by the host (csrc/page_tables.cu).

A :class:`PageTables` deals the pages of one or more caches (one per layer; a page of the tables is that page in each of them) to up to 1024
sequences.  :meth:`PageTables.step` is the one operation: every sequence goes on from the first ``keep`` tokens of its parent and makes room for new
ones.  So a step of beam search is ``step(1, parents=search.parents)``, a decode step ``step(1)``, dropping rejected drafts
``step(0, keep=lengths)``, a request that begins has no parent (-1) and as many tokens as its prompt, one that ends no parent and none.

    tables = PageTables(caches, seqs=requests * beams, tokens=longest)
    tables.step(lengths, parents=nobody)                    # prompts: int32 tensors on the device
    plan = build_plan(caches[0], heads, q_lens, kv_lens, tables)

Whole pages are shared by all sequences that go on from them; the rows of a page that is not full are copied (in all caches), so no sequence
writes where another one reads.  Pages are taken lowest number first, sequence after sequence.  A call runs on the current stream of the
caches' device; the copies are done before the next call on that stream.  A graph with a step reads and writes the tables whenever it is replayed: keep them,
and the caches, as long as the graph.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import c_int, c_void_p
from .paged import PagedCache, _whole

MAX_SEQS, MAX_CACHES = 1024, 256
LAYOUT = 0x70670003          # last word of the tables: the library refuses one whose fields lie elsewhere
_ENTRY: dict = {}


class _Args(ctypes.Structure):
    """``Tables`` of csrc/page_tables.cu."""
    _fields_ = ([(n, c_void_p) for n in ("table", "lens", "refs", "claim", "copies", "count")]
                + [(n, c_int) for n in ("seqs", "width", "pages", "page", "layout")])


def _entry():
    if not _ENTRY:
        lib = _lib.load()
        if lib.snu1_page_tables_bytes() != ctypes.sizeof(_Args):
            raise _lib.NativeLibraryError(f"{_lib.lib_path()} has tables of another size: build it again (python -m sensenova_u1_b200.build)")
        P, I = c_void_p, c_int
        lib.snu1_page_tables_step.argtypes = (P, P, P, P, I, P)
        lib.snu1_page_tables_copy.argtypes = (P, P, I, I, I, P)
        _ENTRY.update(step=lib.snu1_page_tables_step, copy=lib.snu1_page_tables_copy)
    return _ENTRY


def _uses(lens, tables, page: int, pages: int, width: int):
    """Host side of :meth:`PageTables.load`: checks, the table's rows, and how many sequences hold every page."""
    lens = _whole("lengths", lens).reshape(-1)
    if len(tables) != len(lens):
        raise ValueError("one page table per sequence")
    if (lens < 0).any() or (lens > width * page).any():
        raise ValueError(f"a sequence has 0 to {width * page} tokens")
    table, refs, part = torch.full((len(lens), width), -1, dtype=torch.int32), torch.zeros(pages, dtype=torch.int32), []
    for i, n in enumerate(lens.tolist()):
        need = -(-n // page)
        row = _whole("pages", tables[i])[:need] if len(tables[i]) else _whole("pages", [0])[:0]
        if len(row) < need:
            raise ValueError(f"sequence {i} needs {need} pages for {n} tokens, its table has {len(row)}")
        if need and (row.min() < 0 or row.max() >= pages):
            raise ValueError(f"sequence {i} names a page that the caches do not have")
        row = torch.from_numpy(row.astype("int32"))
        if len(row.unique()) != need:
            raise ValueError(f"sequence {i} has a page twice")
        table[i, :need] = row
        refs[row.long()] += 1
        if n % page:
            part.append((i, int(row[-1])))
    for i, p in part:
        if refs[p] != 1:
            raise ValueError(f"the last page of sequence {i} is not full: no other sequence may have it")
    return table, refs


class PageTables:
    """``caches``: all of one geometry and device, one or as many as there are layers.  ``seqs`` sequences of up to ``tokens`` tokens each, all of them
    empty at first.  On the device: ``table`` int32 [seqs, pages of a sequence] (-1: none), ``lens`` int32 [seqs], ``refs`` int32 [pages], how many
    sequences hold a page.  They are read by plans and changed by :meth:`step` and :meth:`load` only."""

    def __init__(self, caches, seqs: int, tokens: int):
        caches = [caches] if isinstance(caches, PagedCache) else list(caches)
        if not 1 <= len(caches) <= MAX_CACHES or not 1 <= seqs <= MAX_SEQS or tokens < 1:
            raise ValueError(f"tables are of 1 to {MAX_CACHES} caches, 1 to {MAX_SEQS} sequences, and at least one token")
        first = caches[0]
        if any(c._key != first._key or c.pages != first.pages for c in caches):
            raise ValueError("the caches of one set of tables have one geometry, type, number of pages and device")
        if len({c.data.data_ptr() for c in caches}) != len(caches):
            raise ValueError("a cache is there twice")
        self.caches, self.device, self.page, self.pages, self.seqs = tuple(caches), first.device, first.page, first.pages, seqs
        self.width = -(-tokens // first.page)
        if self.width * first.page >= 1 << 30:
            raise ValueError("too many tokens for one sequence")
        make = lambda *shape, value=0: torch.full(shape, value, dtype=torch.int32, device=self.device)
        self.table, self.lens, self.refs = make(seqs, self.width, value=-1), make(seqs), make(self.pages)
        self._claim, self._copies, self._count = make(self.pages, value=MAX_SEQS), make(seqs, 4), make(1)
        self._layers = torch.tensor([[c.data.data_ptr() for c in caches], [0 if c.scales is None else c.scales.data_ptr() for c in caches]],
                                    dtype=torch.int64).to(self.device)
        _entry()
        self._args = _Args(*(t.data_ptr() for t in (self.table, self.lens, self.refs, self._claim, self._copies, self._count)),
                           seqs, self.width, self.pages, self.page, LAYOUT)
        self._addr, self._index = ctypes.addressof(self._args), self.device.index

    def load(self, lens, tables) -> None:
        """All sequences' lengths and pages as the host has them: ``tables`` lists of page numbers in order.  Full pages may be in several tables."""
        if len(_whole("lengths", lens).reshape(-1)) != self.seqs:
            raise ValueError(f"the tables have {self.seqs} sequences")
        table, refs = _uses(lens, tables, self.page, self.pages, self.width)
        self.table.copy_(table)
        self.refs.copy_(refs)
        self.lens.copy_(torch.as_tensor(_whole("lengths", lens)).reshape(-1))

    def _per_seq(self, name: str, t):
        if t is None:
            return None
        if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.shape != (self.seqs,) or t.get_device() != self._index or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous int32 [{self.seqs}] on the caches' device")
        return t.data_ptr()

    def step(self, tokens, parents: torch.Tensor | None = None, keep: torch.Tensor | None = None) -> None:
        """Every sequence goes on from the first ``keep`` tokens (default: all) of its parent (int32 [seqs], -1: of nobody; default: itself), as they were
        before the step, and gets pages for ``tokens`` more (one number, or int32 [seqs]).  May be captured in a CUDA graph.

        Where there are not enough free pages, or a sequence would have more tokens than the tables have room for, or a parent does not exist,
        ``check_status`` raises: what is missing stays without a page (-1), and attention and writing report it if they get there."""
        index = self._index
        if index != torch._C._cuda_getDevice():
            with torch.cuda.device(index):
                return self.step(tokens, parents, keep)
        each = 0
        if isinstance(tokens, torch.Tensor):
            more = self._per_seq("tokens", tokens)
        else:
            more, each = None, tokens
            if not isinstance(each, int) or isinstance(each, bool) or not 0 <= each < 1 << 30:
                raise ValueError("tokens is a number of new tokens, or int32 [sequences]")
        parents, keep = self._per_seq("parents", parents), self._per_seq("keep", keep)
        entry, stream = _entry(), torch._C._cuda_getCurrentRawStream(index)
        _lib.LAUNCHES += 1
        rc = entry["step"](self._addr, parents, keep, more, each, stream)
        if rc == 0 and (parents is not None or keep is not None):            # (a sequence that only grows copies nothing)
            first = self.caches[0]
            _lib.LAUNCHES += 1
            rc = entry["copy"](self._addr, self._layers.data_ptr(), len(self.caches), first.kv_heads, first.scales is not None, stream)
        if rc != 0:
            raise _lib.error("page_tables_step", rc)
