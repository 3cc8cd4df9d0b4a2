"""Paged key/value cache and attention over it (csrc/paged_cache.cu, csrc/attn_paged.cu, csrc/attn_paged_sm100.cu).

A :class:`PagedCache` holds the keys and values of one layer in pages of 16, 32, 64 or 128 tokens, as bf16 or as e4m3 codes with
one fp32 scale per token and head (half the memory: 132 bytes of 256).  Codes are finite and scales not negative, as
:func:`paged_write` leaves them; a row that holds a value that is not finite has NaN as its scale.  A sequence owns pages in any order; several sequences may
read the same page (a shared prompt), only one may write it, and at one place of its table.

One :class:`PagedPlan` describes a step: how many new tokens every sequence brings, how many tokens it has then, and its
pages.  The plan is made once per step on the host and serves every layer::

    plan = build_plan(caches[0], heads, q_lens, kv_lens, tables)
    for layer, cache in zip(layers, caches):
        q, k, v = layer.project(x)                     # [rows, heads, 128], rows of all sequences one after another
        paged_write(cache, k, v, plan)
        o = paged_attention(q, cache, plan, scale)

A sequence may bring one token (a decode step), a few (drafted tokens) or thousands (a chunk of its prompt), all in one plan.
For a captured decode loop, ``build_plan(..., grow=n)`` leaves room for ``n`` further tokens and :meth:`PagedPlan.advance` inside
the graph moves every sequence on by one.  A graph reads the plan's arrays whenever it is replayed: keep the plan as long as the graph.

A call runs on the current stream of the tensors' device.  A plan's device arrays belong to the streams that are ordered after
the one it was built on; calls that only read (write into different caches, attention, reading back) may share it.
"""
from __future__ import annotations

import ctypes
import random
from dataclasses import dataclass, field

import numpy as np
import torch

from . import _lib
from ._lib import c_float, c_int, c_ll, c_void_p

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIM = 128
E4M3 = torch.float8_e4m3fn
KEY_TILE = 64            # keys of a stage of the kernel for few rows
FEW_SLOTS = (444, 296)   # its CTAs that run at once: of up to eight rows three on each of 148 SMs, otherwise two
FEW_LEAST = 4            # a part of a sequence has at least this many key tiles
# 17 to 24 rows have a kernel of their own (else that for 32): e4m3 always, bf16 from so many key tiles per CTA on.  Us, 20 rows,
# 32 / 8 heads, the former / the latter: e4m3 1 x 1000 keys 11.3 / 11.8, 8 x 12000 62 / 85; bf16 1 x 1000 12.2 / 10.4, 8 x 1000 15.5 / 14.4,
# 8 x 12000 70.7 / 74.6, 24 x 4000 84 / 88.
FEW_24 = 16
FEW_JOIN = 8             # up to so many rows the parts of few rows join themselves (JOIN_ROWS in attn_paged.cu)
FEW_CLUSTER = 8          # up to so many parts are a cluster, if all sequences can have as many
FEW_TILE = 32            # rows (new tokens x query heads of a group) of one CTA, at most
# More rows of a sequence are a chunk.  Chunk kernel / few rows, us, 32 / 8 heads, sequences of 12000 keys: bf16 1 x 32 rows
# 21 / 23, 8 x 32 86 / 79, 1 x 48 24 / 27, 8 x 48 88 / 135; e4m3 1 x 32 22 / 24, 8 x 32 93 / 86, 24 x 32 of 4000 keys 120 / 108, 8 x 32 of
# 1000 20 / 16, 1 x 48 22 / 32, 8 x 48 93 / 154.
CHUNK_FROM = FEW_TILE
CHUNK_TILE = 128         # keys of a tile of the kernel for chunks, and rows of a row tile
# e4m3 chunks of up to so many rows are widened by the CTAs that read them, one row tile each; longer ones are widened once.
# Us, the former / the latter: 8 sequences of 12000 keys, 128 rows 101 / 202, 256 177 / 234, 512 349 / 330; of 1000 keys 21 / 28, 22 / 32,
# 42 / 34.
ONE_MOST = 256
CHUNK_SLOTS = 148        # its CTAs that run at once
CHUNK_START = 5          # what starting and ending a CTA costs, in key tiles (1.8 us): 8 to 10 us from its start to its end
CHUNK_JOIN = 3           # what a part costs besides: 128 KB written and read again
PREFIX_ROWS = 64         # rows of a CTA of the kernel for shared tokens, which are counted in tiles of 128
PREFIX_LEAST = 2         # a part has at least this many key tiles
# Sharing costs two launches more, so a run has at least so many tokens (bf16, e4m3), or all runs save at least so many tiles of 128 keys of a head.  Us in
# a graph, with / without, 32 / 8 heads: 32 sequences of 512 bf16 tokens 12.6 / 10.9, of 1024 14.0 / 15.8, of 8192 22 / 83; 4 of 2048 10.6 / 11.3, e4m3 11.3 /
# 11.5; 8 of 3200 11.6 / 12.3, e4m3 12.3 / 13.2.  Two sequences alone are even at 3000 (e4m3 3300) tokens, and with 4 heads beyond 4096: from the limit up to there
# sharing takes 0.5 to 2 us more (2 of 2048 10.2 / 8.2; e4m3, 4 heads, 2 of 2560 10.6 / 8.4).
SHARE_TOKENS, SHARE_TILES = (2048, 2560), 1900
# Us on an SM, by type (bf16, e4m3): to start and end a CTA, and one of its tiles.  Of shared tokens: 64 rows, and as chunks 256 (128) rows.  Of
# tails, two or three of which share the SM, both for the CTA's share of it.
PREFIX_COST = ((6.0, 1.5), (6.0, 1.55))
MANY_COST = ((9.0, 1.8), (9.0, 1.75))
TAIL_COST = ((1.7, 1.5), (1.7, 1.05))


_ENTRY: dict = {}         # the entry points that calls go to


def _library():
    """The library, its entry points told the types of their arguments (cheaper than an object per argument and call)."""
    lib = _lib.load()
    if not _ENTRY:
        if lib.snu1_paged_plan_bytes() != ctypes.sizeof(_Args):
            raise _lib.NativeLibraryError(f"{_lib.lib_path()} has plans of another size: build it again (python -m sensenova_u1_b200.build)")
        P, L, I = c_void_p, c_ll, c_int
        lib.snu1_paged_cache_init.argtypes = (P, P, P, I, I, I, I)
        lib.snu1_paged_read.argtypes = (P, P, P, P, P)
        lib.snu1_paged_attention.argtypes = (P, P, P, L, P, L, c_float, P, ctypes.c_ulonglong, P)
        lib.snu1_paged_write.argtypes = (P, P, P, L, P, L, P)
        for name in ("paged_write", "paged_read", "paged_attention"):
            _ENTRY[name] = getattr(lib, "snu1_" + name)
    return lib


class PagedCache:
    """Keys and values of one layer: ``data`` [pages, 2, kv_heads, page, 128] (bf16 or float8_e4m3fn; index 0 of the second
    dimension are the keys), ``scales`` [pages, 2, kv_heads, page] fp32 for e4m3 (value = code * scale), else None."""

    def __init__(self, data: torch.Tensor, scales: torch.Tensor | None = None):
        if data.dim() != 5 or data.shape[1] != 2 or data.shape[4] != HEAD_DIM or data.shape[0] < 1 or data.shape[2] < 1:
            raise ValueError("a paged cache is [pages, 2, kv_heads, page, 128]")
        if data.dtype not in (torch.bfloat16, E4M3):
            raise ValueError("a paged cache holds bfloat16 or float8_e4m3fn")
        if data.shape[3] not in PAGE_SIZES:
            raise ValueError(f"a page holds 16, 32, 64 or 128 tokens, not {data.shape[3]}")
        if (data.dtype == E4M3) != (scales is not None):
            raise ValueError("e4m3 codes, and only they, have scales")
        if not data.is_contiguous() or (scales is not None and not (
                scales.dtype == torch.float32 and scales.shape == data.shape[:4] and scales.is_contiguous()
                and scales.device == data.device)):
            raise ValueError("data and scales [pages, 2, kv_heads, page] (fp32) must be contiguous, on one device")
        if not data.is_cuda:
            raise ValueError("a paged cache is in GPU memory")
        self._data, self._scales = data, scales
        self.pages, _, self.kv_heads, self.page, _ = data.shape
        if self.kv_heads > 1023 or self.pages >= 1 << 31:
            raise ValueError("too many heads or pages")
        self._key = (data.dtype, self.page, self.kv_heads, data.get_device())
        self._desc = ctypes.create_string_buffer(_library().snu1_paged_cache_bytes())
        self._addr = ctypes.addressof(self._desc)
        with torch.cuda.device(data.device):
            _lib.call("paged_cache_init", self._addr, data.data_ptr(), None if scales is None else scales.data_ptr(), self.pages,
                      self.kv_heads, self.page, 0 if scales is None else 1)

    @classmethod
    def empty(cls, pages: int, page: int, kv_heads: int, dtype=torch.bfloat16, device="cuda") -> "PagedCache":
        data = torch.empty(pages, 2, kv_heads, page, HEAD_DIM, dtype=dtype, device=device)
        return cls(data, torch.empty(data.shape[:4], dtype=torch.float32, device=device) if dtype == E4M3 else None)

    @property
    def data(self) -> torch.Tensor:
        return self._data

    @property
    def scales(self) -> torch.Tensor | None:
        return self._scales

    @property
    def device(self) -> torch.device:
        return self._data.device


PLAN_LAYOUT = 0x70670005     # last word of a plan: the library refuses one whose fields lie elsewhere


class _Args(ctypes.Structure):
    """``Plan`` of csrc/paged.cuh."""
    _fields_ = ([(n, c_void_p) for n in ("q_start", "kv_len", "cap", "table", "behind", "row_seq", "k_start", "read_pages", "unpack",
                                         "unpack_first", "few", "chunk", "one", "merge", "skip", "lead", "runs", "prefix", "tail", "joins", "run_start", "run_len", "run_seq",
                                         "many", "own_q_start", "own_kv_len", "own_cap")]
                + [(n, c_int) for n in ("seqs", "rows", "width", "page", "group", "read_count", "few_count", "few_rows", "few_parts", "few_cluster",
                                        "chunk_count", "one_count", "merge_count", "partial_rows", "prefix_count", "tail_count", "tail_rows", "join_count", "many_count",
                                        "unpack_count", "layout")])


@dataclass
class PagedPlan:
    """One step of a batch; see the module's text.  ``kv_len`` is the device's copy of the lengths."""
    heads: int
    kv_heads: int
    page: int
    pages: int
    dtype: torch.dtype            # of the caches
    device: torch.device
    q_lens: list
    kv_lens: list
    rows: int
    keys: int                     # rows that paged_read gives
    scratch: int                  # bytes that attention needs beside its output
    kv_len: torch.Tensor
    grow: int
    _store: torch.Tensor = field(repr=False)
    _args: _Args = field(repr=False)
    _rows: torch.Tensor = field(repr=False)       # sequence of every row
    _ends: torch.Tensor = field(repr=False)       # row behind the last of every sequence
    tables: object = field(default=None, repr=False)      # the PageTables that it reads

    def __post_init__(self):
        self._index = self.device.index
        # what an output and the scratch are like (half the host time of naming shape, type and device)
        like = self._store.view(torch.bfloat16)[:1]
        self._out, self._scratch = like.expand(self.rows, self.heads, HEAD_DIM), like.expand(self.scratch // 2)
        self._read = like.expand(self.keys, self.kv_heads, HEAD_DIM)
        self._key = (self.dtype, self.page, self.kv_heads, self._index)
        self._addr = ctypes.addressof(self._args)

    def advance(self, tokens: int = 1) -> None:
        """Every sequence has ``tokens`` more (up to ``grow`` in all; beyond that nothing is written, attention reads up to the last
        token that the plan has room for, and ``check_status`` raises after either): its new rows are the ``q_len`` last ones of the longer
        sequence.  Runs on the device and may be captured; :func:`paged_read` keeps the lengths that the plan was made with."""
        if self.tables is not None:
            raise RuntimeError("the lengths are those of the plan's tables: their step() moves them on")
        self.kv_len.add_(tokens)

    def positions(self) -> torch.Tensor:
        """Place of every new row in its sequence, int32 on the device (by the lengths that the device has, also in a captured step)."""
        seq = self._rows.long()
        return self.kv_len[seq] - self._ends[seq] + torch.arange(self.rows, dtype=torch.int32, device=self.device)


def _shares(tiles: np.ndarray, heads: int, slots: int, least: int) -> np.ndarray:
    """Into how many parts the key tiles of every work item are split.  ``heads`` CTAs run per part and ``slots`` at once: parts
    are as short as they may be (``least`` tiles) while all of them run in one wave; where even whole items are more than
    that, only items longer than a fair share are split."""
    if not len(tiles):
        return tiles
    tiles = np.maximum(tiles, 1)
    share = max(least, 1)
    if len(tiles) * heads <= slots:
        hi = int(tiles.max())
        lo = share
        while lo < hi:                                        # least share whose parts fit
            mid = (lo + hi) // 2
            if int((-(-tiles // mid)).sum()) * heads <= slots:
                hi = mid
            else:
                lo = mid + 1
        share = max(share, lo)
    else:
        share = max(share, -(-int(tiles.sum()) * heads // slots))
    return -(-tiles // share)


def _whole(what: str, x) -> np.ndarray:
    """``x`` as int64; numbers that are not whole are refused, not cut."""
    a = np.asarray(x)
    if a.size and a.dtype.kind not in "iu":
        raise ValueError(f"{what} must be whole numbers, not {a.dtype}")
    return a.astype(np.int64, copy=False)


def _shared_runs(shared, n: int, q, kv, few, table, page: int):
    """Which sequences read their first tokens together: runs [first sequence, sequences, tokens] of sequences with few rows, tokens in whole
    tiles of 128, and the tokens that each sequence leaves to its run."""
    skip, runs, taken = np.zeros(n, dtype=np.int64), [], np.zeros(n, dtype=bool)
    for entry in shared:
        first, count, tokens = (int(x) for x in _whole("shared", entry).reshape(3))
        if first < 0 or count < 1 or first + count > n or tokens < 0 or taken[first:first + count].any():
            raise ValueError("shared names sequences [first, how many, shared tokens], each at most once")
        taken[first:first + count] = True
        if (kv[first:first + count] < tokens).any():
            raise ValueError("a sequence has fewer tokens than it shares")
        tokens = tokens // CHUNK_TILE * CHUNK_TILE
        if table is not None and (table[first:first + count, :tokens // page] != table[first, :tokens // page]).any():
            raise ValueError("sequences that share tokens must have them in the same pages")
        start = first
        for i in range(first, first + count + 1):             # a chunk reads its keys itself
            if i < first + count and (few[i] or q[i] == 0):
                continue
            if tokens and (q[start:i] > 0).sum() > 1:
                runs.append((start, i - start, tokens))
                skip[start:i] = np.where(q[start:i] > 0, tokens, 0)
            start = i + 1
    return runs, skip


def _lay_out(q_lens, kv_lens, tables, page: int, pages: int, group: int, kv_heads: int, fp8: bool, limits, grow: int, shared=()):
    """Host side of :func:`build_plan`: checks, and every array of the plan as int32.  ``tables`` may be the number of pages of a table on the device."""
    q, kv = _whole("lengths", q_lens).reshape(-1), _whole("lengths", kv_lens).reshape(-1)
    n = len(q)
    if len(kv) != n or (q < 0).any() or (kv < q).any() or grow < 0:
        raise ValueError("every sequence has q_len >= 0 new tokens among its kv_len >= q_len tokens, and grow >= 0")
    if n > 65535 or group > 65535 or (n and (kv.max() + grow >= 1 << 30 or q.sum() * group >= 1 << 31 or kv.sum() >= 1 << 31)):
        raise ValueError("too many sequences or tokens for one plan")
    cap = np.where(q > 0, kv + grow, kv)
    need = -(-cap // page)
    width = max(1, int(need.max()) if n else 1)
    on_device = isinstance(tables, int)
    if on_device:
        if width > tables:
            raise ValueError(f"a sequence has up to {cap.max()} tokens, the tables have room for {tables * page}")
        width, tables = tables, [()] * n
    table = np.zeros((n, 0 if on_device else width), dtype=np.int64)
    if isinstance(tables, torch.Tensor):
        if tables.is_cuda or tables.dim() != 2 or tables.is_floating_point():
            raise ValueError("page tables are lists of page numbers, or one host tensor [sequences, pages]")
        tables = tables.numpy()
    whole = isinstance(tables, np.ndarray) and tables.dtype.kind in "iu"
    if len(tables) != n:
        raise ValueError("one page table per sequence")
    for i in range(0 if on_device else n):
        if len(tables[i]) < need[i]:
            raise ValueError(f"sequence {i} needs {need[i]} pages for {cap[i]} tokens, its table has {len(tables[i])}")
        table[i, :need[i]] = tables[i][:need[i]] if whole else _whole("pages", tables[i][:need[i]])
    if table.size and (table.min() < 0 or table.max() >= pages):          # (places that are not needed hold 0)
        i = int(((table < 0) | (table >= pages)).any(1).argmax())
        raise ValueError(f"sequence {i} names a page that the cache does not have")
    table = table.astype(np.int32)
    rows = int(q.sum())
    row_seq = np.repeat(np.arange(n, dtype=np.int32), q)
    behind = None
    if limits is not None:
        lim = _whole("limits", limits).reshape(-1)
        if grow:
            raise ValueError("limits are fixed: a plan with limits cannot grow")
        if len(lim) != rows or (lim < 0).any() or (lim > kv[row_seq]).any():
            raise ValueError("one limit per row, between 0 and the keys of its sequence")
        behind = (kv[row_seq] - lim).astype(np.int32)
    start = lambda x: np.concatenate([[0], np.cumsum(x)]).astype(np.int32)
    read = -(-kv // page)
    pages_of = lambda c: np.stack([np.repeat(np.arange(n), c), np.arange(int(c.sum())) - np.repeat(np.cumsum(c) - c, c)], 1).astype(np.int32)
    # attention: tiles of rows, split over keys
    q_rows = q * group
    chunked = (q_rows > CHUNK_FROM) & (group <= CHUNK_TILE)
    runs, skip = _shared_runs(shared, n, q, kv, (q_rows > 0) & (q_rows <= FEW_TILE) & ~chunked, None if on_device else table, page)
    if runs and max(t for _, _, t in runs) < SHARE_TOKENS[fp8] and (
            kv_heads * sum((int((q[a:a + c] > 0).sum()) - 1) * t for a, c, t in runs) < SHARE_TILES * CHUNK_TILE):
        runs, skip = [], np.zeros(n, dtype=np.int64)
    few_q = np.where(chunked | (skip > 0), 0, q_rows)
    top = int(few_q.max()) if n else 0
    few_rows = 8 if top <= 8 else 16 if top <= 16 else FEW_TILE
    if 16 < top <= 24 and (fp8 or int((-(-cap[few_q > 0] // KEY_TILE)).sum()) * kv_heads >= FEW_24 * FEW_SLOTS[1]):
        few_rows = 24
    tile_rows = (CHUNK_TILE // group) * group if group <= CHUNK_TILE else 1      # a row tile is made of whole tokens
    single = chunked & fp8 & (q_rows <= ONE_MOST)              # widened by the CTAs that read it

    def tiles_of(q_rows, m):
        count = -(-q_rows // m)
        seq = np.repeat(np.arange(n), count)
        return seq, (np.arange(len(seq)) - np.repeat(np.cumsum(count) - count, count)) * m

    seq, row0 = tiles_of(few_q, few_rows)
    tiles = -(-cap[seq] // KEY_TILE)
    slots = FEW_SLOTS[few_rows > 8]
    parts = _shares(tiles, kv_heads, slots, FEW_LEAST)
    cluster = int(parts.max()) if len(parts) else 1
    if 1 < cluster <= FEW_CLUSTER and len(seq) * cluster * kv_heads <= slots:      # as many parts for everybody, side by side
        part = np.tile(np.arange(cluster), len(seq))
        few = np.stack([np.repeat(seq, cluster), np.repeat(row0, cluster), part | cluster << 16, np.full(len(part), -1)], 1).astype(np.int32)
        merge, partial = np.zeros((0, 4), np.int32), 0
    else:
        few, merge, partial = _items(seq, row0, tiles, parts, few_q, few_rows, 0)
        cluster = 1
    few_parts = partial // few_rows if few_rows <= FEW_JOIN else 0       # parts that join themselves
    merge = [] if few_rows <= FEW_JOIN else [merge]

    def chunks_of(which, m, partial):
        if not which.any():
            return np.zeros((0, 4), np.int32), partial
        seq, row0 = tiles_of(np.where(which, q_rows, 0), m)
        if limits is None:                                    # a row tile reads up to its last token
            last = np.minimum((row0 + m - 1) // group, q[seq] - 1)
            tiles = -(-(cap[seq] - q[seq] + 1 + last) // CHUNK_TILE)
        else:
            tiles = -(-kv[seq] // CHUNK_TILE)
        items, join, partial = _items(seq, row0, tiles, _waves(tiles, kv_heads, CHUNK_SLOTS), q_rows, m, partial)
        merge.append(join)
        return items, partial

    one, partial = chunks_of(single, tile_rows, partial)
    chunk, partial = chunks_of(chunked & ~single, 2 * tile_rows, partial)
    merge = np.concatenate(merge) if merge else np.zeros((0, 4), np.int32)
    together = dict(skip=None, lead=None, runs=None, prefix=None, tail=None, joins=None, run_start=None, run_len=None, run_seq=None, many=None)
    tail_rows = 0
    if runs:
        together, tail_rows, partial = _together(runs, skip, q_rows, cap, start(q), group, kv_heads, fp8, partial)
        if on_device:
            together["lead"] = np.arange(n, dtype=np.int32)
            for first, count, _ in runs:
                together["lead"][first:first + count] = first
    unpack = unpack_first = None
    if fp8 and len(chunk):
        wide = np.where(chunked & ~single, -(-cap // CHUNK_TILE), 0)    # 128-token pages
        unpack, unpack_first = pages_of(wide), start(wide)[:n]
    arrays = dict(q_start=start(q), kv_len=kv.astype(np.int32), cap=cap.astype(np.int32), table=table, behind=behind, row_seq=row_seq,
                  k_start=start(kv), read_pages=pages_of(read), unpack=unpack, unpack_first=unpack_first, few=few, chunk=chunk,
                  one=one, merge=merge, **together)
    if on_device:
        arrays["table"] = arrays["kv_len"] = None
    counts = dict(seqs=n, rows=rows, width=width, page=page, group=group, read_count=int(read.sum()), few_count=len(few),
                  few_rows=few_rows, few_parts=few_parts, few_cluster=cluster, chunk_count=len(chunk), one_count=len(one), merge_count=len(merge),
                  partial_rows=partial, prefix_count=len(together["prefix"]) if runs else 0, tail_count=len(together["tail"]) if runs else 0,
                  tail_rows=tail_rows, join_count=len(together["joins"]) // 2 if runs else 0, many_count=len(together["many"]) if runs else 0,
                  unpack_count=0 if unpack is None else len(unpack), layout=PLAN_LAYOUT)
    return arrays, counts


def _together(runs, skip, q_rows, cap, q_start, group: int, heads: int, fp8: bool, first: int):
    """Work on tokens that runs of sequences share (prefix, and many for runs of more rows than that kernel's CTAs have), on the other tokens of these
    sequences (tail), and the joins of both, [row, head of the group, partial row, parts | partial row, parts, rows of a part, rows of a part of the
    shared tokens] for every row."""
    runs = np.array([[q_start[a], q_start[a + n] - q_start[a], a, t, n] for a, n, t in runs])
    rows, tokens = runs[:, 1] * group, runs[:, 3]
    # (The kernel for chunks holds probabilities over bf16 in one bf16 number, 2^-8 of each, and keys over e4m3 as fp16, where the one for 64 rows has two numbers
    # and the codes: 2.2e-3 of the output's norm instead of 1.7e-3, of which 1.6e-3 are its own rounding.  64 sequences of 32000 tokens 71 us instead of 115.)
    big = (rows > PREFIX_ROWS) & (group <= CHUNK_TILE)
    # tails: sequences, rows of a CTA, items, their tiles and parts
    seqs = np.concatenate([np.arange(a, a + n) for a, n in runs[:, [2, 4]]])
    top = int(q_rows[seqs].max())
    m_tail = 8 if top <= 8 else 16 if top <= 16 else FEW_TILE
    slots = FEW_SLOTS[m_tail > 8]
    tail_count = -(-q_rows[seqs] // m_tail)
    tail_seq = np.repeat(seqs, tail_count)
    tail_tiles = -(-(cap - skip)[tail_seq] // KEY_TILE)
    tail_parts = _shares(tail_tiles, heads, slots, FEW_LEAST)
    tail_us = heads / CHUNK_SLOTS * (tail_parts.sum() * TAIL_COST[fp8][0] + tail_tiles.sum() * KEY_TILE / CHUNK_TILE * TAIL_COST[fp8][1])
    whole = (CHUNK_TILE // group) * group if group <= CHUNK_TILE else 1
    joins = np.zeros((int(rows.sum()), 8), dtype=np.int64)
    of_run = np.repeat(np.arange(len(runs)), rows)
    place = np.arange(len(of_run)) - np.repeat(np.cumsum(rows) - rows, rows)
    joins[:, 0] = runs[of_run, 0] + place // group
    joins[:, 1] = place % group
    # Long runs as chunks or as many items of 64 rows, whichever is done sooner.
    best = None
    for by_chunks in (big, np.zeros_like(big)):
        kinds = []
        for name, which, m, cost in (("many", by_chunks, whole if fp8 else 2 * whole, MANY_COST[fp8]), ("prefix", ~by_chunks, PREFIX_ROWS, PREFIX_COST[fp8])):
            count = np.where(which, -(-rows // m), 0)
            run = np.repeat(np.arange(len(runs)), count)
            kinds.append((name, which, m, count, run, tokens[run] // CHUNK_TILE, cost))
        done, parts = _shared_parts([(k[5], *k[6]) for k in kinds], heads, heads * int(tail_parts.sum()), slots, tail_us)
        if best is None or done < best[0]:
            best = (done, kinds, parts)
    work = {}
    for (name, which, m, count, run, tiles, _), parts in zip(best[1], best[2]):
        row0 = (np.arange(len(run)) - np.repeat(np.cumsum(count) - count, count)) * m
        at = first + np.cumsum(parts * m) - parts * m
        first += int((parts * m).sum())
        i = np.repeat(np.arange(len(run)), parts)
        part = np.arange(len(i)) - np.repeat(np.cumsum(parts) - parts, parts)
        items = np.stack([run[i], row0[i], part | parts[i] << 16, at[i] + part * m], 1).reshape(-1, 4)
        if name == "many":
            items[:, 0] *= 2
        work[name] = items.astype(np.int32)
        here = which[of_run]                                      # every row of such a run: partial rows of its part 0, and parts
        item = ((np.cumsum(count) - count)[of_run] + place // m)[here]
        joins[here, 2] = at[item] + (place % m)[here]
        joins[here, 3] = parts[item]
        joins[here, 7] = m
    row0 = (np.arange(len(tail_seq)) - np.repeat(np.cumsum(tail_count) - tail_count, tail_count)) * m_tail
    at = first + np.cumsum(tail_parts * m_tail) - tail_parts * m_tail
    first += int((tail_parts * m_tail).sum())
    i = np.repeat(np.arange(len(tail_seq)), tail_parts)
    part = np.arange(len(i)) - np.repeat(np.cumsum(tail_parts) - tail_parts, tail_parts)
    tail = np.stack([tail_seq[i], row0[i], part | tail_parts[i] << 16, at[i] + part * m_tail], 1)
    order = np.argsort(-(tail_tiles[i] / tail_parts[i]), kind="stable")
    rows = q_rows[seqs]
    of_seq = np.repeat(np.arange(len(seqs)), rows)
    place = np.arange(len(of_seq)) - np.repeat(np.cumsum(rows) - rows, rows)
    item = (np.cumsum(tail_count) - tail_count)[of_seq] + place // m_tail
    joins[:, 4] = at[item] + place % m_tail
    joins[:, 5] = tail_parts[item]
    joins[:, 6] = m_tail
    twice = lambda x, y: np.stack([x, y], 1).reshape(-1).astype(np.int32)
    return (dict(skip=skip.astype(np.int32), runs=runs[:, :4].astype(np.int32), tail=tail[order].astype(np.int32), joins=joins.reshape(-1, 4).astype(np.int32),
                 run_start=twice(runs[:, 0], runs[:, 0] + runs[:, 1]), run_len=twice(tokens, tokens), run_seq=twice(runs[:, 2], runs[:, 2]), **work),
            m_tail, first)


def _shared_parts(kinds, heads: int, tails: int, slots: int, us: float):
    """Into how many parts the work on shared tokens is split, for every kind [tiles of its items, us to start a CTA, us of a tile], and when all is
    done.  Its CTAs have an SM each.  ``tails`` CTAs, of which ``slots`` fill all SMs, take no time of their own if all of them fit the SMs that are left;
    otherwise most of them run afterwards, ``us`` in all.  (bf16, 32 / 8 heads, by CTAs for shared tokens: 8 sequences of 4200 + 60 tokens 128: 15.8 us, 88: 11.9;
    16 of 32000 + 1000, whose tails need all SMs, 104: 48.9, 144: 44.6.  Over 25 such calls, cut into 3 to 20 parts each, the choice took 1.2 % more than
    the best.  Most of that is calls whose last few tails are alone: 64 of 8000 + 400 50.8, with 88 CTAs 45.5; models of their turns chose worse elsewhere.)

    More CTAs than SMs are taken up where that is clearly sooner: a long run beside many short ones is not left whole (8 sequences of 40000 tokens and 18 runs of
    4 x 2560 363 -> 85 us, 4 x (8 of 3000, 6000, 9000, 12000 and 30000) 323 -> 199).  By less than a tenth the model does not know (30 runs of 8 x 8000, cut in two 202 -> 218)."""
    sizes = [(int(t), int(c), start, tile) for tiles, start, tile in kinds for t, c in zip(*np.unique(tiles, return_counts=True))]
    longest = max((t for t, *_ in sizes), default=1)
    best, share = None, 0
    for cut in range(1, 2 * CHUNK_SLOTS):
        if -(-longest // cut) == share:
            continue
        share = -(-longest // cut)
        split = [(c, -(-t // share), start + -(-t // -(-t // share)) * tile) for t, c, start, tile in sizes]       # items, parts, us of one
        ctas = heads * sum(c * n for c, n, _ in split)
        if best is not None and share < PREFIX_LEAST:
            break
        busy = max(t for *_, t in split)
        if ctas > CHUNK_SLOTS:
            busy = max(busy, heads / CHUNK_SLOTS * sum(c * n * t for c, n, t in split) + busy / 2)
        done = busy + (0.0 if tails <= slots // CHUNK_SLOTS * (CHUNK_SLOTS - ctas) else us + 4.0)
        if best is None or done < (0.9 if ctas > CHUNK_SLOTS else 1.0) * best[0]:
            best = (done, share)
    return best[0], [-(-tiles // best[1]) for tiles, _, _ in kinds]


def _waves(tiles: np.ndarray, heads: int, slots: int) -> np.ndarray:
    """Parts of the chunk kernel's items: of the shares that cut the longest item into up to 16 parts, the one that is done
    first when the CTAs are taken up longest first.  Starting and ending a CTA costs ``CHUNK_START`` key tiles, what a part
    writes and its join reads ``CHUNK_JOIN``."""
    if not len(tiles):
        return tiles
    tiles = np.maximum(tiles, 1)
    best = None
    for cut in range(1, 17):
        share = -(-int(tiles.max()) // cut)
        parts = -(-tiles // share)
        cost = -(-tiles // parts) + CHUNK_START + np.where(parts > 1, CHUNK_JOIN, 0)
        if best is not None and max(int((cost * parts).sum()) * heads / slots, int(cost.max())) + CHUNK_START / 2 >= 0.98 * best[0]:
            continue                                          # could not be done sooner even if every CTA were as long
        cost = np.sort(np.repeat(cost, parts * heads))[::-1]
        if best is not None and len(cost) > 8 * slots:        # so many waves are full enough
            break
        busy = np.zeros(slots)
        for i in range(0, len(cost), slots):                  # the longest that are left go to those that are free first
            wave = cost[i:i + slots]
            busy.sort()
            busy[:len(wave)] += wave
        done = busy.max() + (CHUNK_START / 2 if cut > 1 else 0)
        if best is None or done < 0.98 * best[0]:
            best = (done, parts)
        if share <= 2:
            break
    return best[1]


def _items(seq, row0, tiles, parts, q_rows, m: int, first: int):
    """Work items [sequence, first row, part | parts << 16, partial row or -1], those with most keys first, the joins of the
    items that were split (four rows each), and the rows of partial results up to there."""
    if not len(seq):
        return np.zeros((0, 4), np.int32), np.zeros((0, 4), np.int32), first
    split = parts > 1
    at = first + np.cumsum(np.where(split, parts * m, 0)) - np.where(split, parts * m, 0)
    have = np.minimum(m, q_rows[seq] - row0)                  # rows of an item
    join = np.where(split, -(-have // 4), 0)
    four = 4 * (np.arange(int(join.sum())) - np.repeat(np.cumsum(join) - join, join))
    merge = np.stack([np.repeat(x, join) for x in (seq, row0, parts | m << 16, at)], 1)
    merge[:, 2] |= np.minimum(4, np.repeat(have, join) - four) << 12
    merge[:, 1] += four
    merge[:, 3] += four
    i = np.repeat(np.arange(len(seq)), parts)
    part = np.arange(len(i)) - np.repeat(np.cumsum(parts) - parts, parts)
    items = np.stack([seq[i], row0[i], part | parts[i] << 16, np.where(split[i], at[i] + part * m, -1)], 1)
    order = np.argsort(-(tiles[i] / parts[i]), kind="stable")
    return items[order].astype(np.int32), merge.astype(np.int32), int(first + np.where(split, parts * m, 0).sum())


def build_plan(cache: PagedCache, heads: int, q_lens, kv_lens, tables, limits=None, grow: int = 0, shared=()) -> PagedPlan:
    """Plan of one step, for ``cache`` and every other cache of its geometry on the same device.

    ``heads``: query heads, a multiple of the cache's.  ``q_lens`` / ``kv_lens``: new tokens of every sequence, and all its
    tokens, the new ones (which are its last) among them.  ``tables``: the pages of every sequence in order, as lists or as one
    host tensor [sequences, at least the pages needed].  ``limits``: for every new row, how many of its sequence's first keys it
    may read (0: none, its output is zeros); without it, every row reads up to itself.  A token of a picture, which
    sees the whole picture, has the picture's end as its limit: the picture is then among the keys, written in this step or before.  ``grow``: tokens that :meth:`PagedPlan.advance` may add.

    ``tables`` may be a :class:`~.page_tables.PageTables` of as many sequences: the plan then reads its tables and lengths as they are when a call
    runs, ``kv_lens`` and ``grow`` say up to how many tokens they go, and its ``step`` stands in for ``advance``.

    ``shared``: one [first sequence, how many, tokens] or more, of sequences that begin with the same tokens in the same pages.  Attention
    reads those once for all of them, where that is faster (in tiles of 128 tokens; the rest, and the keys of chunks, are read by each sequence).  Where more
    than 64 rows (sequences x new tokens x heads of a group) share, it may round as it does for chunks.  Over a ``PageTables`` the sequences need not stay
    alike: one that has been cut, has ended or is another request by now reads from its own pages what it does not hold in common with the
    first of them any more, as long as the tables come from ``step``."""
    if heads < 1 or heads % cache.kv_heads != 0:
        raise ValueError("the number of query heads must be a multiple of the cache's heads")
    with torch.cuda.device(cache.device):                     # (the stream that the copy below goes to)
        capturing = torch.cuda.is_current_stream_capturing()
    if capturing:
        raise RuntimeError("a plan is made before a CUDA graph is captured: the graph would copy from host memory that is gone")
    from .page_tables import PageTables
    live = tables if isinstance(tables, PageTables) else None
    if live is not None:
        if live.page != cache.page or live.pages > cache.pages or live.device != cache.device:
            raise ValueError("the tables are of caches of another page size, size or device")
        if live.seqs != len(q_lens):
            raise ValueError(f"the tables have {live.seqs} sequences")
        tables = live.width
    arrays, counts = _lay_out(q_lens, kv_lens, tables, cache.page, cache.pages, heads // cache.kv_heads, cache.kv_heads,
                              cache.scales is not None, limits, grow, () if shared is None else shared)
    # all arrays in one copy from pinned memory that nothing waits for
    at, total = {}, 0
    for name, a in arrays.items():
        if a is not None:
            at[name] = total
            total += -(-a.size // 4) * 4
    host = torch.empty(max(total, 4), dtype=torch.int32, pin_memory=True)
    flat = host.numpy()
    for name, o in at.items():
        flat[o:o + arrays[name].size] = arrays[name].reshape(-1)
    store = host.to(cache.device, non_blocking=True)
    fields = {name: store.data_ptr() + 4 * o for name, o in at.items()}
    n = counts["seqs"]
    if live is None:
        kv_len = store[at["kv_len"]:at["kv_len"] + n]
    else:
        kv_len = live.lens
        fields |= dict(table=live.table.data_ptr(), kv_len=live.lens.data_ptr())
    args = _Args(**fields, **counts)
    joined = counts["partial_rows"] * cache.kv_heads
    scratch = joined * HEAD_DIM * 4 + (joined + counts["few_parts"] * cache.kv_heads + 15) // 16 * 128 + counts["unpack_count"] * cache.kv_heads * (2 * CHUNK_TILE * HEAD_DIM * 2 + 16)
    return PagedPlan(heads, cache.kv_heads, cache.page, cache.pages, cache.data.dtype, cache.device,
                     [int(x) for x in q_lens], [int(x) for x in kv_lens],
                     counts["rows"], int(arrays["k_start"][-1]), scratch, kv_len, grow, store, args,
                     store[at["row_seq"]:at["row_seq"] + counts["rows"]], store[at["q_start"] + 1:at["q_start"] + 1 + n], live)


_BF16 = torch.bfloat16
_words = random.Random()          # never 0, the word of a flag that is not set; of its own: a program that seeds the global one does not repeat them


def _check(cache: PagedCache, plan: PagedPlan) -> None:
    if cache._key != plan._key or cache.pages < plan.pages:
        raise ValueError("the plan was made for caches of another geometry, type or device")


def _row_stride(name: str, t: torch.Tensor, plan: PagedPlan, heads: int) -> int:
    """Elements from one row to the next of a [plan.rows or more, heads, 128] tensor."""
    try:
        rows, n, dim = t.shape
        row, head, one = t.stride()
    except ValueError:                                            # of other dimensions
        rows = -1
    if (rows < plan.rows or n != heads or dim != HEAD_DIM or one != 1 or (head != HEAD_DIM and heads > 1) or t.dtype is not _BF16
            or t.get_device() != plan._index):
        raise ValueError(f"{name} must be bf16 [{plan.rows} or more, {heads}, {HEAD_DIM}] with contiguous heads on the plan's device")
    if row < heads * HEAD_DIM:
        if rows > 1:
            raise ValueError(f"the rows of {name} overlap")
        return heads * HEAD_DIM                                   # (one row's stride says nothing)
    return row


def _call(index: int, name: str, *args) -> None:
    """On the tensors' device, whichever is current.  (What ``_lib.call`` does, without looking the entry point up: 0.5 us of 6.)"""
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return _call(index, name, *args)
    _lib.LAUNCHES += 1
    rc = _ENTRY[name](*args, torch._C._cuda_getCurrentRawStream(index))
    if rc != 0:
        raise _lib.error(name, rc)


def paged_write(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, plan: PagedPlan) -> None:
    """Keys and values of the plan's new rows into their sequences' pages, quantised where the cache holds e4m3.  ``k`` / ``v``:
    [at least plan.rows, kv_heads, 128] bf16, rows may be slices of wider ones; rows behind the last sequence are ignored.  A
    row is scaled so that its largest value is 448, the largest e4m3 value; one that holds a value that is not finite
    reads back as NaN."""
    _check(cache, plan)
    ldk, ldv = _row_stride("k", k, plan, cache.kv_heads), _row_stride("v", v, plan, cache.kv_heads)
    if plan.rows:
        _call(plan._index, "paged_write", cache._addr, plan._addr, k.data_ptr(), ldk, v.data_ptr(), ldv)


def paged_read(cache: PagedCache, plan: PagedPlan) -> tuple[torch.Tensor, torch.Tensor]:
    """The cached keys and values of the plan's sequences, one sequence after another: two tensors [plan.keys, kv_heads, 128] bf16
    (e4m3: code times scale in fp32, rounded to bf16)."""
    _check(cache, plan)
    k, v = torch.empty_like(plan._read), torch.empty_like(plan._read)
    if plan.keys:
        _call(plan._index, "paged_read", cache._addr, plan._addr, k.data_ptr(), v.data_ptr())
    return k, v


def paged_attention(q: torch.Tensor, cache: PagedCache, plan: PagedPlan, scale: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the plan's new rows over their sequences' cached keys, softmax in fp32.  ``q``: [at least plan.rows, heads,
    128] bf16, rows may be slices of wider ones; returns ``out`` (default: new, [plan.rows, heads, 128]), whose rows behind
    the last sequence are left as they are; ``out`` may be ``q``.  ``scale`` is positive.

    A row that may read a key or value that is not finite is NaN, in part or whole; other rows are as if it were not there.
    What lies behind a sequence's last token or in pages of nobody does not matter.  Queries and scores may have any size as long as the
    products of a query and a key and their sum stay within fp32; chunk rows with scores beyond 2^20 (log2 units) take a slow path.

    Over e4m3 a key adds nothing to the output where its probability times the size of its value is below 2^-32 of the largest such
    product, for shared tokens 2^-28 (and has less than 11 bits below 2^-18); there a query's value below 2^-14 of its row's largest has no bits below
    2^-22 of that.  Over shared bf16 tokens a key adds nothing where its probability is below 2^-100 of the largest.  Chunks (more than 32 rows per key/value head) over e4m3 hold 128 cached tokens' values of a head relative to the largest of
    them (less than 2^-80 counts as that): values 2^27 times smaller than that lose bits.  Where the largest value of another 128 tokens is
    2^d times larger, probabilities below 2^(d - 133) of the largest one are lost."""
    _check(cache, plan)
    ldq = _row_stride("q", q, plan, plan.heads)
    if out is None:
        out = torch.empty_like(plan._out)
        ldo = plan.heads * HEAD_DIM
    else:
        ldo = _row_stride("out", out, plan, plan.heads)
    if plan.rows:
        scratch = torch.empty_like(plan._scratch) if plan.scratch else None
        _call(plan._index, "paged_attention", cache._addr, plan._addr, q.data_ptr(), ldq, out.data_ptr(), ldo, scale,
              scratch.data_ptr() if plan.scratch else None, _words.getrandbits(64) | 1)
    return out
