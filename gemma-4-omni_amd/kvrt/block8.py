"""A paged KV cache held in 8 bits with one scale per (page, KV head).

Where a :class:`~kvrt.runtime.KVRuntime` keeps lengths and page tables on the
host, everything here lives on the GPU, so a serving step over requests of
unequal length is captured once and replayed as the lengths move:

* :class:`BlockTables` — page tables, free pages and slot maps, brought to a
  step's request lengths by :meth:`BlockTables.update`;
* :class:`Block8Pool` — one layer's coded pages (int8 or e4m3): ``append``
  codes new rows into them, ``gather`` reads the zero-padded batch back,
  ``attend`` is attention of each request's newest rows.

One set of tables serves the pools of all layers::

    tables = BlockTables(n, max_pages, pool_pages)
    pools = [Block8Pool.zeros(pool_pages, 8, 128) for _ in range(layers)]
    plan = tables.update(lengths, new, rows=total)      # int32 [n] on the GPU
    for pool, (q, k, v) in zip(pools, projections):      # packed rows [total, heads, 128]
        pool.append(k, v, plan.slot_map)
        out = pool.attend(q, tables.table, plan.lengths, plan.starts, scale, max_q=longest,
                          granted=plan.granted)

Rolling back, a finished request (length 0) and growing are all ``update``
calls. The kernels are hand-written for gfx950 behind include/kvrt.h; there
is no PyTorch or CPU path. Calls run on the current torch stream of the
tensors' device. An object's calls belong on one stream at a time (``update``
and ``append`` write its state); ``gather`` and ``attend`` only read a pool and
may overlap, captured or not: each ``attend`` has a workspace of its own. Pools
have their tables' ``block_size``: page ids and slots do not carry it. The
reference holds no paged or block-scaled KV.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib as L
from .runtime import _check, calls, current_stream_handle, require_cuda, tensor_desc

_calls_mod = None


def _calls():
    """The native call module with the entry points of this module connected."""
    global _calls_mod
    if _calls_mod is None:
        lib, mod = L.load(), calls()
        fns = (lib.kvrt_block_tables_update_async, lib.kvrt_block8_append_async, lib.kvrt_block8_gather_async,
               lib.kvrt_block8_attend_async, lib.kvrt_block8_attend_work)
        mod.connect_blocks(*(ctypes.cast(f, ctypes.c_void_p).value for f in fns))
        _calls_mod = mod
    return _calls_mod


_CODES = {torch.int8: L.DT_INT8, torch.float8_e4m3fn: L.DT_E4M3}
_NAMES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_FLOATS = {torch.bfloat16: 0, torch.float32: 1}
_MASKS = {None: 0, torch.bool: 1, torch.float32: 2, torch.bfloat16: 3}
_I32_MAX = 2 ** 31 - 1


def _device(device: torch.device | str | None) -> torch.device:
    dev = torch.device(device if device is not None else "cuda")
    if dev.type != "cuda" or not torch.cuda.is_available():
        raise RuntimeError("8-bit pages need a ROCm GPU (torch.cuda); there is no CPU path")
    return torch.device("cuda", torch.cuda.current_device()) if dev.index is None else dev


def _int32(t: torch.Tensor, name: str, size: int, device: torch.device) -> torch.Tensor:
    """t, checked: a contiguous int32 vector of that size on the device."""
    require_cuda(t, name)
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != size or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor [{size}], got {t.dtype} {tuple(t.shape)}")
    _same(t, name, device)
    return t


def _same(t: torch.Tensor, name: str, device: torch.device) -> None:
    require_cuda(t, name)
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the pages on {device}")


class _on:
    """The device current for a launch (nothing to do where it already is)."""

    __slots__ = ("guard",)

    def __init__(self, device: torch.device) -> None:
        self.guard = None if torch.cuda.current_device() == device.index else torch.cuda.device(device)

    def __enter__(self) -> None:
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc) -> None:
        if self.guard is not None:
            self.guard.__exit__(*exc)


class _Status:
    """The device word in which kernels report what the host cannot check."""

    _status: torch.Tensor

    def status(self) -> int:
        """Wait for the current stream, then return and clear the reported bits:
        0, or ``BLOCK_BAD_INDEX`` (1: a page id, slot, length or row count out of
        range was skipped), ``BLOCK_NO_PAGES`` (2: a request was refused for want
        of pages), ``BLOCK_NOT_FINITE`` (4: an appended value was not finite). One that
        a call on another stream raises meanwhile may be lost."""
        bits = int(self._status.item())
        if bits:
            self._status.zero_()
        return bits


class BlockPlan(NamedTuple):
    """What :meth:`BlockTables.update` found for a step (int32, on the GPU)."""

    starts: torch.Tensor    # [n + 1] first packed row of each request's new rows
    slot_map: torch.Tensor  # [rows] page * block_size + offset of each packed row, -1: none
    lengths: torch.Tensor   # [n] rows each request holds after the step
    granted: torch.Tensor   # [n] new rows that were given pages: all of a request's, or 0


class BlockTables(_Status):
    """Page tables of ``n`` requests over a pool of ``pool_pages`` pages.

    ``table`` int32 [n, max_pages] (-1: unmapped), ``mapped`` [n] pages each
    request holds, ``free`` [pool_pages] and ``free_count`` [1]: the free page
    ids, the next one taken last. They are ordinary tensors: a caller may set
    them up (or save and restore them) between calls.
    """

    def __init__(self, n: int, max_pages: int, pool_pages: int, *, block_size: int = 16,
                 device: torch.device | str | None = None) -> None:
        self._lib = L.load()
        self.n, self.max_pages, self.pool_pages, self.block_size = map(int, (n, max_pages, pool_pages, block_size))
        if not 1 <= self.n <= 65535 or self.max_pages < 1 or self.pool_pages < 1:
            raise ValueError("tables need 1 to 65535 requests and at least one page")
        if self.block_size not in (16, 32, 64, 128):
            raise ValueError(f"block_size must be 16, 32, 64 or 128, got {block_size}")
        if max(self.n * self.max_pages, self.pool_pages * self.block_size) > _I32_MAX or \
                self.max_pages * self.block_size > 2 ** 30:
            raise ValueError("tables number entries and slots in 32 bits, and hold up to 2^30 positions a request")
        self.device = _device(device)
        make = dict(dtype=torch.int32, device=self.device)
        self.table = torch.full((self.n, self.max_pages), -1, **make)
        self.mapped = torch.zeros(self.n, **make)
        self.free = torch.arange(self.pool_pages - 1, -1, -1, **make)  # page 0 is taken first
        self.free_count = torch.full((1,), self.pool_pages, **make)
        self._work = torch.empty(L.block_tables_work(self.n), **make)
        self._status = torch.zeros(1, **make)
        self._call = _calls()
        self._sizes = self._c()  # what calls read beside the four public tensors
        self._sizes_at = ctypes.addressof(self._sizes)

    def _c(self) -> L.KvrtBlockTables:
        for name, size in (("mapped", self.n), ("free", self.pool_pages), ("free_count", 1)):
            _int32(getattr(self, name), name, size, self.device)
        t = self.table
        if t.dtype != torch.int32 or tuple(t.shape) != (self.n, self.max_pages) or not t.is_contiguous():
            raise ValueError(f"table must be a contiguous int32 tensor [{self.n}, {self.max_pages}]")
        _same(t, "table", self.device)
        c = L.KvrtBlockTables()
        c.table, c.mapped, c.free_pages = t.data_ptr(), self.mapped.data_ptr(), self.free.data_ptr()
        c.free_count, c.work, c.status = self.free_count.data_ptr(), self._work.data_ptr(), self._status.data_ptr()
        c.n, c.max_pages, c.pool_pages, c.block = self.n, self.max_pages, self.pool_pages, self.block_size
        return c

    def update(self, lengths: torch.Tensor, new: torch.Tensor, *, rows: int) -> BlockPlan:
        """Bring the tables to a step: request i keeps its first ``lengths[i]`` rows
        and takes ``new[i]`` more (int32 [n] on the GPU); ``rows`` is the size of
        the packed batch the new rows go into.

        Pages past both are released and pages are mapped for the new rows,
        nothing is read back. A request is refused, whole, when the free pages no
        longer suffice for it (``BLOCK_NO_PAGES``), or when its numbers are not
        possible or its rows end past ``rows`` (``BLOCK_BAD_INDEX``): it keeps its pages
        and is granted no row; :meth:`status` tells."""
        got = self._call.block_update(self._sizes_at, current_stream_handle(self.device), self.device.index, self.table,
                                      self.mapped, self.free, self.free_count, lengths, new, rows)
        if type(got) is tuple:
            return BlockPlan._make(got)
        if got < 0:
            _check(got, "kvrt_block_tables_update_async")
        rows = int(rows)
        if rows < 0:
            raise ValueError("rows must not be negative")
        _int32(lengths, "lengths", self.n, self.device)
        _int32(new, "new", self.n, self.device)
        c = self._c()
        with _on(self.device):
            make = dict(dtype=torch.int32, device=self.device)
            plan = BlockPlan(torch.empty(self.n + 1, **make), torch.empty(rows, **make),
                             torch.empty(self.n, **make), torch.empty(self.n, **make))
            _check(self._lib.kvrt_block_tables_update_async(
                ctypes.byref(c), lengths.data_ptr(), new.data_ptr(), rows, plan.starts.data_ptr(),
                plan.slot_map.data_ptr() or None, plan.lengths.data_ptr(), plan.granted.data_ptr(),
                ctypes.c_void_p(current_stream_handle(self.device))), "kvrt_block_tables_update_async")
        return plan


class Block8Pool(_Status):
    """One layer's pages of coded K and V rows.

    ``k``, ``v``: codes [pages, kv_heads, block_size, head_dim], torch.int8 or
    torch.float8_e4m3fn; ``k_scale``, ``v_scale``: fp32 [pages, kv_heads]. A code
    stands for code * scale; scales are read as within [2^-64, 2^32]. They are
    ordinary tensors: each call uses (a captured one keeps) those the pool holds
    when it is made, and others of the same shapes and types may be assigned.
    """

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor) -> None:
        self._lib = L.load()
        require_cuda(k, "k")
        if k.dtype not in _CODES or k.dim() != 4:
            raise ValueError("codes must be int8 or float8_e4m3fn tensors [pages, kv_heads, block_size, head_dim]")
        self.device = k.device
        pages, heads, block, dim = k.shape
        if block not in (16, 32, 64, 128) or dim not in (64, 128, 256, 512) or not 1 <= heads <= 64 or pages < 1:
            raise ValueError("pages need 1 to 64 heads, 16, 32, 64 or 128 rows and head_dim 64, 128, 256 or 512; got "
                             f"{tuple(k.shape)}")
        if pages * heads * block > _I32_MAX:
            raise ValueError("a pool numbers its rows in 32 bits")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.kv_heads, self.block_size, self.head_dim = pages, heads, block, dim
        self._dtype = k.dtype
        with _on(self.device):
            self._status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._call = _calls()
        self._sizes = self._c()  # what calls read beside the four public tensors
        self._sizes_at = ctypes.addressof(self._sizes)

    def _c(self) -> L.KvrtBlock8:
        c = L.KvrtBlock8()
        codes, scales = (self.pages, self.kv_heads, self.block_size, self.head_dim), (self.pages, self.kv_heads)
        for name, want, dtype in (("k", codes, self._dtype), ("v", codes, self._dtype), ("k_scale", scales, torch.float32),
                                  ("v_scale", scales, torch.float32)):
            t = getattr(self, name)
            _same(t, name, self.device)
            if tuple(t.shape) != want or t.dtype != dtype or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous {dtype} tensor {want}")
            setattr(c, name, t.data_ptr())
        c.status = self._status.data_ptr()
        c.dtype, c.pages, c.kv_heads, c.block, c.head_dim = _CODES[self._dtype], *codes
        return c

    @classmethod
    def zeros(cls, pages: int, kv_heads: int, head_dim: int, *, block_size: int = 16, dtype: str = "int8",
              device: torch.device | str | None = None) -> "Block8Pool":
        """An empty pool; ``dtype`` is "int8" or "e4m3"."""
        if dtype not in _NAMES:
            raise ValueError(f"dtype must be one of {sorted(_NAMES)}, got {dtype!r}")
        dev = _device(device)
        shape = (int(pages), int(kv_heads), int(block_size), int(head_dim))
        codes = [torch.zeros(shape, dtype=torch.int8, device=dev).view(_NAMES[dtype]) for _ in range(2)]
        scales = [torch.zeros(shape[:2], dtype=torch.float32, device=dev) for _ in range(2)]
        return cls(*codes, *scales)

    def _table(self, table: torch.Tensor) -> L.KvrtTensor:
        _same(table, "table", self.device)
        if table.dtype != torch.int32 or table.dim() != 2:
            raise ValueError("table must be an int32 tensor [n, max_pages]")
        return tensor_desc(table)

    def append(self, k: torch.Tensor, v: torch.Tensor, slot_map: torch.Tensor) -> None:
        """Code rows k, v [T, kv_heads, head_dim] bf16 into slots ``slot_map`` [T]
        (int32 on the GPU, as :meth:`BlockTables.update` makes it; negative: the row
        is skipped). A page's scale grows with its new rows and the rows before
        them are coded anew; rows behind them (rolled back) are dropped. A page
        takes one run of consecutive slots per call; a slot map that names a slot
        twice or enters a page twice leaves that page undefined."""
        rc = self._call.block_append(self._sizes_at, current_stream_handle(self.device), self.device.index, self.k, self.v,
                                     self.k_scale, self.v_scale, k, v, slot_map)
        if rc <= 0:
            return _check(rc, "kvrt_block8_append_async")
        c = self._c()
        for t, name in ((k, "k"), (v, "v")):
            _same(t, name, self.device)
        _int32(slot_map, "slot_map", int(k.shape[0]), self.device)
        with _on(self.device):
            _check(self._lib.kvrt_block8_append_async(
                ctypes.byref(c), ctypes.byref(tensor_desc(k)), ctypes.byref(tensor_desc(v)), slot_map.data_ptr() or None,
                ctypes.c_void_p(current_stream_handle(self.device))), "kvrt_block8_append_async")

    def gather(self, table: torch.Tensor, lengths: torch.Tensor, lmax: int | None = None, *,
               start_pos: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16,
               mask_dtype: torch.dtype | None = torch.bool, out: tuple | None = None) -> tuple:
        """Zero-padded batch K, V [n, kv_heads, Lmax, head_dim] of ``dtype`` (bf16, as
        ``attend_tensors`` takes it, or fp32) and mask [n, Lmax] of the requests'
        positions ``start_pos[i]`` (int32 [n] on the GPU, default 0) on.
        ``out``: (K, V) or (K, V, mask) destinations instead of new tensors (strided
        views with a contiguous last dimension); they then set Lmax and dtype."""
        if out is None and dtype in _FLOATS and mask_dtype in _MASKS:
            got = self._call.block_gather_new(self._sizes_at, current_stream_handle(self.device), self.device.index, self.k, self.v,
                                              self.k_scale, self.v_scale, table, lengths, start_pos, lmax, _FLOATS[dtype],
                                              _MASKS[mask_dtype])
            if type(got) is tuple:
                return got
            if got < 0:
                _check(got, "kvrt_block8_gather_async")
        elif out is not None and lmax is None:
            rc = self._call.block_gather(self._sizes_at, current_stream_handle(self.device), self.device.index, self.k, self.v,
                                         self.k_scale, self.v_scale, table, lengths, start_pos, out[0], out[1],
                                         out[2] if len(out) > 2 else None)
            if rc <= 0:
                _check(rc, "kvrt_block8_gather_async")
                return out[0], out[1], out[2] if len(out) > 2 else None
        c, td = self._c(), self._table(table)
        n = int(table.shape[0])
        _int32(lengths, "lengths", n, self.device)
        if start_pos is not None:
            _int32(start_pos, "start_pos", n, self.device)
        with _on(self.device):
            mask = None
            if out is not None:
                out_k, out_v = out[0], out[1]
                mask = out[2] if len(out) > 2 else None
                if lmax is not None and int(lmax) != out_k.shape[2]:
                    raise ValueError(f"lmax {lmax} does not match out, which holds {out_k.shape[2]} rows")
                for t, name in ((out_k, "out K"), (out_v, "out V"), (mask, "out mask")):
                    if t is not None:
                        _same(t, name, self.device)
            else:
                if lmax is None or int(lmax) < 0:
                    raise ValueError("gather needs lmax (or out): lengths stay on the GPU")
                shape = (n, self.kv_heads, int(lmax), self.head_dim)
                out_k = torch.empty(shape, dtype=dtype, device=self.device)
                out_v = torch.empty(shape, dtype=dtype, device=self.device)
                if mask_dtype is not None:
                    mask = torch.empty(shape[:1] + shape[2:3], dtype=mask_dtype, device=self.device)
            md = None if mask is None else ctypes.byref(tensor_desc(mask))
            _check(self._lib.kvrt_block8_gather_async(
                ctypes.byref(c), ctypes.byref(td), lengths.data_ptr(), None if start_pos is None else start_pos.data_ptr(),
                ctypes.byref(tensor_desc(out_k)), ctypes.byref(tensor_desc(out_v)), md,
                ctypes.c_void_p(current_stream_handle(self.device))), "kvrt_block8_gather_async")
        return out_k, out_v, mask

    def attend(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor, scale: float,
               *, max_q: int, granted: torch.Tensor | None = None, window: int = 0,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of packed query rows q [T, Hq, head_dim] bf16 over the pages.

        Request i's rows are ``starts[i]`` up to ``starts[i + 1]`` (or ``granted[i]`` of
        them, as an update's plan gives them), at its last positions: row r of m
        sits at ``lengths[i] - m + r`` and sees keys up to itself, with ``window`` W
        only the last W of them. A row that sees no key becomes zeros; rows of no
        request are left as they are (undefined in a new ``out``). ``max_q``: the
        most rows of one request (more raise ``BLOCK_BAD_INDEX``, the first
        ``max_q`` are computed). ``out`` shares no memory with ``q``. The same inputs
        give the same bits, captured or not, whatever was called before."""
        got = self._call.block_attend(self._sizes_at, current_stream_handle(self.device), self.device.index, self.k, self.v,
                                      self.k_scale, self.v_scale, float(scale), window, max_q, q, table, lengths, starts,
                                      granted, out)
        if type(got) is not int:
            return got
        if got < 0:
            _check(got, "kvrt_block8_attend_async")
        c, td = self._c(), self._table(table)
        n = int(table.shape[0])
        _same(q, "q", self.device)
        _int32(lengths, "lengths", n, self.device)
        _int32(starts, "starts", n + 1, self.device)
        if granted is not None:
            _int32(granted, "granted", n, self.device)
        if q.dim() != 3:
            raise ValueError(f"q must be [T, Hq, {self.head_dim}], got {tuple(q.shape)}")
        # brought into 32 bits: a window past every key is none, negative numbers are refused
        max_q, window = max(-1, min(int(max_q), int(q.shape[0]))), max(-1, min(int(window), _I32_MAX))
        if out is not None:
            _same(out, "out", self.device)
        with _on(self.device):
            if out is None:
                out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
            size = self._lib.kvrt_block8_attend_work(ctypes.byref(c), n, int(table.shape[1]), int(q.shape[0]), int(q.shape[1]),
                                                     max_q)
            work = torch.empty(size, dtype=torch.uint8, device=self.device) if size else None
            _check(self._lib.kvrt_block8_attend_async(
                ctypes.byref(c), ctypes.byref(tensor_desc(q)), ctypes.byref(td), lengths.data_ptr(), starts.data_ptr(),
                None if granted is None else granted.data_ptr(), ctypes.byref(tensor_desc(out)), float(scale),
                window, max_q, None if work is None else work.data_ptr(), size,
                ctypes.c_void_p(current_stream_handle(self.device))), "kvrt_block8_attend_async")
        return out
