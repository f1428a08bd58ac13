"""A paged cache of keys and values in 8 bits for a batch of requests, and attention over it (nnq_kv_* of the C ABI).

``KvCache`` holds one layer's blocks, ``KvBatch`` the block tables and the slot map that the layers of a step share:

    batch = KvBatch(requests, max_blocks, rows, block=32)
    batch.build(past, count, free)                    # tables, slots and positions of the step's packed rows
    cache.append(k, v, batch.slot)                    # [rows, kv_heads, dim] -> codes
    y = cache.attend(q, batch, max_rows=1)            # [rows, heads, dim]

The reference keeps one sequence's keys and values in f32 (``KvCacheLayer``,
crates/nn-core/src/layers/generation/kv_cache.rs:132) and attends with ``sdpa``
(crates/nn-core/src/layers/attention/sdpa.rs:42-118). Tensors are torch CUDA tensors of the backend's device; calls run on the
current stream of that device, allocate through torch alone and may be captured in a CUDA graph.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

from . import api

INT8, E4M3 = 0, 1   # nnq_kv_format


class _Cache(ctypes.Structure):
    _fields_ = [("format", ctypes.c_int32), ("kv_heads", ctypes.c_int32), ("dim", ctypes.c_int32), ("block", ctypes.c_int32), ("blocks", ctypes.c_int64),
                ("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_exp", ctypes.c_void_p), ("v_exp", ctypes.c_void_p)]


class _Batch(ctypes.Structure):
    _fields_ = [("length", ctypes.c_void_p), ("row_start", ctypes.c_void_p), ("table", ctypes.c_void_p), ("requests", ctypes.c_int64),
                ("table_ld", ctypes.c_int64), ("rows", ctypes.c_int64), ("max_rows", ctypes.c_int64)]


def _int32(t, name: str, shape, index: int):
    torch = api._torch()
    if t.dtype != torch.int32 or not t.is_cuda or t.get_device() != index or not t.is_contiguous():
        raise api.InvalidArgument(f"{name}: expected a contiguous int32 tensor on cuda:{index}, got {t.dtype} on {t.device}")
    if t.shape != shape:
        raise api.ShapeMismatch(f"{name}: expected {tuple(shape)}, got {tuple(t.shape)}")
    return t


class _InPlace:
    """Tensors whose memory the calls rely on are filled in place (``copy_``), not replaced."""
    _fixed = frozenset()

    def __setattr__(self, name, value):
        if name in self._fixed:
            raise AttributeError(f"{type(self).__name__}.{name} is filled in place, not replaced")
        object.__setattr__(self, name, value)

    def _place(self, **tensors):
        for name, value in tensors.items():
            object.__setattr__(self, name, value)


class KvBatch(_InPlace):
    """Block tables [requests, max_blocks], lengths, packed rows (row_start), and slot and position of every row, on the device. The tensors
    are filled in place, not replaced."""

    _fixed = frozenset(("table", "length", "row_start", "slot", "position", "used", "rows"))

    def __init__(self, requests: int, max_blocks: int, rows: int, block: int = 16, backend: Optional[api.Backend] = None):
        if requests < 1 or max_blocks < 1 or rows < 0:
            raise api.InvalidArgument(f"a batch of {requests} requests, {max_blocks} blocks each, {rows} rows")
        torch = api._torch()
        b = backend or api.gpu_backend()
        self.backend, self.block = b, int(block)
        self.device = torch.device("cuda", b.device)
        z = lambda *s: torch.zeros(s, dtype=torch.int32, device=self.device)  # noqa: E731
        self._place(table=torch.full((requests, max_blocks), -1, dtype=torch.int32, device=self.device), length=z(requests), row_start=z(requests + 1),
                    slot=z(rows), position=z(rows), used=z(1), rows=int(rows))

    @classmethod
    def from_tensors(cls, table, length, row_start, block: int, slot=None, position=None, backend: Optional[api.Backend] = None) -> "KvBatch":
        """A batch over tables that exist already (int32, on the device); without a slot map it can be attended to, not built."""
        torch = api._torch()
        self = cls.__new__(cls)
        b = self.backend = backend or api.gpu_backend()
        self.device, self.block = torch.device("cuda", b.device), int(block)
        if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1:
            raise api.ShapeMismatch(f"table: expected [requests, blocks], got {tuple(table.shape)}")
        n = table.shape[0]
        rows = 0 if slot is None else slot.numel()
        self._place(table=_int32(table, "table", table.shape, b.device), length=_int32(length, "length", (n,), b.device),
                    row_start=_int32(row_start, "row_start", (n + 1,), b.device), slot=None if slot is None else _int32(slot, "slot", (rows,), b.device),
                    position=None if position is None else _int32(position, "position", (position.numel() if slot is None else rows,), b.device),
                    used=torch.zeros(1, dtype=torch.int32, device=self.device), rows=rows)
        return self

    @property
    def requests(self) -> int:
        return self.table.shape[0]

    def build(self, past, count, free, skip=None):
        """Tables and slots for `count` new tokens behind `past` ones, int32 [requests] each. `free`: numbers of free blocks (int32), of which
        the first `skip` (int32 [1], None: none) are taken; `self.used` is skip plus the blocks taken here. `past` may be
        ``self.length`` and `skip` ``self.used``: a captured step then advances the batch. Rows behind the last request get slot -1,
        and so do tokens for whose block the list or the table had no room (``used`` then exceeds the list)."""
        if self.slot is None or self.position is None:
            raise api.InvalidArgument("a batch without slot and position tensors cannot be built")
        n, b = self.table.shape[0], self.backend
        past, count = _int32(past, "past", (n,), b.device), _int32(count, "count", (n,), b.device)
        free = _int32(free, "free", (free.numel(),), b.device)
        if skip is not None:
            _int32(skip, "skip", (1,), b.device)
        st = b._lib.nnq_kv_tables(b._ctx, past.data_ptr(), count.data_ptr(), n, free.data_ptr(), free.numel(), None if skip is None else skip.data_ptr(), self.block,
                                  self.table.data_ptr(), self.table.shape[1], self.length.data_ptr(), self.row_start.data_ptr(), self.slot.data_ptr(),
                                  self.position.data_ptr(), self.rows, self.used.data_ptr(), api._stream_ptr(None, b.device))
        if st:
            b.check(st)
        return self


class KvCache(_InPlace):
    """One layer's keys and values: codes uint8 [blocks, kv_heads, block, dim] (``k``, ``v``) and exponent bytes uint8 [blocks, kv_heads]
    (``k_exp``, ``v_exp``); value = code * 2^(byte - 127). A saved cache is brought back with ``copy_`` into these tensors."""

    _fixed = frozenset(("k", "v", "k_exp", "v_exp"))

    def __init__(self, blocks: int, kv_heads: int, dim: int, block: int = 16, fmt: int = INT8, backend: Optional[api.Backend] = None):
        torch = api._torch()
        if fmt not in (INT8, E4M3):
            raise api.InvalidArgument(f"unknown cache format {fmt}")
        if dim not in (64, 128, 192, 256):
            raise api.Unsupported(f"heads of a cache must be 64, 128, 192 or 256 wide (got {dim})")
        if block not in (16, 32, 64, 128, 256):
            raise api.Unsupported(f"blocks of a cache must hold 16, 32, 64, 128 or 256 tokens (got {block})")
        if blocks < 1 or kv_heads < 1 or blocks * block >= 1 << 31:
            raise api.InvalidArgument(f"a cache of {blocks} blocks of {block} tokens, {kv_heads} heads")
        b = self.backend = backend or api.gpu_backend()
        self.blocks, self.kv_heads, self.dim, self.block, self.fmt = int(blocks), int(kv_heads), int(dim), int(block), int(fmt)
        self.device = torch.device("cuda", b.device)
        z = lambda *s: torch.zeros(s, dtype=torch.uint8, device=self.device)  # noqa: E731
        self._place(k=z(blocks, kv_heads, block, dim), v=z(blocks, kv_heads, block, dim), k_exp=z(blocks, kv_heads).fill_(127),
                    v_exp=z(blocks, kv_heads).fill_(127))
        self._need = {}   # workspace by numbers of query heads and rows
        self._c = _Cache(self.fmt, self.kv_heads, self.dim, self.block, self.blocks, self.k.data_ptr(), self.v.data_ptr(), self.k_exp.data_ptr(), self.v_exp.data_ptr())
        self._ref = ctypes.byref(self._c)

    def memory_bytes(self) -> int:
        return 2 * self.blocks * self.kv_heads * (self.block * self.dim + 1)

    def _rows(self, x, name: str, heads: int):
        """A [rows, heads, dim] tensor as the kernels read it: rows may lie apart (a slice of a wider product), heads not."""
        torch = api._torch()
        shape = x.shape
        if len(shape) != 3 or shape[1] != heads or shape[2] != self.dim:
            raise api.ShapeMismatch(f"{name}: expected [rows, {heads}, {self.dim}], got {tuple(shape)}")
        if not x.is_cuda or x.get_device() != self.backend.device:
            raise api.InvalidArgument(f"{name}: expected a tensor on {self.device}, got {x.device}")
        if x.is_contiguous() and (x.dtype == torch.float32 or x.dtype == torch.bfloat16) and x.data_ptr() % 16 == 0:
            return x
        if x.dtype not in (torch.float32, torch.bfloat16):
            x = x.float()
        size = x.element_size()
        # (a single row may have any stride; row strides must not fold rows onto each other)
        if x.stride(2) != 1 or x.stride(1) != self.dim or (x.shape[0] > 1 and x.stride(0) < heads * self.dim) or x.stride(0) * size % 16 or x.data_ptr() % 16:
            x = x.contiguous()
            if x.data_ptr() % 16:
                x = x.clone()
        return x

    def append(self, k, v, slots):
        """Quantizes rows of keys and values [rows, kv_heads, dim] into their slots (int32 [rows], -1: skipped). A block's tokens are
        consecutive rows. Non-finite values are stored as 0 or the largest code and reported by ``Backend.device_status``."""
        b = self.backend
        k, v = self._rows(k, "k", self.kv_heads), self._rows(v, "v", self.kv_heads)
        if k.dtype != v.dtype:
            k, v = k.float(), v.float()
        n = k.shape[0]
        _int32(slots, "slots", (n,), b.device)
        if v.shape[0] != n:
            raise api.ShapeMismatch(f"{n} keys and {v.shape[0]} values")
        ld = self.kv_heads * self.dim
        st = b._lib.nnq_kv_append(b._ctx, self._ref, k.data_ptr(), k.stride(0) if n > 1 else ld, v.data_ptr(), v.stride(0) if n > 1 else ld,
                                  api._dtype_code(k), slots.data_ptr(), n, api._stream_ptr(None, b.device))
        if st:
            b.check(st)

    def read(self, slots, dtype=None):
        """(keys, values) of given slots, [rows, kv_heads, dim], f32 (default) or bf16: exact in both; zeros for slot -1."""
        torch = api._torch()
        dtype = dtype or torch.float32
        if dtype not in (torch.float32, torch.bfloat16):
            raise api.Unsupported(f"a cache is read as float32 or bfloat16, not {dtype}")
        b = self.backend
        _int32(slots, "slots", (slots.numel(),), b.device)
        n = slots.numel()
        k = torch.empty((n, self.kv_heads, self.dim), dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        st = b._lib.nnq_kv_read(b._ctx, self._ref, slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), api._dtype_code(k), api._stream_ptr(None, b.device))
        if st:
            b.check(st)
        return k, v

    def attend(self, q, batch: KvBatch, scale: Optional[float] = None, window: int = 0, max_rows: int = 1, out=None):
        """Softmax attention of the batch's packed rows q [rows, heads, dim] to the positions up to their own (the last `window` of them, 0:
        all), in out's dtype, without one in q's where that is float32 or bfloat16 (others are taken as float32). `scale` defaults to dim^-1/2.
        `max_rows`: rows of the request with the most, for the choice of kernels: with the default a prompt is right but many times slower.
        `out` must not overlap q. Rows behind the last request are left as `out` has them."""
        torch = api._torch()
        b = self.backend
        heads = q.shape[1] if q.dim() == 3 else 0
        q = self._rows(q, "q", heads)
        n, ld = q.shape[0], heads * self.dim
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
        elif out.shape != q.shape or out.device != self.device or out.dtype not in (torch.float32, torch.bfloat16) or out.stride(2) != 1 or out.stride(1) != self.dim:
            raise api.ShapeMismatch(f"out: expected {tuple(q.shape)}, heads next to each other, on {self.device}")
        if not 0 <= window < 1 << 31:   # (the C call would take what is left of it in 32 bits)
            raise api.InvalidArgument(f"a window of {window}")
        if batch.block != self.block or batch.backend.device != b.device:
            raise api.InvalidArgument(f"a batch of blocks of {batch.block} on {batch.device} for a cache of blocks of {self.block} on {self.device}")
        table = batch.table
        c = _Batch(batch.length.data_ptr(), batch.row_start.data_ptr(), table.data_ptr(), *table.shape, n, max(int(max_rows), 1))
        need = self._need.get((heads, c.max_rows))
        if need is None:
            size = ctypes.c_size_t()
            b.check(b._lib.nnq_kv_attention_workspace(b._ctx, self._ref, ctypes.byref(c), heads, ctypes.byref(size)))
            need = self._need[heads, c.max_rows] = size.value
        work = torch.empty(need, dtype=torch.uint8, device=self.device)
        st = b._lib.nnq_kv_attention(b._ctx, self._ref, ctypes.byref(c), q.data_ptr(), api._dtype_code(q), q.stride(0) if n > 1 else ld, heads,
                                     1.0 / math.sqrt(self.dim) if scale is None else float(scale), int(window), out.data_ptr(), api._dtype_code(out),
                                     out.stride(0) if n > 1 else ld, work.data_ptr(), need, api._stream_ptr(None, b.device))
        if st:
            b.check(st)
        return out
