"""Paged key/value cache of a serving loop (xpu_kv_* in include/xpu_cuda.h).

Many sequences share one pool of pages. Tables, lengths and reference counts
live on the device and every operator changes them there, so a loop of
``append``, ``kernels.tree_attention``, ``trim``, ``fork`` and ``compact``
never waits for the host. A request that cannot be met changes nothing and
sets a bit that ``status`` reads.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib, kernels

EXHAUSTED, BAD_SEQUENCE, SHARED_CUT, BAD_INDEX, TIMEOUT = 1, 2, 4, 8, 16  # XPU_KV_*


class KvCache:
    """Keys and values [layers, pages, kv_heads, page_size, head_dim]; tables
    [sequences, width] of page ids (-1: none), lens [sequences], refs [pages]
    (users of each page), all int32."""

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, sequences: int,
                 max_positions: int, dtype=torch.bfloat16, device="cuda"):
        shape = (layers, pages, kv_heads, page_size, head_dim)
        width = max(1, -(-max_positions // page_size))
        self._bind(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device),
                   torch.full((sequences, width), -1, dtype=torch.int32, device=device),
                   torch.zeros(sequences, dtype=torch.int32, device=device),
                   torch.zeros(pages, dtype=torch.int32, device=device))

    @classmethod
    def wrap(cls, k: torch.Tensor, v: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor,
             refs: torch.Tensor) -> "KvCache":
        """A cache over tensors that the caller has (and keeps consistent)."""
        self = cls.__new__(cls)
        self._bind(k, v, tables, lens, refs)
        return self

    def _bind(self, k, v, tables, lens, refs):
        if k.dim() != 5 or k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("k and v are [layers, pages, kv_heads, page_size, head_dim] of one dtype")
        if tables.dim() != 2 or any(t.dtype != torch.int32 for t in (tables, lens, refs)):
            raise ValueError("tables is [sequences, width]; tables, lens and refs are int32")
        if lens.shape != tables.shape[:1] or refs.shape != k.shape[1:2]:
            raise ValueError("lens has an entry per sequence, refs one per page")
        self.k, self.v, self.tables, self.lens, self.refs = k, v, tables, lens, refs
        self.layers, self.pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.dtype = k.dtype
        self._status = torch.zeros(1, dtype=torch.int32, device=k.device)
        size = int(_lib.load().xpu_kv_workspace_size(self.pages))
        self._workspace = torch.zeros(size // 4, dtype=torch.int32, device=k.device)
        self._c = _lib.KvCacheC(*(kernels._ptr(t) for t in (k, v, tables, lens, refs, self._status, self._workspace)),
                                kernels._dtype_code(k), self.layers, self.pages, self.page_size, self.kv_heads,
                                self.head_dim, *tables.shape)
        self.handle = ctypes.addressof(self._c)

    def status(self) -> int:
        """Bits that refused requests have set (EXHAUSTED, BAD_SEQUENCE,
        SHARED_CUT, BAD_INDEX, TIMEOUT), cleared by reading; waits for the device.
        After a TIMEOUT the workspace is made ready again."""
        torch.cuda.synchronize(self._status.device)  # the operators may have run on any stream
        bits = int(self._status.item())
        if bits:
            self._status.zero_()
            if bits & TIMEOUT:
                self._workspace.zero_()
            torch.cuda.synchronize(self._status.device)  # before a call on any stream can set a bit again
        return bits

    @staticmethod
    def _ids(t: torch.Tensor) -> int:
        if t.dtype != torch.int32 or not t.is_cuda or not t.is_contiguous():
            raise ValueError("ids, offsets and lengths are contiguous int32 CUDA tensors")
        return t.data_ptr()

    def _list(self, sequences, other, more=0):
        count = sequences.numel()
        if other.numel() != count + more:
            raise ValueError("one entry per sequence" + (" and one more" if more else ""))
        return self._ids(sequences), self._ids(other), count

    def _rows(self, k, v, rows, lead):
        shape = k.shape
        if k.dtype != self.dtype or v.dtype != self.dtype or shape != v.shape:
            raise ValueError("k and v must have the cache's dtype and one shape")
        if len(shape) != 4 or shape[0] != lead or shape[2] != self.kv_heads or shape[3] != self.head_dim:
            raise ValueError(f"k and v must be [{lead}, rows, {self.kv_heads}, {self.head_dim}]")
        held, row = shape[1], self.kv_heads * self.head_dim
        layer = held * row
        if not k.is_contiguous() or not v.is_contiguous():
            row = kernels._packed("k and v", k[0], self.kv_heads, self.head_dim)  # too short a stride is refused below
            layer = k.stride(0) if lead > 1 else 0
            if kernels._packed("k and v", v[0], self.kv_heads, self.head_dim) != row or lead > 1 and v.stride(0) != layer:
                raise ValueError("k and v must have one layout")
        if not k.is_cuda or not v.is_cuda:
            raise ValueError("libxpu_cuda entry points take CUDA tensors")
        tokens, at = (held, None) if rows is None else (rows.numel(), self._ids(rows))
        return tokens, at, k.data_ptr(), v.data_ptr(), held, layer, row

    def extend(self, sequences: torch.Tensor, starts: torch.Tensor, stream=None) -> None:
        """Lengthens sequences[i] by starts[i+1] - starts[i] positions,
        taking the lowest free pages (xpu_kv_extend)."""
        _lib.call("xpu_kv_extend", self.handle, *self._list(sequences, starts, 1), kernels._stream(stream))

    def write(self, layer: int, sequences: torch.Tensor, starts: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
              rows: torch.Tensor | None = None, stream=None) -> None:
        """Writes the positions that the last ``extend`` of the same list
        added, in one layer: k and v [rows, kv_heads, head_dim], token t from
        row rows[t], or t (xpu_kv_write)."""
        tokens, at, pk, pv, held, layer_stride, row = self._rows(k[None], v[None], rows, 1)
        _lib.call("xpu_kv_write", self.handle, *self._list(sequences, starts, 1), tokens, at, pk, pv, held, 0, row, layer, 1,
                  kernels._stream(stream))

    def append(self, sequences: torch.Tensor, starts: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
               rows: torch.Tensor | None = None, stream=None) -> None:
        """``extend`` and ``write`` of every layer: k and v [layers, rows,
        kv_heads, head_dim] (xpu_kv_append)."""
        tokens, at, pk, pv, held, layer_stride, row = self._rows(k, v, rows, self.layers)
        _lib.call("xpu_kv_append", self.handle, *self._list(sequences, starts, 1), tokens, at, pk, pv, held, layer_stride, row,
                  kernels._stream(stream))

    def trim(self, sequences: torch.Tensor, lens: torch.Tensor, stream=None) -> None:
        """Shortens sequences[i] to lens[i] positions and lets go of the pages
        behind them; 0 frees the sequence (xpu_kv_trim)."""
        _lib.call("xpu_kv_trim", self.handle, *self._list(sequences, lens), kernels._stream(stream))

    def fork(self, parents: torch.Tensor, children: torch.Tensor, stream=None) -> None:
        """Makes the empty sequence children[i] a copy of parents[i]: full
        pages are shared, the rest is copied (xpu_kv_fork)."""
        _lib.call("xpu_kv_fork", self.handle, *self._list(parents, children), kernels._stream(stream))

    def compact(self, stream=None) -> None:
        """Moves the pages in use to the front of the pool (xpu_kv_compact)."""
        _lib.call("xpu_kv_compact", self.handle, kernels._stream(stream))
