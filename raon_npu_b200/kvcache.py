"""The paged 4-bit KV cache and the attention that reads it.

``KvCache`` is a pool of pages of keys and values in q4nx groups (32 values:
4-bit codes, bf16 scale and min) for every layer of a model, ``KvBatch`` the
sequences of one call.  A layer of a decode or prefill step is::

    cache.append(layer, qkv, batch, q, q_heads=32, q_norm=wq, k_norm=wk, rope=table)
    cache.attend(layer, q, batch, out)

Page management (``new``, ``extend``, ``fork``, ``trim``, ``free``,
``compact``, ``batch``) is optional: a program that keeps its own page tables
passes them to ``KvBatch``.

Buffers are torch tensors on the context's device; 16-bit rows may be
``torch.bfloat16`` or bf16 bits in an integer type.  Launches go to ``stream``
(a raw handle; default: the current torch stream) and return at once.  Tensors
passed with a ``stream`` that is not the current one must stay alive until it
has used them (``Tensor.record_stream``).

``attend`` uses scratch of the context: calls of one context that may run at
the same time, on two streams or in two graphs, give wrong results.  Order
them, or give each stream a ``Context`` and a ``KvCache`` on one ``pool``.
"""

from __future__ import annotations

import ctypes
import operator

import numpy as np
import torch

from . import _lib
from ._lib import check
from .device import CUDA_STREAM_LEGACY, Context, _ptr

# A decode step makes one or two of these calls a layer, so the checks below
# are written for the host's time: get_device() (-1 on the CPU) instead of
# device objects, is_contiguous() before strides.
_raw_stream = torch._C._cuda_getCurrentRawStream
_BF16 = frozenset((torch.bfloat16, torch.int16, torch.uint16))   # bf16 values, or their bits
_F32 = frozenset((torch.float32,))
_float32 = torch.float32


def rope_table(positions: int, rope_dim: int, base: float = 10000.0) -> np.ndarray:
    """f32 [positions, rope_dim]: cos | sin of position * base^(-2i/rope_dim), computed in 64 bits."""
    if rope_dim < 2 or rope_dim % 2:
        raise ValueError(f"rope_dim must be even, got {rope_dim}")
    ang = np.arange(positions, dtype=np.float64)[:, None] * base ** (-np.arange(0, rope_dim, 2) / rope_dim)
    return np.concatenate([np.cos(ang), np.sin(ang)], axis=1).astype(np.float32)


def _ints(t, ndim: int, what: str):
    if t.dtype is not torch.int32 or t.dim() != ndim or not t.is_cuda or (t.shape[-1] > 1 and t.stride(-1) != 1):
        raise ValueError(f"{what} must be an int32 CUDA tensor of {ndim} dimension(s), contiguous in the last")
    return t


def _rows(t, width: int, what: str, dev: int, types=_BF16):
    """(rows, row stride in elements) of [rows, width] or [rows, heads, head_dim] values."""
    shape = t.shape
    if len(shape) == 2 and shape[1] == width and t.is_contiguous() and t.dtype in types and t.get_device() == dev:
        return shape[0], width
    if t.dtype not in types or t.get_device() != dev:
        raise ValueError(f"{what} must be a {'bf16' if types is _BF16 else 'f32'} tensor on cuda:{dev}, got {t.dtype} on {t.device}")
    if len(shape) == 2:
        inner = shape[1] == width and (t.is_contiguous() or width == 1 or t.stride(1) == 1)
    elif len(shape) == 3:
        inner = shape[1] * shape[2] == width and (t.is_contiguous() or (
            (shape[2] == 1 or t.stride(2) == 1) and (shape[1] == 1 or t.stride(1) == shape[2])))
    else:
        inner = False
    if not inner:
        raise ValueError(f"{what} must hold rows of {width} contiguous values, got {tuple(shape)} "
                         f"with strides {tuple(t.stride())}")
    rows = shape[0]
    ld = t.stride(0) if rows > 1 else width
    if ld < width:
        raise ValueError(f"{what}: rows overlap (stride {ld} of {width} values)")
    return rows, ld


def _whole(numbers, what: str) -> np.ndarray:
    """int32 array of whole numbers of any integer type."""
    try:
        return np.asarray([operator.index(n) for n in numbers], dtype=np.int32)
    except (TypeError, OverflowError) as e:
        raise ValueError(f"{what} must be whole 32-bit numbers: {e}") from None


class KvBatch:
    """The sequences of a call, as device arrays the caller may update in place
    between calls (a captured step reads them anew).

    ``table`` int32 [sequences, columns]: page ids; ``kv_len`` int32
    [sequences]: tokens of each sequence, this call's included; ``q_off`` int32
    [sequences + 1]: first row of each sequence (None: one row each); ``max_q``:
    an upper bound of the rows of a sequence.
    """

    def __init__(self, table, kv_len, q_off=None, max_q: int = 1):
        self.table = _ints(table, 2, "table")
        self.kv_len = _ints(kv_len, 1, "kv_len")
        self.n_seqs, self.columns = int(table.shape[0]), int(table.shape[1])
        if int(kv_len.shape[0]) != self.n_seqs:
            raise ValueError(f"kv_len has {kv_len.shape[0]} entries for {self.n_seqs} sequences")
        self.ld = int(table.stride(0)) if self.n_seqs > 1 else self.columns
        if self.ld < self.columns:
            raise ValueError(f"table: rows overlap (stride {self.ld} of {self.columns} columns)")
        self.q_off = q_off
        if q_off is not None:
            _ints(q_off, 1, "q_off")
            if int(q_off.shape[0]) != self.n_seqs + 1:
                raise ValueError(f"q_off has {q_off.shape[0]} entries for {self.n_seqs} sequences")
        dev = table.get_device()
        if kv_len.get_device() != dev or (q_off is not None and q_off.get_device() != dev):
            raise ValueError(f"table, kv_len and q_off must be on one device, cuda:{dev} as the table")
        if max_q < 1 or (q_off is None and max_q != 1):
            raise ValueError(f"max_q {max_q}: at least 1, and 1 without q_off")
        self.max_q = int(max_q)


class KvCache:
    """Pages of 4-bit keys and values on one device.

    ``pool``: a uint8 CUDA tensor of at least ``KvCache.pool_bytes(...)`` bytes
    to live in (the layout is given in include/raon_cuda.h); None: memory of
    the library's own.
    """

    def __init__(self, ctx: Context, layers: int, kv_heads: int, head_dim: int, pages: int, page_size: int = 64,
                 pool=None):
        self.ctx, self.lib, self.device = ctx, ctx.lib, ctx.device
        self.layers, self.kv_heads, self.head_dim = int(layers), int(kv_heads), int(head_dim)
        self.pages, self.page_size = int(pages), int(page_size)
        self.scale = self.head_dim ** -0.5
        nbytes = 0
        if pool is not None:
            if not pool.is_cuda or not pool.is_contiguous() or pool.device.index != ctx.device:
                raise ValueError(f"pool must be a contiguous tensor on cuda:{ctx.device}")
            nbytes = pool.numel() * pool.element_size()
        self.pool = pool
        h = ctypes.c_void_p()
        check(self.lib.rc_kv_create(ctx.handle, layers, pages, kv_heads, head_dim, page_size, _ptr(pool) or None, nbytes,
                                    ctypes.byref(h)), "rc_kv_create")
        self.handle = h
        self._pages = None
        ctx._adopt(self)

    @staticmethod
    def pool_bytes(layers: int, kv_heads: int, head_dim: int, pages: int, page_size: int = 64) -> int:
        n = ctypes.c_size_t()
        check(_lib.load().rc_kv_pool_bytes(layers, pages, kv_heads, head_dim, page_size, ctypes.byref(n)),
              "rc_kv_pool_bytes")
        return n.value

    def close(self) -> None:
        if self.handle and self.ctx.handle:
            self.lib.rc_kv_destroy(self.handle)
        self.handle = None
        self.pool = None

    release = close

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _norm(self, w, name: str) -> int:
        if w.dtype in _BF16 and w.get_device() == self.device and w.numel() == self.head_dim and w.is_contiguous():
            return w.data_ptr()
        raise ValueError(f"{name} must hold {self.head_dim} bf16 values on the device")

    def _batch_args(self, batch: KvBatch, rows: int, what: str):
        q_off = batch.q_off
        if batch.table.get_device() != self.device:
            raise ValueError(f"{what}: the batch is on {batch.table.device}, the cache on cuda:{self.device}")
        if q_off is None and rows != batch.n_seqs:
            raise ValueError(f"{what}: {rows} rows for {batch.n_seqs} sequences without q_off")
        return batch.table.data_ptr(), batch.kv_len.data_ptr(), None if q_off is None else q_off.data_ptr()

    def _stream(self, stream) -> int:
        """The stream to launch on; torch's default stream is the legacy one (0 is the context's own in the C ABI)."""
        return int(stream) if stream is not None else _raw_stream(self.device) or CUDA_STREAM_LEGACY

    def _torch_stream(self, handle: int):
        """The torch stream of a handle as the C ABI takes it (0: the context's own)."""
        dev = torch.device("cuda", self.device)
        if handle == CUDA_STREAM_LEGACY:
            return torch.cuda.default_stream(dev)
        return torch.cuda.ExternalStream(handle or self.ctx.stream, dev)

    # ---------------------------------------------------------- operators --
    def append(self, layer: int, x, batch: KvBatch, q_out=None, q_heads: int = 0, q_norm=None, k_norm=None,
               eps: float = 1e-6, rope=None, interleaved: bool = False, stream: int | None = None) -> None:
        """Store the keys and values of ``x``'s rows and write its queries, normalised and rotated, to ``q_out``.

        x [rows, (q_heads + 2 kv_heads) * head_dim] bf16 or f32: the q, k and v
        heads of each row.  q_norm, k_norm bf16 [head_dim]: RMS norm weights of
        the query and key heads (None: no norm).  rope f32 [positions,
        rope_dim]: cos | sin of every position (None: no rotation)."""
        width = (q_heads + 2 * self.kv_heads) * self.head_dim
        dev = self.device
        f32 = x.dtype is _float32
        rows, ldx = _rows(x, width, "x", dev, _F32 if f32 else _BF16)
        ldq = 0
        if q_heads:
            if q_out is None:
                raise ValueError("append: q_out is missing")
            n, ldq = _rows(q_out, q_heads * self.head_dim, "q_out", dev)
            if n != rows:
                raise ValueError(f"append: x has {rows} rows, q_out {n}")
        q_w = None if q_norm is None else self._norm(q_norm, "q_norm")
        k_w = None if k_norm is None else self._norm(k_norm, "k_norm")
        rope_rows = rope_dim = 0
        if rope is not None:
            if rope.dtype is not _float32 or rope.dim() != 2 or rope.get_device() != dev or not rope.is_contiguous():
                raise ValueError(f"rope must be a contiguous f32 tensor [positions, rope_dim] on cuda:{dev}")
            rope_rows, rope_dim = rope.shape
        table, kv_len, q_off = self._batch_args(batch, rows, "append")
        rc = self.lib.rc_kv_append(
            self.handle, layer, x.data_ptr(), _lib.RC_DTYPE_F32 if f32 else _lib.RC_DTYPE_BF16, ldx, q_heads, rows,
            table, batch.columns, batch.ld, kv_len, q_off, batch.n_seqs, q_w, k_w, eps, None if rope is None else rope.data_ptr(), rope_rows,
            rope_dim, 1 if interleaved else 0, q_out.data_ptr() if q_heads else None, ldq, self._stream(stream))
        if rc:
            check(rc, "rc_kv_append")

    def attend(self, layer: int, q, batch: KvBatch, out, scale: float | None = None, window: int = 0, sinks: int = 0,
               stream: int | None = None) -> None:
        """Attention of ``q`` [rows, heads * head_dim] bf16 over the batch's cached tokens into ``out``.

        scale: of the scores (default 1 / sqrt(head_dim)).  window > 0: a row
        sees itself, the window - 1 tokens before it and the first ``sinks``
        tokens of its sequence; 0: every token up to itself.  One call of a
        context at a time, whatever the streams."""
        dev = self.device
        shape = q.shape
        width = shape[1] if len(shape) == 2 else shape[1] * shape[2] if len(shape) == 3 else 0
        heads = width // self.head_dim
        rows, ldq = _rows(q, heads * self.head_dim, "q", dev)
        n, ldo = _rows(out, width, "out", dev)
        if n != rows:
            raise ValueError(f"attend: q has {rows} rows, out {n}")
        table, kv_len, q_off = self._batch_args(batch, rows, "attend")
        rc = self.lib.rc_kv_attend(
            self.handle, layer, q.data_ptr(), ldq, heads, rows, table, batch.columns, batch.ld, kv_len, q_off,
            batch.n_seqs, batch.max_q, self.scale if scale is None else scale, window, sinks, out.data_ptr(), ldo,
            self._stream(stream))
        if rc:
            check(rc, "rc_kv_attend")

    def read(self, layer: int, batch: KvBatch, k_out, v_out, stream: int | None = None) -> None:
        """The cached keys and values of the batch's rows in bf16: k_out, v_out [rows, kv_heads, head_dim], contiguous."""
        width = self.kv_heads * self.head_dim
        rows, ldk = _rows(k_out, width, "k_out", self.device)
        n, ldv = _rows(v_out, width, "v_out", self.device)
        if n != rows or ldk != width or ldv != width:
            raise ValueError("read: k_out and v_out must be contiguous and of one shape")
        table, kv_len, q_off = self._batch_args(batch, rows, "read")
        rc = self.lib.rc_kv_read(self.handle, layer, rows, table, batch.columns, batch.ld, kv_len, q_off, batch.n_seqs,
                                 k_out.data_ptr(), v_out.data_ptr(), self._stream(stream))
        if rc:
            check(rc, "rc_kv_read")

    def move_pages(self, src, dst, table=None, stream: int | None = None) -> None:
        """Copy pages src[i] -> dst[i] in every layer and rewrite ``table``'s entries accordingly, in one launch.

        src, dst int32 [n] on the device; a page is not both a source and a
        destination, nor twice a destination (nor, with a table, twice a source)."""
        _ints(src, 1, "src")
        _ints(dst, 1, "dst")
        if src.shape != dst.shape:
            raise ValueError(f"move_pages: {src.shape[0]} sources, {dst.shape[0]} destinations")
        rows = cols = ld = 0
        if table is not None:
            _ints(table, 2, "table")
            if table.get_device() != self.ctx.device:
                raise ValueError(f"move_pages: the table must be on cuda:{self.ctx.device}")
            rows, cols = table.shape
            ld = table.stride(0) if rows > 1 else cols
        if src.get_device() != self.ctx.device or dst.get_device() != self.ctx.device:
            raise ValueError(f"move_pages: the moves must be on cuda:{self.ctx.device}")
        rc = self.lib.rc_kv_move_pages(self.handle, src.data_ptr(), dst.data_ptr(), src.shape[0],
                                       None if table is None else table.data_ptr(), rows, cols, ld, self._stream(stream))
        if rc:
            check(rc, "rc_kv_move_pages")

    # ------------------------------------------------------------- pages --
    @property
    def page_pool(self) -> "PagePool":
        """The pages as sequences own them (made on first use)."""
        if self._pages is None:
            self._pages = PagePool(self.pages, self.page_size)
        return self._pages

    def new(self) -> int:
        """A sequence without tokens; ``extend`` gives it room."""
        return self.page_pool.new()

    def extend(self, seqs, n, stream: int | None = None) -> None:
        """Room for ``n`` more tokens (a number, or one for each) in every sequence of ``seqs``.

        Tails shared with a fork are copied first.  Raises ``CacheFull`` and
        changes nothing when the pool cannot hold them all."""
        self._move(self.page_pool.extend(seqs, n), stream)

    def fork(self, seq: int) -> int:
        """A second sequence with the same tokens; nothing is copied until one of the two grows."""
        return self.page_pool.fork(seq)

    def trim(self, seq: int, n: int) -> None:
        """Keep the first ``n`` tokens."""
        self.page_pool.trim(seq, n)

    def free(self, seq: int) -> None:
        self.page_pool.free(seq)

    def compact(self, stream: int | None = None) -> int:
        """Move the pages in use to the lowest ids; returns how many moved.  Tables made before are stale."""
        moves = self.page_pool.compact()
        self._move(moves, stream)
        return len(moves)

    def batch(self, seqs, rows=None, columns: int | None = None) -> KvBatch:
        """Device tables of ``seqs``; rows: how many of each sequence's last tokens are this call's (None: one)."""
        seqs = list(seqs)
        table, kv_len = self.page_pool.table(seqs, columns)
        dev = torch.device("cuda", self.ctx.device)
        q_off, max_q = None, 1
        if rows is not None:
            rows = _whole(rows, "batch: rows")
            if rows.shape != kv_len.shape or (rows < 0).any() or (rows > kv_len).any():
                raise ValueError("batch: rows must be between 0 and each sequence's tokens")
            q_off = torch.from_numpy(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)).to(dev)
            max_q = max(1, int(rows.max(initial=0)))
        return KvBatch(torch.from_numpy(table).to(dev), torch.from_numpy(kv_len).to(dev), q_off, max_q)

    def _move(self, moves, stream) -> None:
        if moves:
            dev = torch.device("cuda", self.ctx.device)
            m = torch.tensor(moves, dtype=torch.int32).t().contiguous().to(dev)
            if stream is not None:
                # the ids live on the current stream and are dropped here, maybe long before ``stream`` gets to them
                m.record_stream(self._torch_stream(int(stream)))
            self.move_pages(m[0], m[1], stream=stream)


class PagePool:
    """Which pages each sequence holds (host only; ``KvCache`` launches the copies it asks for)."""

    def __init__(self, pages: int, page_size: int):
        self.lib = _lib.load()
        self.handle = None
        h = ctypes.c_void_p()
        check(self.lib.rc_pages_create(pages, page_size, ctypes.byref(h)), "rc_pages_create")
        self.handle = h
        self.pages, self.page_size = int(pages), int(page_size)

    def __del__(self):
        if getattr(self, "handle", None):
            self.lib.rc_pages_destroy(self.handle)
            self.handle = None

    def new(self) -> int:
        s = ctypes.c_int()
        check(self.lib.rc_pages_new(self.handle, ctypes.byref(s)), "rc_pages_new")
        return s.value

    def extend(self, seqs, n) -> list[tuple[int, int]]:
        """n more tokens (a number, or one for each) for every sequence; the (source, destination) page copies to
        launch before anything is written to them."""
        ids = _whole(seqs, "extend: sequences")
        one = not hasattr(n, "__iter__") or getattr(n, "ndim", 1) == 0
        counts = _whole([n] * len(ids) if one else n, "extend: counts")
        if counts.shape != ids.shape:
            raise ValueError(f"extend: {len(ids)} sequences, {len(counts)} counts")
        src, dst, k = np.empty(len(ids), np.int32), np.empty(len(ids), np.int32), ctypes.c_int()
        check(self.lib.rc_pages_extend(self.handle, ids.ctypes.data, counts.ctypes.data, len(ids), src.ctypes.data,
                                       dst.ctypes.data, ctypes.byref(k)), "rc_pages_extend")
        return list(zip(src[:k.value].tolist(), dst[:k.value].tolist()))

    def fork(self, seq: int) -> int:
        s = ctypes.c_int()
        check(self.lib.rc_pages_fork(self.handle, seq, ctypes.byref(s)), "rc_pages_fork")
        return s.value

    def trim(self, seq: int, n: int) -> None:
        check(self.lib.rc_pages_trim(self.handle, seq, n), "rc_pages_trim")

    def free(self, seq: int) -> None:
        check(self.lib.rc_pages_free(self.handle, seq), "rc_pages_free")

    def compact(self) -> list[tuple[int, int]]:
        src, dst = np.empty(self.pages, np.int32), np.empty(self.pages, np.int32)
        n = ctypes.c_int()
        check(self.lib.rc_pages_compact(self.handle, src.ctypes.data, dst.ctypes.data, ctypes.byref(n)),
              "rc_pages_compact")
        return list(zip(src[:n.value].tolist(), dst[:n.value].tolist()))

    def info(self) -> tuple[int, int]:
        """(free pages, one past the highest page in use)."""
        f, h = ctypes.c_int(), ctypes.c_int()
        check(self.lib.rc_pages_info(self.handle, ctypes.byref(f), ctypes.byref(h)), "rc_pages_info")
        return f.value, h.value

    def tokens(self, seq: int) -> int:
        n = ctypes.c_int()
        check(self.lib.rc_pages_len(self.handle, seq, ctypes.byref(n)), "rc_pages_len")
        return n.value

    def table(self, seqs, columns: int | None = None) -> tuple[np.ndarray, np.ndarray]:
        """int32 [sequences, columns] page ids (-1 past a sequence's pages) and int32 token counts."""
        ids = _whole(seqs, "table: sequences")
        if columns is None:
            columns = max([1] + [-(-self.tokens(int(s)) // self.page_size) for s in ids])
        table, kv_len = np.empty((len(ids), columns), np.int32), np.empty(len(ids), np.int32)
        check(self.lib.rc_pages_table(self.handle, ids.ctypes.data, len(ids), table.ctypes.data, columns,
                                      kv_len.ctypes.data), "rc_pages_table")
        return table, kv_len
