"""The KV cache in 8 bits: codes and a scale for each (position, kv head) of K and of V, in pages, with the calls that store new
rows, attend to the cache and read it back (jg_kvq_* in include/jsgrad_cuda.h).

The reference keeps K and V in the model's 16-bit type (Attention.cache_kv, jsgrad/models/llama.ts:78-90); ``KVCache`` in llama.py is
that cache, ``QuantKVCache`` takes 0.51 of its memory (and of what a decode step reads) for an error of K and V of about 0.7 %
("int8") or 2.6 % ("fp8") of a normally distributed row.  ``Llama3(kv_dtype="int8")`` puts it under a model.

Rows are fp16 tensors [rows, columns] whose first columns are used: wq|wk|wv outputs [(H + 2G) * hd], queries and results [H * hd],
read-back K and V [G * hd].  `pos`, `seq`, `count`, `first` are int32 tensors on the device; what they name outside the cache
is not followed (include/jsgrad_cuda.h says what comes back instead).  One or two rows of a model's decode are faster with the fp16 cache, whose steps are a
single kernel.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import ffi
from .device import CUDA, Tensor

FORMATS = {"int8": ffi.KVQ_INT8, "fp8": ffi.KVQ_E4M3}


def _ints(dev: CUDA, name: str, t: Tensor | None, n: int) -> int:
    """Its address, or 0 where it is not given."""
    if t is None:
        return 0
    buf = t.buf
    if buf.dev is not dev:
        raise ValueError(f"{name} lies on {buf.dev.device}, the cache on {dev.device}")
    if buf.dtype != "int32":
        raise TypeError(f"{name} is {buf.dtype}, not int32")
    if buf.size < n:
        raise ValueError(f"{name} has {buf.size} entries, {n} are needed")
    return buf.ptr


def _rows(dev: CUDA, name: str, t: Tensor, columns: int, rows: int = 0) -> tuple[int, int, int]:
    """(address, row stride, rows) of a tensor of fp16 rows."""
    buf, ld = t.buf, t.shape[-1]
    if buf.dev is not dev:
        raise ValueError(f"{name} lies on {buf.dev.device}, the cache on {dev.device}")
    if buf.dtype != "float16":
        raise TypeError(f"{name} is {buf.dtype}, not float16")
    if ld < columns:
        raise ValueError(f"{name} has rows of {ld}, {columns} are needed")
    have = buf.size // ld
    if have < rows:
        raise ValueError(f"{name} has {have} rows, {rows} are needed")
    return buf.ptr, ld, have


class QuantKVCache:
    """A paged cache of `max_batch` slots of up to `max_context` positions, dtype "int8" or "fp8" (e4m3).  Every slot owns its
    pages unless `n_pages` gives the pool another size and `set_block_table` deals them out."""

    def __init__(self, dev: CUDA, n_layers: int, n_heads: int, n_kv_heads: int, head_dim: int, max_context: int, max_batch: int,
                 page_size: int = 64, dtype: str = "int8", n_pages: int | None = None):
        if dtype not in FORMATS:
            raise ValueError(f"dtype={dtype!r}: expected one of {', '.join(map(repr, FORMATS))}")
        self.dev, self.dtype = dev, dtype
        self.n_heads, self.n_kv_heads, self.head_dim, self.page_size = n_heads, n_kv_heads, head_dim, page_size
        self.max_pages_per_seq = (max_context + page_size - 1) // page_size
        self.n_pages = n_pages if n_pages is not None else self.max_pages_per_seq * max_batch
        self.max_batch = max_batch
        self._q, self._kv, self._qkv = n_heads * head_dim, n_kv_heads * head_dim, (n_heads + 2 * n_kv_heads) * head_dim  # columns
        d = ffi.KvDesc(n_layers, n_kv_heads, head_dim, page_size, self.n_pages, max_batch, self.max_pages_per_seq, n_heads, 0)
        self.handle = C.c_void_p()
        ffi.call("jg_kvq_create", dev.handle, C.byref(d), FORMATS[dtype], C.byref(self.handle))

    def set_block_table(self, table: np.ndarray) -> None:
        """Pages of every slot: int32 [max_batch, max_pages_per_seq]."""
        table = np.ascontiguousarray(table, dtype=np.int32)
        if table.shape != (self.max_batch, self.max_pages_per_seq):
            raise ValueError(f"block table of shape {table.shape}, not {(self.max_batch, self.max_pages_per_seq)}")
        ffi.call("jg_kvq_set_block_table", self.handle, table.ctypes.data_as(C.c_void_p))

    def nbytes(self) -> int:
        """Of codes, scales and block table."""
        out = C.c_uint64(0)
        ffi.call("jg_kvq_bytes", self.handle, C.byref(out))
        return out.value

    def write(self, layer: int, qkv: Tensor, pos: Tensor, seq: Tensor | None = None, freqs_cis: Tensor | None = None,
              q_out: Tensor | None = None) -> None:
        """Rotates Q and K of every row of `qkv` (by `freqs_cis`, or not at all) and stores K and V: row r is position pos[r] of slot
        seq[r] (None: slot r).  Rotated Q goes to `q_out`, which may be `qkv`.  The rows name different positions."""
        x, ldx, R = _rows(self.dev, "qkv", qkv, self._qkv)
        to, ldq, _ = _rows(self.dev, "q_out", q_out, self._q, R) if q_out is not None else (0, 0, 0)
        if to == x and ldq != ldx and R > 1:  # its rows would be written over those of qkv that are still to be read
            raise ValueError(f"q_out is qkv, with rows of {ldq} and not {ldx}")
        table, n = self._table(freqs_cis)
        self.dev.call("jg_kvq_write", self.handle, layer, to, ldq, x, ldx, table, n, _ints(self.dev, "pos", pos, R), _ints(self.dev, "seq", seq, R), R, self.n_heads)

    def decode(self, layer: int, qkv: Tensor, pos: Tensor, freqs_cis: Tensor | None = None, seq: Tensor | None = None,
               out: Tensor | None = None) -> Tensor:
        """One new token for each row of `qkv`, rows in different slots: stores it as `write` does and attends to positions 0 .. pos[b].
        `qkv` is left as it is.  A row whose position lies outside the cache gets zeros."""
        x, ldx, B = _rows(self.dev, "qkv", qkv, self._qkv)
        if out is None:
            out = Tensor.empty((B, self._q), "float16", self.dev)
        to, ldo, _ = _rows(self.dev, "out", out, self._q, B)
        table, n = self._table(freqs_cis)
        self.dev.call("jg_kvq_decode", self.handle, layer, to, ldo, x, ldx, table, n, _ints(self.dev, "pos", pos, B), _ints(self.dev, "seq", seq, B), B, self.n_heads)
        return out

    def attend(self, layer: int, q: Tensor, pos: Tensor, count: Tensor | None = None, first: Tensor | None = None,
               seq: Tensor | None = None, max_count: int | None = None, step: int | None = None, out: Tensor | None = None) -> Tensor:
        """Attention of a chunk of new positions of each of len(pos) sequences, whose K and V `write` has stored: position pos[b] + i, i <
        count[b], is row first[b] + i * step of `q` (rotated) and of `out`, and sees positions 0 .. pos[b] + i of slot seq[b].
        Defaults: max_count positions each (all rows, dealt evenly), in position-major order (row i * B + b).  A ragged batch
        has running sums in `first`, step=1, and the largest count as `max_count`.  Rows that no sequence names stay as they are (zeros where
        `out` is not given); a row whose position or slot lies outside the cache gets zeros."""
        x, ldq, R = _rows(self.dev, "q", q, self._q)
        if out is None:
            out = Tensor.zeros((R, self._q), "float16", self.dev)
        to, ldo, _ = _rows(self.dev, "out", out, self._q, R)
        self.dev.call("jg_kvq_attn", self.handle, layer, to, ldo, x, ldq, R, *self._where(R, pos, count, first, seq, max_count, step), self.n_heads)
        return out

    def read(self, layer: int, pos: Tensor, count: Tensor | None = None, first: Tensor | None = None, seq: Tensor | None = None,
             max_count: int | None = None, step: int | None = None, k: Tensor | None = None, v: Tensor | None = None,
             rows: int | None = None) -> tuple[Tensor, Tensor]:
        """K and V of stretches of the cache as fp16 rows, named as in `attend`; `rows` of them are made where `k` and `v` are not given."""
        if (k is None) != (v is None):
            raise ValueError("k and v are given together")
        if k is None:
            if rows is None:
                raise ValueError("give k and v, or the number of rows")
            k, v = (Tensor.zeros((rows, self._kv), "float16", self.dev) for _ in range(2))
        to_k, ld, R = _rows(self.dev, "k", k, self._kv)
        to_v, ldv, _ = _rows(self.dev, "v", v, self._kv, R)
        if ldv != ld:
            raise ValueError(f"k has rows of {ld}, v of {ldv}")
        self.dev.call("jg_kvq_read", self.handle, layer, to_k, to_v, ld, R, *self._where(R, pos, count, first, seq, max_count, step))
        return k, v

    def _table(self, freqs_cis: Tensor | None) -> tuple[int, int]:
        if freqs_cis is None:
            return 0, 0
        shape = freqs_cis.shape
        if freqs_cis.buf.dev is not self.dev:
            raise ValueError(f"freqs_cis lies on {freqs_cis.buf.dev.device}, the cache on {self.dev.device}")
        if freqs_cis.buf.dtype != "float16" or len(shape) != 3 or shape[2] != 2 or shape[1] * 2 != self.head_dim:
            raise ValueError(f"freqs_cis is {freqs_cis.dtype} {tuple(shape)}, not float16 [positions, {self.head_dim // 2}, 2]")
        return freqs_cis.buf.ptr, shape[0]

    def _where(self, R: int, pos: Tensor, count, first, seq, max_count: int | None, step: int | None) -> tuple:
        """(pos, count, first, seq, sequences, max_count, step) of a call."""
        B = pos.buf.size
        if max_count is None:
            if R % B or count is not None or first is not None:
                raise ValueError("max_count is needed where sequences have different numbers of rows")
            max_count = R // B
        if step is None:
            step = B if first is None else 1
        return _ints(self.dev, "pos", pos, B), _ints(self.dev, "count", count, B), _ints(self.dev, "first", first, B), _ints(self.dev, "seq", seq, B), B, max_count, step

    def close(self) -> None:
        if self.handle:
            ffi.call("jg_kvq_destroy", self.handle)
            self.handle = None

    def __del__(self):
        try:
            if self.dev.handle is not None:
                self.close()
        except Exception:
            pass
