"""The attention half of a decoder layer: per-head norm and rotation, the paged 4-bit cache, attention over it.

Python-side callers of padra_qk_norm_rope, padra_kv_append, padra_kv_read and padra_attention_q4 (formulas, cache format and
contracts: include/padra_b200.h).  `KvCache` owns one layer's pool, `Sequences` describes the rows of a call, `Rotary` the position
rotation; `AttentionKernels` passes their pointers through.  The reference's counterparts are its attention_*, kv_* and
qk_rope_* kernels (src/cuda/), which neither run on this GPU nor know pages or a 4-bit cache.
"""
from __future__ import annotations

import ctypes as C
import threading

import torch

from . import binding as B

GROUP = 32  # values that share an FP16 scale
NO_WINDOW = 2 ** 31 - 1  # as wide as an int goes, wider than any context
ROWS_TYPE = {torch.bfloat16: B.ROWS_BF16, torch.float16: B.ROWS_F16, torch.float32: B.ROWS_F32}


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


class KvCache:
    """One layer's cache: `pages` pages of `page_size` tokens for `kv_heads` KV heads, 4.5 bits per value."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, device="cuda"):
        _need(head_dim in (64, 128), "head_dim is 64 or 128")
        self._set(torch.zeros((pages, kv_heads, self.block_bytes(page_size, head_dim)), dtype=torch.uint8, device=device), page_size, head_dim)

    @staticmethod
    def block_bytes(page_size: int, head_dim: int) -> int:
        """Bytes of one page of one KV head."""
        return page_size * (head_dim + head_dim // 8)

    @classmethod
    def over(cls, pool: torch.Tensor, page_size: int, head_dim: int) -> "KvCache":
        """A cache in memory that the caller has: pool [pages][kv_heads][block bytes], uint8."""
        self = cls.__new__(cls)
        self._set(pool, page_size, head_dim)
        return self

    def _set(self, pool, page_size, head_dim):
        _need(pool.dtype == torch.uint8 and pool.dim() == 3 and pool.is_contiguous() and pool.shape[2] == self.block_bytes(page_size, head_dim),
              "pool is a contiguous uint8 tensor [pages][kv_heads][block bytes]")
        self.pool, self.page_size, self.head_dim = pool, page_size, head_dim
        self.pages, self.kv_heads = pool.shape[:2]
        self.device_index = pool.get_device()
        self.struct = B.KvCacheStruct(pool.data_ptr(), self.pages, page_size, self.kv_heads, head_dim)
        self.ref = C.addressof(self.struct)


class Sequences:
    """Whose rows a call works on: page_table [count][stride], row_begin [count + 1], context [count], all int32 on the device.
    `rows` is the number of rows of the row arrays, `max_rows` the most that one sequence has; both are known on the host,
    so that nothing has to be read back and a captured call can be replayed with new contents of the three tensors."""

    def __init__(self, page_table: torch.Tensor, row_begin: torch.Tensor, context: torch.Tensor, rows: int, max_rows: int):
        count = context.numel()
        for t in (page_table, row_begin, context):
            _need(t.dtype == torch.int32 and t.is_contiguous() and t.device == context.device, "page_table, row_begin and context are contiguous int32 tensors of one device")
        _need(page_table.dim() == 2 and page_table.shape[0] == count and row_begin.numel() == count + 1, "page_table [count][stride], row_begin [count + 1], context [count]")
        self.page_table, self.row_begin, self.context, self.rows, self.max_rows = page_table, row_begin, context, rows, max_rows
        self.device_index = context.get_device()
        self.struct = B.SequencesStruct(page_table.data_ptr(), row_begin.data_ptr(), context.data_ptr(), count, page_table.shape[1], rows, max_rows)
        self.ref = C.addressof(self.struct)


class Rotary:
    """Rotation of the first 2 * len(inv_freq) values of a head; inv_freq (float64, device) in radians per position."""

    def __init__(self, inv_freq: torch.Tensor, interleaved: bool = False, amplitude: float = 1.0):
        _need(inv_freq.dtype == torch.float64 and inv_freq.dim() == 1 and inv_freq.is_contiguous(), "inv_freq is a contiguous float64 vector")
        self.inv_freq = inv_freq
        self.device_index = inv_freq.get_device()
        self.struct = B.RotaryStruct(inv_freq.data_ptr(), amplitude, 2 * inv_freq.numel(), int(interleaved))
        self.ref = C.addressof(self.struct)


def _row_stride(x: torch.Tensor, rows: int, dim: int, dtype: torch.dtype, what: str, device: int) -> int:
    """Checks a [rows][heads][dim] row array on a device, whose heads lie side by side, and returns its stride per row."""
    shape = x.shape
    if x.get_device() != device:
        raise ValueError(f"{what}: on {x.device}, wanted cuda:{device}")
    if len(shape) != 3 or shape[0] != rows or shape[2] != dim or x.dtype is not dtype:
        raise ValueError(f"{what}: want [{rows}][heads][{dim}] of {dtype}, got {list(shape)} of {x.dtype}")
    if x.is_contiguous():
        return shape[1] * dim
    stride = x.stride()
    if stride[2] != 1 or (shape[1] > 1 and stride[1] != dim):
        raise ValueError(f"{what}: the heads of a row lie side by side")
    return stride[0]


def _empty(shape, dtype: torch.dtype, device, stream) -> torch.Tensor:
    """Memory for a call on `stream` (None: the current one): taken there, since work on the current stream may still be using what
    the current stream has given back."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def _weight(w: torch.Tensor | None, dim: int, device: int) -> int | None:
    if w is None:
        return None
    if w.get_device() != device or (w.dtype is not torch.bfloat16 and w.dtype is not torch.uint16) or w.numel() != dim or not w.is_contiguous():
        raise ValueError(f"norm weights are BF16 vectors of head_dim values on cuda:{device}")
    return w.data_ptr()


class AttentionKernels:
    """Callers of the C ABI on the current stream (or `stream`) of the current device."""

    def __init__(self, device="cuda"):
        self.lib = B.load()
        self.bad = torch.zeros(1, dtype=torch.int32, device=device)
        self._bad, self._device = self.bad.data_ptr(), self.bad.get_device()
        self._workspace = {}  # (stream, head_dim) -> workspace: calls on one stream follow one another
        self._making = threading.Lock()  # of a workspace: two threads' first calls on a stream have to get the same

    def reset_bad(self):
        self.bad.zero_()

    def bad_flag(self) -> int:
        return int(self.bad.item())

    def _stream(self, stream) -> int:
        # the library launches on the current device
        if torch._C._cuda_getDevice() != self._device:
            raise ValueError(f"the current device is not cuda:{self._device}, which these kernels were made for")
        return torch._C._cuda_getCurrentRawStream(self._device) if stream is None else stream.cuda_stream

    def _here(self, *parts) -> int:
        """The kernels' device, after a check that caches, sequences and rotations are there too."""
        for p in parts:
            if p is not None and p.device_index != self._device:
                raise ValueError(f"{type(p).__name__} on device {p.device_index}, wanted cuda:{self._device}")
        return self._device

    def qk_norm_rope(self, q, k, positions, rotary=None, q_weight=None, k_weight=None, eps=1e-6, q_out=None, k_out=None, stream=None):
        """Per-head RMS norm (where a weight is given) and rotation of q and k (k may be None); returns (q_out, k_out)."""
        rows, q_heads, dim = q.shape
        dtype, at = q.dtype, self._here(rotary)
        if q_out is None:
            q_out = _empty(q.shape, dtype, q.device, stream)
        _need(q_out.shape[1] == q_heads, "q_out has as many heads as q")
        if positions is not None:
            _need(positions.dtype is torch.int32 and positions.numel() == rows and positions.is_contiguous() and positions.get_device() == at, "positions: int32 [rows] on the kernels' device")
        if k is not None:
            if k_out is None:
                k_out = _empty(k.shape, dtype, k.device, stream)
            k_heads = k.shape[1]
            _need(k_out.shape[1] == k_heads, "k_out has as many heads as k")
            k_args = (k.data_ptr(), k_out.data_ptr(), _row_stride(k, rows, dim, dtype, "k", at), _row_stride(k_out, rows, dim, dtype, "k_out", at), k_heads)
        else:
            k_args = (None, None, 0, 0, 0)
        status = self.lib.padra_qk_norm_rope(
            q.data_ptr(), q_out.data_ptr(), _row_stride(q, rows, dim, dtype, "q", at), _row_stride(q_out, rows, dim, dtype, "q_out", at), q_heads, *k_args,
            _weight(q_weight, dim, at), _weight(k_weight, dim, at), eps, None if positions is None else positions.data_ptr(), rotary and rotary.ref, rows, dim,
            ROWS_TYPE.get(dtype, -1), self._bad, self._stream(stream))
        if status:
            raise B.PadraError(status, "padra_qk_norm_rope")
        return q_out, k_out

    def append(self, cache, sequences, k, v, rotary=None, k_weight=None, eps=1e-6, q=None, q_weight=None, q_out=None, stream=None):
        """Appends the rows' K (normed, rotated) and V; with q also norms and rotates the rows' queries and returns them."""
        rows, dim, dtype, at = sequences.rows, cache.head_dim, k.dtype, self._here(cache, sequences, rotary)
        _need(k.shape[1] == cache.kv_heads and v.shape[1] == cache.kv_heads, "k and v have the cache's heads")
        if q is not None:
            if q_out is None:
                q_out = _empty(q.shape, dtype, q.device, stream)
            q_heads = q.shape[1]
            _need(q_out.shape[1] == q_heads, "q_out has as many heads as q")
            q_args = (q.data_ptr(), q_out.data_ptr(), _row_stride(q, rows, dim, dtype, "q", at), _row_stride(q_out, rows, dim, dtype, "q_out", at), q_heads,
                      _weight(q_weight, dim, at))
        else:
            q_args = (None, None, 0, 0, 0, None)
        status = self.lib.padra_kv_append(
            cache.ref, sequences.ref, k.data_ptr(), v.data_ptr(), _row_stride(k, rows, dim, dtype, "k", at), _row_stride(v, rows, dim, dtype, "v", at),
            _weight(k_weight, dim, at), eps, rotary and rotary.ref, *q_args, ROWS_TYPE.get(dtype, -1), self._bad, self._stream(stream))
        if status:
            raise B.PadraError(status, "padra_kv_append")
        return q_out

    def read(self, cache, sequences, k_out=None, v_out=None, dtype=torch.bfloat16, stream=None):
        """The values of the cached tokens at the rows' positions; returns (k_out, v_out)."""
        rows, heads, dim, at = sequences.rows, cache.kv_heads, cache.head_dim, self._here(cache, sequences)
        if k_out is None:
            k_out = _empty((rows, heads, dim), dtype, cache.pool.device, stream)
        if v_out is None:
            v_out = _empty((rows, heads, dim), k_out.dtype, cache.pool.device, stream)
        dtype = k_out.dtype
        _need(k_out.shape[1] == heads and v_out.shape[1] == heads, "k_out and v_out have the cache's heads")
        status = self.lib.padra_kv_read(
            cache.ref, sequences.ref, k_out.data_ptr(), v_out.data_ptr(), _row_stride(k_out, rows, dim, dtype, "k_out", at),
            _row_stride(v_out, rows, dim, dtype, "v_out", at), ROWS_TYPE.get(dtype, -1), self._bad, self._stream(stream))
        if status:
            raise B.PadraError(status, "padra_kv_read")
        return k_out, v_out

    def workspace(self, head_dim, handle, stream=None):
        """(address, bytes) of the workspace of calls on `stream` (None: the current one), whose handle is given: calls on one
        stream follow one another.  It is made by the first call on the stream, which therefore comes before any capture;
        captured calls keep using it, so graphs captured on one stream are not to be replayed side by side, nor beside calls on it."""
        found = self._workspace.get((handle, head_dim))
        if found is None:
            with self._making:
                found = self._workspace.get((handle, head_dim)) or self._make_workspace(head_dim, handle, stream)
        return found[:2]

    def _make_workspace(self, head_dim, handle, stream):
        with torch.cuda.stream(stream):
            _need(not torch.cuda.is_current_stream_capturing(), "the first attention call on a stream allocates its workspace: make it before capturing")
        n = self.lib.padra_attention_q4_workspace_bytes(head_dim)
        ws = _empty((n,), torch.uint8, self.bad.device, stream)
        self._workspace[handle, head_dim] = made = ws.data_ptr(), n, ws
        return made

    def attention(self, cache, sequences, q, scale, window=0, out=None, stream=None):
        """softmax(scale q k^T) v over the cache, causal, with window > 0 over the last `window` tokens only.  The longest sequence of rows
        chooses the kernel for all: many decode rows are faster in a call of their own than beside a chunk."""
        rows, dim, dtype, heads, at = sequences.rows, cache.head_dim, q.dtype, q.shape[1], self._here(cache, sequences)
        if out is None:
            out = _empty(q.shape, dtype, q.device, stream)
        _need(out.shape[1] == heads, "out has as many heads as q")
        handle = self._stream(stream)
        status = self.lib.padra_attention_q4(
            cache.ref, sequences.ref, q.data_ptr(), out.data_ptr(), _row_stride(q, rows, dim, dtype, "q", at), _row_stride(out, rows, dim, dtype, "out", at), heads,
            ROWS_TYPE.get(dtype, -1), scale, min(window, NO_WINDOW), *self.workspace(dim, handle, stream), self._bad, handle)
        if status:
            raise B.PadraError(status, "padra_attention_q4")
        return out
