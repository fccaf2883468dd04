"""A paged key-value cache and the attention of one new token over it.

The reference keeps no cache: it observes a backend that grows one by concatenation, per token and layer
(/root/reference/whisper_timestamped/transcribe.py:783-793).  ``PagedKVCache`` is the device-side store next to the capture
rings of ``capture.py`` and ``streams.py``: sequences of different lengths share it and step together, a token is written
once, nothing that is there moves, and the pages may hold 8-bit codes with one power of two per (token, head).

    cache = PagedKVCache.allocate(n_pages=512, n_heads=8, head_dim=64, page_size=16, dtype=torch.float16, device="cuda")
    cache.append(k, v, table, positions)          # one new token of every sequence (k, v: (B, 8, 64))
    out = cache.attend(q, table, lengths)         # (B, 8, 64): each over its own positions 0 ... lengths[b] - 1
    k_rows, v_rows = cache.gather(table, positions, sequences=seq)

``table`` (int32, (B, width)): row b lists the pages of sequence b in order; entries behind its last page are never read.
Everything runs on the current stream of the cache's device and reads tables, positions and lengths on the device: a
captured graph follows them from replay to replay.  ``check()`` (which waits for the device) raises if a call since the
last check met a sequence, position, length or page outside of its range; such a call reads and writes nothing there
and returns NaN for what it could not compute.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import WtError

_DTYPES = {torch.float32: _lib.WT_DTYPE_F32, torch.float16: _lib.WT_DTYPE_F16, torch.bfloat16: _lib.WT_DTYPE_BF16}
_PAGE_DTYPES = {**_DTYPES, torch.float8_e4m3fn: _lib.WT_DTYPE_E4M3}
HEAD_DIMS = (32, 64, 96, 128, 256)


def _overlaps(t):
    """May two elements of t share a place?  (A dimension of size one has no stride to speak of.)"""
    extent = 1
    for stride, size in sorted((t.stride(i), t.shape[i]) for i in range(t.dim()) if t.shape[i] > 1):
        if stride < extent:
            return True
        extent += stride * (size - 1)
    return False


def _check_pages(t, name):
    """(pages, heads, slots, head_dim), values of a row side by side, 16-byte steps, no two elements in one place."""
    if not isinstance(t, torch.Tensor) or t.dim() != 4 or t.dtype not in _PAGE_DTYPES:
        raise WtError(f"{name}: a 4-dimensional tensor (pages, heads, slots, head_dim) of float32, float16, bfloat16 or float8_e4m3fn")
    if min(t.shape) < 1 or t.shape[3] not in HEAD_DIMS:
        raise WtError(f"{name}: shape {tuple(t.shape)}; head_dim is one of {HEAD_DIMS}, nothing is empty")
    if t.stride(3) != 1 or t.data_ptr() % 16 or any(t.stride(i) * t.element_size() % 16 for i in range(3) if t.shape[i] > 1):
        raise WtError(f"{name}: rows must be contiguous and start on 16-byte steps (strides {t.stride()})")
    if _overlaps(t):
        raise WtError(f"{name}: rows overlap (strides {t.stride()})")


class PagedKVCache:
    """Over tensors the caller owns: ``k``, ``v`` (pages, heads, slots, head_dim), in float32, float16 or bfloat16, or in
    float8_e4m3fn with ``k_exp``, ``v_exp`` (pages, heads, slots) uint8: value = code * 2 ** (exp - 127)."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_exp: torch.Tensor | None = None, v_exp: torch.Tensor | None = None):
        _check_pages(k, "k")
        _check_pages(v, "v")
        if k.shape != v.shape or k.dtype != v.dtype:
            raise WtError(f"k and v differ: {tuple(k.shape)} {k.dtype}, {tuple(v.shape)} {v.dtype}")
        if k.data_ptr() == v.data_ptr():
            raise WtError("k and v are the same memory")
        quantised = k.dtype == torch.float8_e4m3fn
        for name, e in (("k_exp", k_exp), ("v_exp", v_exp)):
            if quantised != (e is not None):
                raise WtError(f"{name}: a float8_e4m3fn cache has exponents, another has none")
            if quantised and (e.shape != k.shape[:3] or e.dtype != torch.uint8 or not e.is_contiguous() or e.data_ptr() % 16):
                raise WtError(f"{name}: contiguous uint8 of shape {tuple(k.shape[:3])}, 16-byte aligned")
        if quantised and k_exp.data_ptr() == v_exp.data_ptr():
            raise WtError("k_exp and v_exp are the same memory")
        if k.shape[0] > 2 ** 31 - 1 or k.shape[1] > 65535 or k.shape[2] > 2 ** 31 - 1:
            raise WtError(f"k: shape {tuple(k.shape)} is beyond 32-bit page and slot numbers or 65535 heads")
        _lib._need_cuda(k, "k")
        _lib.same_device(k, v, k_exp, v_exp)
        self.k, self.v, self.k_exp, self.v_exp = k, v, k_exp, v_exp
        self.device, self.dtype = k.device, k.dtype
        self.n_pages, self.n_heads, self.page_size, self.head_dim = k.shape
        self.error = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._lib = _lib.load()

        def strides(t):    # (a dimension of size one has no stride to speak of)
            return [t.stride(i) if t.shape[i] > 1 else 0 for i in range(3)]

        self._desc = _lib.KvCache(k.data_ptr(), v.data_ptr(), _lib._ptr(k_exp) or None, _lib._ptr(v_exp) or None, *strides(k), *strides(v),
                                  self.n_pages, self.n_heads, self.page_size, self.head_dim, _PAGE_DTYPES[k.dtype], 0,
                                  self.error.data_ptr())
        self._p = ctypes.addressof(self._desc)

    @classmethod
    def allocate(cls, n_pages: int, n_heads: int, head_dim: int, page_size: int = 64, dtype=torch.float16, device="cuda"):
        """Zeroed pages, laid out (page, head, slot); ``dtype=torch.float8_e4m3fn``: with exponents."""
        shape = (int(n_pages), int(n_heads), int(page_size), int(head_dim))
        if dtype == torch.float8_e4m3fn:
            k, v, ke, ve = (torch.zeros(s, dtype=torch.uint8, device=device) for s in (shape, shape, shape[:3], shape[:3]))
            return cls(k.view(dtype), v.view(dtype), ke, ve)
        return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))

    # --- arguments
    def _dtype(self, t_dtype, name):
        """An 8-bit cache takes and gives any of the three types, another only its own."""
        if t_dtype not in _DTYPES or (self.k_exp is None and t_dtype != self.dtype):
            raise WtError(f"{name}: {t_dtype} with a cache of {self.dtype}")
        return _DTYPES[t_dtype]

    def _int32(self, t, name, shape=None):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.device != self.device or not t.is_contiguous() or \
                (shape is not None and t.shape != shape):
            raise WtError(f"{name}: contiguous int32 on {self.device}" + (f" of shape {tuple(shape)}" if shape is not None else ""))
        return t.data_ptr()

    def _table(self, table):
        if not isinstance(table, torch.Tensor) or table.dim() != 2 or table.dtype != torch.int32 or table.device != self.device or \
                table.shape[1] < 1 or table.stride(1) != 1 or (table.shape[0] > 1 and table.stride(0) < table.shape[1]):
            raise WtError(f"page table: int32 (sequences, pages) on {self.device}, the pages of a sequence side by side")
        n, width = table.shape
        if width * self.page_size > 2 ** 31 - 1:
            raise WtError(f"page table: {width} pages of {self.page_size} are beyond 32-bit positions")
        return table.data_ptr(), table.stride(0) if n > 1 else width, n, width

    def _rows_of(self, positions, sequences, n_seqs):
        if not isinstance(positions, torch.Tensor) or positions.dim() != 1:
            raise WtError("positions: one int32 per row")
        n = positions.shape[0]
        pos = self._int32(positions, "positions")
        if sequences is None and n > n_seqs:
            raise WtError(f"{n} rows for {n_seqs} sequences: say whose they are (sequences=)")
        return n, None if sequences is None else self._int32(sequences, "sequences", positions.shape), pos

    def _new(self, t, name, n):
        if not isinstance(t, torch.Tensor) or t.shape != (n, self.n_heads, self.head_dim) or t.device != self.device:
            raise WtError(f"{name}: ({n}, {self.n_heads}, {self.head_dim}) on {self.device}")
        item = t.element_size()
        if n and (t.stride(2) != 1 or t.data_ptr() % 16 or (n > 1 and t.stride(0) * item % 16) or (self.n_heads > 1 and t.stride(1) * item % 16)):
            raise WtError(f"{name}: rows must be contiguous and start on 16-byte steps (strides {t.stride()})")
        return t.data_ptr(), t.stride(0) if n > 1 else 0, t.stride(1) if self.n_heads > 1 else 0

    # --- operators
    def append(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, positions: torch.Tensor, sequences: torch.Tensor | None = None):
        """Writes rows ``k[r]``, ``v[r]`` (heads, head_dim; any row and head strides of whole 16 bytes) at ``positions[r]``
        of sequence ``sequences[r]`` (None: of sequence r).  A negative position marks a padded row: not written.  No
        two rows of a call may name the same place."""
        tp, ts, n_seqs, width = self._table(table)
        n, seq, pos = self._rows_of(positions, sequences, n_seqs)
        if k.dtype != v.dtype:
            raise WtError(f"k and v differ: {k.dtype}, {v.dtype}")
        dt = self._dtype(k.dtype, "k, v")
        kp, k_row, k_head = self._new(k, "k", n)
        vp, v_row, v_head = self._new(v, "v", n)
        if n == 0:
            return
        with _lib.on_device(self.k) as st:
            rc = self._lib.wt_kv_append(self._p, kp, vp, dt, k_row, k_head, v_row, v_head, n, tp, ts, n_seqs, width, seq, pos, st)
        _lib._check(rc, "wt_kv_append")

    def gather(self, table: torch.Tensor, positions: torch.Tensor, sequences: torch.Tensor | None = None, dtype=None, out=None):
        """-> (k, v), each (rows, heads, head_dim): the rows at ``positions[r]`` of sequence ``sequences[r]``, in the cache's
        type, or from an 8-bit cache in ``dtype`` (default float32).  A negative position reads as zeros.  ``out``: two
        contiguous tensors to write instead of new ones."""
        tp, ts, n_seqs, width = self._table(table)
        n, seq, pos = self._rows_of(positions, sequences, n_seqs)
        if out is None:
            dtype = dtype if dtype is not None else (torch.float32 if self.k_exp is not None else self.dtype)
            dt = self._dtype(dtype, "dtype")
            out = tuple(torch.empty((n, self.n_heads, self.head_dim), dtype=dtype, device=self.device) for _ in range(2))
        else:
            k, v = out
            if k.dtype != v.dtype or (dtype is not None and k.dtype != dtype):
                raise WtError(f"out: {k.dtype} and {v.dtype}" + (f", not {dtype}" if dtype is not None else ""))
            dt = self._dtype(k.dtype, "out")
            for name, t in (("out[0]", k), ("out[1]", v)):
                self._new(t, name, n)
                if not t.is_contiguous():
                    raise WtError(f"{name}: not contiguous")
            if n and k.data_ptr() == v.data_ptr():
                raise WtError("out: the same memory twice")
        if n:
            with _lib.on_device(self.k) as st:
                rc = self._lib.wt_kv_gather(self._p, out[0].data_ptr(), out[1].data_ptr(), dt, n, tp, ts, n_seqs, width, seq, pos, st)
            _lib._check(rc, "wt_kv_gather")
        return out

    def attend(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, scale: float | None = None,
               out: torch.Tensor | None = None, return_lse: bool = False):
        """One new token of every sequence: q (B, query heads, head_dim) over the sequence's positions 0 ... lengths[b] - 1;
        query head h reads key head h // (query heads // heads).  -> (B, query heads, head_dim) in q's type, with
        ``return_lse`` also the float32 (B, query heads) logarithm of its sum of exponentials.  A length of zero gives
        zeros (and -inf).  ``scale``: default head_dim ** -0.5.  ``out`` may be q itself."""
        tp, ts, n_seqs, width = self._table(table)
        if not isinstance(q, torch.Tensor) or q.dim() != 3 or q.shape[0] != n_seqs or q.shape[2] != self.head_dim or \
                q.shape[1] < 1 or q.shape[1] % self.n_heads or q.device != self.device or q.stride(2) != 1:
            raise WtError(f"q: ({n_seqs}, a multiple of {self.n_heads}, {self.head_dim}) on {self.device}, a head's values side by side")
        dt = self._dtype(q.dtype, "q")
        lp = self._int32(lengths, "lengths", (n_seqs,))
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
        elif out.shape != q.shape or out.dtype != q.dtype or out.device != self.device or out.stride(2) != 1 or \
                _overlaps(out):
            raise WtError(f"out: {tuple(q.shape)} of {q.dtype} on {self.device}, a head's values side by side, no two in one place")
        hq = q.shape[1]
        lse = torch.empty((n_seqs, hq), dtype=torch.float32, device=self.device) if return_lse else None
        if n_seqs:
            with _lib.on_device(self.k) as st:
                ws, ws_bytes = self._captured_workspace(n_seqs, hq, width)
                rc = self._lib.wt_kv_attend(self._p, q.data_ptr(), dt, q.stride(0), q.stride(1), n_seqs, hq,
                                            self.head_dim ** -0.5 if scale is None else float(scale), tp, ts, width, lp, out.data_ptr(),
                                            out.stride(0), out.stride(1), lse.data_ptr() if return_lse else None, _lib._ptr(ws) or None, ws_bytes, st)
            _lib._check(rc, "wt_kv_attend")
        return (out, lse) if return_lse else out

    def _captured_workspace(self, n_seqs, n_q_heads, width):
        """A call that is being captured has a workspace in its graph's own memory, its counters cleared in every replay: two
        graphs never share one.  Others use the library's arena of their stream."""
        if not torch.cuda.is_current_stream_capturing():
            return None, 0
        n = self._lib.wt_kv_attend_workspace(self._p, n_seqs, n_q_heads, width)
        if n < 0:
            _lib._check(n, "wt_kv_attend_workspace")
        if n == 0:
            return None, 0
        ws = torch.empty(n, dtype=torch.uint8, device=self.device)
        ws[:_lib.WT_KV_WORKSPACE_ZEROED].zero_()
        return ws, n

    def check(self):
        """Waits for the device; raises if a call since the last check met something outside of its range."""
        bits = int(self.error.item())
        if bits:
            self.error.zero_()
            said = {_lib.WT_KV_BAD_POSITION: "a position or length beyond the page table", _lib.WT_KV_BAD_PAGE: "a page outside of the cache",
                    _lib.WT_KV_BAD_SEQUENCE: "a sequence outside of the page table"}
            raise WtError("paged cache: " + ", ".join(s for b, s in said.items() if bits & b))
