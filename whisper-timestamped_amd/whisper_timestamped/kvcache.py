"""A paged key-value cache and the attention of one new token over it.

The reference keeps no cache: it observes a backend that grows one by concatenation, per token and layer
(/root/reference/whisper_timestamped/transcribe.py:783-793).  ``PagedKVCache`` is the device-side store next to the capture
rings of ``capture.py`` and ``streams.py``: sequences of different lengths share it and step together, a token is written
once, nothing that is there moves, and the pages may hold 8-bit codes with one power of two per (token, head).

    cache = PagedKVCache.allocate(n_pages=512, n_heads=8, head_dim=64, page_size=16, dtype=torch.float16, device="cuda")
    cache.append(k, v, table, positions)          # one new token of every sequence (k, v: (B, 8, 64))
    out = cache.attend(q, table, lengths)         # (B, 8, 64): each over its own positions 0 ... lengths[b] - 1
    k_rows, v_rows = cache.gather(table, positions, sequences=seq)

``table`` (int32, (B, width)): row b lists the pages of sequence b in order; entries behind its last page may be read, but are never followed.
Everything runs on the current stream of the cache's device and reads tables, positions and lengths on the device: a
captured graph follows them from replay to replay.  ``check()`` (which waits for the device) raises if a call since the
last check met a sequence, position, length or page outside of its range; such a call reads and writes nothing there
and returns NaN for what it could not compute.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from ._lib import WtError

HEAD_DIMS = (32, 64, 96, 128, 256)


@functools.lru_cache(maxsize=None)
def _calls():
    """The module of the calls, on the entries of the library that ``_lib`` has loaded."""
    L = _lib.load()
    missing = [n for n in _lib.KV_EXPORTS if not hasattr(L, n)]
    if missing:
        raise ImportError(f"{_lib.LIB_PATH} lacks {', '.join(missing)}: rebuild it (`make -C {_lib._PKG_ROOT}/csrc`)")
    try:
        from . import _kvcalls
    except ImportError as err:
        raise ImportError(f"{err}: build it with `make -C {_lib._PKG_ROOT}/csrc`") from err
    entries = (L.wt_kv_append, L.wt_kv_gather, L.wt_kv_attend, L.wt_kv_attend_workspace, L.wt_last_error)
    _kvcalls.setup(WtError, *(ctypes.cast(f, ctypes.c_void_p).value for f in entries))
    return _kvcalls


class PagedKVCache:
    """Over tensors the caller owns: ``k``, ``v`` (pages, heads, slots, head_dim), in float32, float16 or bfloat16, or in
    float8_e4m3fn with ``k_exp``, ``v_exp`` (pages, heads, slots) uint8: value = code * 2 ** (exp - 127)."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_exp: torch.Tensor | None = None, v_exp: torch.Tensor | None = None):
        self._calls = _calls()
        self._handle, self.error = self._calls.make(k, v, k_exp, v_exp, False)
        self.k, self.v, self.k_exp, self.v_exp = k, v, k_exp, v_exp
        self.device, self.dtype = k.device, k.dtype
        self.n_pages, self.n_heads, self.page_size, self.head_dim = k.shape

    @classmethod
    def allocate(cls, n_pages: int, n_heads: int, head_dim: int, page_size: int = 64, dtype=torch.float16, device="cuda"):
        """Zeroed pages, laid out (page, head, slot); ``dtype=torch.float8_e4m3fn``: with exponents."""
        shape = (int(n_pages), int(n_heads), int(page_size), int(head_dim))
        if dtype == torch.float8_e4m3fn:
            k, v, ke, ve = (torch.zeros(s, dtype=torch.uint8, device=device) for s in (shape, shape, shape[:3], shape[:3]))
            return cls(k.view(dtype), v.view(dtype), ke, ve)
        return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))

    # --- operators (argument checks, results and launches: csrc/wt_kv_calls.cpp)
    def append(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, positions: torch.Tensor, sequences: torch.Tensor | None = None):
        """Writes rows ``k[r]``, ``v[r]`` (heads, head_dim; any row and head strides of whole 16 bytes) at ``positions[r]``
        of sequence ``sequences[r]`` (None: of sequence r).  A negative position marks a padded row: not written.  No
        two rows of a call may name the same place, and ``k`` and ``v`` are not the cache's own memory."""
        self._calls.append(self._handle, k, v, table, positions, sequences)

    def gather(self, table: torch.Tensor, positions: torch.Tensor, sequences: torch.Tensor | None = None, dtype=None, out=None):
        """-> (k, v), each (rows, heads, head_dim): the rows at ``positions[r]`` of sequence ``sequences[r]``, in the cache's
        type, or from an 8-bit cache in ``dtype`` (default float32).  A negative position reads as zeros.  ``out``: two
        contiguous tensors to write instead of new ones (not the cache's own memory)."""
        return self._calls.gather(self._handle, table, positions, sequences, dtype, out)

    def attend(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, scale: float | None = None,
               out: torch.Tensor | None = None, return_lse: bool = False, workspace: torch.Tensor | None = None):
        """One new token of every sequence: q (B, query heads, head_dim) over the sequence's positions 0 ... lengths[b] - 1;
        query head h reads key head h // (query heads // heads).  -> (B, query heads, head_dim) in q's type, with
        ``return_lse`` also the float32 (B, query heads) logarithm of its sum of exponentials.  A length of zero gives
        zeros (and -inf).  ``scale``: default head_dim ** -0.5.  ``out`` may be q itself, and shares no memory with it otherwise.

        Long sequences are split over workgroups that meet in a workspace: the library's own of the current stream, or
        ``workspace`` (from ``attend_workspace``).  Calls that may run at the same time need one each.  A call that is being
        captured into a graph has none of the stream's: without ``workspace`` it takes one in the graph's memory, which
        costs every replay a small kernel that clears its counters."""
        return self._calls.attend(self._handle, q, table, lengths, scale, out, return_lse, workspace)

    def attend_workspace(self, n_q_heads: int, table: torch.Tensor) -> torch.Tensor | None:
        """A workspace for ``attend`` calls with this many query heads and tables of this shape (or fewer sequences, or fewer
        pages): made ready once, left ready by every call.  None: such calls need none."""
        return self._calls.workspace(self._handle, table, n_q_heads)

    def check(self):
        """Waits for the device, all of its streams; raises if a call since the last check met something outside of its range."""
        torch.cuda.synchronize(self.device)
        bits = int(self.error.item())
        if bits:
            self.error.zero_()
            torch.cuda.synchronize(self.device)          # (cleared before a call on another stream can report again)
            said = {_lib.WT_KV_BAD_POSITION: "a position or length beyond the page table", _lib.WT_KV_BAD_PAGE: "a page outside of the cache",
                    _lib.WT_KV_BAD_SEQUENCE: "a sequence outside of the page table"}
            raise WtError("paged cache: " + ", ".join(s for b, s in said.items() if bits & b))
