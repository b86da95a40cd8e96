"""Pages of a paged key/value cache, given out and taken back on the GPU, on libgemma4_qmm.

A :class:`PagePool` keeps which pages are free, how many tokens each request holds and the
requests' tables.  Before a step :meth:`PagePool.reserve` finds pages for its new tokens and
fills the arrays of the step's batch; after it :meth:`PagePool.release` keeps what is known to
stay (all of a prompt, the accepted ones of drafted tokens, nothing of a request that is done)
and takes the other pages back.  Both read lengths on the device, so a captured step can hold
them::

    pool = PagePool.allocate(num_pages, 64, requests=32, pages_per_request=512)
    positions, slots = pool.reserve(new_tokens, rows)      # int32 [32] on the GPU
    q = cache.append(k, v, pool.batch, rope=rope, q=q)     # caches of pool.num_pages pages
    y = cache.attend(q, pool.batch)
    pool.release(pool.lens + kept)

One pool serves every layer whose pages go by the same lengths and window.  Errors surface as
:class:`~helios_amd.qmm.Gemma4Error`; there is no fallback.
"""

from __future__ import annotations

import ctypes

from . import qmm
from .attention import KVBatch, _int32, _invalid, _new, _on
from .qmm import Gemma4Error, Status

_u32, _vp = ctypes.c_uint32, ctypes.c_void_p


class _Pool(ctypes.Structure):
    _fields_ = [("free_pages_dev", _vp), ("free_count_dev", _vp), ("lens_dev", _vp), ("block_tables_dev", _vp), ("num_pages", _u32),
                ("page_size", _u32), ("requests", _u32), ("pages_per_request", _u32), ("table_stride", _u32)]


class PagePool:
    """Free pages, lengths and tables of ``lens.numel()`` requests over pages of ``page_size``
    tokens: int32 GPU tensors free_pages [num_pages] (its first free_count [1] entries are the
    free pages, the last given out next), lens [R], block_tables [R, pages]; kept, not copied.
    A page is in one table, or free.  ``batch`` is the :class:`KVBatch` of the last ``reserve``,
    over the same tables; ``granted`` says which requests got their pages."""

    def __init__(self, free_pages, free_count, lens, block_tables, page_size: int):
        import torch

        self.free_pages, self.free_count = _int32(free_pages, "free_pages", 1), _int32(free_count, "free_count", 1)
        self.lens, self.block_tables = _int32(lens, "lens", 1), _int32(block_tables, "block_tables", 2)
        self.requests, self.num_pages, self.page_size = lens.shape[0], free_pages.shape[0], int(page_size)
        self._device = lens.get_device()
        if free_count.shape[0] != 1:
            raise _invalid("free_count must have one entry")
        for t in (free_pages, free_count, block_tables):
            if t.get_device() != self._device:
                raise _invalid("free_pages, free_count, lens and block_tables must be on one device")
        if not 0 < self.page_size < 1 << 32:  # the rest is the library's to check
            raise _invalid("page_size must be positive and fit 32 bits")
        ints = lambda n: torch.zeros(n, dtype=torch.int32, device=lens.device)  # noqa: E731
        self.granted = ints(self.requests)
        # also checks the shapes; batch.kv_lens is what reserve writes, not what is held
        self.batch = KVBatch(ints(self.requests + 1), ints(self.requests), block_tables)
        width, stride = self.batch._table
        self._lib = qmm.load_library()
        self._c = _Pool(free_pages.data_ptr(), free_count.data_ptr(), lens.data_ptr(), block_tables.data_ptr(), self.num_pages,
                        self.page_size, self.requests, width, stride)
        self._ref = ctypes.byref(self._c)
        self._outs = (self.batch.query_starts.data_ptr(), self.batch.kv_lens.data_ptr(), self.granted.data_ptr())

    @classmethod
    def allocate(cls, num_pages: int, page_size: int, requests: int, pages_per_request: int, device="cuda"):
        """A pool whose pages are all free, page 0 given out first, and whose requests are empty."""
        import torch

        ints = {"dtype": torch.int32, "device": device}
        return cls(torch.arange(num_pages - 1, -1, -1, **ints), torch.full((1,), num_pages, **ints), torch.zeros(requests, **ints),
                   torch.full((requests, pages_per_request), -1, **ints), page_size)

    def reserve(self, new_tokens, rows: int | None = None, stream=None):
        """Finds pages for new_tokens[r] tokens (int32 [R]) after the lens[r] that request r holds,
        in the order of the requests, each request's whole or not at all (``granted``), and sets
        ``batch`` to the step's.  With ``rows`` (the rows of q, padding included) returns
        (positions int32 [rows], slots int64 [rows]): each row's position in its request and
        page * page_size + slot, -1 where there is no page; else (None, None).  ``lens`` stays."""
        import torch

        self._lens(new_tokens, "new_tokens")
        positions = slots = None
        if rows is not None:
            if not 0 <= rows < 1 << 24:
                raise Gemma4Error(Status.UNSUPPORTED_CONFIG, "rows must be 0 to 2^24 - 1")
            positions = _new(self.lens, (rows,), torch.int32, stream)
            slots = _new(self.lens, (rows,), torch.int64, stream)
        _on(self._device, (new_tokens,), ())
        status = self._lib.gemma4_kv_reserve(self._ref, new_tokens.data_ptr(), *self._outs, rows or 0,
                                             positions.data_ptr() if rows else None, slots.data_ptr() if rows else None,
                                             qmm._stream_ptr(stream, self._device))
        if status != 0:
            qmm.check(status, self._lib)
        return positions, slots

    def release(self, lens, window: int = 0, stream=None):
        """Keeps lens[r] tokens (int32 [R]; 0: done) of request r: sets ``lens``, and takes back
        the pages behind them and, with ``window``, those before what the next token sees."""
        self._lens(lens, "lens")
        if window < 0:
            raise _invalid("window must be >= 0 (0: none)")
        if window > 1 << 30:  # the library's limit, checked here: a larger one does not reach it whole
            raise Gemma4Error(Status.UNSUPPORTED_CONFIG, "window exceeds 2^30 (0: none)")
        _on(self._device, (lens,), ())
        status = self._lib.gemma4_kv_release(self._ref, lens.data_ptr(), window, qmm._stream_ptr(stream, self._device))
        if status != 0:
            qmm.check(status, self._lib)

    def _lens(self, t, what: str):
        _int32(t, what, 1)
        if t.shape[0] != self.requests:
            raise _invalid(f"{what} must have {self.requests} entries")
