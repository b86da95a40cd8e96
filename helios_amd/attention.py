"""Attention over a paged key/value cache, on libgemma4_qmm.

What a layer does between its q|k|v and o projections, for a batch of requests with one
or many new tokens each (the reference: ``fast::rms_norm``, ``fast::rope`` and
``fast::scaled_dot_product_attention`` around a cache per request,
``native/gemma4_mlx/src/native_model.cc:808-881``):

* :func:`qk_norm_rope` — RMS norm of each query and key head and the position rotation;
* :meth:`PagedKVCache.append` — the same for a batch's keys, stored with the values into
  the cache's pages (and for its queries, in the same launch);
* :meth:`PagedKVCache.attend` — causal attention of the batch's queries over the cache.

One layer of a decoding step, from the fused projection's rows to o's input::

    cache = PagedKVCache(k_pages, v_pages)                  # kept, one per layer
    batch = KVBatch(query_starts, kv_lens, block_tables)    # kept; updated on the device
    qkv = qkv_proj(x)
    q, k, v = (qkv[:, a:b].unflatten(1, (-1, 256)) for a, b in ((0, 4096), (4096, 6144), (6144, 8192)))
    q = cache.append(k, v, batch, rope=rope, k_norm=k_norm, v_norm=v_norm, q=q, q_norm=q_norm)
    y = o_proj(cache.attend(q, batch, scale=1.0, window=1024).flatten(1))

Tensors are bf16 on the GPU (pages may be ``float8_e4m3fn``).  The device arrays of a
batch are read when the kernels run, so a captured graph follows what is written to them.
With ``stream`` a call runs there instead of on torch's current stream: its inputs must be
ready on that stream and stay until it is done with them, and the outputs it makes belong to
that stream's memory (use them elsewhere after waiting for it).
Errors surface as :class:`~helios_amd.qmm.Gemma4Error`; there is no fallback.
"""

from __future__ import annotations

import ctypes
import struct

from . import qmm
from .qmm import Gemma4Error, Status

KV_BF16 = 0
KV_E4M3 = 1

_u32, _u64, _vp = ctypes.c_uint32, ctypes.c_uint64, ctypes.c_void_p


class _Pages(ctypes.Structure):
    _fields_ = [("k_dev", _vp), ("v_dev", _vp), ("page_stride", _u64), ("token_stride", _u64), ("head_stride", _u64),
                ("num_pages", _u32), ("page_size", _u32), ("kv_heads", _u32), ("head_dim", _u32), ("dtype", _u32),
                ("k_scale", ctypes.c_float), ("v_scale", ctypes.c_float)]


class _Scales(ctypes.Structure):
    _fields_ = [("k_dev", _vp), ("v_dev", _vp), ("page_stride", _u64), ("head_stride", _u64), ("block", _u32)]


class _Batch(ctypes.Structure):
    _fields_ = [("query_starts_dev", _vp), ("kv_lens_dev", _vp), ("block_tables_dev", _vp), ("requests", _u32),
                ("tokens", _u32), ("pages_per_request", _u32), ("table_stride", _u32)]


class _Rope(ctypes.Structure):
    _fields_ = [("inv_freq_dev", _vp), ("pairs", _u32), ("distance", _u32)]


class _Heads(ctypes.Structure):
    _fields_ = [("x_dev", _vp), ("out_dev", _vp), ("weight_dev", _vp), ("x_stride", _u64), ("out_stride", _u64),
                ("count", _u32), ("norm", _u32), ("eps", ctypes.c_float)]


# _Batch and _Heads as bytes: packing takes a quarter of a ctypes structure's time, and these
# two are made for every call (bytes pass as the pointers the calls declare)
_pack_batch = struct.Struct("PPPIIII").pack
_pack_heads = struct.Struct("PPPQQIIf4x").pack


def _invalid(message: str):
    return Gemma4Error(Status.INVALID_ARGUMENT, message)


def _int32(t, what: str, dims: int):
    import torch

    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.dim() != dims or not t.is_cuda:
        raise _invalid(f"{what} must be a {dims}-dimensional int32 tensor on the GPU")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise _invalid(f"{what} must have its last dimension contiguous")
    return t


def _heads_tensor(t, what: str, head_dim: int | None = None):
    """The shape and row stride of a [rows, heads, head_dim] bf16 tensor whose heads lie next
    to each other in a row."""
    import torch

    if not isinstance(t, torch.Tensor) or t.dtype != torch.bfloat16 or t.dim() != 3 or not t.is_cuda:
        raise _invalid(f"{what} must be a bfloat16 tensor [rows, heads, head_dim] on the GPU")
    shape = t.shape
    rows, heads, dim = shape
    row_stride, head_stride, one = t.stride()
    if head_dim is not None and dim != head_dim:
        raise _invalid(f"{what} has head_dim {dim}, expected {head_dim}")
    if one != 1 or (heads > 1 and head_stride != dim):
        raise _invalid(f"{what} must have its heads contiguous within a row")
    # a single row's stride says nothing
    return shape, row_stride if rows > 1 else heads * dim


def _on(index, tensors, held):
    """Every tensor, and what the rotations, norms and batches hold, must live on GPU `index`,
    which must be the current device."""
    import torch

    for t in tensors:
        if t is not None and t.get_device() != index:
            raise _invalid("all tensors must be on one device")
    for h in held:
        if h is not None and h._device not in (index, None):
            raise _invalid(f"a {type(h).__name__} is on cuda:{h._device}, the other tensors on cuda:{index}")
    if torch.cuda.current_device() != index:
        raise _invalid(f"the tensors are on cuda:{index}, which is not the current device")


class Rope:
    """Rotation by ``position * inv_freq[i]`` of elements (i, i + distance) of each head,
    i < len(inv_freq); the others pass.  ``distance`` defaults to len(inv_freq) (the first
    2 len(inv_freq) elements, in halves); head_dim / 2 pairs across the whole head, and 1
    means adjacent pairs (2i, 2i + 1)."""

    def __init__(self, inv_freq, distance: int | None = None):
        import torch

        if not isinstance(inv_freq, torch.Tensor) or inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_cuda:
            raise _invalid("inv_freq must be a one-dimensional float32 tensor on the GPU")
        self.inv_freq = inv_freq.contiguous()
        self._device = inv_freq.get_device()
        pairs = inv_freq.numel()
        self.distance = pairs if distance is None else int(distance)
        if not 0 <= self.distance < 1 << 32:  # the rest is checked with the head_dim
            raise _invalid("distance must be positive and fit 32 bits")
        self._c = _Rope(self.inv_freq.data_ptr(), pairs, self.distance)
        self._ref = ctypes.byref(self._c)


class HeadNorm:
    """RMS norm over each head: x / sqrt(mean(x^2) + eps) * weight (None: ones)."""

    def __init__(self, weight=None, eps: float = 1e-6):
        import torch

        if weight is not None:
            if not isinstance(weight, torch.Tensor) or weight.dtype != torch.bfloat16 or weight.dim() != 1 or not weight.is_cuda:
                raise _invalid("a head norm's weight must be a one-dimensional bfloat16 tensor on the GPU")
            weight = weight.contiguous()
        self.weight = weight
        self.eps = float(eps)
        self.size = 0 if weight is None else weight.numel()
        self._ptr = 0 if weight is None else weight.data_ptr()
        self._device = None if weight is None else weight.get_device()  # None: on any


class KVBatch:
    """The new tokens of a batch: request r's rows are query_starts[r] up to
    query_starts[r + 1] of q, k and v, the last at position kv_lens[r] - 1; position p
    lies in page block_tables[r, p // page_size] (an entry outside the cache's pages is an
    absent page).  int32 GPU tensors [R + 1], [R] and [R, pages]; they are kept, not
    copied, and read when the kernels run.  Rows past query_starts[-1] are padding."""

    def __init__(self, query_starts, kv_lens, block_tables):
        self.query_starts = _int32(query_starts, "query_starts", 1)
        self.kv_lens = _int32(kv_lens, "kv_lens", 1)
        self.block_tables = _int32(block_tables, "block_tables", 2)
        n = kv_lens.shape[0]
        if query_starts.shape[0] != n + 1 or block_tables.shape[0] != n:
            raise _invalid(f"query_starts must have one entry more than kv_lens and block_tables as many rows ({n})")
        width = block_tables.shape[1]
        stride = block_tables.stride(0) if n > 1 else width  # a single row's stride says nothing
        if stride < width:
            raise _invalid("block_tables' rows overlap")
        self.requests = n
        self._device = kv_lens.get_device()
        if query_starts.get_device() != self._device or block_tables.get_device() != self._device:
            raise _invalid("query_starts, kv_lens and block_tables must be on one device")
        self._fields = (query_starts.data_ptr(), kv_lens.data_ptr(), block_tables.data_ptr(), n)
        self._table = (width, stride)
        self._packed = (-1, b"")

    def _struct(self, tokens: int):
        # replaced as a whole: two threads may use one batch with different row counts
        packed = self._packed
        if packed[0] != tokens:
            packed = self._packed = (tokens, _pack_batch(*self._fields, tokens, *self._table))
        return packed[1]


def _heads(t, shape, stride, norm, out, out_stride):
    if norm is None:
        return _pack_heads(t.data_ptr(), out, 0, stride, out_stride, shape[1], 0, 0.0)
    if norm.weight is not None and norm.size != shape[2]:
        raise _invalid(f"the norm's weight has {norm.size} values, head_dim is {shape[2]}")
    return _pack_heads(t.data_ptr(), out, norm._ptr, stride, out_stride, shape[1], 1, norm.eps)


def _new(like, shape, dtype, stream):
    """A tensor that `stream` writes, from its memory: that of torch's current stream may still
    be in use there."""
    import torch

    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    with torch.cuda.stream(stream):
        return like.new_empty(shape, dtype=dtype)


def _output(out, shape, like, what: str, stream):
    """(tensor, row stride) of an output of `shape` that `stream` writes."""
    if out is None:
        return _new(like, shape, None, stream), shape[1] * shape[2]
    got, stride = _heads_tensor(out, what)
    if got != shape:
        raise _invalid(f"{what} has the wrong shape")
    return out, stride


def set_attention_kernel(kernel: int) -> int:
    """Pins the attention kernel for this process: 0 (the default) chooses by the rows of each
    request and the work of the call, 1 the 128-row tiles for every request with rows enough,
    2 the 16-row tiles only.  Returns the previous setting."""
    if int(kernel) not in (0, 1, 2):
        raise ValueError(f"kernel must be 0, 1 or 2, got {kernel}")
    return int(qmm.load_library().gemma4_kv_set_attention_kernel(int(kernel)))


def qk_norm_rope(q, k, positions, rope=None, q_norm=None, k_norm=None, out_q=None, out_k=None, stream=None):
    """Norms (where given) and rotates the heads of q [rows, heads, head_dim] and, unless
    None, of k, in one launch.  ``positions``: int32 [rows].  Returns (q, k) in new
    tensors, or in ``out_q`` and ``out_k`` (which may be q and k themselves)."""
    lib = qmm.load_library()
    shape, q_stride = _heads_tensor(q, "q")
    rows, _, head_dim = shape
    if k is not None:
        k_shape, k_stride = _heads_tensor(k, "k", head_dim)
        if k_shape[0] != rows:
            raise _invalid("q and k must have the same rows")
    if rope is not None:
        _int32(positions, "positions", 1)
        if positions.shape[0] != rows:
            raise _invalid(f"positions must have {rows} entries")
    else:
        positions = None
    out_q, out_stride = _output(out_q, shape, q, "out_q", stream)
    of_q = _heads(q, shape, q_stride, q_norm, out_q.data_ptr(), out_stride)
    of_k = None
    if k is not None:
        out_k, out_stride = _output(out_k, k_shape, k, "out_k", stream)
        of_k = _heads(k, k_shape, k_stride, k_norm, out_k.data_ptr(), out_stride)
    else:
        out_k = None
    _on(q.get_device(), (k, positions, out_q, out_k), (rope, q_norm, k_norm))
    status = lib.gemma4_qk_norm_rope(of_q, of_k, None if rope is None else rope._ref,
                                     None if positions is None else positions.data_ptr(), rows, head_dim,
                                     qmm._stream_ptr(stream))
    if status != 0:
        qmm.check(status, lib)
    return out_q, out_k


def _block_scales(k_scale, v_scale, k, h: int, s: int):
    """The blocks' scales of pages k, whose dims h and s are the heads and the slots."""
    import torch

    kinds = (torch.uint8, torch.float8_e8m0fnu)
    for t in (k_scale, v_scale):
        if not isinstance(t, torch.Tensor) or t.dim() != 3 or not t.is_cuda or t.dtype not in kinds:
            raise _invalid("block scales must be two float8_e8m0fnu (or uint8) tensors [pages, kv_heads, blocks] on the GPU")
    if k.dtype != torch.float8_e4m3fn:
        raise _invalid("block scales belong to float8_e4m3fn pages")
    if k_scale.shape != v_scale.shape or k_scale.stride() != v_scale.stride() or k_scale.device != k.device or v_scale.device != k.device:
        raise _invalid("the block scales must have the same shape and strides, and the pages' device")
    pages, heads, per = k_scale.shape
    if pages != k.shape[0] or heads != k.shape[h] or per == 0 or k.shape[s] % per:
        raise _invalid(f"block scales must be [{k.shape[0]}, {k.shape[h]}, a divisor of {k.shape[s]}]")
    if per > 1 and k_scale.stride(2) != 1:
        raise _invalid("a page's block scales must lie side by side")
    # the stride of an axis of one says nothing
    strides = [k_scale.stride(i) if k_scale.shape[i] > 1 else per for i in (0, 1)]
    return _Scales(k_scale.data_ptr(), v_scale.data_ptr(), *strides, k.shape[s] // per)


class PagedKVCache:
    """Keys and values of many requests in pages: two tensors [pages, kv_heads, page_size,
    head_dim] (``layout`` "phsd") or [pages, page_size, kv_heads, head_dim] ("pshd"), bf16
    or float8_e4m3fn, of equal strides.  e4m3 pages hold value / scale: one scale for all, or,
    with float8_e8m0fnu (or uint8) tensors [pages, kv_heads, page_size // block] of equal
    strides, a power of two for each ``block`` consecutive tokens (16 to 256) of a page and
    KV head, which ``append`` sets from the values it stores.  Tokens that are dropped again (drafts
    that fell) leave a scale that they raised, and the tokens before them in the block rounded by
    it.  The tensors are the caller's;
    ``PagedKVCache.allocate`` makes them."""

    def __init__(self, k, v, k_scale=1.0, v_scale=1.0, layout: str = "phsd"):
        import torch

        kinds = {torch.bfloat16: KV_BF16, torch.float8_e4m3fn: KV_E4M3}
        for t, what in ((k, "k"), (v, "v")):
            if not isinstance(t, torch.Tensor) or t.dim() != 4 or not t.is_cuda or t.dtype not in kinds:
                raise _invalid(f"{what} must be a 4-dimensional bfloat16 or float8_e4m3fn tensor on the GPU")
        if layout not in ("phsd", "pshd"):
            raise _invalid("layout must be 'phsd' or 'pshd'")
        if k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype or k.device != v.device:
            raise _invalid("k and v must have the same shape, strides, dtype and device")
        if k.numel() == 0 or k.stride(3) != 1:
            raise _invalid("k and v must not be empty and must have head_dim contiguous")
        self.k, self.v = k, v
        h, s = (1, 2) if layout == "phsd" else (2, 1)
        self._scales = None
        if isinstance(k_scale, torch.Tensor) or isinstance(v_scale, torch.Tensor):
            self._scales = _block_scales(k_scale, v_scale, k, h, s)
            self._scales_ref = ctypes.byref(self._scales)
            self.k_scale, self.v_scale = k_scale, v_scale
        else:
            self.k_scale, self.v_scale = float(k_scale), float(v_scale)
        self.kv_heads, self.page_size, self.head_dim = k.shape[h], k.shape[s], k.shape[3]
        self.num_pages = k.shape[0]
        self.device = k.device
        self._device = k.get_device()
        self._lib = qmm.load_library()
        # the stride of an axis of one says nothing
        strides = [k.stride(i) if k.shape[i] > 1 else self.head_dim for i in (0, s, h)]
        self._c = _Pages(k.data_ptr(), v.data_ptr(), *strides, self.num_pages, self.page_size, self.kv_heads,
                         self.head_dim, kinds[k.dtype], *((1.0, 1.0) if self._scales else (self.k_scale, self.v_scale)))
        self._ref = ctypes.byref(self._c)

    @classmethod
    def allocate(cls, num_pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=None, k_scale: float = 1.0,
                 v_scale: float = 1.0, device="cuda", scale_block: int = 0):
        """A cache of new, uninitialised pages (unused slots are never read into a result).  With
        ``scale_block`` (float8_e4m3fn pages) each block of so many tokens has a scale."""
        import torch

        shape = (num_pages, kv_heads, page_size, head_dim)
        k, v = (torch.empty(shape, dtype=dtype or torch.bfloat16, device=device) for _ in range(2))
        if scale_block:
            if scale_block < 0 or page_size % scale_block:
                raise _invalid("scale_block must divide page_size")
            if k_scale != 1.0 or v_scale != 1.0:
                raise _invalid("k_scale and v_scale belong to caches without scale_block")
            k_scale, v_scale = (torch.empty((num_pages, kv_heads, page_size // scale_block), dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu)
                                for _ in range(2))
        return cls(k, v, k_scale, v_scale)

    def append(self, k, v, batch: KVBatch, rope=None, k_norm=None, v_norm=None, q=None, q_norm=None, out_q=None,
               stream=None):
        """Stores the batch's k and v [rows, kv_heads, head_dim]: k normed and rotated, v
        normed, each where given.  k and v may be the same tensor.  With q [rows, heads,
        head_dim] the same launch norms and rotates it; returns it (or None), in a new tensor or in
        ``out_q``, which may be q itself but not lie over k or v.  With block scales the cache's k and
        v, and their scales, must not share memory."""
        shape, k_stride = _heads_tensor(k, "k", self.head_dim)
        v_shape, v_stride = (shape, k_stride) if v is k else _heads_tensor(v, "v", self.head_dim)
        rows = shape[0]
        if v_shape != shape or shape[1] != self.kv_heads:
            raise _invalid(f"k and v must be [rows, {self.kv_heads}, {self.head_dim}]")
        of_q = None
        if q is not None:
            q_shape, q_stride = _heads_tensor(q, "q", self.head_dim)
            if q_shape[0] != rows:
                raise _invalid("q, k and v must have the same rows")
            out_q, out_stride = _output(out_q, q_shape, q, "out_q", stream)
            of_q = _heads(q, q_shape, q_stride, q_norm, out_q.data_ptr(), out_stride)
        else:
            out_q = None
        _on(self._device, (k, v, q, out_q), (batch, rope, k_norm, v_norm, q_norm))
        args = (batch._struct(rows), of_q, _heads(k, shape, k_stride, k_norm, 0, 0), _heads(v, v_shape, v_stride, v_norm, 0, 0),
                None if rope is None else rope._ref, qmm._stream_ptr(stream))
        if self._scales is None:
            status = self._lib.gemma4_kv_append(self._ref, *args)
        else:
            status = self._lib.gemma4_kv_append_scaled(self._ref, self._scales_ref, *args)
        if status != 0:
            qmm.check(status, self._lib)
        return out_q

    def attend(self, q, batch: KVBatch, scale: float | None = None, window: int = 0, out=None, return_lse: bool = False,
               stream=None):
        """softmax(scale q . K) V of q [rows, heads, head_dim] over the keys each row sees:
        those up to its own position and, with ``window``, the last ``window`` of them.
        ``scale`` defaults to head_dim ** -0.5.  Returns out (a row with no visible key is
        zeros), and with ``return_lse`` also the log-sum-exp, float32 [rows, heads]."""
        import torch

        shape, q_stride = _heads_tensor(q, "q", self.head_dim)
        rows, heads, _ = shape
        if window < 0:
            raise _invalid("window must be >= 0 (0: none)")
        if window > 1 << 30:  # the library's limit, checked here: a larger one does not reach it whole
            raise Gemma4Error(Status.UNSUPPORTED_CONFIG, "window exceeds 2^30 (0: none)")
        out, out_stride = _output(out, shape, q, "out", stream)
        lse = _new(q, (rows, heads), torch.float32, stream) if return_lse else None
        _on(self._device, (q, out), (batch,))
        args = (batch._struct(rows), q.data_ptr(), q_stride, heads, self.head_dim ** -0.5 if scale is None else scale, window,
                out.data_ptr(), out_stride, None if lse is None else lse.data_ptr(), qmm._stream_ptr(stream))
        if self._scales is None:
            status = self._lib.gemma4_kv_attention(self._ref, *args)
        else:
            status = self._lib.gemma4_kv_attention_scaled(self._ref, self._scales_ref, *args)
        if status != 0:
            qmm.check(status, self._lib)
        return (out, lse) if return_lse else out
