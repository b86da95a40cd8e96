"""Tokens from logits, and drafted tokens checked against them, on libgemma4_qmm.

* :func:`sample` — a token from each row of the head's logits;
* :func:`verify_drafts` — which of a batch's drafted tokens stand, so that the tokens kept are
  distributed as the target's own, and the token that follows them.

Random numbers are inputs (uniforms of the caller's generator), so a call has one answer, and
a captured graph draws anew when they are refilled.  Probabilities and their sums are 64 bits
wide.  (The reference drafts and checks greedily, ``crates/gemma4d-engine/src/lib.rs:175-300``:
a temperature of 0 here.)  Errors surface as :class:`~helios_amd.qmm.Gemma4Error`.
"""

from __future__ import annotations

import ctypes
import math

from . import qmm
from .attention import _int32, _invalid, _new, _on

_u32, _u64, _vp, _f32 = ctypes.c_uint32, ctypes.c_uint64, ctypes.c_void_p, ctypes.c_float


class _Logits(ctypes.Structure):
    _fields_ = [("x_dev", _vp), ("stride", _u64), ("dtype", _u32), ("softcap", _f32)]


def _number(v, what: str, zero: str):
    """A finite v >= 0 that is not 0 for the library, which takes float32, alone."""
    v = float(v)
    if not 0.0 <= v < math.inf:
        raise _invalid(f"{what} must be finite and >= 0 (0: {zero})")
    if 0.0 < v <= 2.0 ** -150:
        raise _invalid(f"{what} must be 0 ({zero}) or over 2^-150: a smaller one is 0 in float32")
    return v


def _logits(t, what: str, softcap):
    import torch

    kind = {torch.bfloat16: 0, torch.float32: 1}.get(t.dtype) if isinstance(t, torch.Tensor) else None
    if kind is None or t.dim() != 2 or not t.is_cuda:
        raise _invalid(f"{what} must be a bfloat16 or float32 tensor [rows, vocab] on the GPU")
    rows, vocab = t.shape
    if vocab > 1 and t.stride(1) != 1:
        raise _invalid(f"{what} must have each row contiguous")
    softcap = _number(softcap, f"{what}' softcap", "none")
    # a single row's stride says nothing
    return _Logits(t.data_ptr(), t.stride(0) if rows > 1 else vocab, kind, softcap)


def _floats(t, what: str, shape):
    import torch

    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or not t.is_cuda or tuple(t.shape) != shape or not t.is_contiguous():
        raise _invalid(f"{what} must be a contiguous float32 tensor {list(shape)} on the GPU")
    return t


def _temperature(t, requests: int):
    """(number for all, tensor or None)."""
    import torch

    if isinstance(t, torch.Tensor):
        return 0.0, _floats(t, "temperature", (requests,))
    return _number(t, "temperature", "greedy"), None


def _ptr(t):
    return None if t is None else t.data_ptr()


def sample(logits, uniforms, temperature=1.0, softcap: float = 0.0, stream=None):
    """A token from softmax(logits / temperature) of each row of logits [rows, vocab], bf16 or
    float32: the first whose cumulative probability exceeds uniforms[row] (float32 [rows] in
    [0, 1)); the first largest logit where the temperature (a number or float32 [rows]) is 0.
    ``softcap`` puts cap * tanh(x / cap) in the logits' place.  Logits of -inf are never taken;
    int32 [rows], -1 where nothing can be."""
    import torch

    lib = qmm.load_library()
    of = _logits(logits, "logits", softcap)
    rows, vocab = logits.shape
    _floats(uniforms, "uniforms", (rows,))
    heat, heats = _temperature(temperature, rows)
    device = logits.get_device()
    _on(device, (uniforms, heats), ())
    out = _new(logits, (rows,), torch.int32, stream)
    status = lib.gemma4_sample(ctypes.byref(of), rows, vocab, uniforms.data_ptr(), heat, _ptr(heats), out.data_ptr(), qmm._stream_ptr(stream, device))
    if status != 0:
        qmm.check(status, lib)
    return out


def verify_drafts(logits, tokens, query_starts, uniforms, temperature=1.0, draft_logits=None, softcap: float = 0.0,
                  draft_softcap: float = 0.0, stream=None):
    """Which drafts stand.  Request r's rows are query_starts[r] up to query_starts[r + 1] (int32
    [R + 1], as a :class:`~helios_amd.attention.KVBatch`'s) of logits [rows, vocab] and tokens
    (int32 [rows], those fed: the last known one, then its drafts).  The draft in row i + 1 stands
    while uniforms[i, 0] * q < p, its probabilities under row i of draft_logits and of logits
    (q = 1 without draft_logits); at the first that falls a token is drawn from max(p - q, 0) by
    uniforms[i, 1], and if all stand from the last row's p.  Temperature (a number or float32 [R])
    0: p and q are 1 at the first largest logit.

    Returns (out int32 [rows], accepted int32 [R]): from each request's first row on its accepted
    drafts and the drawn token, accepted + 1 in all, then -1."""
    import torch

    lib = qmm.load_library()
    of = _logits(logits, "logits", softcap)
    rows, vocab = logits.shape
    draft = None
    if draft_logits is not None:
        draft = _logits(draft_logits, "draft_logits", draft_softcap)
        if draft_logits.shape != logits.shape or draft_logits.dtype != logits.dtype:
            raise _invalid("draft_logits must have logits' shape and type")
    _int32(tokens, "tokens", 1)
    _int32(query_starts, "query_starts", 1)
    requests = query_starts.shape[0] - 1
    if tokens.shape[0] != rows:
        raise _invalid(f"tokens must have {rows} entries")
    if requests < 1:
        raise _invalid("query_starts must have an entry more than there are requests, one at least")
    _floats(uniforms, "uniforms", (rows, 2))
    heat, heats = _temperature(temperature, requests)
    device = logits.get_device()
    _on(device, (draft_logits, tokens, query_starts, uniforms, heats), ())
    out = _new(logits, (rows,), torch.int32, stream)
    accepted = _new(logits, (requests,), torch.int32, stream)
    if rows == 0:
        with qmm._made_on(stream):
            return out, accepted.zero_()
    status = lib.gemma4_verify_drafts(ctypes.byref(of), None if draft is None else ctypes.byref(draft), tokens.data_ptr(),
                                      query_starts.data_ptr(), requests, rows, vocab, uniforms.data_ptr(), heat, _ptr(heats),
                                      out.data_ptr(), accepted.data_ptr(), qmm._stream_ptr(stream, device))
    if status != 0:
        qmm.check(status, lib)
    return out, accepted
