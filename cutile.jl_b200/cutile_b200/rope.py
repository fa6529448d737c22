"""Rotary positions: queries and keys turned pair by pair by an angle that grows with their token's position, and the gradient.

Queries (D, Heads, SeqLen, Batch) are torch [Batch, SeqLen, Heads, D], or [tokens, Heads, D], with any strides but contiguous heads (the
arrays of `fmha` are passed as Q.transpose(1, 2)); keys the same with heads of their own.  Positions are [Batch, SeqLen] or [tokens].
"""
import ctypes as C
import math

import torch

from . import _host, _lib
from ._util import dense, dtype_code, handles, ids_bits, ptr


def rope_frequencies(rotary_dim, base=10000.0, scaling=None, factor=1.0, original_length=None, low=1.0, high=4.0):
    """Angles per position of the rotary_dim / 2 pairs, f64 on the host: base ** (-2 i / rotary_dim), scaled for contexts longer than a
    model was trained for (by `factor`):
      "linear"  all of them divided by the factor;
      "base"    by a base that is larger by factor ** (rotary_dim / (rotary_dim - 2)): the first pair as it is, the last divided by the factor;
      "parts"   pairs that make `high` turns or more over the original length as they are, those with `low` or fewer divided by the
                factor, and in between by the share of the way."""
    if int(rotary_dim) != rotary_dim or rotary_dim <= 0 or rotary_dim % 2:
        raise _lib.CtbError(_lib.BAD_ARG, f"rotary_dim must be even and positive, got {rotary_dim}")
    if not (math.isfinite(base) and base > 0 and math.isfinite(factor) and factor > 0):
        raise _lib.CtbError(_lib.BAD_ARG, "base and factor must be positive numbers")
    if scaling not in (None, "linear", "base", "parts"):
        raise _lib.CtbError(_lib.BAD_ARG, f"scaling must be None, 'linear', 'base' or 'parts', got {scaling!r}")
    share = torch.arange(0, int(rotary_dim), 2, dtype=torch.float64) / rotary_dim
    if scaling == "base":
        if rotary_dim <= 2:
            raise _lib.CtbError(_lib.BAD_ARG, "scaling by the base needs more than one pair")
        return (base * factor ** (rotary_dim / (rotary_dim - 2))) ** -share
    f = base ** -share
    if scaling == "linear":
        return f / factor
    if scaling == "parts":
        if original_length is None or not original_length > 0 or not high > low:
            raise _lib.CtbError(_lib.BAD_ARG, "scaling by parts needs original_length > 0 and high > low")
        keep = ((original_length * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        return f * keep + f / factor * (1 - keep)
    return f


def _tokens(t, what):
    """A [.., Heads, D] tensor as one of [batch, seq, heads, D]."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise _lib.CtbError(_lib.BAD_ARG, "expected a CUDA tensor (device array); host arrays are not accepted")
    if t.dim() not in (3, 4) or (t.shape[-1] > 1 and t.stride(-1) != 1):
        raise _lib.CtbError(_lib.BAD_ARG, f"{what}: expected [Batch, SeqLen, Heads, D] or [tokens, Heads, D] with contiguous heads")
    return t if t.dim() == 4 else t.unsqueeze(0)


def _like(out, x, what):
    if out is None:
        return torch.empty_like(x)
    if not isinstance(out, torch.Tensor) or out.device != x.device or out.shape != x.shape or out.dtype != x.dtype:
        raise _lib.CtbError(_lib.BAD_ARG, f"{what} must have the shape, type and device of its input")
    return out


def _rope(who, q, k, positions, frequencies, interleaved, scale, out_q, out_k, inverse, hints):
    if not hints:
        r = _host.rope(q, k, positions, frequencies, interleaved, scale, out_q, out_k, inverse)
        if r is not None:
            return r
    ctx, stream = handles(q, hints)
    q4 = _tokens(q, "q")
    shape = tuple(q.shape[:-2])
    if k is not None:
        k4 = _tokens(k, "k")
        if k.device != q.device or k.dtype != q.dtype or tuple(k.shape[:-2]) != shape or k.shape[-1] != q.shape[-1]:
            raise _lib.CtbError(_lib.BAD_ARG, f"{who}: k must have the tokens, head size, type and device of q")
    bits = ids_bits(dense(positions, shape, "positions", q), "positions")
    if not isinstance(frequencies, torch.Tensor) or frequencies.dim() != 1:
        raise _lib.CtbError(_lib.BAD_ARG, "frequencies: expected a tensor of one dimension")
    dense(frequencies, frequencies.shape, "frequencies", q, torch.float64)
    oq = _like(out_q, q, "out_q")
    ok = None if k is None else _like(out_k, k, "out_k")
    strides = list(_tokens(oq, "out_q").stride()[:3]) + list(q4.stride()[:3])
    if k is not None:
        strides += list(_tokens(ok, "out_k").stride()[:3]) + list(k4.stride()[:3])
    _lib.check(_lib.lib.ctb_rope(ctx, stream, ptr(oq), ptr(q), ptr(ok), ptr(k), ptr(positions), bits, ptr(frequencies), q4.shape[0], q4.shape[1],
                                 q4.shape[2], 0 if k is None else k4.shape[2], q4.shape[3], 2 * frequencies.shape[0],
                                 (C.c_int64 * 12)(*strides), int(bool(interleaved)), int(inverse), float(scale), dtype_code(q)))
    return oq, ok


def rope_fwd(q, k, positions, frequencies, interleaved=False, scale=1.0, out_q=None, out_k=None, **hints):
    """Turns pair i of every head of a token at position n by n * frequencies[i]: (x1, x2) -> scale * (x1 cos - x2 sin, x1 sin + x2
    cos).  Pairs are elements (2 i, 2 i + 1) with `interleaved`, else (i, i + len(frequencies)); elements behind the last pair are copied.
    q and k (or None) in f32, f16 or bf16; positions int32 or int64, frequencies f64 on the device (rope_frequencies).  out_q and out_k
    may be q and k.  Returns (q, k) turned."""
    return _rope("rope_fwd", q, k, positions, frequencies, interleaved, scale, out_q, out_k, False, hints)


def rope_bwd(d_q, d_k, positions, frequencies, interleaved=False, scale=1.0, out_q=None, out_k=None, **hints):
    """Gradients of rope_fwd's q and k from the gradients of its results: a turn by the opposite angles.  Options as there."""
    return _rope("rope_bwd", d_q, d_k, positions, frequencies, interleaved, scale, out_q, out_k, True, hints)
