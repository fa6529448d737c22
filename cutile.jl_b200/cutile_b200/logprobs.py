"""Log probabilities of given tokens, entropies and the most probable alternatives of rows of logits, with their gradient.

Logits (V, T) are torch [T, V]: T rows of V contiguous elements in f32, f16 or bf16 with any row stride; results per row are [T], lists of
alternatives (top, T) are torch [T, top].  Ids are 1-based, 0 is no token.
"""
from typing import NamedTuple, Optional

import torch

from . import _host, _lib
from ._util import dense, dtype_code, gradient_of, handles, ids_bits, ptr, rows


class TokenLogprobs(NamedTuple):
    """Results of token_logprobs, f32; None for what was not asked for.  The three vectors may share an allocation."""
    logprobs: Optional[torch.Tensor]      # [T] of the given tokens
    entropy: Optional[torch.Tensor]       # [T]
    lse: torch.Tensor                     # [T] log of the sum of exponentials
    top_logprobs: Optional[torch.Tensor]  # [T, top], descending
    top_ids: Optional[torch.Tensor]       # [T, top] int32


def token_logprobs(logits, tokens=None, top=0, temperature=1.0, entropy=True, **hints):
    """Log probabilities under softmax(logits / temperature) of `tokens` ([T] int32 or int64; a row with token 0 is padding:
    it is not read and its results are 0), the entropies, and the `top` (up to 32) most probable elements of every row, equal ones
    by ascending id.  Returns a TokenLogprobs."""
    if not hints:
        r = _host.token_logprobs(logits, tokens, top, temperature, entropy)
        if r is not None:
            return TokenLogprobs._make(r)
    ctx, stream = handles(logits, hints)
    ld, T, V = rows(logits, "logits")

    def new(*shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device=logits.device)
    top = int(top)
    r = TokenLogprobs(None if tokens is None else new(T), new(T) if entropy else None, new(T), new(T, max(top, 0)) if top else None,
                      new(T, max(top, 0), dtype=torch.int32) if top else None)
    bits = 64 if tokens is None else ids_bits(dense(tokens, (T,), "tokens", logits), "tokens")
    _lib.check(_lib.lib.ctb_token_logprobs(ctx, stream, ptr(logits), ptr(tokens), bits, ptr(r.logprobs), ptr(r.entropy), ptr(r.lse),
                                           ptr(r.top_logprobs), ptr(r.top_ids), V, T, ld, top, float(temperature), dtype_code(logits)))
    return r


def token_logprobs_bwd(logits, tokens, lse, entropy, d_logprobs=None, d_entropy=None, top_ids=None, d_top_logprobs=None, temperature=1.0,
                       out=None, **hints):
    """Gradient of the logits, [T, V] in their type, from the gradients of the results of token_logprobs (any of them None) and
    its lse, entropy (needed with d_entropy) and top_ids (needed with d_top_logprobs).  `out` may be the logits themselves."""
    if not hints:
        r = _host.token_logprobs_bwd(logits, tokens, lse, entropy, d_logprobs, d_entropy, top_ids, d_top_logprobs, temperature, out)
        if r is not None:
            return r if out is None else out
    ctx, stream = handles(logits, hints)
    ld, T, V = rows(logits, "logits")
    bits = 64 if tokens is None else ids_bits(dense(tokens, (T,), "tokens", logits), "tokens")
    top = 0
    if d_top_logprobs is not None:
        if top_ids is None or top_ids.dim() != 2:
            raise _lib.CtbError(_lib.BAD_ARG, "token_logprobs_bwd: d_top_logprobs needs top_ids of shape [T, top]")
        top = top_ids.shape[1]
        dense(top_ids, (T, top), "top_ids", logits, torch.int32)
        dense(d_top_logprobs, (T, top), "d_top_logprobs", logits, torch.float32)
    if d_entropy is not None and entropy is None:
        raise _lib.CtbError(_lib.BAD_ARG, "token_logprobs_bwd: d_entropy needs entropy")
    for t, what in ((lse, "lse"), (entropy, "entropy"), (d_logprobs, "d_logprobs"), (d_entropy, "d_entropy")):
        if t is not None:
            dense(t, (T,), what, logits, torch.float32)
    out, ld_out = gradient_of(logits, out)
    _lib.check(_lib.lib.ctb_token_logprobs_bwd(ctx, stream, ptr(out), ptr(logits), ptr(tokens), bits, ptr(lse), ptr(entropy),
                                               ptr(d_logprobs), ptr(d_entropy), ptr(top_ids if top else None),
                                               ptr(d_top_logprobs if top else None), V, T, ld_out, ld, top, float(temperature),
                                               dtype_code(logits)))
    return out
