"""Distillation of a student from a teacher's top logits, with its gradient.

The student's logits (V, T) are torch [T, V]: T rows of V contiguous elements in f32, f16 or bf16 with any row stride; a teacher's list
(entries, T) is torch [T, entries].  Ids are 1-based, 0 is an unused entry, and a row without used ones is padding.

Without teacher_lse the teacher's probabilities q are the softmax of its listed values / temperature, and the loss of a row is
sum q_j (log q_j - log p_j).  With teacher_lse [T], the log of the sum of exponentials of ALL its logits / temperature (what
`logprobs.token_logprobs` returns; 0 for a list of log probabilities), q_j = exp(value_j / temperature - teacher_lse), and what that
leaves of the teacher's probability stands against what the student gives to all ids that are not listed.
"""
import torch

from . import _host, _lib
from ._util import dense, dtype_code, gradient_of, handles, ids_bits, ptr, rows


def _teacher(logits, T, ids, values, lse):
    """(entries, id bits, type of the values) of a checked list."""
    if not isinstance(ids, torch.Tensor) or ids.dim() != 2:
        raise _lib.CtbError(_lib.BAD_ARG, "teacher_ids: expected a tensor of shape [T, entries]")
    entries = ids.shape[1]
    bits = ids_bits(dense(ids, (T, entries), "teacher_ids", logits), "teacher_ids")
    dense(values, (T, entries), "teacher_values", logits)
    if lse is not None:
        dense(lse, (T,), "teacher_lse", logits, torch.float32)
    return entries, bits, dtype_code(values)


def distill_fwd(logits, teacher_ids, teacher_values, teacher_lse=None, temperature=1.0, **hints):
    """Returns (loss [T] f32, saved [T, 8] f32); saved is what distill_bwd needs."""
    if not hints:
        r = _host.distill_fwd(logits, teacher_ids, teacher_values, teacher_lse, temperature)
        if r is not None:
            return r
    ctx, stream = handles(logits, hints)
    ld, T, V = rows(logits, "logits")
    entries, bits, values_code = _teacher(logits, T, teacher_ids, teacher_values, teacher_lse)
    loss = torch.empty(T, dtype=torch.float32, device=logits.device)
    saved = torch.empty((T, 8), dtype=torch.float32, device=logits.device)
    _lib.check(_lib.lib.ctb_distill_fwd(ctx, stream, ptr(logits), ptr(teacher_ids), bits, ptr(teacher_values), values_code,
                                        ptr(teacher_lse), ptr(loss), ptr(saved), V, T, ld, entries, float(temperature),
                                        dtype_code(logits)))
    return loss, saved


def distill_bwd(logits, teacher_ids, teacher_values, saved, d_loss, temperature=1.0, out=None, **hints):
    """Gradient of the logits, [T, V] in their type, from d_loss [T] f32 and what distill_fwd saved.  `out` may be the logits."""
    if not hints:
        r = _host.distill_bwd(logits, teacher_ids, teacher_values, saved, d_loss, temperature, out)
        if r is not None:
            return r if out is None else out
    ctx, stream = handles(logits, hints)
    ld, T, V = rows(logits, "logits")
    entries, bits, values_code = _teacher(logits, T, teacher_ids, teacher_values, None)
    dense(saved, (T, 8), "saved", logits, torch.float32)
    dense(d_loss, (T,), "d_loss", logits, torch.float32)
    out, ld_out = gradient_of(logits, out)
    _lib.check(_lib.lib.ctb_distill_bwd(ctx, stream, ptr(out), ptr(logits), ptr(teacher_ids), bits, ptr(teacher_values), values_code,
                                        ptr(saved), ptr(d_loss), V, T, ld_out, ld, entries, float(temperature), dtype_code(logits)))
    return out


def distill_fwd_bwd(logits, teacher_ids, teacher_values, d_loss, teacher_lse=None, temperature=1.0, out=None, **hints):
    """Loss and gradient in one call, for a d_loss [T] f32 that is known beforehand (the rows' weights); rows of 32 to 128 KB, or
    of up to 512 KB when there are many, are read once.  Returns (loss [T] f32, gradient [T, V]); `out` may be the logits."""
    if not hints:
        r = _host.distill_fwd_bwd(logits, teacher_ids, teacher_values, d_loss, teacher_lse, temperature, out)
        if r is not None:
            return r if out is None else (r[0], out)
    ctx, stream = handles(logits, hints)
    ld, T, V = rows(logits, "logits")
    entries, bits, values_code = _teacher(logits, T, teacher_ids, teacher_values, teacher_lse)
    dense(d_loss, (T,), "d_loss", logits, torch.float32)
    out, ld_out = gradient_of(logits, out)
    loss = torch.empty(T, dtype=torch.float32, device=logits.device)
    saved = torch.empty((T, 8), dtype=torch.float32, device=logits.device)
    _lib.check(_lib.lib.ctb_distill_fwd_bwd(ctx, stream, ptr(out), ptr(logits), ptr(teacher_ids), bits, ptr(teacher_values), values_code,
                                            ptr(teacher_lse), ptr(loss), ptr(saved), ptr(d_loss), V, T, ld_out, ld, entries,
                                            float(temperature), dtype_code(logits)))
    return loss, out
