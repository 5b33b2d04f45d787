"""Distillation of a student from a teacher's top logits, beside the losses of noise_amd.dust.

  distill_loss(logits, teacher_logits, teacher_index, ...)                per-token losses; differentiable in the logits
  distill_loss_grad(logits, teacher_logits, teacher_index, weight, ...)   losses and the weighted sum's gradient in one pass

The logits are the head's raw ones (utils/model.py:204-206) with its soft cap as an option. The calls are
torch.ops.noise_amd operators too. Derivatives are taken backwards and once, as in noise_amd.sinks.
"""
import torch

from . import _lib
from .sinks import F32, TYPES, _call, _new, _no_tangents

MAX_ENTRIES = 1024


def _operands(fn, logits, teacher_logits, teacher_index, vocab, temperature, softcap):
    if logits.dtype not in TYPES or logits.dim() < 1:
        raise ValueError(f'{fn}: bfloat16 or float32 logits [..., width], got {logits.dtype} {tuple(logits.shape)}')
    shape, width = logits.shape[:-1], logits.shape[-1]
    vocab = width if vocab is None else int(vocab)
    if not 0 < vocab <= width:
        raise ValueError(f'{fn}: vocab must be 1 .. {width}, got {vocab}')
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f'{fn}: temperature must be 1e-6 .. 1e6, got {temperature}')
    if softcap is not None and not 1e-6 <= softcap <= 1e6:
        raise ValueError(f'{fn}: softcap must be 1e-6 .. 1e6 (None: no cap), got {softcap}')
    if teacher_logits.shape != teacher_index.shape or teacher_logits.shape[:-1] != shape or teacher_logits.shape[-1] == 0:
        raise ValueError(f'{fn}: teacher logits and indices must be [{", ".join(map(str, shape))}, entries], got '
                         f'{tuple(teacher_logits.shape)} and {tuple(teacher_index.shape)}')
    if teacher_index.shape[-1] > MAX_ENTRIES:
        raise ValueError(f'{fn}: at most {MAX_ENTRIES} teacher entries per token, got {teacher_index.shape[-1]}')
    if teacher_index.dtype not in (torch.int32, torch.int64):
        raise ValueError(f'{fn}: teacher indices must be int32 or int64, got {teacher_index.dtype}')
    if teacher_logits.dtype not in TYPES:
        raise ValueError(f'{fn}: bfloat16 or float32 teacher logits, got {teacher_logits.dtype}')
    if teacher_logits.device != logits.device or teacher_index.device != logits.device:
        raise ValueError(f'{fn}: tensors on {logits.device}, {teacher_logits.device} and {teacher_index.device}')
    x = logits if logits.dim() == 2 else logits.reshape(-1, width)
    if x.stride(1) != 1 and width > 1 or x.stride(0) < 0:
        x = x.contiguous()
    return x, *(t if t.is_contiguous() else t.contiguous() for t in (teacher_logits, teacher_index)), vocab


def distill(fn, logits, teacher_logits, teacher_index, weight, vocab, temperature, softcap, with_grad):
    """(losses, gradient of sum weight * loss or None); weight None: ones"""
    x, t, i, vocab = _operands(fn, logits, teacher_logits, teacher_index, vocab, temperature, softcap)
    _no_tangents(fn, logits, teacher_logits, weight)
    rows, width = x.shape
    if weight is not None:
        if weight.shape != logits.shape[:-1] or weight.device != logits.device:
            raise ValueError(f'{fn}: weights must be {tuple(logits.shape[:-1])} on {logits.device}, got '
                             f'{tuple(weight.shape)} on {weight.device}')
        if weight.dtype != F32 or not weight.is_contiguous():
            weight = weight.to(F32).contiguous()
    loss = x.new_empty(logits.shape[:-1], dtype=F32)
    grad = _new(logits) if with_grad else None
    if rows:
        _call('noise_distill', x.device, x.data_ptr(), TYPES[x.dtype], rows, vocab, x.stride(0), t.data_ptr(),
              TYPES[t.dtype], i.data_ptr(), int(i.dtype == torch.int64), t.shape[-1], _lib.ptr(weight),
              float(temperature), float(softcap or 0.0), loss.data_ptr(), _lib.ptr(grad), width, width)
    return loss, grad


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_logits, teacher_index, vocab, temperature, softcap):
        ctx.save_for_backward(logits, teacher_logits, teacher_index)
        ctx.more = (vocab, temperature, softcap)
        return distill('distill_loss', logits, teacher_logits, teacher_index, None, vocab, temperature, softcap, False)[0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, weight):
        logits, teacher_logits, teacher_index = ctx.saved_tensors
        return (distill('distill_loss', logits, teacher_logits, teacher_index, weight, *ctx.more, True)[1],
                None, None, None, None, None)


def distill_loss(logits, teacher_logits, teacher_index, vocab=None, temperature=1.0, softcap=None):
    """Per-token distillation losses, fp32 [...], from raw logits [..., width] (bfloat16 or float32, the first `vocab` in use)
    and the teacher's top logits and their indices [..., entries]:

        z = cap(logits) / temperature,  cap(x) = softcap * tanh(x / softcap),  p = softmax(teacher / temperature)
        loss = temperature^2 * sum_k p_k (log p_k - log softmax(z)[index_k])

    with p over the entries in use: an index outside 0 .. vocab - 1 or a teacher logit of -inf leaves its entry out, and a
    token without entries has loss and gradient 0; at most 1024 entries (a gradient's work grows with their square: past 256 of
    them it outweighs a row of 4096). The same index may stand in several entries. Statistics and sums are in fp32.
    Differentiable in the logits (once); the teacher has no gradient."""
    if torch.compiler.is_compiling():
        return torch.ops.noise_amd.distill_loss(logits, teacher_logits, teacher_index,
                                                logits.shape[-1] if vocab is None else int(vocab), float(temperature), softcap)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _Distill.apply(logits, teacher_logits, teacher_index, vocab, float(temperature), softcap)
    return distill('distill_loss', logits, teacher_logits, teacher_index, None, vocab, temperature, softcap, False)[0]


def distill_loss_grad(logits, teacher_logits, teacher_index, weight=None, vocab=None, temperature=1.0, softcap=None):
    """(losses, gradient) of distill_loss in one pass over the logits, for a training step that knows its weights before
    the loss: the gradient, of the logits' shape and type, is that of sum(weight * loss), weight [...] (None: ones).
    Columns from `vocab` on get zeros. Both results are plain tensors, for logits that require a gradient too
    (logits.backward(gradient) goes on from there)."""
    if torch.compiler.is_compiling():
        return torch.ops.noise_amd.distill_loss_grad(logits, teacher_logits, teacher_index, weight,
                                                     logits.shape[-1] if vocab is None else int(vocab), float(temperature),
                                                     softcap)
    return distill('distill_loss_grad', logits, teacher_logits, teacher_index, weight, vocab, temperature, softcap, True)
