"""The cross entropy of a linear head over a vocabulary of any size, without its logits in memory, beside noise_amd.dust's
forward-only head_loss of the fixed model.

  linear_cross_entropy(x, weight, targets, vocab, softcap)       per-token losses; differentiable in x and weight
  linear_cross_entropy_grad(x, weight, targets, token_weight, vocab, softcap)
                                                                 losses and the weighted sum's gradients in one call

The head is utils/model.py:204-206's with its soft cap as an option, the loss that of train/val/run.py:89-94. The calls are
torch.ops.noise_amd operators too. Derivatives are taken backwards and once, as in noise_amd.sinks.
"""
import functools
from array import array

import torch

from . import _lib
from .sinks import F32, TYPES, _call, _new, _no_tangents

MAX_VOCAB, MAX_DIM, MAX_ROWS = 1 << 22, 1 << 16, 1 << 30


def _rows(t):
    """t [rows, dim], or a copy of it, with unit inner stride and rows after one another"""
    return t if (t.stride(1) == 1 or t.shape[1] == 1) and (t.stride(0) >= t.shape[1] or t.shape[0] == 1) else t.contiguous()


def _operands(fn, x, weight, targets, vocab, softcap):
    """x [rows, dim], the weight and targets as the kernels take them, copies among them; then vocab and softcap"""
    if x.dtype not in TYPES or x.dim() < 1 or weight.dtype != x.dtype or weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError(f'{fn}: bfloat16 or float32 x [..., dim] and weight [width, dim] of its type, got {x.dtype} '
                         f'{tuple(x.shape)} and {weight.dtype} {tuple(weight.shape)}')
    width, dim = weight.shape
    vocab = width if vocab is None else int(vocab)
    if not 0 < vocab <= min(width, MAX_VOCAB):
        raise ValueError(f'{fn}: vocab must be 1 .. {min(width, MAX_VOCAB)}, got {vocab}')
    if not 0 < dim <= MAX_DIM:
        raise ValueError(f'{fn}: dim must be 1 .. {MAX_DIM}, got {dim}')
    if softcap is not None and not 1e-6 <= softcap <= 1e6:
        raise ValueError(f'{fn}: softcap must be 1e-6 .. 1e6 (None: no cap), got {softcap}')
    if targets.shape != x.shape[:-1] or targets.dtype not in (torch.int32, torch.int64):
        raise ValueError(f'{fn}: targets must be int32 or int64 of shape {tuple(x.shape[:-1])}, got {targets.dtype} '
                         f'{tuple(targets.shape)}')
    if weight.device != x.device or targets.device != x.device:
        raise ValueError(f'{fn}: tensors on {x.device}, {weight.device} and {targets.device}')
    _no_tangents(fn, x, weight)
    x = _rows(x if x.dim() == 2 else x.reshape(-1, dim))
    if x.shape[0] > MAX_ROWS:
        raise ValueError(f'{fn}: at most {MAX_ROWS} tokens, got {x.shape[0]}')
    return x, _rows(weight), targets if targets.is_contiguous() else targets.contiguous(), vocab, float(softcap or 0.0)


def _table(x, weight, targets, vocab, with_grad):
    """A noise_vocab_t, its address (the array holds it for as long as it lives), a workspace and its bytes"""
    (rows, dim), width, kind, at = x.shape, weight.shape[0], TYPES[x.dtype], weight.data_ptr()
    pitch = weight.stride(0) if width > 1 else dim
    table = array('q', (x.data_ptr(), x.stride(0) if rows > 1 else dim, at, pitch, targets.data_ptr(),
                        int(targets.dtype == torch.int64), rows, dim, vocab, kind))
    need = _workspace(at % 16, pitch, rows, dim, vocab, kind, with_grad)
    return table, table.buffer_info()[0], x.new_empty(need, dtype=torch.uint8), need


@functools.lru_cache(maxsize=1024)
def _workspace(offset, pitch, rows, dim, vocab, kind, with_grad):
    # (of addresses like these, of which none is read)
    table = array('q', (4096, dim, 4096 + offset, pitch, 4096, 0, rows, dim, vocab, kind))
    return _lib.lib().noise_vocab_workspace_bytes(table.buffer_info()[0], with_grad)


def _forward(shape, x, weight, targets, vocab, softcap, with_lse):
    """(losses, lse or None) of checked operands"""
    loss = x.new_empty(shape, dtype=F32)
    lse = torch.empty_like(loss) if with_lse else None
    if x.shape[0]:
        table, at, work, need = _table(x, weight, targets, vocab, 0)
        _call('noise_vocab_loss', x.device, at, softcap, loss.data_ptr(), _lib.ptr(lse), work.data_ptr(), need)
    return loss, lse


def _gradients(fn, shape, token_weight, lse, x, weight, targets, vocab, softcap, need_x, need_weight):
    """(losses or, where lse is given, None; dx [rows, dim]; dweight) of checked operands"""
    _no_tangents(fn, token_weight)
    if token_weight is not None:
        if token_weight.shape != shape or token_weight.device != x.device:
            raise ValueError(f'{fn}: token weights must be {tuple(shape)} on {x.device}, got {tuple(token_weight.shape)} on '
                             f'{token_weight.device}')
        if token_weight.dtype != F32 or not token_weight.is_contiguous():
            token_weight = token_weight.to(F32).contiguous()
    loss = x.new_empty(shape, dtype=F32) if lse is None else None
    dx = _new(x) if need_x else None
    dw = _new(weight) if need_weight else None
    if x.shape[0]:
        table, at, work, need = _table(x, weight, targets, vocab, 1)
        _call('noise_vocab_grad', x.device, at, softcap, _lib.ptr(token_weight), _lib.ptr(lse), _lib.ptr(loss), _lib.ptr(dx),
              _lib.ptr(dw), weight.shape[0], work.data_ptr(), need)
    elif dw is not None:
        dw.zero_()
    return loss, dx, dw


def forward(x, weight, targets, vocab, softcap, with_lse):
    """(losses, lse or None)"""
    return _forward(targets.shape, *_operands('linear_cross_entropy', x, weight, targets, vocab, softcap), with_lse)


def gradients(fn, x, weight, targets, token_weight, lse, vocab, softcap, need_x=True, need_weight=True):
    """(losses or, where lse is given, None; dx; dweight)"""
    operands = _operands(fn, x, weight, targets, vocab, softcap)
    loss, dx, dw = _gradients(fn, targets.shape, token_weight, lse, *operands, need_x, need_weight)
    return loss, None if dx is None else dx.view(x.shape), dw


class _Head(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, targets, vocab, softcap):
        ctx.shapes = x.shape, targets.shape
        x, weight, targets, *ctx.more = _operands('linear_cross_entropy', x, weight, targets, vocab, softcap)
        loss, lse = _forward(ctx.shapes[1], x, weight, targets, *ctx.more, True)
        # (what the kernels take is saved: the tensors themselves, or the copies made of them)
        ctx.save_for_backward(lse, x, weight, targets)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        _, dx, dw = _gradients('linear_cross_entropy', ctx.shapes[1], dloss, *ctx.saved_tensors, *ctx.more,
                               *ctx.needs_input_grad[:2])
        return None if dx is None else dx.view(ctx.shapes[0]), dw, None, None, None


def linear_cross_entropy(x, weight, targets, vocab=None, softcap=None):
    """Per-token cross entropies, fp32 [...], of hidden states x [..., dim] under the head weight [width, dim] (both bfloat16 or
    both float32, the weight's first `vocab` rows in use) against targets [...] (int32 or int64):

        z = cap(x weight^T),  cap(z) = softcap * tanh(z / softcap),  loss = log sum exp z - z[target]

    A token whose target lies outside 0 .. vocab - 1 has loss 0 and no gradient, whatever its x holds. The logits are formed a
    tile at a time and never stored; their products, sums and softmax are in fp32, float32 operands with 21 bits in the products.
    Rows may lie at any distance from each other. Differentiable in x and weight (once): the backward pass forms the logits again.

    Their gradients are held in 16 bits, as bfloat16 beside bfloat16 operands (up to 32 tokens: as a sum of two, 16 bits of a
    value) and two times 16 beside float32 ones, for at most 2 GiB of tokens and vocabulary at a time, or for 256 tokens where
    those take more (float32 of more than 2^21 entries: up to 4 GiB). Up to 64 tokens have logits in float32 and their gradients
    twice instead, 2 GiB at most together; many tokens of a small vocabulary may have logits in float32 besides, 1 GiB at most.

    float32 values below 2^-38 of their tensor's largest, the tokens' weights among those tensors, count as 0. So a column that
    takes entries out of the vocabulary, beside a column of ones in x, should hold values like -1e4 or, for losses, -inf in
    float32, not the type's lowest, beside which all other weights are 0; bfloat16 weights may hold either. (An infinite weight
    makes its column of dx NaN, as 0 times infinity.) A token's probabilities are off by 2^-24 of its largest logit's size."""
    if torch.compiler.is_compiling():
        return torch.ops.noise_amd.linear_cross_entropy(x, weight, targets, weight.shape[0] if vocab is None else int(vocab),
                                                        softcap)[0]
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return _Head.apply(x, weight, targets, vocab, softcap)
    return forward(x, weight, targets, vocab, softcap, False)[0]


def linear_cross_entropy_grad(x, weight, targets, token_weight=None, vocab=None, softcap=None):
    """(losses, dx, dweight) of linear_cross_entropy in one call, for a training step that knows its tokens' weights before the
    losses: the gradients, of x's and weight's shapes and type, are those of sum(token_weight * loss), token_weight [...] (None:
    ones). Rows of dweight from `vocab` on are zeros. (Of many bfloat16 tokens, entries whose exponentials are below 2^-62 of the
    largest of their 128 have no part in a token's gradients; backward() keeps those too.) The results are plain tensors, for
    operands that require a gradient too (x.backward(dx) goes on from there)."""
    if torch.compiler.is_compiling():
        # (the operator has no backward pass, and its results would ask for one)
        return torch.ops.noise_amd.linear_cross_entropy_grad(x.detach(), weight.detach(), targets,
                                                             None if token_weight is None else token_weight.detach(),
                                                             weight.shape[0] if vocab is None else int(vocab), softcap)
    return gradients('linear_cross_entropy_grad', x, weight, targets, token_weight, None, vocab, softcap)
