"""Attention layers of a model trained with exact gradients and served past its window.

  qk_norm_rotary(q, k, cos, sin, ...)          norm of every head's queries and keys, rotated, in one pass; differentiable
  qk_norm_rotary_append(q, k, v, cos, sin, k_cache, v_cache, start, ...)   the same for new tokens, into a cache
  sink_attention(q, k, v, window, sinks, lengths)   a sliding window and first tokens that stay visible; differentiable
  sink_attention_decode(q, k_cache, v_cache, start, window, sinks)         a few new tokens against a cache

Tensors are [batch, token, head, dim] with dim 64 or 128, as in utils/model.py; the queries' heads are a multiple of the
keys' (query head h reads key head h // (H // Hk)). The norm and rotation are those of utils/model.py:46-47, 55-58 and
88-94 (rotated halves; without learned weights the rotation and the norm commute), the mask that of utils/model.py:17-21
with the first `sinks` tokens beside the window. The same calls are torch.ops.noise_amd operators, which compiled callers trace.

Derivatives are taken backwards and once; tensors with forward-mode tangents (torch.autograd.forward_ad) are refused.
"""
import functools
from array import array

import torch
from torch.autograd import forward_ad

from . import _lib

BF16, F32 = torch.bfloat16, torch.float32
EPS = torch.finfo(F32).eps   # utils/model.py:46-47 under fp32 statistics
TYPES = {BF16: _lib.TYPE_BF16, F32: _lib.TYPE_FP32}
FAR = 2 ** 62                # windows from here on are all the same, whatever the cache
MAX_NEW = 16                 # new tokens per sequence of one sink_attention_decode call


def _check(fn, q, k, v=None):
    """(B, T, H, D, T', Hk) of [B, T, H, D] and [B, T', Hk, D] of one device, type and head dim"""
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4 or qs[0] != ks[0] or qs[3] != ks[3]:
        raise ValueError(f'{fn}: q and k must be [batch, token, head, dim] of one batch and dim, got {tuple(qs)} and '
                         f'{tuple(ks)}')
    B, T, H, D = qs
    _, S, Hk, _ = ks
    if D != 64 and D != 128:
        raise ValueError(f'{fn}: head dim must be 64 or 128, got {D}')
    if Hk == 0 or H == 0 or H % Hk:
        raise ValueError(f'{fn}: {H} query heads are no multiple of {Hk} key heads')
    device = q.device
    if k.device != device or (v is not None and v.device != device):
        raise ValueError(f'{fn}: tensors on {device}, {k.device}' + (f' and {v.device}' if v is not None else ''))
    return B, T, H, D, S, Hk


def _strides(t):
    """The strides of t's batch, tokens and heads, 0 where there is one of them (torch keeps any number there)"""
    (B, T, H, _), (a, b, c, _) = t.shape, t.stride()
    return a if B > 1 else 0, b if T > 1 else 0, c if H > 1 else 0


def _rows(t):
    """t with unit inner stride and rows of whole 16 B at 16 B addresses, less than 2^25 elements from token to token (copied
    if it has not)."""
    if t.is_contiguous() and not t.data_ptr() % 16:
        return t
    (a, b, c), unit = _strides(t), 16 // t.element_size()
    if t.stride(3) != 1 or (a | b | c) % unit or b >= 1 << 25 or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
    return t


def _cache_rows(fn, cache):
    (a, b, c, one), unit = cache.stride(), 16 // cache.element_size()
    if (a | b | c) % unit:
        a, b, c = _strides(cache)
    if one != 1 or (a | b | c) % unit or cache.data_ptr() % 16:
        raise ValueError(f'{fn}: cache rows must be whole 16 B at 16 B addresses with unit inner stride')


def _no_tangents(fn, *tensors):
    """Refuses tensors that carry forward-mode tangents, which would otherwise be dropped and read as derivatives of 0"""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f'{fn}: forward-mode derivatives are not implemented')


def _no_gradients(fn, *tensors):
    """Refuses tensors whose gradient a call without a backward pass would drop"""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f'{fn}: not differentiable, and a tensor requires a gradient: call it under torch.no_grad()')


def _span(shape, strides):
    """(elements from a tensor's first to behind its last, its (stride, size) from the outermost dimension in), or None where it
    is not made of dimensions inside one another: where a step along one lands on what the shorter steps reach"""
    end, dims = 1, sorted((s, n) for s, n in zip(strides, shape) if n > 1)
    for s, n in dims:
        if s < end:
            return None
        end += s * (n - 1)
    return end, dims[::-1]


@functools.lru_cache(maxsize=1024)
def _spans(shape, strides, others):
    return _span(shape, strides), _span(shape, others)


def _own_memory(fn, k_cache, v_cache):
    """Refuses caches of one shape and type in which two slots are the same memory (or may be: where the caches' ranges meet and
    their strides differ)"""
    k, v = _spans(k_cache.shape, k_cache.stride(), v_cache.stride())
    if k is None or v is None:
        raise ValueError(f'{fn}: slots of a cache overlap (a broadcast cache has none of its own to write to)')
    off = (v_cache.data_ptr() - k_cache.data_ptr()) // k_cache.element_size()
    if -v[0] < off < k[0] and k_cache.numel() and (k[1] != v[1] or _reach(off, k[1])):
        raise ValueError(f'{fn}: k_cache and v_cache have slots in the same memory')


def _reach(off, dims):
    """Whether two elements of such a tensor lie `off` apart: a dimension's steps miss `off` by less than one of them, which
    leaves two numbers of steps, and the rest to the dimensions inside"""
    if not dims:
        return off == 0
    (s, n), *inner = dims
    return any(abs(d) < n and _reach(off - d * s, inner) for d in (off // s, off // s + 1))


_HEADS = 5 * 8   # bytes of a noise_heads_t: five 64-bit numbers


def _table(*tensors, pointers=()):
    """noise_heads_t of each tensor, one after the other, then the tensors' or None's addresses in `pointers`; and the address of
    the first (the array holds them for as long as it lives)"""
    flat = []
    for t in tensors:
        a, b, c, _ = t.stride()
        if (a | b | c) % 8 or b >= 1 << 25:
            a, b, c = _strides(t)
        flat += (t.data_ptr(), a, b, c, t.size(2))
    for t in pointers:
        flat.append(0 if t is None else t.data_ptr())
    table = array('q', flat)
    return table, table.buffer_info()[0]


def _new(t):
    """an uninitialised contiguous tensor like t"""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _call(name, device, *args):
    """The entry point on `device`'s current stream (made the current device for the launch)."""
    index = device.index
    if index is None:
        raise ValueError(f'{name}: tensors must be on a GPU, got {device}')
    if torch._C._cuda_getDevice() == index:
        return _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(index))
    with torch.cuda.device(device):
        return _lib.call(name, *args, _lib.stream_ptr(device))


def _ints(fn, name, t, batch, device):
    """[batch] int32 or int64 on the device, contiguous, and whether it is int64."""
    if t.dtype not in (torch.int32, torch.int64) or t.shape != (batch,) or t.device != device:
        raise ValueError(f'{fn}: {name} must be int32 or int64 of shape [{batch}] on {device}, got {t.dtype} '
                         f'{tuple(t.shape)} on {t.device}')
    return t if t.is_contiguous() else t.contiguous(), int(t.dtype == torch.int64)


# --- norm and rotation ---


def _tables(fn, cos, sin, D, device):
    if cos.shape != sin.shape or cos.dim() != 2 or cos.shape[1] != D // 2 or cos.shape[0] == 0:
        raise ValueError(f'{fn}: cos and sin must be [positions, {D // 2}], got {tuple(cos.shape)} and {tuple(sin.shape)}')
    if cos.device != device or sin.device != device:
        raise ValueError(f'{fn}: rotation tables on {cos.device} and {sin.device}, tensors on {device}')
    return _plain(cos), _plain(sin)


def _plain(t):
    """t in fp32, contiguous, at a 16 B address"""
    if t.dtype != F32 or not t.is_contiguous():
        t = t.to(F32).contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _weight(fn, w, D, device):
    if w is None:
        return None
    if w.shape != (D,) or w.device != device:
        raise ValueError(f'{fn}: weights must be [{D}] on {device}, got {tuple(w.shape)} on {w.device}')
    return _plain(w)


def _norm_operands(fn, q, k, cos, sin, q_weight, k_weight, start):
    """(cos, sin, q_weight, k_weight, start, start is int64) as the kernels take them"""
    _check(fn, q, k)
    if q.shape[1] != k.shape[1] or q.dtype != k.dtype:
        raise ValueError(f'{fn}: q and k must have one length and type, got {tuple(q.shape)} {q.dtype} and '
                         f'{tuple(k.shape)} {k.dtype}')
    if q.dtype not in TYPES:
        raise ValueError(f'{fn}: bfloat16 or float32 tensors, got {q.dtype}')
    _no_tangents(fn, q, k, cos, sin, q_weight, k_weight)
    B, T, _, D = q.shape
    cos, sin = _tables(fn, cos, sin, D, q.device)
    wide = 0
    if start is not None:
        start, wide = _ints(fn, 'start', start, B, q.device)
    elif T > cos.shape[0]:
        raise ValueError(f'{fn}: {T} tokens but rotation tables of {cos.shape[0]} positions')
    return cos, sin, _weight(fn, q_weight, D, q.device), _weight(fn, k_weight, D, q.device), start, wide


def _norm_forward(q, k, cos, sin, qw, kw, start, wide, eps):
    """qk_norm_rotary of checked operands"""
    B, T, _, D = q.shape
    out = _new(q), _new(k)
    x = _rows(q), _rows(k)   # (copies among them, and the table, live until the launch)
    table, at = _table(*x, *out, pointers=(qw, kw))
    _call('noise_qk_norm_rotary', q.device, at, at + 2 * _HEADS, at + 4 * _HEADS, None, None, cos.data_ptr(),
          sin.data_ptr(), cos.size(0), None if start is None else start.data_ptr(), wide, B, T, 0, D, TYPES[q.dtype], eps)
    return out


@functools.lru_cache(maxsize=None)
def _norm_workspace(D):
    return _lib.lib().noise_qk_norm_rotary_bwd_workspace_bytes(D)


def _norm_backward(dq, dk, q, k, cos, sin, qw, kw, start, wide, eps):
    """Gradients of q, k and (fp32; None for absent ones) of the weights, of checked operands"""
    _no_tangents('qk_norm_rotary', dq, dk)
    B, T, _, D = q.shape
    dt = q.dtype
    dx = _new(q), _new(k)
    x = _rows(q), _rows(k), _rows(dq if dq.dtype == dt else dq.to(dt)), _rows(dk if dk.dtype == dt else dk.to(dt))
    need, work, dqw, dkw = 0, None, None, None
    if qw is not None or kw is not None:
        need = _norm_workspace(D)
        work = q.new_empty(need, dtype=torch.uint8)
        dqw = None if qw is None else torch.empty_like(qw)
        dkw = None if kw is None else torch.empty_like(kw)
    table, at = _table(*x, *dx, pointers=(qw, kw, dqw, dkw))
    _call('noise_qk_norm_rotary_bwd', q.device, at, at + 2 * _HEADS, at + 4 * _HEADS, at + 6 * _HEADS,
          at + 6 * _HEADS + 16, cos.data_ptr(), sin.data_ptr(), cos.size(0), None if start is None else start.data_ptr(), wide,
          B, T, D, TYPES[dt], eps, None if work is None else work.data_ptr(), need)
    return dx[0], dx[1], dqw, dkw


def _as(grad, like):
    return grad if grad is None or grad.dtype == like.dtype else grad.to(like.dtype)


def norm_forward(q, k, cos, sin, q_weight, k_weight, start, eps):
    return _norm_forward(q, k, *_norm_operands('qk_norm_rotary', q, k, cos, sin, q_weight, k_weight, start), eps)


def norm_backward(dq, dk, q, k, cos, sin, q_weight, k_weight, start, eps):
    """Gradients of q, k and (in their types; None for absent ones) of the weights."""
    operands = _norm_operands('qk_norm_rotary', q, k, cos, sin, q_weight, k_weight, start)
    dq, dk, dqw, dkw = _norm_backward(dq, dk, q, k, *operands, eps)
    return dq, dk, _as(dqw, q_weight), _as(dkw, k_weight)


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, cos, sin, q_weight, k_weight, start, eps):
        cos, sin, qw, kw, start, wide = _norm_operands('qk_norm_rotary', q, k, cos, sin, q_weight, k_weight, start)
        # (what the kernels take is saved: the tensors themselves, or the fp32 copies made of them)
        ctx.save_for_backward(q, k, cos, sin, qw, kw, start)
        ctx.more = wide, eps
        ctx.types = None if q_weight is None else q_weight.dtype, None if k_weight is None else k_weight.dtype
        return _norm_forward(q, k, cos, sin, qw, kw, start, wide, eps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        dq, dk, dqw, dkw = _norm_backward(dq, dk, *ctx.saved_tensors, *ctx.more)
        a, b = ctx.types
        return (dq, dk, None, None, dqw if a is None or a == F32 else dqw.to(a),
                dkw if b is None or b == F32 else dkw.to(b), None, None)


def qk_norm_rotary(q, k, cos, sin, q_weight=None, k_weight=None, start=None, eps=EPS):
    """(q', k'): every row of q [B, T, H, D] and k [B, T, Hk, D] normed to RMS 1 over D (fp32 statistics), times its
    weight [D] if there is one, and rotated for its position: t, or start[b] + t with start [B] (int32 or int64). cos and
    sin are tables [positions, D / 2] over absolute positions (used in fp32); a token whose position lies outside them
    gets zeros (and has no gradient). q and k are bfloat16 or float32, and so are q' and k' (contiguous), rounded once.
    Differentiable in q, k and the weights (once); the weights' gradients are summed in fp32 in a fixed order."""
    if torch.compiler.is_compiling():
        return torch.ops.noise_amd.qk_norm_rotary(q, k, cos, sin, q_weight, k_weight, start, float(eps))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or (q_weight is not None and q_weight.requires_grad)
                                    or (k_weight is not None and k_weight.requires_grad)):
        return _Norm.apply(q, k, cos, sin, q_weight, k_weight, start, float(eps))
    return norm_forward(q, k, cos, sin, q_weight, k_weight, start, float(eps))


def qk_norm_rotary_append(q, k, v, cos, sin, k_cache, v_cache, start, q_weight=None, k_weight=None, eps=EPS):
    """q' of qk_norm_rotary for new tokens at positions start[b] + t, with k' and v [B, T, Hk, D] written to those slots of
    k_cache and v_cache [B, capacity, Hk, D] (of k's type) in the same launch. A token whose position lies outside the
    cache or the tables gets zeros in q' and leaves the cache as it is, so an idle sequence has a start of -T; no other
    slot is touched. The caches may be views of one buffer (refused where their slots overlap); q, k and v must not share
    memory with them. Not differentiable (it writes in place): while gradients are recorded, tensors that require one are
    refused."""
    if torch.compiler.is_compiling():
        return torch.ops.noise_amd.qk_norm_rotary_append(q, k, v, cos, sin, k_cache, v_cache, start, q_weight, k_weight,
                                                         float(eps))
    fn = 'qk_norm_rotary_append'
    cos, sin, qw, kw, start, wide = _norm_operands(fn, q, k, cos, sin, q_weight, k_weight, start)
    B, T, H, D = q.shape
    if start is None:
        raise ValueError(f'{fn}: start is required')
    if v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
        raise ValueError(f"{fn}: v must have k's shape, type and device, got {tuple(v.shape)} {v.dtype} on {v.device}")
    _no_tangents(fn, v, k_cache, v_cache)
    _no_gradients(fn, q, k, v, k_cache, v_cache, q_weight, k_weight)
    S = k_cache.shape[1] if k_cache.dim() == 4 else 0
    for c in (k_cache, v_cache):
        if c.shape != (B, S, k.shape[2], D) or c.dtype != k.dtype or c.device != k.device or S == 0:
            raise ValueError(f'{fn}: caches must be [{B}, capacity, {k.shape[2]}, {D}] {k.dtype} on {k.device}, got '
                             f'{tuple(c.shape)} {c.dtype} on {c.device}')
        _cache_rows(fn, c)
    _own_memory(fn, k_cache, v_cache)
    out = _new(q)
    q, k, v = _rows(q), _rows(k), _rows(v)
    table, at = _table(q, k, out, k_cache, v, v_cache, pointers=(qw, kw))
    _call('noise_qk_norm_rotary', q.device, at, at + 2 * _HEADS, at + 6 * _HEADS, at + 4 * _HEADS, at + 5 * _HEADS,
          cos.data_ptr(), sin.data_ptr(), cos.size(0), start.data_ptr(), wide, B, T, S, D, TYPES[q.dtype], float(eps))
    torch.autograd.graph.increment_version((k_cache, v_cache))   # (a graph that holds them refuses its backward pass)
    return out


# --- attention ---


def _attend_operands(fn, q, k, v, window, sinks, lengths):
    _check(fn, q, k, v)
    if v.shape != k.shape or q.shape[1] != k.shape[1]:
        raise ValueError(f'{fn}: k and v must have one shape and the length of q, got {tuple(q.shape)}, '
                         f'{tuple(k.shape)}, {tuple(v.shape)}')
    if q.dtype != BF16 or k.dtype != BF16 or v.dtype != BF16:
        raise ValueError(f'{fn}: bfloat16 tensors, got {q.dtype}, {k.dtype}, {v.dtype}')
    if window < 0 or sinks < 0:
        raise ValueError(f'{fn}: window and sinks must not be negative, got {window} and {sinks}')
    _no_tangents(fn, q, k, v)
    return (None, 0) if lengths is None else _ints(fn, 'lengths', lengths, q.shape[0], q.device)


def _attend_forward(q, k, v, window, sinks, lengths, wide, training):
    """(out, what its rounding left out or None, lse or None) of checked operands"""
    B, T, H, D = q.shape
    out, rest, lse = _new(q), None, None
    q, k, v = _rows(q), _rows(k), _rows(v)
    if training:
        rest, lse = torch.empty_like(out), q.new_empty((B, H, T), dtype=F32)
    table, at = _table(q, k, v, out, *((rest,) if training else ()))
    _call('noise_sink_attention_fwd', q.device, at, at + _HEADS, at + 2 * _HEADS, at + 3 * _HEADS,
          at + 4 * _HEADS if training else None, lse.data_ptr() if training else None,
          None if lengths is None else lengths.data_ptr(), wide, B, T, D, window, sinks, D ** -0.5)
    return out, rest, lse


@functools.lru_cache(maxsize=1024)
def _attend_workspace(*sizes):
    return _lib.lib().noise_sink_attention_bwd_workspace_bytes(*sizes)


def _attend_backward(dout, q, k, v, out, rest, lse, window, sinks, lengths, wide):
    _no_tangents('sink_attention', dout)
    B, T, H, D = q.shape
    grads = [_new(q), _new(k), _new(v)]
    x = _rows(q), _rows(k), _rows(v), _rows(out), rest, _rows(dout if dout.dtype == BF16 else dout.to(BF16))
    table, at = _table(*x, *grads)
    need = _attend_workspace(B, T, H, k.size(2), D, window, sinks)
    work = q.new_empty(max(need, 0), dtype=torch.uint8)
    _call('noise_sink_attention_bwd', q.device, *range(at, at + 6 * _HEADS, _HEADS), lse.data_ptr(),
          *range(at + 6 * _HEADS, at + 9 * _HEADS, _HEADS), None if lengths is None else lengths.data_ptr(), wide, B, T, D,
          window, sinks, D ** -0.5, work.data_ptr(), need)
    return grads


def attend_forward(q, k, v, window, sinks, lengths, training):
    """(out, rest, lse): with `training` what attend_backward takes beside the output, else None"""
    return _attend_forward(q, k, v, window, sinks, *_attend_operands('sink_attention', q, k, v, window, sinks, lengths),
                           training)


def attend_backward(dout, q, k, v, out, rest, lse, window, sinks, lengths):
    operands = _attend_operands('sink_attention', q, k, v, window, sinks, lengths)
    return _attend_backward(dout, q, k, v, out, rest, lse, window, sinks, *operands)


class _Attend(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, lengths):
        lengths, wide = _attend_operands('sink_attention', q, k, v, window, sinks, lengths)
        out, rest, lse = _attend_forward(q, k, v, window, sinks, lengths, wide, True)
        ctx.save_for_backward(q, k, v, out, rest, lse, lengths)
        ctx.more = window, sinks, wide
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, out, rest, lse, lengths = ctx.saved_tensors
        window, sinks, wide = ctx.more
        return (*_attend_backward(dout, q, k, v, out, rest, lse, window, sinks, lengths, wide), None, None, None)


def sink_attention(q, k, v, window, sinks=0, lengths=None):
    """Causal attention in which token i sees the tokens j <= i with i - j <= window or j < sinks, [B, T, H, D] from q
    [B, T, H, D] and k, v [B, T, Hk, D] in bfloat16 (fp32 scores and sums; the weights and, in the backward pass, the scores'
    gradients are rounded to bfloat16 for their products). lengths [B] (int32 or int64): the batch is padded; tokens from
    lengths[b] on are seen by none, get zeros, have no gradient, and may hold anything. Tokens of the sequence itself
    are taken to be finite, with scores (q . k / sqrt(D)) below 2^28 in size; gradients take the scores' exponents from fp32
    sums, whose steps are 2^-7 of a weight at scores of 2^15. Differentiable in q, k and v (once), with sums in a fixed order."""
    window, sinks = min(int(window), FAR), min(int(sinks), FAR)
    training = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if torch.compiler.is_compiling():
        if training:
            return torch.ops.noise_amd.sink_attention(q, k, v, window, sinks, lengths)[0]
        return torch.ops.noise_amd.sink_attention_output(q, k, v, window, sinks, lengths)
    if training:
        return _Attend.apply(q, k, v, window, sinks, lengths)
    return attend_forward(q, k, v, window, sinks, lengths, False)[0]


@functools.lru_cache(maxsize=1024)
def _decode_workspace(*sizes):
    return _lib.lib().noise_sink_decode_workspace_bytes(*sizes)


def sink_attention_decode(q, k_cache, v_cache, start, window, sinks=0):
    """sink_attention of T new tokens (1 to 16) against a cache: q [B, T, H, D], k_cache and v_cache [B, capacity, Hk, D]
    in bfloat16, whose slots hold the positions 0, 1, ... (every position has its slot: the window saves reading, not room);
    token t of sequence b stands at position start[b] + t (its own key already in the cache, as qk_norm_rotary_append leaves
    it) and sees the slots up to there that the window and the sinks allow. A token at a negative position (an idle sequence
    has a start of -T) gets zeros. Slots that no token of the call sees may hold anything. Not differentiable: while gradients
    are recorded, tensors that require one are refused."""
    if torch.compiler.is_compiling():
        return torch.ops.noise_amd.sink_attention_decode(q, k_cache, v_cache, start, min(int(window), FAR), min(int(sinks), FAR))
    fn = 'sink_attention_decode'
    window, sinks = min(int(window), FAR), min(int(sinks), FAR)
    B, T, H, D, S, Hk = _check(fn, q, k_cache, v_cache)
    if S == 0 or v_cache.shape != k_cache.shape:
        raise ValueError(f'{fn}: caches must have one shape and some capacity, got {tuple(k_cache.shape)} and '
                         f'{tuple(v_cache.shape)}')
    if q.dtype != BF16 or k_cache.dtype != BF16 or v_cache.dtype != BF16:
        raise ValueError(f'{fn}: bfloat16 tensors, got {q.dtype}, {k_cache.dtype}, {v_cache.dtype}')
    if T > MAX_NEW:
        raise ValueError(f'{fn}: at most {MAX_NEW} new tokens, got {T}')
    if window < 0 or sinks < 0:
        raise ValueError(f'{fn}: window and sinks must not be negative, got {window} and {sinks}')
    _no_tangents(fn, q, k_cache, v_cache)
    _no_gradients(fn, q, k_cache, v_cache)
    start, wide = _ints(fn, 'start', start, B, q.device)
    _cache_rows(fn, k_cache)
    _cache_rows(fn, v_cache)
    out = _new(q)
    need = _decode_workspace(B, T, H, Hk, S, D, window, sinks)
    work = q.new_empty(need, dtype=torch.uint8) if need > 0 else None
    q = _rows(q)
    table, at = _table(q, k_cache, v_cache, out)
    _call('noise_sink_decode', q.device, at, at + _HEADS, at + 2 * _HEADS, at + 3 * _HEADS, start.data_ptr(), wide, B, T, S, D,
          window, sinks, D ** -0.5, None if work is None else work.data_ptr(), need)
    return out
