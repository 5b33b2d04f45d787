"""The residual stream between two blocks of a model trained with exact gradients.

  residual_norm(x, y, x0, scale, x0_scale, gate, y_weight, weight, norm_y)   a block's output onto the stream, and the norm that
                                                                             the next block reads, in one pass; differentiable

The mixing is that of the forward that train/val/eggroll.py:77-94 repeats (x = resid_lambda x + x0_lambda x0, h = norm(x)), the
norm that of utils/model.py:46-47; the learned weights, the gate and the norm of the block's output are options. The call is a
torch.ops.noise_amd operator too. Derivatives are taken backwards and once, as in noise_amd.sinks.
"""
import functools
import math
from array import array

import torch

from . import _lib
from .sinks import BF16, EPS, F32, TYPES, _call, _new, _no_tangents

MAX_DIM = 8192


def _vector(fn, name, w, D, device):
    """The weight in fp32, contiguous"""
    if w is None:
        return None
    if w.shape != (D,) or w.device != device or not w.is_floating_point():
        raise ValueError(f'{fn}: {name} must be [{D}] on {device}, got {w.dtype} {tuple(w.shape)} on {w.device}')
    return w if w.dtype == F32 and w.is_contiguous() else w.to(F32).contiguous()


def _scalar(fn, name, s, device):
    """The scalar in fp32"""
    if s is None:
        return None
    if not isinstance(s, torch.Tensor):
        raise ValueError(f'{fn}: {name} must be a tensor of one value on {device}, got {s!r}')
    if s.numel() != 1 or s.device != device or not s.is_floating_point():
        raise ValueError(f'{fn}: {name} must be one value on {device}, got {s.dtype} {tuple(s.shape)} on {s.device}')
    return s if s.dtype == F32 else s.to(F32)


def _rows(t, D):
    """(t, or a copy of it, with its rows at one distance from each other and unit inner stride; that distance)"""
    if t.is_contiguous():
        return t, D
    dims = [(n, s) for n, s in zip(t.shape[:-1], t.stride()) if n > 1]
    if (t.stride(-1) == 1 or D == 1) and all(s == n * r for (_, s), (n, r) in zip(dims, dims[1:])):
        return t, dims[-1][1] if dims else D
    return t.contiguous(), D


def _gate(fn, gate, x):
    """(gate as contiguous rows of D, rows of x that share one)"""
    shape, full = gate.shape, x.shape
    if gate.device != x.device or gate.dtype not in TYPES:
        raise ValueError(f'{fn}: gate must be bfloat16 or float32 on {x.device}, got {gate.dtype} on {gate.device}')
    n, same = len(full), 0
    over = (1,) * (n - len(shape)) + tuple(shape)
    # as x up to some dimension, ones from there on
    while same < n - 1 and over[same] == full[same]:
        same += 1
    if not 1 <= len(shape) <= n or shape[-1] != full[-1] or any(s != 1 for s in over[same:n - 1]):
        raise ValueError(f'{fn}: gate must be [{full[-1]}], or as x with ones from some dimension on, got {tuple(shape)} for '
                         f'{tuple(full)}')
    return gate if gate.is_contiguous() else gate.contiguous(), math.prod(full[same:n - 1])


def _operands(fn, x, y, x0, scale, x0_scale, gate, y_weight, weight, norm_y, dtype):
    """The operands as the kernels take them, copies among them, and what else goes into a noise_residual_t"""
    shape, device, xt = x.shape, x.device, x.dtype
    if xt not in TYPES or not shape:
        raise ValueError(f'{fn}: bfloat16 or float32 x [..., dim], got {xt} {tuple(shape)}')
    D = shape[-1]
    if not 0 < D <= MAX_DIM:
        raise ValueError(f'{fn}: dim must be 1 .. {MAX_DIM}, got {D}')
    for name, t in (('y', y), ('x0', x0)):
        if t is not None and (t.shape != shape or t.device != device):
            raise ValueError(f'{fn}: {name} must be {tuple(shape)} on {device}, got {tuple(t.shape)} on {t.device}')
    if x0 is not None and x0.dtype != xt:
        raise ValueError(f'{fn}: x and x0 must have one type, got {xt} and {x0.dtype}')
    if y is None and (gate is not None or norm_y):
        raise ValueError(f'{fn}: a gate or norm of y without y')
    if y_weight is not None and not norm_y:
        raise ValueError(f"{fn}: y_weight is the weight of y's norm, which norm_y=True asks for")
    if x0 is None and x0_scale is not None:
        raise ValueError(f'{fn}: x0_scale without x0')
    if dtype is None:
        dtype = xt if y is None else y.dtype
    if dtype not in TYPES or (y is not None and y.dtype != dtype) or (xt == BF16 and dtype == F32):
        raise ValueError(f'{fn}: h has the type of y, bfloat16, or float32 where x is float32; got x {xt}, '
                         f'y {None if y is None else y.dtype} and {dtype}')
    _no_tangents(fn, x, y, x0, scale, x0_scale, gate, y_weight, weight)
    rows = x.numel() // D
    x, sx = _rows(x, D)
    sy = s0 = 0
    if y is not None:
        y, sy = _rows(y, D)
    if x0 is not None:
        x0, s0 = _rows(x0, D)
    gate_rows, gate_type = rows, BF16
    if gate is not None:
        gate, gate_rows = _gate(fn, gate, x)
        gate_type = gate.dtype
    tensors = (x, y, x0, _scalar(fn, 'scale', scale, device), _scalar(fn, 'x0_scale', x0_scale, device), gate,
               _vector(fn, 'y_weight', y_weight, D, device), _vector(fn, 'weight', weight, D, device))
    return tensors, (sx, sy, s0), (rows, gate_rows, D, TYPES[xt], TYPES[dtype], TYPES[gate_type], int(norm_y)), dtype


def _table(tensors, strides, numbers):
    """A noise_residual_t, and its address (the array holds it for as long as it lives)"""
    p = [0 if t is None else t.data_ptr() for t in tensors]
    table = array('q', (*p[:3], *strides, *p[3:], *numbers))
    return table, table.buffer_info()[0]


def _forward(tensors, strides, numbers, dtype, eps):
    """residual_norm of checked operands"""
    x = tensors[0]
    out = _new(x)
    h = torch.empty_like(out, dtype=dtype)
    if numbers[0]:
        table, at = _table(tensors, strides, numbers)
        _call('noise_residual_norm', x.device, at, out.data_ptr(), h.data_ptr(), eps)
    return out, h


@functools.lru_cache(maxsize=1024)
def _workspace(rows, gate_rows, D):
    return _lib.lib().noise_residual_norm_bwd_workspace_bytes(rows, gate_rows, D)


def _upstream(grad, dtype):
    if grad is None:
        return None
    grad = grad if grad.dtype == dtype else grad.to(dtype)
    return grad if grad.is_contiguous() else grad.contiguous()


def _backward(dout, dh, tensors, strides, numbers, dtype, eps, needs):
    """The gradients of checked operands, None where `needs` says False; the scalars' and weights' in fp32"""
    _no_tangents('residual_norm', dout, dh)
    x = tensors[0]
    if not numbers[0] or (dout is None and dh is None):
        return [torch.zeros_like(t) if n and t is not None else None for t, n in zip(tensors, needs)]
    dout, dh = _upstream(dout, x.dtype), _upstream(dh, dtype)
    grads = [_new(t) if n and t is not None else None for t, n in zip(tensors, needs)]
    need, work = 0, None
    if any([g is not None for g in grads[3:]]):
        need = _workspace(*numbers[:3])
        work = x.new_empty(need, dtype=torch.uint8)
    table, at = _table(tensors, strides, numbers)
    to = array('q', [0 if g is None else g.data_ptr() for g in grads])
    _call('noise_residual_norm_bwd', x.device, at, _lib.ptr(dout), _lib.ptr(dh), to.buffer_info()[0], eps, _lib.ptr(work), need)
    return grads


def forward(x, y, x0, scale, x0_scale, gate, y_weight, weight, norm_y, dtype, eps):
    return _forward(*_operands('residual_norm', x, y, x0, scale, x0_scale, gate, y_weight, weight, norm_y, dtype), eps)


def backward(dout, dh, x, y, x0, scale, x0_scale, gate, y_weight, weight, norm_y, dtype, eps, needs):
    """The gradients of x, y, x0, scale, x0_scale, gate, y_weight and weight in their types, None where `needs` says False"""
    given = x, y, x0, scale, x0_scale, gate, y_weight, weight
    grads = _backward(dout, dh, *_operands('residual_norm', *given, norm_y, dtype), eps, needs)
    return [g if g is None or g.dtype == t.dtype else g.to(t.dtype) for g, t in zip(grads, given)]


class _Residual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, x0, scale, x0_scale, gate, y_weight, weight, norm_y, dtype, eps):
        tensors, *more = _operands('residual_norm', x, y, x0, scale, x0_scale, gate, y_weight, weight, norm_y, dtype)
        # (what the kernels take is saved: the tensors themselves, or the copies made of them)
        ctx.save_for_backward(*tensors)
        ctx.more = *more, eps
        ctx.types = [None if t is None or t.dtype == F32 else t.dtype for t in (scale, x0_scale, y_weight, weight)]
        ctx.set_materialize_grads(False)
        return _forward(tensors, *more, eps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dh):
        grads = _backward(dout, dh, ctx.saved_tensors, *ctx.more, ctx.needs_input_grad)
        for i, t in zip((3, 4, 6, 7), ctx.types):
            if t is not None and grads[i] is not None:
                grads[i] = grads[i].to(t)
        return (*grads, None, None, None)


def residual_norm(x, y=None, x0=None, scale=None, x0_scale=None, gate=None, y_weight=None, weight=None, norm_y=False, dtype=None,
                  eps=EPS):
    """(x', h): the residual stream x [..., D] with a block's output y on it, and its norm, which the next block reads:

        b  = y,  or with norm_y  y / sqrt(mean y^2 + eps) y_weight
        x' = scale (x + gate b) + x0_scale x0
        h  = x' / sqrt(mean x'^2 + eps) weight

    What is None is left out. x and x0 (the stream's beginning, mixed in again) are float32 or bfloat16 and so is x'; y and h are
    of x's type, or bfloat16 beside a float32 stream (`dtype`: h's type where there is no y). scale and x0_scale are tensors of
    one value; y_weight and weight [D]; gate is [D], of x's shape (a gate per token), or as x with ones from some dimension on
    ([batch, 1, D]: one per sequence), float32 or bfloat16. D is at most 8192. Everything is computed in fp32 and rounded once; h
    is the norm of x' before x' is rounded. Rows may lie at any distance from each other. Differentiable in every tensor (once);
    gradients of what several rows share are summed in fp32 in a fixed order, the two scalars' in fp64."""
    if torch.compiler.is_compiling():
        return torch.ops.noise_amd.residual_norm(x, y, x0, scale, x0_scale, gate, y_weight, weight, bool(norm_y), dtype,
                                                 float(eps))
    if torch.is_grad_enabled():
        for t in (x, y, x0, scale, x0_scale, gate, y_weight, weight):
            if isinstance(t, torch.Tensor) and t.requires_grad:
                return _Residual.apply(x, y, x0, scale, x0_scale, gate, y_weight, weight, bool(norm_y), dtype, float(eps))
    return forward(x, y, x0, scale, x0_scale, gate, y_weight, weight, bool(norm_y), dtype, float(eps))
