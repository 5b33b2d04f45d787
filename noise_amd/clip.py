"""Clipping of a training step's gradients.

  clip_gradients(gradients, max_norm)   their global norm, and the gradients scaled to a bound on it, in place

The call is a torch.ops.noise_amd operator too, which compiled callers trace. Eggroll.step takes a bound as an option.
"""
from array import array

import torch

from . import _lib
from .sinks import F32, TYPES, _call, _no_gradients, _no_tangents


def clip(fn, gradients, max_norm):
    gradients = [g for g in gradients if g is not None]
    if not gradients:
        raise ValueError(f'{fn}: no gradients')
    if not max_norm >= 0:
        raise ValueError(f'{fn}: max_norm must be 0 or more, got {max_norm}')
    device, flat = gradients[0].device, []
    for g in gradients:
        if g.dtype not in TYPES:
            raise ValueError(f'{fn}: bfloat16 or float32 gradients, got {g.dtype}')
        if g.device != device:
            raise ValueError(f'{fn}: gradients on {device} and {g.device}')
        # (elements in any order: a transposed gradient is as good as another)
        if not g.is_contiguous() and not torch.ops.aten.is_non_overlapping_and_dense(g):
            raise ValueError(f'{fn}: a gradient of shape {tuple(g.shape)} and strides {g.stride()} has gaps or overlaps itself')
        flat += (g.data_ptr(), g.numel(), TYPES[g.dtype])
    _no_tangents(fn, *gradients)
    _no_gradients(fn, *gradients)
    table = array('q', flat)
    need = _lib.lib().noise_clip_workspace_bytes(len(gradients))
    norm = torch.empty((), dtype=F32, device=device)
    work = torch.empty(need, dtype=torch.uint8, device=device)
    _call('noise_clip_gradients', device, table.buffer_info()[0], len(gradients), float(max_norm),
          norm.data_ptr(), work.data_ptr(), need)
    if max_norm != float('inf'):
        torch.autograd.graph.increment_version(gradients)
    return norm


def clip_gradients(gradients, max_norm):
    """The norm of all gradients taken together (fp32, without dimensions), and the gradients scaled in place where it is above
    `max_norm`:

        norm = sqrt(sum of all squares),  g <- g min(1, max_norm / (norm + 1e-6))

    `gradients` are bfloat16 and float32 tensors of any sizes on one device (None is left out), their elements in any order but
    without gaps, no two of them in the same memory. Squares are summed in 64 bits, in a fixed order. The norm is rounded to
    float32 (infinite past its range, where the gradients are scaled as ever), the factor to 24 bits, its products to float32 and
    then to the gradients' type. An infinite `max_norm` leaves the gradients as they are. A NaN among them makes the norm and all
    of them NaN; an infinity makes the norm infinite, the finite ones 0 and the infinite ones NaN. Nothing waits for the device:
    the norm stays on it."""
    if torch.compiler.is_compiling():
        return torch.ops.noise_amd.clip_gradients([g for g in gradients if g is not None], float(max_norm))
    return clip('clip_gradients', gradients, max_norm)
