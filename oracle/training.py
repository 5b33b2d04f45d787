"""The ends of a training step in 64 bits, from their definitions: the residual stream between two blocks, the cross entropy of a
linear head, clipping. Gradients by differentiating the definitions."""
import math

import torch


def rms_norm(x, weight=None, eps=0.0):
    n = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    return n if weight is None else n * weight


def residual(x, y=None, x0=None, scale=None, x0_scale=None, gate=None, y_weight=None, weight=None, norm_y=False, eps=0.0):
    """(x', h) of double tensors"""
    t = x
    if y is not None:
        b = rms_norm(y, y_weight, eps) if norm_y else y
        t = t + (b if gate is None else gate * b)
    if scale is not None:
        t = scale * t
    if x0 is not None:
        t = t + (x0 if x0_scale is None else x0_scale * x0)
    return t, rms_norm(t, weight, eps)


def linear_cross_entropy(x, weight, targets, vocab, softcap=None, token_weight=None):
    """(losses [R], dx, dweight) of 2-D x and weight: the gradients of sum token_weight * loss. Rows without a target in
    0 .. vocab - 1 take no part, whatever stands in them."""
    loss = torch.zeros(len(x), dtype=torch.float64, device=x.device)
    dx, dw = torch.zeros(x.shape, dtype=torch.float64, device=x.device), torch.zeros(weight.shape, dtype=torch.float64, device=x.device)
    live = ((targets >= 0) & (targets < vocab)).nonzero()[:, 0]
    if not len(live):
        return loss, dx, dw
    with torch.enable_grad():
        xs, w = x[live].double().requires_grad_(), weight[:vocab].double().requires_grad_()
        z = xs @ w.t()
        if softcap is not None:
            z = softcap * torch.tanh(z / softcap)
        part = torch.logsumexp(z, -1) - z.gather(1, targets[live].long()[:, None])[:, 0]
        by = torch.ones_like(part) if token_weight is None else token_weight[live].double()
        dx[live], dw[:vocab] = torch.autograd.grad((part * by).sum(), (xs, w))
    loss[live] = part.detach()
    return loss, dx, dw


def clip(gradients, max_norm):
    """(norm, clipped gradients)"""
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in gradients))
    factor = max_norm / (norm + 1e-6)
    if factor >= 1:
        factor = 1.0
    return norm, [g.double() * factor for g in gradients]
