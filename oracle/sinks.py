"""The attention operators in 64 bits, from their definitions, on whatever device the inputs are on.

  norm_rotary       a head norm with weights, rotated (utils/model.py:46-47, 55-58)
  attend, attend_grads   a window and first tokens that stay visible, over a padded batch; with what bf16 weights add
  decode            the same of new tokens against a cache
"""
import math

import torch

F64 = torch.float64


def norm_rotary(x, w, cos, sin, start, eps):
    """x [B, T, H, D], positions start[b] + t; zeros outside the tables. The second result bounds the roundings' scale:
    the sum of the absolute values that each element adds up."""
    B, T, H, D = x.shape
    pos = torch.arange(T, device=x.device) + (0 if start is None else start.long()[:, None])
    pos = pos.expand(B, T)
    inside = ((pos >= 0) & (pos < cos.shape[0]))[..., None, None]
    at = pos.clamp(0, cos.shape[0] - 1)
    c, s = cos.double()[at][:, :, None], sin.double()[at][:, :, None]
    u = x.double() * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + eps)
    if w is not None:
        u = u * w.double()
    u1, u2 = u[..., :D // 2], u[..., D // 2:]
    y = torch.cat([u1 * c + u2 * s, u2 * c - u1 * s], -1)
    scale = torch.cat([(u1 * c).abs() + (u2 * s).abs(), (u2 * c).abs() + (u1 * s).abs()], -1)
    return y * inside, (scale * inside).detach()


def visible(i, j, window, sinks):
    """Does the query at position i [.., 1] see key j?"""
    return (j <= i) & ((i - j <= window) | (j < sinks))


def attend(q, k, v, window, sinks, lengths=None):
    """(out, sum of p |v|) of [B, T, H, D] inputs, in 64 bits; zeros past the lengths."""
    B, T, H, D = q.shape
    G = H // k.shape[2]
    out = torch.zeros(q.shape, dtype=F64, device=q.device)
    weight = torch.zeros_like(out)
    for b in range(B):
        n = T if lengths is None else min(T, max(0, int(lengths[b])))
        if n == 0:
            continue
        j = torch.arange(n, device=q.device)
        hidden = ~visible(j[:, None], j, window, sinks)
        for h in range(H):
            qh, kh, vh = q[b, :n, h].double(), k[b, :n, h // G].double(), v[b, :n, h // G].double()
            p = torch.softmax((qh @ kh.t() / math.sqrt(D)).masked_fill(hidden, -math.inf), -1)
            out[b, :n, h] = p @ vh
            weight[b, :n, h] = p @ vh.abs()
    return out, weight


def attend_grads(q, k, v, dout, window, sinks, lengths=None, unit=2.0 ** -8):
    """(dq, dk, dv) in 64 bits, and for each how far off it may be when the weights p, the scores' gradients and the
    output that goes into sum(dout * out) are rounded to a type whose half step is `unit`, and the results too."""
    B, T, H, D = q.shape
    G, scale = H // k.shape[2], 1 / math.sqrt(D)
    grads = [torch.zeros(t.shape, dtype=F64, device=q.device) for t in (q, k, v)]
    slack = [torch.zeros_like(t) for t in grads]
    for b in range(B):
        n = T if lengths is None else min(T, max(0, int(lengths[b])))
        if n == 0:
            continue
        j = torch.arange(n, device=q.device)
        hidden = ~visible(j[:, None], j, window, sinks)
        for h in range(H):
            qh, kh, vh = q[b, :n, h].double(), k[b, :n, h // G].double(), v[b, :n, h // G].double()
            do = dout[b, :n, h].double()
            p = torch.softmax((qh @ kh.t() * scale).masked_fill(hidden, -math.inf), -1)
            o = p @ vh
            ds = p * (do @ vh.t() - (do * o).sum(-1, keepdim=True))
            grads[0][b, :n, h] = scale * ds @ kh
            grads[1][b, :n, h // G] += scale * ds.t() @ qh
            grads[2][b, :n, h // G] += p.t() @ do
            off = unit * (ds.abs() + p * (do.abs() * (o.abs() + p @ vh.abs())).sum(-1, keepdim=True))
            slack[0][b, :n, h] = scale * off @ kh.abs()
            slack[1][b, :n, h // G] += scale * off.t() @ qh.abs()
            slack[2][b, :n, h // G] += unit * p.t() @ do.abs()
    return grads, [s + unit * g.abs() for s, g in zip(slack, grads)]


def decode(q, k_cache, v_cache, start, window, sinks):
    """(out, sum of p |v|) of new tokens at positions start[b] + t; zeros where no slot is seen."""
    B, T, H, D = q.shape
    S, Hk = k_cache.shape[1:3]
    out = torch.zeros(q.shape, dtype=F64, device=q.device)
    weight = torch.zeros_like(out)
    j = torch.arange(S, device=q.device)
    for b in range(B):
        for t in range(T):
            seen = visible(int(start[b]) + t, j, window, sinks)
            if not bool(seen.any()):
                continue
            kb, vb = k_cache[b, seen].double(), v_cache[b, seen].double()
            for h in range(H):
                p = torch.softmax(kb[:, h * Hk // H] @ q[b, t, h].double() / math.sqrt(D), -1)
                out[b, t, h] = p @ vb[:, h * Hk // H]
                weight[b, t, h] = p @ vb[:, h * Hk // H].abs()
    return out, weight
