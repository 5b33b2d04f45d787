"""linear_cross_entropy over more tokens and vocabulary entries than one piece of dZ holds (2 GiB: 768 tokens of 1300001 entries in
bf16, 256 in fp32, in pieces of one size: 512 and 256): pieces that masks leave empty or in part, gradients in one call and through
autograd, soft caps, a weight with rows past the vocabulary.

Bounds as test_vocab_gpu's, with the largest error ez of any logit: F (dim / 16 + 24) of its terms' sizes (fp32: three times the steps,
2^-21 of them and 2^-38 dim of the tensors' largest), and 2^-21 of the cap. A loss: 2 ez + F (80 + V / 128 + 8 A). dZ is off by its
exponent's error, the slope's 4 ez / cap and its rounding, 2^-8 or 2^-21, of itself and in fp32 by 2^-38 of the largest token's weight;
dx by that of its terms, their sum's V / 16 + 88 steps (three times V / 16 in fp32) and half a step of its own; dW likewise with the
tokens for V. One bf16 call may leave out exponentials below 2^-62 of their segment's largest, which sums up to 2^-55 of a token's weight
(128 entries a segment, the segments' largest at most 1 together) in dx, and counts the others' 2^-11 beside 2^-8."""
import math

import pytest
import torch
from test_vocab_gpu import BF16, DEV, F, F32, HALF, make

pytestmark = pytest.mark.gpu
V, D = 1300001, 8


def want_of(x, weight, targets, w, cap):
    """Losses, dx and the sizes of its terms, dweight and the sizes of its, in 64 bits, some tokens at a time; the largest size of a
    logit's terms, the largest logit, the smallest slope"""
    R, ws = len(x), weight[:V].double()
    loss = torch.zeros(R, dtype=torch.float64, device=DEV)
    dx, size = torch.zeros(R, D, dtype=torch.float64, device=DEV), torch.zeros(R, D, dtype=torch.float64, device=DEV)
    dw, size_w = torch.zeros_like(ws), torch.zeros_like(ws)
    N, A, least = 0.0, 0.0, 1.0
    for rows in ((targets >= 0) & (targets < V)).nonzero()[:, 0].split(100):
        if not len(rows):
            break
        xs, at = x[rows].double(), targets[rows]
        N = max(N, float((xs.abs() @ ws.abs().t()).max()))
        z = xs @ ws.t()
        if cap:
            z = torch.tanh(z / cap) * cap
        A = max(A, float(z.abs().max()) + math.log(V) + 1)
        log_p = torch.log_softmax(z, -1)
        loss[rows] = -log_p.gather(1, at[:, None])[:, 0]
        p = log_p.exp_()
        p[torch.arange(len(rows), device=DEV), at] -= 1
        p *= w[rows].double()[:, None]
        if cap:
            slope = z.div_(cap).square_().neg_().add_(1)
            least = min(least, float(slope.min()))
            p *= slope
            del slope
        del z
        dx[rows], size[rows] = p @ ws, p.abs() @ ws.abs()
        dw += p.t() @ xs
        size_w += p.abs().t() @ xs.abs()
        del log_p, p
    return loss, dx, size, dw, size_w, N, A, least


@pytest.mark.parametrize('cap', [None, 15.0])
@pytest.mark.parametrize('live', [0, 1, 256, 300, 512, 600, 900])
@pytest.mark.parametrize('dtype', [BF16, F32])
def test_masked_pieces(dtype, live, cap):
    """The tokens with a target, `live` of 900, fill some pieces; the others hold NaN."""
    from noise_amd.vocab import linear_cross_entropy, linear_cross_entropy_grad
    R, split = 900, dtype == F32
    x, weight, targets, w = make(R, V, D, dtype, live, V + 3)
    gone = torch.randperm(R, device=DEV, generator=torch.Generator(DEV).manual_seed(live))[live:]
    targets[gone] = torch.tensor([-100, V, V + 2], device=DEV)[gone % 3]
    top = float(x.abs().max() * weight[:V].abs().max())
    x[gone], w[gone] = float('nan'), float('nan')
    loss64, dx64, size, dw64, size_w, N, A, least = want_of(x, weight, targets, w, cap)
    ez = F * ((3 if split else 1) * D / 16 + 24) * N + (2.0 ** -21 * N + 2.0 ** -38 * D * top if split else 0) + 2.0 ** -21 * (cap or 0)
    eloss = 2 * ez + F * (80 + V / 128 + 8 * A)
    each = ez + eloss + (4 * ez / cap / least if cap else 0) + 12 * F + (2.0 ** -21 if split else 2.0 ** -8 + 2.0 ** -11)
    steps = F * ((3 if split else 1) * V / 16 + 88)
    most, far = float(w.nan_to_num().max()), float(x.nan_to_num().abs().max())
    rest = most * float(weight[:V].abs().max()) * (2.0 ** -38 * V if split else 2.0 ** -55)
    rest_w = most * far * live * 2.0 ** (-38 if split else -62)
    leaves = x.detach().requires_grad_(), weight.detach().requires_grad_()
    for how in ('one call', 'backward'):
        if how == 'one call':
            loss, dx, dw = linear_cross_entropy_grad(x, weight, targets, w, vocab=V, softcap=cap)
        else:
            by = linear_cross_entropy(*leaves, targets, vocab=V, softcap=cap)
            loss, (dx, dw) = by.detach(), torch.autograd.grad(by, leaves, w)
            del by
        assert ((loss - loss64).abs() <= eloss).all(), how
        assert not loss[gone].any() and not dx[gone].any() and not dw[V:].any()
        off = (dx.double() - dx64).abs()
        assert (off <= (each + steps) * size + rest + HALF[dtype] * dx64.abs()).all(), (how, (off / size.clamp(min=1e-30)).max())
        off = (dw[:V].double() - dw64).abs()
        assert (off <= (each + F * ((3 if split else 1) * R / 16 + 88)) * size_w + rest_w + HALF[dtype] * dw64.abs()).all(), how
        del loss, dx, dw, off
