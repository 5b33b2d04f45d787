"""The second part of dZ beside bf16 operands of up to 32 tokens. A sum of two bf16 values is off by 2^-16 of itself at most (the rest,
2^-8 of it or less, rounded by 2^-8), one value by 2^-8. So dx and dW are bounded as in test_vocab_gpu, but with 2^-16 in place of that
2^-8, and with half a step of bf16 at the result's own power of two for their rounding, which is all that is left to see: a part that
is lost or read as zeros moves results by up to half a step more."""
import pytest
import torch
from test_vocab_gpu import BF16, DEV, HALF, bounds, make

from oracle import training as oracle


def half_step(v):
    """Of bf16, 8 bits, at the power of two of |v|"""
    return torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=1e-37))) - 8)


def limits(x, weight, targets, w, V, cap, want):
    """The bounds of dx and dW before they are rounded, and with it"""
    _, ex, ew = bounds(x, weight, targets, w, V, cap, *want)
    used = (targets >= 0) & (targets < V)
    xs, ws = torch.where(used[:, None], x, 0).double(), weight[:V].double()
    z, slope = xs @ ws.t(), 1.0
    if cap:
        z = cap * torch.tanh(z / cap)
        slope = 1 - (z / cap) ** 2
    p = torch.softmax(z, -1)
    p.scatter_add_(1, torch.where(used, targets, 0).long()[:, None], -torch.ones_like(p[:, :1]))
    dz = (torch.where(used, w.double(), 0.0)[:, None] * p * slope).abs()
    out = []
    for e, value, size in ((ex, want[1], dz @ ws.abs()), (ew[:V], want[2][:V], dz.t() @ xs.abs())):
        e = (e - HALF[BF16] * value.abs()) / (1 + HALF[BF16]) - (2.0 ** -8 - 2.0 ** -16) * size
        out.append(e + half_step(value.abs() + e))
    return out


@pytest.mark.gpu
@pytest.mark.parametrize('cap', [None, 15.0])
@pytest.mark.parametrize('V,D', [(700, 64), (2000, 203), (131, 1000)])
@pytest.mark.parametrize('R', [1, 2, 15, 16, 17, 31, 32])
def test_second_part(R, V, D, cap):
    from noise_amd.vocab import linear_cross_entropy, linear_cross_entropy_grad
    for seed in range(3):
        x, weight, targets, w = make(R, V, D, BF16, seed, V + 3, masked=R > 2)
        want = oracle.linear_cross_entropy(x, weight, targets, V, cap, w)
        ex, ew = limits(x, weight, targets, w, V, cap, want)
        leaves = x.detach().requires_grad_(), weight.detach().requires_grad_()
        both = torch.autograd.grad(linear_cross_entropy(*leaves, targets, vocab=V, softcap=cap), leaves, w)
        for how, (dx, dw) in (('one call', linear_cross_entropy_grad(x, weight, targets, w, vocab=V, softcap=cap)[1:]), ('backward', both)):
            for name, a, b, c in (('dx', dx, want[1], ex), ('dweight', dw[:V], want[2][:V], ew)):
                off = (a.double() - b).abs()
                assert (off <= c).all(), (how, name, (off - c).max(), (off / c).max())
