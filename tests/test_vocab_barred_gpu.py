"""linear_cross_entropy where a column of the weight, beside a column of ones in x, takes vocabulary entries out: single ones, and whole
runs of 128 of them. Such an entry counts as 0, so losses and gradients are those of the other entries alone, within their bounds
(test_vocab_gpu's): what is added for it is 0 exactly. In fp32 a value of 200 beside the others' 2 adds 2^-38 200 dim |x| to a logit's
error, less than a hundredth of what the bound holds of it, which is multiplied by 1.01."""
import math

import pytest
import torch
from test_vocab_gpu import BF16, DEV, F32, bounds, make

from oracle import training as oracle

pytestmark = pytest.mark.gpu
INF = math.inf
LOWEST = torch.finfo(BF16).min
# few tokens; tokens and entries whose logits come in tiles, the last one of a single entry among them
SIZES = [(30, 1000, 64), (300, 1000, 72), (6000, 5003, 64), (60000, 129, 64)]
RUNS = {'last': lambda V: [(V - 1, V)], 'runs': lambda V: [(0, 128)] if V < 256 else [(128, 256), (V // 128 * 128 - 128, V)],
        'first': lambda V: [(0, 128)], 'scattered': lambda V: [(v, v + 1) for v in range(0, V, 17)]}


def off_bounds(name, a, b, c):
    off = (a.double() - b).abs()
    assert (off <= 1.01 * c).all(), (name, (off - 1.01 * c).max(), off.max(), b.abs().max())


def check(R, V, D, dtype, value, runs):
    from noise_amd.vocab import linear_cross_entropy, linear_cross_entropy_grad
    x, weight, targets, w = make(R, V, D, dtype, V)
    keep = torch.ones(V, dtype=torch.bool, device=DEV)
    for a, b in RUNS[runs](V):
        keep[a:b] = False
    kept = keep.nonzero()[:, 0]
    targets = kept[targets % len(kept)]
    x[:, -1] = 1
    weight[:, -1] = 0
    alone = weight[keep]
    place = torch.cumsum(keep, 0)[targets] - 1
    want = oracle.linear_cross_entropy(x, alone, place, len(kept), None, w)
    limit = bounds(x, alone, place, w, len(kept), None, *want)
    weight[~keep, -1] = value
    with torch.no_grad():
        off_bounds('alone', linear_cross_entropy(x, weight, targets), want[0], limit[0])
    leaves = x.detach().requires_grad_(), weight.detach().requires_grad_()
    loss = linear_cross_entropy(*leaves, targets)
    for how, got in (('one call', linear_cross_entropy_grad(x, weight, targets, w)),
                     ('backward', (loss.detach(), *torch.autograd.grad(loss, leaves, w)))):
        off_bounds((how, 'loss'), got[0], want[0], limit[0])
        # (the column itself: 0 times an infinity, as in a product of the probabilities and the weight)
        end = D - 1 if math.isinf(value) else D
        off_bounds((how, 'dx'), got[1][:, :end], want[1][:, :end], limit[1][:, :end])
        off_bounds((how, 'dweight'), got[2][keep], want[2], limit[2])
        assert not got[2][~keep].any(), how


@pytest.mark.parametrize('runs', RUNS)
@pytest.mark.parametrize('value', [-200.0, -1e10, LOWEST, -INF])
def test_entries_taken_out(value, runs):
    for size in SIZES:
        check(*size, BF16, value, runs)


@pytest.mark.parametrize('runs', RUNS)
def test_entries_taken_out_fp32(runs):
    for size in SIZES:
        check(*size, F32, -200.0, runs)


@pytest.mark.parametrize('dtype,shift', [(BF16, 1e5), (BF16, -1e5), (F32, 1e5), (F32, -1e5), (BF16, 1e10), (BF16, -1e10)])
def test_logits_with_a_large_common_part(dtype, shift):
    """Within the bounds, which grow with the logits, while these say anything of the losses; further out at least finite."""
    from noise_amd.vocab import linear_cross_entropy, linear_cross_entropy_grad
    for R, V, D in SIZES[:3]:
        x, weight, targets, w = make(R, V, D, dtype, V)
        x[:, -1] = 1
        weight[:, -1] = shift
        leaves = x.detach().requires_grad_(), weight.detach().requires_grad_()
        loss = linear_cross_entropy(*leaves, targets)
        one, two = linear_cross_entropy_grad(x, weight, targets, w), (loss.detach(), *torch.autograd.grad(loss, leaves, w))
        assert all(torch.isfinite(t).all() for t in (*one, *two))
        if abs(shift) < 1e6:
            want = oracle.linear_cross_entropy(x, weight, targets, V, None, w)
            limit = bounds(x, weight, targets, w, V, None, *want)
            for got in (one, two):
                for name, a, b, c in zip(('loss', 'dx', 'dweight'), got, want, limit):
                    off_bounds(name, a, b, c)


@pytest.mark.parametrize('runs', RUNS)
def test_infinite_weights_fp32(runs):
    """Held as two values too: the infinity must meet one value of x alone, whose sign is x's."""
    for size in SIZES:
        check(*size, F32, -INF, runs)


@pytest.mark.parametrize('cap', [None, 80.0])
@pytest.mark.parametrize('R,V,D', [(75, 35534, 391), (168, 37229, 772), (259, 30247, 200), (3000, 9001, 64)])
def test_improbable_entries(R, V, D, cap):
    """Logits some 80 apart: an improbable entry's gradients are as near as another's, in the call that keeps the exponentials as well,
    whose 2^-11 is counted beside the bounds' 2^-8. That call may leave out exponentials below 2^-62 of the largest of 128 entries."""
    from noise_amd.vocab import linear_cross_entropy, linear_cross_entropy_grad
    x, weight, targets, w = make(R, V, D, BF16, R, V + 5, scale=10.0)
    want = oracle.linear_cross_entropy(x, weight, targets, V, cap, w)
    limit = [1.125 * b for b in bounds(x, weight, targets, w, V, cap, *want)]
    leaves = x.detach().requires_grad_(), weight.detach().requires_grad_()
    loss = linear_cross_entropy(*leaves, targets, vocab=V, softcap=cap)
    most = 2.0 ** -62 * w.double()
    left = 0.0, 128 * most[:, None] * weight[:V].double().abs().max(), most @ x.double().abs()
    for how, got in (('backward', (loss.detach(), *torch.autograd.grad(loss, leaves, w))),
                     ('one call', linear_cross_entropy_grad(x, weight, targets, w, vocab=V, softcap=cap))):
        for name, a, b, c, d in zip(('loss', 'dx', 'dweight'), got, want, limit, left):
            off = (a.double() - b).abs()
            c = c + d if how == 'one call' else c
            assert (off <= c).all(), (how, name, (off - c).max(), off.max(), int((off > c).sum()), b.numel())
