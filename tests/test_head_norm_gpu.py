"""qk_norm_rotary and its gradients against the 64-bit definition.

Bounds: a result is a sum of two products; each carries the row's 1 / rms (a sum of 128 squares in 3 + 8 levels of lanes and
16 terms in turn, halved by the root, 1 ulp for the root), the weight and the table: fewer than 32 roundings of 2^-24 of
the products' absolute sum, then the output's half step. The input gradient adds a mean of 128 products of the same kind."""
import math

import pytest
import torch

from oracle import sinks as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda', 0)
EPS = torch.finfo(torch.float32).eps
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
F = 2.0 ** -24


def tables(n, D):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    return a.cos().float().to(DEV), a.sin().float().to(DEV)


def make(B, T, H, Hk, D, dtype, seed, weights=True):
    g = torch.Generator(DEV).manual_seed(seed)
    t = [torch.randn(B, T, h, D, device=DEV, generator=g).to(dtype) for h in (H, Hk, H, Hk)]
    t[0] *= torch.linspace(0.01, 3, T, device=DEV)[:, None, None].to(dtype)
    w = [1 + 0.3 * torch.randn(D, device=DEV, generator=g) for _ in range(2)] if weights else [None, None]
    return t, w


def check_all(q, k, dq, dk, cos, sin, w, start=None, eps=EPS):
    from noise_amd.sinks import qk_norm_rotary
    leaves = [t.detach().requires_grad_() for t in (q, k, *w) if t is not None]
    outs = qk_norm_rotary(*leaves[:2], cos, sin, *(leaves[2:] or [None, None]), start=start, eps=eps)
    grads = torch.autograd.grad(outs, leaves, (dq, dk))
    half = HALF[q.dtype]
    for i, (x, dy) in enumerate(((q, dq), (k, dk))):
        x64 = x.double().requires_grad_()
        w64 = None if w[i] is None else w[i].double().requires_grad_()
        want, scale = oracle.norm_rotary(x64, w64, cos, sin, start, eps)
        off = (outs[i].detach().double() - want.detach()).abs()
        assert outs[i].dtype == q.dtype and outs[i].is_contiguous()
        assert (off <= half * want.detach().abs() + 32 * F * scale).all(), off.max()
        wants = torch.autograd.grad(want, [x64] if w64 is None else [x64, w64], dy.double())
        # dx = r (g - n mean(g n)): every term is below r max|w dy| (|c| + |s|) (1 + max|n|) <= the bound below
        r = torch.rsqrt(x.double().square().mean(-1, keepdim=True) + eps)
        n = x.double() * r
        g = 2 ** 0.5 * dy.double().abs().amax(-1, keepdim=True) * (1 if w64 is None else w[i].double().abs().max())
        bound = half * wants[0].abs() + 64 * F * r * g * (1 + n.abs() * n.abs().mean(-1, keepdim=True))
        off = (grads[i].double() - wants[0]).abs()
        assert (off <= bound).all(), (off - bound).max()
        if w64 is not None:
            # a sum over the rows in two levels: rows / 512 / 64 terms in turn, then 64, then 512 / 8 and 8, of
            # products with up to 16 roundings each
            total = (2 ** 0.5 * dy.double().abs().amax(-1, keepdim=True) * n.abs()).sum((0, 1, 2))
            off = (grads[2 + i].double() - wants[1]).abs()
            assert (off <= (200 * F) * total + 1e-30).all(), (off / total).max()
    return outs, grads


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('B,T,H,Hk', [(1, 1, 1, 1), (2, 7, 4, 2), (3, 33, 8, 8), (1, 257, 5, 1), (4, 100, 16, 4),
                                      (2, 1111, 8, 2)])
def test_shapes(B, T, H, Hk, D, dtype):
    for weights in (True, False):
        t, w = make(B, T, H, Hk, D, dtype, T, weights)
        check_all(*t, *tables(T, D), w)


def test_many_rows():
    """More rows than the partial sums' workgroups take at once."""
    t, w = make(4, 2048, 16, 4, 64, torch.bfloat16, 1)
    check_all(*t, *tables(2048, 64), w)


@pytest.mark.parametrize('wide', [torch.int32, torch.int64])
def test_positions(wide):
    """Positions before and past the tables: zeros, and no gradient from there."""
    t, w = make(5, 20, 4, 2, 64, torch.float32, 2)
    start = torch.tensor([0, 31, 40, -5, 50], device=DEV, dtype=wide)
    outs, grads = check_all(*t, *tables(50, 64), w, start)
    assert (outs[0][2, 10:] == 0).all() and (outs[0][3, :5] == 0).all() and (outs[1][4] == 0).all()
    assert (grads[0][2, 10:] == 0).all() and (grads[1][4] == 0).all()
    if wide == torch.int64:
        check_all(*t, *tables(50, 64), w, torch.tensor([2 ** 40, -2 ** 40, 1, 2, 2 ** 63 - 21], device=DEV))


def test_rows_outside_the_tables_may_hold_anything():
    from noise_amd.sinks import qk_norm_rotary
    t, w = make(2, 6, 2, 2, 64, torch.bfloat16, 3)
    for x in t:
        x[1] = math.nan
    leaves = [x.detach().requires_grad_() for x in (*t[:2], *w)]
    outs = qk_norm_rotary(*leaves[:2], *tables(6, 64), *leaves[2:], start=torch.tensor([0, -6], device=DEV))
    for x in (*outs, *torch.autograd.grad(outs, leaves, t[2:])):
        assert torch.isfinite(x).all()


def test_strides_zeros_and_eps():
    B, T, D = 2, 40, 64
    g = torch.Generator(DEV).manual_seed(4)
    qkv = torch.randn(B, T, 12, D, device=DEV, generator=g)
    dy = torch.randn(B, T, 1, D, device=DEV, generator=g)
    cos, sin = tables(T, D)
    for x in (qkv, qkv.bfloat16()):
        q, k, _ = x.split([6, 3, 3], 2)
        check_all(q, k, dy.to(x.dtype).expand(B, T, 6, D), dy.to(x.dtype).expand(B, T, 3, D), cos, sin, [None, None])
        t = x.transpose(1, 2).contiguous().transpose(1, 2)
        check_all(t[:, :, :6], t[:, :, 6:9], q, k, cos, sin, [None, None], eps=1e-2)
    odd = torch.randn(B, T, 4, D + 1, device=DEV, generator=g)[..., 1:]
    check_all(odd, odd[:, :, :2], odd, odd[:, :, 2:], cos, sin, [None, None])
    from noise_amd.sinks import qk_norm_rotary
    zero = torch.zeros(1, 3, 2, D, device=DEV)
    out, _ = qk_norm_rotary(zero, zero, cos, sin)
    assert (out == 0).all()


def test_against_the_model_layer():
    """Without weights: the rotation and norm of utils/model.py:88-94 (rotary, then norm) on the model's own tables."""
    from noise_amd.model import rotary_tables
    from noise_amd.sinks import qk_norm_rotary
    from oracle import model as om
    t, _ = make(2, 300, 8, 8, 64, torch.float32, 5)
    cos, sin = rotary_tables(300)
    q, k = qk_norm_rotary(*t[:2], cos.to(DEV), sin.to(DEV))
    for got, x in ((q, t[0]), (k, t[1])):
        want = om.norm(om.apply_rotary_emb(x.cpu().double(), cos.double(), sin.double()))
        # (bf16 tables do not turn rows exactly: their squares sum to 1 within 2^-8, which the norm after the turn removes)
        assert (got.cpu().double() - want).abs().max() <= 2.0 ** -7 * want.abs().max()


def test_gradients_against_differences():
    from noise_amd.sinks import qk_norm_rotary
    t, w = make(1, 5, 2, 1, 64, torch.float32, 6)
    cos, sin = tables(5, 64)
    leaves = [x.detach().requires_grad_() for x in (*t[:2], *w)]
    grads = torch.autograd.grad(qk_norm_rotary(*leaves[:2], cos, sin, *leaves[2:]), leaves, t[2:])
    for i, grad in enumerate(grads):
        d = grad.double()
        h = 1e-5 / d.abs().max()

        def at(step):
            x = [y.double() + (step * d if n == i else 0) for n, y in enumerate((*t[:2], *w))]
            return sum((oracle.norm_rotary(x[j], x[2 + j], cos, sin, None, EPS)[0] * t[2 + j].double()).sum() for j in (0, 1))
        slope = (at(h) - at(-h)) / (2 * h)
        assert abs(slope - d.square().sum()) <= 1e-5 * d.square().sum()


def test_repeats_graphs_and_the_operator():
    from noise_amd.sinks import norm_backward, norm_forward, qk_norm_rotary
    t, w = make(3, 500, 8, 2, 64, torch.bfloat16, 7)
    cos, sin = tables(500, 64)
    step = lambda: (*norm_forward(*t[:2], cos, sin, *w, None, EPS),
                    *norm_backward(t[2], t[3], *t[:2], cos, sin, *w, None, EPS))
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        t[0].mul_(-0.5)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want))
    leaves = [x.detach().requires_grad_() for x in (*t[:2], *w)]
    y = torch.ops.noise_amd.qk_norm_rotary(*leaves[:2], cos, sin, *leaves[2:], None, EPS)
    got = (*y, *torch.autograd.grad(y, leaves, t[2:]))
    assert all(torch.equal(x, z) for x, z in zip(got, step()))
    half = [x.detach().requires_grad_() for x in (*t[:2], w[0].bfloat16(), w[1].bfloat16())]
    y = qk_norm_rotary(*half[:2], cos, sin, *half[2:])
    assert [g.dtype for g in torch.autograd.grad(y, half, t[2:])] == [torch.bfloat16] * 4
