"""The training operators together: a step of a small model of this kind with exact gradients, out of residual_norm, qk_norm_rotary,
sink_attention, linear_cross_entropy and clip_gradients, and its head's form with the gradients in one call.

The step is compared with itself in 64 bits. What bf16 operands may cost it is taken from the same step in elementary torch
operations on the same roundings of operands (products of bf16 values in fp32, results rounded where the operators round): the
operators' gradients may be off by twice what that step's are."""
import math

import pytest
import torch

from oracle import training as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda', 0)
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
LAYERS, HEADS, DIM, WIDTH, VOCAB, CAP = 3, 4, 64, 256, 600, 15.0


def parameters(seed=0):
    g = torch.Generator(DEV).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device=DEV, generator=g)
    p = dict(wte=randn(VOCAB, WIDTH), head=randn(VOCAB, WIDTH) * 2 / math.sqrt(WIDTH), resid=1 - 0.1 * torch.rand(LAYERS, device=DEV, generator=g),
             x0=0.1 * torch.rand(LAYERS, device=DEV, generator=g), last=1 + 0.1 * randn(WIDTH))
    for i in range(LAYERS):
        for n in 'qkvo':
            p[f'{i}.{n}'] = randn(WIDTH, WIDTH) / math.sqrt(WIDTH)
        p[f'{i}.fc'], p[f'{i}.proj'] = randn(2 * WIDTH, WIDTH) / math.sqrt(WIDTH), randn(WIDTH, 2 * WIDTH) / math.sqrt(2 * WIDTH)
        p[f'{i}.gate'], p[f'{i}.after'] = 0.5 + 0.1 * randn(WIDTH), 1 + 0.1 * randn(WIDTH)
    return p


def tables(T, dtype=F32):
    inv = 10000.0 ** (-torch.arange(0, DIM, 2, device=DEV, dtype=F64) / DIM)
    angle = torch.arange(T, device=DEV, dtype=F64)[:, None] * inv
    return angle.cos().to(dtype), angle.sin().to(dtype)


class Own:
    """The framework's operators, under autocast's types: fp32 stream, bf16 branches"""

    def round(self, t):
        return t.to(BF16)

    def linear(self, x, w):
        return torch.nn.functional.linear(x, w.to(BF16))

    def norm(self, *args, **kw):
        from noise_amd.residual import residual_norm
        return residual_norm(*args, **kw)

    def attend(self, q, k, v):
        from noise_amd.sinks import qk_norm_rotary, sink_attention
        q, k = qk_norm_rotary(q, k, *tables(q.shape[1]))
        return sink_attention(q, k, v, 40, 2)

    def loss(self, h, w, targets):
        from noise_amd.vocab import linear_cross_entropy
        return linear_cross_entropy(h, w.to(BF16), targets, softcap=CAP)


class Plain:
    """Elementary operations in `wide`, with results rounded where the operators round them"""

    def __init__(self, wide, rounding):
        self.wide, self.rounding = wide, rounding

    def round(self, t):
        return t.to(BF16).to(self.wide) if self.rounding else t.to(self.wide)

    def linear(self, x, w):
        return self.round(x @ self.round(w).t())

    def norm(self, x, y=None, x0=None, scale=None, x0_scale=None, gate=None, y_weight=None, weight=None, norm_y=False, dtype=None):
        out, h = oracle.residual(x, y, x0, scale, x0_scale, gate, y_weight, weight, norm_y, torch.finfo(F32).eps)
        return out, self.round(h)

    def attend(self, q, k, v):
        T = q.shape[1]
        cos, sin = (t[:, None] for t in tables(T, self.wide))

        def turn(x):
            a, b = oracle.rms_norm(x, None, torch.finfo(F32).eps).chunk(2, -1)
            return self.round(torch.cat([a * cos + b * sin, b * cos - a * sin], -1))
        q, k, v = (t.transpose(1, 2).contiguous() for t in (turn(q), turn(k), v))
        at = torch.arange(T, device=DEV)
        hidden = (at[:, None] < at) | ((at[:, None] - at > 40) & (at >= 2))
        p = torch.softmax((torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(DIM)).masked_fill(hidden, -math.inf), -1)
        return self.round(torch.matmul(self.round(p), v).transpose(1, 2))

    def loss(self, h, w, targets):
        z = CAP * torch.tanh(h.reshape(-1, WIDTH) @ self.round(w).t() / CAP)
        t = targets.reshape(-1)
        live = t >= 0
        at = torch.where(live, t, 0)
        return torch.where(live, torch.logsumexp(z, -1) - z.gather(1, at[:, None])[:, 0], 0.0).view(targets.shape)


def hidden(ops, p, tokens):
    B, T = tokens.shape
    x = ops.norm(p['wte'][tokens], dtype=F32)[1] if isinstance(ops, Own) else oracle.rms_norm(p['wte'][tokens], None, torch.finfo(F32).eps)
    x0, y, more = x, None, {}
    for i in range(LAYERS):
        x, h = ops.norm(x, y, x0, p['resid'][i], p['x0'][i], dtype=BF16, **more)
        q, k, v = (ops.linear(h, p[f'{i}.{n}']).view(B, T, HEADS, DIM) for n in 'qkv')
        a = ops.linear(ops.attend(q, k, v).reshape(B, T, WIDTH), p[f'{i}.o'])
        x, h = ops.norm(x, a)
        y = ops.linear(ops.linear(h, p[f'{i}.fc']).relu().square(), p[f'{i}.proj'])
        more = dict(gate=p[f'{i}.gate'], y_weight=p[f'{i}.after'], norm_y=True)
    return ops.norm(x, y, weight=p['last'], **more)[1]


def data(seed=0, B=3, T=130):
    g = torch.Generator(DEV).manual_seed(seed)
    tokens = torch.randint(VOCAB, (B, T + 1), device=DEV, generator=g)
    targets = tokens[:, 1:].clone()
    targets[0, :50] = -100
    targets[2, 90:] = -100
    return tokens[:, :-1], targets


def step(ops, p, tokens, targets):
    loss = ops.loss(hidden(ops, p, tokens), p['head'], targets)
    return loss, torch.autograd.grad(loss.sum() / (targets >= 0).sum(), list(p.values()))


def test_step():
    from noise_amd.clip import clip_gradients
    base, (tokens, targets) = parameters(), data()
    results = {}
    for name, ops, dtype in (('own', Own(), F32), ('plain', Plain(F32, True), F32), ('exact', Plain(F64, False), F64)):
        p = {n: t.to(dtype).requires_grad_() for n, t in base.items()}
        loss, grads = step(ops, p, tokens, targets)
        results[name] = loss.detach().double(), [g.double() for g in grads]
        if name == 'own':
            norm, want = clip_gradients(list(grads), 0.01), grads
    exact = results['exact']
    for name in ('own', 'plain'):
        results[name + ' off'] = [(results[name][0] - exact[0]).norm() / exact[0].norm()] + \
            [(a - b).norm() / b.norm() for a, b in zip(results[name][1], exact[1])]
    for n, a, b in zip(('loss', *base), results['own off'], results['plain off']):
        assert a <= 2 * b + 1e-6, (n, a.item(), b.item())
    assert (results['own'][0][targets < 0] == 0).all()
    # the clipped gradients are those, scaled to the bound
    before, clipped = oracle.clip(results['own'][1], 0.01)
    assert abs(norm.item() - before) <= 1e-6 * before
    for a, b in zip(want, clipped):
        assert ((a.double() - b).abs() <= 2.0 ** -21 * b.abs() + 1e-45).all()


def test_head_gradients_in_one_call():
    """The hidden states' and the head's gradients of linear_cross_entropy_grad go on as those of the loss do."""
    from noise_amd.vocab import linear_cross_entropy_grad
    base, (tokens, targets) = parameters(1), data(1)
    p = {n: t.clone().requires_grad_() for n, t in base.items()}
    loss, want = step(Own(), p, tokens, targets)
    h = hidden(Own(), p, tokens)
    weight = torch.full(targets.shape, 1.0, device=DEV) / (targets >= 0).sum()
    own, dh, dhead = linear_cross_entropy_grad(h.detach(), p['head'].detach().to(BF16), targets, weight, softcap=CAP)
    assert torch.equal(own, loss.detach())
    got = torch.autograd.grad(h, [t for n, t in p.items() if n != 'head'], dh)
    want = dict(zip(p, want))
    for (n, w), g in zip(((n, w) for n, w in want.items() if n != 'head'), got):
        # (dZ's exponentials carry one more rounding, 2^-11, beside dZ's own 2^-8)
        assert (g - w).norm() <= 2.0 ** -7 * w.norm(), n
    assert (dhead.float() - want['head']).norm() <= 2.0 ** -7 * want['head'].norm()


def test_captured_steps():
    """Forward, backward and clipping in one graph, replayed on new tokens with eager steps between."""
    from noise_amd.clip import clip_gradients
    p = {n: t.requires_grad_() for n, t in parameters(2).items()}
    tokens, targets = data(2)

    def clipped():
        loss, grads = step(Own(), p, tokens, targets)
        return (loss.detach(), clip_gradients(grads, 0.05), *grads)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            clipped()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = clipped()
    for seed in range(3):
        a, b = data(10 + seed)
        tokens.copy_(a)
        targets.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for n, x, y in zip(('loss', 'norm', *p), got, clipped()):
            # (torch's own products and the embedding's gradient may differ between the two)
            assert (x.double() - y.double()).norm() <= 1e-3 * y.double().norm(), n
