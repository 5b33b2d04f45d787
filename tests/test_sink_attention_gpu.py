"""sink_attention and its gradients against the 64-bit definition, element by element.

Bounds (bf16's half step u = 2^-8): the weights p are rounded once for p v and the result once, so an output is off by at
most u (sum p |v| + |o|). For the gradients oracle.sinks.attend_grads adds up the same roundings of p, of the scores'
gradients and of the output. fp32 sums of at most some thousand terms and exponents of scores below 2^7 add less than
2^-14 of the same sums: 2 % of u."""
import math

import pytest
import torch

from oracle import sinks as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda', 0)
U = 2.0 ** -8
MORE = 1.02
TINY = 1e-30


def inputs(B, T, H, Hk, D, seed, n=3):
    g = torch.Generator(DEV).manual_seed(seed)
    q, *rest = (torch.randn(B, T, H if i in (0, 3) else Hk, D, device=DEV, generator=g) for i in range(n))
    rest[0][:, :2] *= 1.5     # first keys that draw attention
    return [t.bfloat16() for t in (q, *rest)]


def check(got, want, bound, what):
    assert got.shape == want.shape and got.dtype == torch.bfloat16
    off = (got.double() - want).abs()
    worst = (off - MORE * bound - TINY).max().item()
    assert worst <= 0 and bool(torch.isfinite(got).all()), f'{what}: {off.max().item()} off, {worst} past its bound'


def check_all(q, k, v, dout, window, sinks, lengths=None):
    from noise_amd.sinks import sink_attention
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = sink_attention(*leaves, window, sinks, lengths)
    want, weight = oracle.attend(q, k, v, window, sinks, lengths)
    check(out.detach(), want, U * (weight + want.abs()), 'out')
    check(sink_attention(q, k, v, window, sinks, lengths), want, U * (weight + want.abs()), 'out without gradients')
    grads = torch.autograd.grad(out, leaves, dout)
    wants, bounds = oracle.attend_grads(q, k, v, dout, window, sinks, lengths)
    for name, got, want, bound in zip('qkv', grads, wants, bounds):
        check(got, want, bound, f'd{name}')
    return out.detach(), grads


@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('T', [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300, 513, 777])
def test_lengths_of_the_sequence(T, D):
    for H, Hk, window, sinks in ((1, 1, T, 0), (2, 1, 40, 3), (6, 2, 0, 1), (3, 3, 70, 100)):
        print(T, D, H, Hk, window, sinks, flush=True)
        check_all(*inputs(2, T, H, Hk, D, T, 4), window, sinks)


@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('window', [0, 1, 31, 32, 63, 64, 65, 200, 10 ** 9])
@pytest.mark.parametrize('sinks', [0, 1, 4, 32, 63, 64, 65, 130, 10 ** 9])
def test_masks(window, sinks, D):
    print(window, sinks, D, flush=True)
    check_all(*inputs(1, 421, 2, 1, D, 7, 4), window, sinks)


@pytest.mark.parametrize('D', [64, 128])
def test_a_long_sequence(D):
    check_all(*inputs(1, 2100, 4, 2, D, 1, 4), 300, 70)
    check_all(*inputs(1, 2100, 4, 1, D, 1, 4), 3, 1500)
    check_all(*inputs(1, 2100, 2, 2, D, 1, 4), 10, 1)


@pytest.mark.parametrize('wide', [torch.int32, torch.int64])
@pytest.mark.parametrize('D', [64, 128])
def test_padded_batch(D, wide):
    """Rows past the lengths hold NaN, infinities and the type's lowest value; lengths of 0 and 1, past the tensors and
    negative."""
    T = 333
    lengths = torch.tensor([T, 0, 1, 64, 200, T + 5, -3, 65], device=DEV, dtype=wide)
    q, k, v, dout = inputs(8, T, 4, 2, D, 3, 4)
    clean = check_all(q, k, v, dout, 50, 3, lengths)
    bad = [math.nan, math.inf, -math.inf, torch.finfo(torch.bfloat16).min]
    for t in (q, k, v, dout):
        for b in range(8):
            n = min(T, max(0, int(lengths[b])))
            t[b, n:] = torch.tensor(bad, device=DEV).repeat(D // 4).bfloat16()
    from noise_amd.sinks import sink_attention
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = sink_attention(*leaves, 50, 3, lengths)
    for got, want in zip((out, *torch.autograd.grad(out, leaves, dout)), (clean[0], *clean[1])):
        assert torch.equal(got, want)


def test_strides_and_views():
    B, T, H, D = 2, 150, 4, 64
    g = torch.Generator(DEV).manual_seed(5)
    packed = torch.randn(B, T, 3 * H + 1, D, device=DEV, generator=g).bfloat16()
    q, k, v = packed[:, :, :H], packed[:, :, H:2 * H], packed[:, :, 2 * H:3 * H]
    dout = torch.randn(B, H, T, D, device=DEV, generator=g).bfloat16().transpose(1, 2)
    check_all(q, k, v, dout, 60, 5)
    wide = torch.randn(B, T, H, D + 1, device=DEV, generator=g).bfloat16()
    check_all(wide[..., 1:], k[:, :, :2], wide[..., :2 * 64][:, :, :2, 1:], dout, 60, 5)   # odd addresses: copied
    check_all(q[:1].expand(B, T, H, D), k[:1].expand(B, T, H, D), v, dout, 60, 5)          # a broadcast batch
    check_all(q, k[:, :, :1].expand(B, T, 2, D), v[:, :, :2], dout, 60, 5)                 # a broadcast head
    check_all(q, k, v, dout[:, :1].expand(B, T, H, D), 60, 5)


def test_gradients_of_broadcast_inputs_add_up():
    from noise_amd.sinks import sink_attention
    q, k, v, dout = inputs(3, 70, 4, 2, 64, 2, 4)
    one = k[:1].clone().requires_grad_()
    sink_attention(q, one.expand(3, 70, 2, 64), v, 30, 2).backward(dout)
    each = k[:1].expand(3, 70, 2, 64).clone().requires_grad_()
    sink_attention(q, each, v, 30, 2).backward(dout)
    assert torch.allclose(one.grad.float(), each.grad.float().sum(0, keepdim=True), rtol=2 * U, atol=4 * U)


def test_gradients_against_differences():
    """The step's change of sum(dout * out), by the 64-bit definition, over a step along each gradient's own direction."""
    from noise_amd.sinks import sink_attention
    q, k, v, dout = inputs(1, 90, 4, 2, 64, 11, 4)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(sink_attention(*leaves, 25, 2), leaves, dout)
    bounds = oracle.attend_grads(q, k, v, dout, 25, 2)[1]
    for i in range(3):
        d = grads[i].double()
        at = lambda step: (oracle.attend(*[t.double() + (step * d if n == i else 0) for n, t in enumerate((q, k, v))],
                                         25, 2)[0] * dout.double()).sum()
        h = 1e-4 / d.abs().max()
        slope = (at(h) - at(-h)) / (2 * h)
        # the slope along d is d . (true gradient): off from d . d by at most |d| . bound (and the difference's h^2)
        assert abs(slope - d.square().sum()) <= MORE * (d.abs() * bounds[i]).sum() + 1e-5 * d.square().sum()


def test_empty():
    from noise_amd.sinks import sink_attention
    for shape in ((0, 5, 4, 64), (2, 0, 4, 64)):
        q = torch.empty(shape, device=DEV, dtype=torch.bfloat16, requires_grad=True)
        out = sink_attention(q, q[:, :, :2], q[:, :, 2:], 10, 2)
        assert out.shape == shape
        out.sum().backward()
        assert q.grad.shape == shape


@pytest.mark.parametrize('D', [64, 128])
def test_gradients_of_weights_close_to_one(D):
    """Rows that give nearly all their weight to one key: dP - dO . out nearly cancels there. Relative to the whole gradient, its
    parts' roundings of 2^-9 (rms 2^-9 / sqrt 3 each: of the scores' gradients, of the weights in the output, of the
    result) leave less than 3 2^-9; the output's own rounding in dO . out would leave several times that."""
    q, k, v, dout = inputs(1, 300, 2, 1, D, 9, 4)
    k[:, 0] = (q.float().mean((1, 2), keepdim=True)[:, 0] * 40).bfloat16()
    k[:, 7] = k[:, 0]
    for scale, window, sinks in ((0.4, 3, 1), (1.0, 3, 1), (1.0, 100, 8)):
        keys = (k.float() * scale).bfloat16()
        from noise_amd.sinks import sink_attention
        leaves = [t.detach().requires_grad_() for t in (q, keys, v)]
        grads = torch.autograd.grad(sink_attention(*leaves, window, sinks), leaves, dout)
        for got, want in zip(grads, oracle.attend_grads(q, keys, v, dout, window, sinks)[0]):
            rel = ((got.double() - want).norm() / want.norm()).item()
            print(D, scale, window, sinks, rel, flush=True)
            assert rel <= 3 * 2.0 ** -9


@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('B,T,window,padded', [(8, 2500, 2100, False), (32, 1100, 200, False), (32, 1100, 200, True)])
def test_enough_rows(B, T, window, padded, D):
    """Rows enough for the larger workgroups (256 queries with a long window, 128 keys), lengths off their tiles, first tokens past
    the window; against the 64-bit definition on some heads of some sequences."""
    from noise_amd.sinks import sink_attention
    q, k, v, dout = inputs(B, T, 8, 4, D, 21, 4)
    lengths = torch.tensor([(T, 700, 0, 129)[b % 4] for b in range(B)], device=DEV) if padded else None
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = sink_attention(*leaves, window, 70, lengths)
    plain = sink_attention(q, k, v, window, 70, lengths)
    grads = torch.autograd.grad(out, leaves, dout)
    for b, h in ((0, 0), (5, 3), (2, 1), (7, 2)):
        heads = [t[b:b + 1, :, 2 * h:2 * h + 2] for t in (q, dout)]
        kv = [t[b:b + 1, :, h:h + 1] for t in (k, v)]
        n = None if lengths is None else lengths[b:b + 1]
        want, weight = oracle.attend(heads[0], *kv, window, 70, n)
        for got in (out.detach(), plain):
            check(got[b:b + 1, :, 2 * h:2 * h + 2], want, U * (weight + want.abs()), 'out')
        wants, bounds = oracle.attend_grads(heads[0], *kv, heads[1], window, 70, n)
        check(grads[0][b:b + 1, :, 2 * h:2 * h + 2], wants[0], bounds[0], 'dq')
        for i in (1, 2):
            check(grads[i][b:b + 1, :, h:h + 1], wants[i], bounds[i], 'dk, dv')


@pytest.mark.parametrize('D', [64, 128])
def test_a_padded_batch_with_a_long_window(D):
    """The 256-query workgroups (8 sequences of 8 heads, a window past 2048) over sequences that end in their first tile, at and
    behind a tile's and a wave's edge, and nowhere; rows past the lengths hold NaN."""
    from noise_amd.sinks import sink_attention
    T, window, sinks = 2500, 2100, 70
    q, k, v, dout = inputs(8, T, 8, 4, D, 22, 4)
    lengths = torch.tensor([T, 1, 64, 65, 129, 257, 700, 0], device=DEV)
    for b, n in enumerate(lengths.tolist()):
        for t in (q, k, v, dout):
            t[b, n:] = math.nan
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = sink_attention(*leaves, window, sinks, lengths)
    plain = sink_attention(q, k, v, window, sinks, lengths)
    grads = torch.autograd.grad(out, leaves, dout)
    for b in range(8):
        h = b % 4
        print(D, b, h, flush=True)
        heads = [t[b:b + 1, :, 2 * h:2 * h + 2] for t in (q, dout)]
        kv = [t[b:b + 1, :, h:h + 1] for t in (k, v)]
        n = lengths[b:b + 1]
        want, weight = oracle.attend(heads[0], *kv, window, sinks, n)
        for got in (out.detach(), plain):
            check(got[b:b + 1, :, 2 * h:2 * h + 2], want, U * (weight + want.abs()), 'out')
        wants, bounds = oracle.attend_grads(heads[0], *kv, heads[1], window, sinks, n)
        check(grads[0][b:b + 1, :, 2 * h:2 * h + 2], wants[0], bounds[0], 'dq')
        for i in (1, 2):
            check(grads[i][b:b + 1, :, h:h + 1], wants[i], bounds[i], 'dk, dv')


def test_growing_scores():
    """Scores far apart, and rows whose largest weight stands in the last tile or the first key."""
    q, k, v, dout = inputs(1, 400, 2, 2, 64, 8, 4)
    k = (k.float() * torch.linspace(0.1, 9, 400, device=DEV)[None, :, None, None]).bfloat16()
    check_all(q, k, v, dout, 390, 0)
    check_all(q, k.flip(1).contiguous(), v, dout, 100, 7)


def test_repeats_and_streams():
    from noise_amd.sinks import sink_attention
    q, k, v, dout = inputs(2, 700, 8, 2, 128, 4, 4)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    run = lambda: (lambda o: (o, *torch.autograd.grad(o, leaves, dout)))(sink_attention(*leaves, 100, 70))
    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        others = [run() for _ in range(3)]
    here = [run() for _ in range(3)]
    torch.cuda.synchronize()
    for results in (*others, *here):
        assert all(torch.equal(x, y) for x, y in zip(first, results))


def test_captured_graphs():
    """Forward and backward captured twice; the replays, in turn with eager calls on other inputs, give the eager bits."""
    from noise_amd.sinks import attend_backward, attend_forward, sink_attention
    q, k, v, dout = inputs(2, 500, 4, 2, 64, 6, 4)

    def step():
        out, *more = attend_forward(q, k, v, 90, 4, None, True)
        return (out, *attend_backward(dout, q, k, v, out, *more, 90, 4, None))

    step()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    for n in range(3):
        for t, x in zip((q, k, v, dout), inputs(2, 500, 4, 2, 64, 50 + n, 4)):
            t.copy_(x)
        want = step()
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(out, want))
        sink_attention(q[:1], k[:1], v[:1], 3)


def test_compiled_operator():
    q, k, v, dout = inputs(2, 130, 4, 2, 64, 12, 4)
    from noise_amd.sinks import sink_attention
    results = []
    for f in (lambda *t: torch.ops.noise_amd.sink_attention(*t, 40, 3, None)[0], lambda *t: sink_attention(*t, 40, 3)):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = f(*leaves)
        results.append((out, *torch.autograd.grad(out, leaves, dout)))
    assert all(torch.equal(x, y) for x, y in zip(*results))


def test_far_scores():
    """Scores of 2^27 and their negatives (a single product of powers of two and bf16 values: exact in fp32): the key with the
    largest, or those that tie for it, take all the weight, and nothing overflows on the way."""
    from noise_amd.sinks import sink_attention, sink_attention_decode
    B, T, H, D = 1, 150, 2, 64
    g = torch.Generator(DEV).manual_seed(1)
    v = torch.randn(B, T, H, D, device=DEV, generator=g).bfloat16()
    q = torch.zeros(B, T, H, D, device=DEV, dtype=torch.bfloat16)
    k = torch.zeros_like(q)
    q[..., 0] = 2.0 ** 15
    for sign in (1, -1):
        k[..., 0] = (sign * 2.0 ** 15 * (1 + torch.arange(T, device=DEV)[None, :, None] / 256)).bfloat16()
        want, weight = oracle.attend(q, k, v, 60, 3)
        check(sink_attention(q, k, v, 60, 3), want, U * (weight + want.abs()), 'out')
        start = torch.tensor([T - 1], device=DEV)
        check(sink_attention_decode(q[:, -1:], k, v, start, 60, 3), want[:, -1:], (U * (weight + want.abs()))[:, -1:], 'decode')


def test_compiled_step():
    """The operators in a compiled function (forward and backward traced, no graph break) give the eager bits."""
    from noise_amd.distill import distill_loss
    from noise_amd.sinks import qk_norm_rotary, sink_attention
    q, k, v, _ = inputs(2, 64, 4, 2, 64, 13, 4)
    angle = torch.rand(64, 32, device=DEV)
    cos, sin = angle.cos(), angle.sin()
    w = torch.rand(64, device=DEV)
    t, i = torch.randn(2, 64, 4, 3, device=DEV), torch.randint(0, 64, (2, 64, 4, 3), device=DEV)

    def step(q, k, v, w):
        q, k = torch.ops.noise_amd.qk_norm_rotary(q, k, cos, sin, w, None, None, 1e-6)
        out = torch.ops.noise_amd.sink_attention(q, k, v, 20, 2, None)[0]
        return torch.ops.noise_amd.distill_loss(out, t, i, 64, 1.0, 15.0)

    def plain(q, k, v, w):
        q, k = qk_norm_rotary(q, k, cos, sin, w, eps=1e-6)
        return distill_loss(sink_attention(q, k, v, 20, 2), t, i, softcap=15.0)

    results = []
    for f in (torch.compile(step, backend='aot_eager', fullgraph=True), plain):
        leaves = [x.detach().requires_grad_() for x in (q, k, v, w)]
        loss = f(*leaves)
        results.append((loss, *torch.autograd.grad(loss.sum(), leaves)))
    assert all(torch.equal(x, y) for x, y in zip(*results))


def test_many_sequences():
    """More sequences than a grid's second dimension holds, each of a few tokens, with cut lists."""
    B, T = 70000, 3
    q, k, v, dout = inputs(B, T, 1, 1, 64, 14, 4)
    from noise_amd.sinks import sink_attention
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = sink_attention(*leaves, 1, 1)
    grads = torch.autograd.grad(out, leaves, dout)
    some = torch.tensor([0, 1, 65534, 65535, 65536, B - 1], device=DEV)
    mine = [t[some].detach().requires_grad_() for t in (q, k, v)]
    part = sink_attention(*mine, 1, 1)
    want, weight = oracle.attend(q[some], k[some], v[some], 1, 1)
    check(out[some].detach(), want, U * (weight + want.abs()), 'out')
    for x, y in zip(grads, torch.autograd.grad(part, mine, dout[some])):
        assert torch.equal(x[some], y)
