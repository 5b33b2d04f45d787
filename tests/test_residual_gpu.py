"""residual_norm and its gradients against the 64-bit definition.

Bounds. Sums over a row run over at most 16 elements in a lane and then up to 9 pairwise steps, so a sum of squares is off by at most
25 F of itself (F = 2^-24) and r = rsqrt by 16 F. x' has fewer than 24 roundings of parts no larger than A = |s| (|x| + |g b|) +
|s0 x0| (b's own norm among them): off by 24 F A. Through r that also moves n by up to 24 F rms(A) r = 24 F K of itself, so h is off
by 48 F (r |w| A + |h| (1 + K)). A gradient's terms are at most M = |dx'| + r (|u| + |n| mean |u n|) with the same two sources of
error, and the norm of y adds its own (the factor 4): 128 F (1 + K) M, times what it is multiplied by. Sums over rows run over at most
64 rows in a lane and 64 partial sums: 256 F (1 + K) of the sum of their terms' sizes. Results in bf16 add half a step."""
import itertools

import pytest
import torch

from oracle import training as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda', 0)
BF16, F32 = torch.bfloat16, torch.float32
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}
F = 2.0 ** -24
EPS = torch.finfo(F32).eps
NAMES = ('x', 'y', 'x0', 'scale', 'x0_scale', 'gate', 'y_weight', 'weight')


def make(shape, xt, yt, seed, parts=NAMES, gate=(), gate_type=F32):
    g = torch.Generator(DEV).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device=DEV, generator=g)
    D = shape[-1]
    t = dict(x=randn(*shape).to(xt), y=(2 * randn(*shape)).to(yt), x0=randn(*shape).to(xt), scale=0.9 + 0.1 * randn(()),
             x0_scale=0.2 + 0.1 * randn(()), gate=(0.5 + 0.3 * randn(*gate, D)).to(gate_type), y_weight=1 + 0.2 * randn(D),
             weight=1 + 0.2 * randn(D))
    up = randn(*shape).to(xt), randn(*shape).to(yt)
    return {n: v for n, v in t.items() if n in parts}, up


def bounds(t, up, norm_y, eps):
    """The sizes that the errors go by, in the order of the results: x', h, then the tensors' gradients"""
    d = {n: v.double().abs() for n, v in t.items()}
    s, s0, g = d.get('scale', 1.0), d.get('x0_scale', 1.0), d.get('gate', 1.0)
    one = torch.ones((), device=DEV, dtype=torch.float64)
    zero = torch.zeros_like(d['x'])
    by = zero
    if 'y' in d:
        ry = (1 / (d['y'].square().mean(-1, keepdim=True) + eps).sqrt()) if norm_y else one
        by = d['y'] * ry * (d.get('y_weight', 1.0) if norm_y else 1.0)
    inner = d['x'] + g * by
    A = s * inner + s0 * d.get('x0', zero)
    out, h = oracle.residual(**{n: v.double() for n, v in t.items()}, norm_y=norm_y, eps=eps)
    r = 1 / (out.square().mean(-1, keepdim=True) + eps).sqrt()
    K = A.square().mean(-1, keepdim=True).sqrt() * r
    w = d.get('weight', 1.0)
    sizes = [24 * A, 48 * (r * w * A + h.abs() * (1 + K))]
    dout, dh = (u.double().abs() if u is not None else zero for u in up)
    n, u = (out * r).abs(), dh * w
    M = (1 + K) * (dout + r * (u + (n + r * A) * (u * (n + r * A)).mean(-1, keepdim=True)))
    over = lambda v, like: v if v.shape == like.shape else v.sum_to_size(like.shape) * 2
    for name, v in t.items():
        if name == 'x':
            sizes.append(128 * s * M)
        elif name == 'y':
            e = s * g * M
            if norm_y:
                e, ny = e * d.get('y_weight', 1.0), d['y'] * ry
                e = 4 * ry * (e + ny * (e * ny).mean(-1, keepdim=True))
            sizes.append(128 * e)
        elif name == 'x0':
            sizes.append(128 * s0 * M)
        elif name == 'scale':
            sizes.append(256 * (M * inner).sum())
        elif name == 'x0_scale':
            sizes.append(256 * (M * d['x0']).sum())
        elif name == 'gate':
            sizes.append(128 * over(s * M * by, v))
        elif name == 'y_weight':
            sizes.append(256 * over(s * g * M * d['y'] * ry, v))
        elif name == 'weight':
            sizes.append(256 * over((1 + K) * dh * (n + r * A), v))
    return sizes


def check(t, up, norm_y=False, eps=EPS):
    from noise_amd.residual import residual_norm
    wide = {n: v.double().requires_grad_() for n, v in t.items()}
    outs = oracle.residual(**wide, norm_y=norm_y, eps=eps)
    used = [(o, u.double()) for o, u in zip(outs, up) if u is not None]
    want = [o.detach() for o in outs]
    want += torch.autograd.grad([o for o, _ in used], list(wide.values()), [u for _, u in used], materialize_grads=True)
    leaves = {n: v.detach().requires_grad_() for n, v in t.items()}
    got = residual_norm(**leaves, norm_y=norm_y, eps=eps)
    plain = residual_norm(**t, norm_y=norm_y, eps=eps)
    assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1])
    used = [(o, u) for o, u in zip(got, up) if u is not None]
    got = [o.detach() for o in got] + list(torch.autograd.grad([o for o, _ in used], list(leaves.values()), [u for _, u in used],
                                                               materialize_grads=True))
    types = [t['x'].dtype, t['y'].dtype if 'y' in t else t['x'].dtype, *(v.dtype for v in t.values())]
    for name, a, b, size, dt in zip(("x'", 'h', *t), got, want, bounds(t, up, norm_y, eps), types):
        assert a.dtype == dt and a.shape == b.shape, (name, a.dtype, a.shape)
        off, bound = (a.double() - b).abs(), HALF[dt] * b.abs() * (1 + 2 ** -8) + F * size + 1e-37
        assert (off <= bound).all(), (name, (off / bound).max(), a.shape)
    return got


DIMS = [1, 2, 7, 8, 9, 64, 127, 128, 129, 255, 512, 513, 1001, 1024, 1025, 2047, 2048, 2056, 4095, 4096, 4104, 5000, 8191, 8192]


@pytest.mark.parametrize('D', DIMS)
def test_widths(D):
    """Every part of the formula, both forms of the block's output, each pair of types."""
    for seed, (xt, yt, norm_y) in enumerate(itertools.product((BF16, F32), (BF16, F32), (False, True))):
        if (xt, yt) == (BF16, F32):
            continue
        parts = NAMES if norm_y else tuple(n for n in NAMES if n != 'y_weight')
        check(*make((3, 5, D), xt, yt, seed, parts), norm_y)


@pytest.mark.parametrize('shape', [(1, 512), (2, 1, 512), (3, 700, 512), (1, 2500, 64), (4000, 16), (2, 300, 2048), (130, 4096)])
def test_rows(shape):
    for norm_y in (False, True):
        check(*make(shape, F32, BF16, 1, NAMES if norm_y else NAMES[:6] + NAMES[7:]), norm_y)


@pytest.mark.parametrize('parts', [p for n in range(8) for p in itertools.combinations(NAMES[1:], n)
                                   if ('y' in p or not {'gate', 'y_weight'} & set(p)) and ('x0' in p or 'x0_scale' not in p)],
                         ids='-'.join)
def test_parts_left_out(parts):
    """Every combination of what may be None, with the norm of y wherever its weight is there."""
    check(*make((2, 9, 96), BF16, BF16, len(parts), ('x', *parts)), 'y_weight' in parts)
    if 'y' in parts:
        check(*make((2, 9, 96), BF16, BF16, len(parts), ('x', *parts)), True)


@pytest.mark.parametrize('lead,gate', [((4, 6), ()), ((4, 6), (1, 1)), ((4, 6), (4, 1)), ((4, 6), (4, 6)), ((1, 6), (1, 1)),
                                       ((4, 1), (4, 1)), ((5, 3, 7), (5, 3, 1)), ((5, 3, 7), (5, 1, 1)), ((2500, 2), (2500, 1)),
                                       ((3, 1111), (3, 1)), ((1, 1), (1, 1)), ((70000, 1, 2), (70000, 1, 1)), ((7,), ())])
@pytest.mark.parametrize('gate_type', [F32, BF16])
def test_gates(lead, gate, gate_type):
    """A gate per channel, per sequence, per token and in between; more gates than one launch dimension has workgroups."""
    D = 8 if lead[0] == 70000 else 200
    for norm_y in (False, True):
        check(*make((*lead, D), F32, BF16, 3, NAMES if norm_y else NAMES[:6] + NAMES[7:], gate, gate_type), norm_y)


def test_upstream_gradients_left_out():
    for keep in ((True, False), (False, True)):
        t, up = make((3, 50, 256), F32, BF16, 5)
        check(t, [u if k else None for u, k in zip(up, keep)], True)


def test_gradients_asked_for_one_by_one():
    """Each tensor's gradient alone is the one it has among all of them."""
    from noise_amd.residual import residual_norm
    t, up = make((3, 50, 256), F32, BF16, 6)
    every = check(t, up, True)[2:]
    for i, name in enumerate(t):
        leaves = {n: v.detach().requires_grad_(n == name) for n, v in t.items()}
        got, = torch.autograd.grad(residual_norm(**leaves, norm_y=True), leaves[name], up)
        assert torch.equal(got, every[i]), name


def test_strides():
    """Rows at other distances, at odd addresses, transposed batches, broadcast rows; gradients of other layouts."""
    from noise_amd.residual import residual_norm
    t, up = make((4, 6, 100), F32, BF16, 7)
    base = residual_norm(**t, norm_y=True)

    def wider(v, off):
        buf = torch.empty(*v.shape[:-1], v.shape[-1] + 13, dtype=v.dtype, device=DEV)
        buf[..., off:off + v.shape[-1]] = v
        return buf[..., off:off + v.shape[-1]]
    forms = [lambda v: wider(v, 1), lambda v: wider(v, 8), lambda v: v.transpose(0, 1).contiguous().transpose(0, 1),
             lambda v: v.transpose(1, 2).contiguous().transpose(1, 2)]
    for form in forms:
        s = {n: form(v) if n in ('x', 'y', 'x0') else v for n, v in t.items()}
        got = residual_norm(**s, norm_y=True)
        assert torch.equal(got[0], base[0]) and torch.equal(got[1], base[1])
        check(s, [form(u) for u in up], True)
    row = {**t, 'x': t['x'][:1, :1].expand(4, 6, 100), 'y': t['y'][:, :1].expand(4, 6, 100)}
    check(row, up, True)


def test_values():
    """Rows of zeros, very large and very small values, NaN and infinities stay in their rows."""
    from noise_amd.residual import residual_norm
    t, up = make((1, 12, 512), F32, F32, 8, ('x', 'y', 'weight'))
    t['x'][0, 0], t['y'][0, 0] = 0, 0
    t['x'][0, 1] *= 1e15
    t['x'][0, 2] *= 1e-15
    t['y'][0, 2] *= 1e-15
    want = check({n: v[:, :4] if n != 'weight' else v for n, v in t.items()}, [u[:, :4] for u in up])
    t['x'][0, 4, 7], t['x'][0, 5, 3], t['y'][0, 6, 500] = float('nan'), float('inf'), float('-inf')
    out, h = residual_norm(**t)
    for row in (4, 5, 6):
        assert not torch.isfinite(h[0, row]).all()
    assert torch.equal(out[0, :4], want[0][0]) and torch.equal(h[0, :4], want[1][0])
    assert torch.isfinite(h[0, 7:]).all()
    leaves = {n: v.detach().requires_grad_() for n, v in t.items()}
    dx, = torch.autograd.grad(residual_norm(**leaves), leaves['x'], up)
    assert torch.isfinite(dx[0, :4]).all() and torch.isfinite(dx[0, 7:]).all()


def test_differences():
    """The gradients along a direction against a difference quotient of the outputs (fp32, step 2^-10: off by the second
    differences, 2^-20 of the third derivatives, and the outputs' roundings over the step)."""
    from noise_amd.residual import residual_norm
    t, up = make((2, 3, 40), F32, F32, 9)
    leaves = {n: v.detach().requires_grad_() for n, v in t.items()}
    grads = torch.autograd.grad(residual_norm(**leaves, norm_y=True), list(leaves.values()), up)
    value = lambda s: sum((o.double() * u.double()).sum() for o, u in zip(residual_norm(**s, norm_y=True), up)).item()
    g = torch.Generator(DEV).manual_seed(1)
    for (name, v), d in zip(t.items(), grads):
        along, h = torch.randn(v.shape, device=DEV, generator=g), 2.0 ** -10
        quotient = (value({**t, name: v + h * along}) - value({**t, name: v - h * along})) / (2 * h)
        size = sum(o.abs().double().mul(u.abs()).sum() for o, u in zip(residual_norm(**t, norm_y=True), up)).item()
        assert abs(quotient - (d.double() * along).sum().item()) <= 64 * F * size / h + 2.0 ** -20 * 64 * size, name


def test_no_rows():
    from noise_amd.residual import residual_norm
    t, up = make((0, 5, 64), F32, BF16, 1)
    leaves = {n: v.requires_grad_() for n, v in t.items()}
    outs = residual_norm(**leaves, norm_y=True)
    assert outs[0].shape == outs[1].shape == (0, 5, 64)
    for d, v in zip(torch.autograd.grad(outs, list(leaves.values()), up), leaves.values()):
        assert d.shape == v.shape and not d.any()


def test_past_32_bits():
    """More than 2^31 elements: a row's results are those of a call of its own; the weight's gradient is off by its sums, of at most
    rows / 2048 rows in a lane (512 workgroups of 4 teams) and 64 more steps, and its terms' own 256 F (1 + K)."""
    from noise_amd.residual import residual_norm
    R, D = 2 ** 22 + 1001, 512
    t, up = make((R, D), BF16, BF16, 3, ('x', 'y', 'scale', 'weight'))
    leaves = {n: v.requires_grad_() for n, v in t.items()}
    outs = residual_norm(**leaves, norm_y=True)
    grads = torch.autograd.grad(outs, list(leaves.values()), up)
    sums, sizes = torch.zeros(D, device=DEV, dtype=torch.float64), torch.zeros(D, device=DEV, dtype=torch.float64)
    for rows in torch.arange(R, device=DEV).tensor_split(16):
        a, b = int(rows[0]), int(rows[-1]) + 1
        own = {n: (v.detach()[a:b] if v.dim() == 2 else v.detach()).requires_grad_() for n, v in leaves.items()}
        part = residual_norm(**own, norm_y=True)
        assert torch.equal(outs[0][a:b], part[0]) and torch.equal(outs[1][a:b], part[1])
        dx, dy = torch.autograd.grad(part, (own['x'], own['y']), (up[0][a:b], up[1][a:b]))
        assert torch.equal(grads[0][a:b], dx) and torch.equal(grads[1][a:b], dy)
        exact, _ = oracle.residual(own['x'].double(), own['y'].double(), scale=own['scale'].double(), norm_y=True, eps=EPS)
        terms = oracle.rms_norm(exact, eps=EPS) * up[1][a:b].double()
        sums += terms.sum(0).detach()
        sizes += terms.abs().sum(0).detach()
        del part, own, exact, terms
    # K: the parts of x' do not cancel to less than a tenth of their sizes
    assert ((grads[3] - sums).abs() <= F * (R / 2048 + 64 + 256 * 11) * sizes).all()


def test_other_types_of_weights_and_dtype():
    """Weights and scalars in bf16 are taken at their value, their gradients come in their type; h in bf16 without y."""
    from noise_amd.residual import residual_norm
    t, up = make((2, 30, 128), F32, BF16, 4)
    low = {n: v.to(BF16) if n in ('scale', 'x0_scale', 'y_weight', 'weight') else v for n, v in t.items()}
    same = {n: v.float() if n in ('scale', 'x0_scale', 'y_weight', 'weight') else v for n, v in low.items()}
    a, b = ({n: v.detach().requires_grad_() for n, v in s.items()} for s in (low, same))
    oa, ob = residual_norm(**a, norm_y=True), residual_norm(**b, norm_y=True)
    assert torch.equal(oa[0], ob[0]) and torch.equal(oa[1], ob[1])
    for n, u, v in zip(t, torch.autograd.grad(oa, list(a.values()), up), torch.autograd.grad(ob, list(b.values()), up)):
        assert u.dtype == low[n].dtype and torch.equal(u, v.to(u.dtype)), n
    out, h = residual_norm(t['x'], x0=t['x0'], scale=t['scale'], x0_scale=t['x0_scale'], dtype=BF16)
    assert out.dtype == F32 and h.dtype == BF16
    full = residual_norm(t['x'], x0=t['x0'], scale=t['scale'], x0_scale=t['x0_scale'])
    assert torch.equal(full[0], out) and torch.equal(full[1].to(BF16), h)


def test_graph_and_streams():
    """A captured step, replayed with new values in its tensors, and a call on another stream than the tensors' own."""
    from noise_amd.residual import residual_norm
    t, up = make((3, 200, 512), F32, BF16, 10)
    leaves = {n: v.detach().clone().requires_grad_() for n, v in t.items()}

    def step():
        outs = residual_norm(**leaves, norm_y=True)
        return (*outs, *torch.autograd.grad(outs, list(leaves.values()), up))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(3):
        new, _ = make((3, 200, 512), F32, BF16, 20 + seed)
        with torch.no_grad():
            for n, v in leaves.items():
                v.copy_(new[n])
        graph.replay()
        torch.cuda.synchronize()
        got = [o.detach().clone() for o in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b.detach())
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.current_stream())
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(other, got):
        assert torch.equal(a.detach(), b)


def test_compiled():
    from noise_amd.residual import residual_norm
    t, up = make((3, 40, 512), F32, BF16, 11)

    def step(t):
        return residual_norm(**t, norm_y=True)
    a, b = ({n: v.detach().requires_grad_() for n, v in t.items()} for _ in range(2))
    oa, ob = step(a), torch.compile(step, fullgraph=True)(b)
    ga, gb = torch.autograd.grad(oa, list(a.values()), up), torch.autograd.grad(ob, list(b.values()), up)
    for x, y in zip((*oa, *ga), (*ob, *gb)):
        assert torch.equal(x, y)
