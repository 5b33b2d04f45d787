"""linear_cross_entropy and its gradients against the 64-bit definition.

Bounds, with F = 2^-24, N = |x| |W|^T (the sizes of a logit's terms) and A the largest |z| of a row plus log V:
  a logit: products are exact in fp32 for bf16 operands and are added in at most dim / 16 + 24 steps; fp32 operands, held as two fp16
    values, miss 2^-21 of a term and 2^-38 of the tensors' largest values, and take three times the steps; the soft cap adds 2^-21 of
    itself, or past 32 of thrice the logit where that is less: ez
  a loss: two logits, and the maximum, the sum's (V / 128 + 40 steps) and the logarithm's roundings: 2 max ez + F (80 + V / 128 + 8 A)
  dZ = weight (p - 1[t]) cap': p is off by its exponent's error, ez + the loss's, cap' by 4 cap's; then dZ is rounded to bf16 (2^-8) or to
    two fp16 values (2^-21, and 2^-38 of the largest weight): ed
  dx, dW: the products with ed, their sums (steps as above, over V and rows, and up to 64 joined parts), the other operand's 2^-21,
    and half a step of the result."""
import math

import pytest
import torch

from oracle import training as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda', 0)
BF16, F32 = torch.bfloat16, torch.float32
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}
F = 2.0 ** -24


def make(R, V, D, dtype, seed=0, width=None, masked=False, scale=2.0):
    g = torch.Generator(DEV).manual_seed(seed)
    W = width or V
    weight = torch.randn(W, D, device=DEV, generator=g).mul_(scale / math.sqrt(D))
    targets = torch.randint(V, (R,), device=DEV, generator=g)
    x = torch.randn(R, D, device=DEV, generator=g) + weight[targets]
    token_weight = torch.rand(R, device=DEV, generator=g) / max(R, 1)
    x, weight = x.to(dtype), weight.to(dtype)
    if masked:
        gone = torch.rand(R, device=DEV, generator=g) < 0.4
        targets[gone] = torch.tensor([-100, -1, V, V + 7, 2 ** 31 - 1], device=DEV)[torch.arange(int(gone.sum()), device=DEV) % 5]
        x[gone] = torch.tensor([float('nan'), float('inf'), 1.0, -3e38], device=DEV).to(dtype)[
            torch.arange(int(gone.sum()), device=DEV) % 4][:, None]
    weight[V:] = float('nan')
    return x, weight, targets, token_weight


def bounds(x, weight, targets, w, V, cap, loss, dx, dw):
    dtype, (R, D) = x.dtype, x.shape
    split = dtype == F32
    used = (targets >= 0) & (targets < V)
    xs = torch.where(used[:, None], x, 0).double()
    ws = weight[:V].double()
    at = torch.where(used, targets, 0).long()[:, None]
    raw = xs @ ws.t()
    N = xs.abs() @ ws.abs().t()
    steps = (3 if split else 1) * (D / 16) + 24
    ez = F * steps * N
    if split:
        ez = ez + 2.0 ** -21 * N + 2.0 ** -38 * D * xs.abs().max() * ws.abs().max()
    z, slope, eslope = raw, 1.0, 0.0
    if cap:
        z = cap * torch.tanh(raw / cap)
        slope = 1 - (z / cap) ** 2
        ez = ez * slope + 2.0 ** -21 * (torch.clamp(3 * z.abs(), max=cap) if cap > 32 else cap) + ez ** 2 / cap
        eslope = 4 * ez / cap
    A = z.abs().amax(-1) + math.log(V) + 1
    eloss = 2 * ez.amax(-1) + F * (80 + V / 128 + 8 * A)
    p = torch.softmax(z, -1)
    w = torch.where(used, w.double() if w is not None else 1.0, 0.0)[:, None]
    dp = p.clone()
    dp.scatter_add_(1, at, -torch.ones_like(at, dtype=torch.float64))
    dz = (w * dp * slope).abs()
    ed = w.abs() * (p * (ez + eloss[:, None] + 8 * F) + 4 * F * dp.abs()) * slope + w.abs() * dp.abs() * eslope
    ed = ed + (2.0 ** -21 * dz + 2.0 ** -38 * w.abs().max() if split else 2.0 ** -8 * dz)
    of = lambda n: F * ((3 if split else 1) * n / 16 + 24 + 64) + (2.0 ** -21 if split else 0)
    ex = ed @ ws.abs() + of(V) * (dz @ ws.abs()) + (2.0 ** -38 * V * w.abs().max() * ws.abs().max() if split else 0)
    ew = ed.t() @ xs.abs() + of(R) * (dz.t() @ xs.abs()) + (2.0 ** -38 * R * w.abs().max() * xs.abs().max() if split else 0)
    full = torch.zeros(dw.shape, dtype=torch.float64, device=DEV)
    full[:V] = ew
    tiny = 1e-37
    return (eloss + F * loss.abs()) * used, ex * (1 + HALF[dtype]) + HALF[dtype] * dx.abs() + tiny, \
        full * (1 + HALF[dtype]) + HALF[dtype] * dw.abs() + tiny


def check(x, weight, targets, w, V, cap=None):
    from noise_amd.vocab import linear_cross_entropy, linear_cross_entropy_grad
    want = oracle.linear_cross_entropy(x, weight, targets, V, cap, w)
    loss, dx, dw = linear_cross_entropy_grad(x, weight, targets, w, vocab=V, softcap=cap)
    assert loss.dtype == F32 and dx.dtype == dw.dtype == x.dtype and loss.shape == x.shape[:-1]
    limit = bounds(x, weight, targets, w, V, cap, *want)
    for name, a, b, c in zip(('loss', 'dx', 'dweight'), (loss, dx, dw), want, limit):
        off = (a.double() - b).abs()
        assert (off <= c).all(), (name, (off - c).max(), off.max(), b.abs().max())
    assert (dw[V:] == 0).all()
    with torch.no_grad():
        plain = linear_cross_entropy(x, weight, targets, vocab=V, softcap=cap)
    off = (plain.double() - want[0]).abs()
    assert (off <= limit[0]).all(), ('plain', (off - limit[0]).max())
    leaves = x.detach().requires_grad_(), weight.detach().requires_grad_()
    by = linear_cross_entropy(*leaves, targets, vocab=V, softcap=cap)
    off = (by.detach().double() - want[0]).abs()
    assert (off <= limit[0]).all()
    grads = torch.autograd.grad(by, leaves, torch.ones_like(by) if w is None else w)
    for name, a, b, c in zip(('dx', 'dweight'), grads, want[1:], limit[1:]):
        off = (a.double() - b).abs()
        assert a.dtype == x.dtype and (off <= c).all(), ('backward', name, (off - c).max(), off.max(), b.abs().max())
    return loss, dx, dw


@pytest.mark.parametrize('dtype', [BF16, F32])
@pytest.mark.parametrize('V', [1, 2, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 1000, 4096, 5003])
def test_vocabularies(V, dtype):
    for cap, width in ((None, V), (15.0, V + 5)):
        check(*make(70, V, 64, dtype, V, width), V, cap)


@pytest.mark.parametrize('dtype', [BF16, F32])
@pytest.mark.parametrize('D', [1, 7, 8, 9, 63, 64, 65, 127, 128, 200, 255, 256, 257, 320, 512, 776, 1000, 1024, 2048])
def test_widths(D, dtype):
    check(*make(40, 300, D, dtype, D), 300, 15.0 if D % 2 else None)


@pytest.mark.parametrize('dtype', [BF16, F32])
@pytest.mark.parametrize('R', [1, 2, 3, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 600, 2049])
def test_rows(R, dtype):
    check(*make(R, 700, 128, dtype, R, masked=R % 2 == 1), 700, None if R % 3 else 15.0)


@pytest.mark.parametrize('dtype', [BF16, F32])
@pytest.mark.parametrize('V', [17, 32767, 32768, 40001])
def test_few_rows(V, dtype):
    """Up to 256 tokens may have kernels of their own, by the sizes: next to those of more."""
    for R, D in ((1, 1), (4, 130), (16, 128), (17, 7), (31, 257), (33, 96), (64, 1000), (65, 64), (129, 2000), (200, 776), (256, 64), (257, 72)):
        check(*make(R, V, D, dtype, R, V + R % 3, masked=R % 2 == 1), V, 15.0 if R % 4 == 0 else None)


@pytest.mark.parametrize('dtype', [BF16, F32])
@pytest.mark.parametrize('R,V,D', [(793, 119, 4096), (257, 2, 2000), (2000, 33, 1001), (5000, 1, 64), (70000, 3, 40), (400, 1500, 3000)])
def test_many_rows_of_few_entries(R, V, D, dtype):
    """Whose logits may be formed as those of few rows are."""
    check(*make(R, V, D, dtype, R, V + 2, masked=R % 2 == 1), V, 15.0 if R % 4 == 0 else None)


@pytest.mark.parametrize('dtype', [BF16, F32])
def test_few_rows_of_a_large_weight(dtype):
    """Gradients past the caches' size, of rows of whole lines and of others."""
    for D in (1024, 1032, 1001):
        check(*make(20, 140000, D, dtype, D, 140003, masked=True), 140000, 15.0)


@pytest.mark.parametrize('dtype', [BF16, F32])
@pytest.mark.parametrize('cap', [1e-6, 0.01, 1.0, 32.0, 33.0, 100.0, 1e3, 1e6])
def test_caps(cap, dtype):
    """Of the whole range, for few rows and for many: far above the logits they leave these as they are."""
    for R in (9, 300):
        check(*make(R, 700, 128, dtype, R, masked=R == 300), 700, cap)


@pytest.mark.parametrize('dtype', [BF16, F32])
def test_masks(dtype):
    """Rows without a target hold NaN and infinities; all of them, all but one; weights with NaN there; int32 targets."""
    x, weight, targets, w = make(300, 500, 96, dtype, 3, 520, masked=True)
    used = (targets >= 0) & (targets < 500)
    w[~used] = float('nan')
    a = check(x, weight, targets, w, 500, 15.0)
    b = check(x, weight, targets.clamp(-2 ** 31, 2 ** 31 - 1).int(), w, 500, 15.0)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert not a[0][~used].any() and not a[1][~used].any()
    # (how sums are cut, and which kernels form the logits, goes by the number of rows: the rows in use alone need not give the same bits)
    check(x[used], weight, targets[used], w[used], 500, 15.0)
    for keep in (0, 1):
        t = torch.full_like(targets, -100)
        t[200:200 + keep] = 7
        x[200] = 1
        w[200] = 0.5
        out = check(x, weight, t, w, 500)
        assert keep or not any(o.any() for o in out)


@pytest.mark.parametrize('dtype', [BF16, F32])
def test_shapes_and_strides(dtype):
    """Batches of sequences, views with other distances between rows, transposed ones; weights None."""
    from noise_amd.vocab import linear_cross_entropy, linear_cross_entropy_grad
    x, weight, targets, w = make(60, 130, 64, dtype, 4)
    base = check(x, weight, targets, None, 130)
    forms = [(x.view(3, 20, 64), weight), (torch.cat([x, x], 1)[:, 64:], torch.cat([weight, weight], 1)[:, :64]),
             (x.t().contiguous().t(), weight.t().contiguous().t()), (torch.cat([x, x[:, :3]], 1)[:, :64], torch.cat([weight, weight[:, :1]], 1)[:, :64]),
             (torch.cat([x[:, :1], x], 1)[:, 1:], torch.cat([weight[:, :1], weight], 1)[:, 1:])]
    for a, b in forms:
        t = targets.view(a.shape[:-1])
        got = linear_cross_entropy_grad(a, b, t)
        assert all(torch.equal(p.reshape(q.shape), q) for p, q in zip(got, base))
        assert torch.equal(linear_cross_entropy(a, b, t).reshape(-1), linear_cross_entropy(x, weight, targets))
    row = x[:1].expand(60, 64)
    check(row, weight, targets, w, 130)
    one = linear_cross_entropy(x[5], weight, targets[5])
    assert one.shape == () and abs(one.item() - base[0][5].item()) <= 1e-4


@pytest.mark.parametrize('dtype', [BF16, F32])
def test_pieces(dtype):
    """More tokens times vocabulary than one piece of dZ holds."""
    R, V, D = (900, 1300001, 8) if dtype == BF16 else (500, 1300001, 8)
    x, weight, targets, w = make(R, V, D, dtype, 5)
    from noise_amd.vocab import linear_cross_entropy_grad
    loss, dx, dw = linear_cross_entropy_grad(x, weight, targets, w)
    ws, tol = weight.double(), HALF[BF16] if dtype == BF16 else 2.0 ** -18
    # dx: sums of V terms in V / 16 + 88 steps (three times V / 16 in fp32), as the bounds above count them
    steps = (1 if dtype == BF16 else 3) * V / 16 + 88
    want_dw = torch.zeros(V, D, dtype=torch.float64, device=DEV)
    for rows in torch.arange(R, device=DEV).split(150):
        xs = x[rows].double()
        log_p = torch.log_softmax(xs @ ws.t(), -1)
        want = -log_p.gather(1, targets[rows][:, None])[:, 0]
        assert ((loss[rows].double() - want).abs() <= F * (80 + V / 128 + 200)).all()
        p = log_p.exp_()
        p[torch.arange(len(rows), device=DEV), targets[rows]] -= 1
        p *= w[rows].double()[:, None]
        size = p.abs() @ ws.abs()
        assert ((dx[rows].double() - p @ ws).abs() <= (2 * tol + steps * F) * size + HALF[dtype] * (p @ ws).abs()).all()
        want_dw += p.t() @ xs
        del log_p, p
    norm = (dw.double() - want_dw).norm() / want_dw.norm()
    assert norm <= (2 * HALF[BF16] if dtype == BF16 else 2.0 ** -18), norm


@pytest.mark.parametrize('dtype', [BF16, F32])
def test_weight_past_32_bits(dtype):
    """A weight of more than 2^31 elements, zero but for some rows at its ends and in its middle. z: F (steps as above) and 2^-21 of
    |x| |W|^T, from which p and so a gradient's terms are off by that of themselves."""
    from noise_amd.vocab import linear_cross_entropy_grad
    V, D = 33000, 65536
    at = torch.cat([torch.tensor([0, 1, 16384, 32768]), torch.arange(V - 60, V)]).to(DEV)
    g = torch.Generator(DEV).manual_seed(11)
    some = (torch.randn(len(at), D, device=DEV, generator=g) / 256).to(dtype)
    weight = torch.zeros(V, D, device=DEV, dtype=dtype)
    weight[at] = some
    some = some.double()
    for R in (20, 300):
        x = torch.randn(R, D, device=DEV, generator=g).to(dtype)
        which, w = torch.randint(len(at), (R,), device=DEV, generator=g), torch.rand(R, device=DEV, generator=g)
        loss, dx, dw = linear_cross_entropy_grad(x, weight, at[which], w)
        z = x.double() @ some.t()
        lse = torch.log(z.exp().sum(-1) + V - len(at))
        ez = (F * ((3 if dtype == F32 else 1) * D / 16 + 24) + 2.0 ** -21) * (x.double().abs() @ some.abs().t()).max()
        want = lse - z.gather(1, which[:, None])[:, 0]
        assert ((loss - want).abs() <= 2 * ez + F * (80 + V / 128 + 200)).all()
        p = (z - lse[:, None]).exp()
        p[torch.arange(R, device=DEV), which] -= 1
        p *= w.double()[:, None]
        tol = 2 * ez + 2 * (HALF[BF16] if dtype == BF16 else 2.0 ** -18)
        for name, a, b in (('dx', dx, p @ some), ('dweight', dw[at], p.t() @ x.double()),
                           ('elsewhere', dw[[2, 20000, 32769, V - 61]], ((w * (-lse).exp())[None] @ x.double()).expand(4, D))):
            assert (a - b).norm() <= tol * b.norm(), (name, (a - b).norm() / b.norm(), tol)
        del loss, dx, dw


def test_rows_past_32_bits():
    """More than 2^31 elements of x: the last tokens' results are those of a call of their own, dW the calls' sum."""
    from noise_amd.vocab import linear_cross_entropy_grad
    R, V, D, N = 2 ** 20 + 4321, 200, 2048, 8
    g = torch.Generator(DEV).manual_seed(12)
    x = torch.randn(R, D, device=DEV, generator=g, dtype=BF16)
    weight = (torch.randn(V, D, device=DEV, generator=g) / 32).to(BF16)
    targets, w = torch.randint(V, (R,), device=DEV, generator=g), torch.rand(R, device=DEV, generator=g) / R
    loss, dx, dw = linear_cross_entropy_grad(x, weight, targets, w)
    total = torch.zeros(V, D, device=DEV, dtype=torch.float64)
    for rows in torch.arange(R, device=DEV).tensor_split(N):
        a, b = int(rows[0]), int(rows[-1]) + 1
        part = linear_cross_entropy_grad(x[a:b], weight, targets[a:b], w[a:b])
        # (the same products in the same order, but for dx where its k may be cut)
        assert torch.equal(loss[a:b], part[0])
        assert (dx[a:b].float() - part[1].float()).norm() <= HALF[BF16] * part[1].float().norm()
        total += part[2].double()
    assert (dw - total).norm() <= 2 * HALF[BF16] * total.norm()


def test_values():
    """Logits far apart, certain and hopeless predictions, soft-capped ones past the cap; infinite and NaN rows stay theirs."""
    from noise_amd.vocab import linear_cross_entropy, linear_cross_entropy_grad
    for dtype in (BF16, F32):
        for scale in (1e-3, 30.0, 300.0):
            for cap in (None, 15.0, 0.5):
                check(*make(50, 400, 64, dtype, 6, scale=scale), 400, cap)
        x, weight, targets, w = make(50, 400, 64, dtype, 7)
        clean = linear_cross_entropy_grad(x, weight, targets, w)
        bad = x.clone()
        bad[10, 3], bad[20, 5] = float('nan'), float('inf')
        loss = linear_cross_entropy(bad, weight, targets)
        dx = linear_cross_entropy_grad(bad, weight, targets, w)[1]
        rest = [r for r in range(50) if r not in (10, 20)]
        assert not torch.isfinite(loss[[10, 20]]).any() and torch.equal(loss[rest], linear_cross_entropy(x, weight, targets)[rest])
        assert torch.isnan(dx[10]).all() and torch.equal(dx[rest], clean[1][rest])
    # tensors of very different sizes in fp32
    x, weight, targets, w = make(50, 400, 64, F32, 8)
    check(x * 1e-20, weight * 1e20, targets, w, 400)
    check(x * 1e12, weight * 1e-12, targets, w * 1e-20, 400)


@pytest.mark.parametrize('D', [8, 40, 72, 200, 776])
def test_what_stands_beside_the_weight(D):
    """Rows that end inside a stage, with NaN between them and behind the last; a logit of -inf leaves its token's loss finite."""
    from noise_amd.vocab import linear_cross_entropy, linear_cross_entropy_grad
    for R in (30, 300):
        x, weight, targets, w = make(R, 500, D, BF16, D)
        wide = torch.full((500, D + 16), float('nan'), device=DEV, dtype=BF16)
        wide[:, :D] = weight
        base = check(x, weight, targets, w, 500)
        for a, b in zip(base, linear_cross_entropy_grad(x, wide[:, :D], targets, w)):
            assert torch.equal(a, b)
        x, targets = x.abs() + 1, targets % 499
        weight[499, D - 1] = -float('inf')
        loss = linear_cross_entropy(x, weight, targets)
        weight[499] = -1e4
        assert torch.isfinite(loss).all() and torch.equal(loss, linear_cross_entropy(x, weight, targets))


def test_repetition_and_streams():
    """The same bits every time and on another stream."""
    from noise_amd.vocab import linear_cross_entropy_grad
    x, weight, targets, w = make(1000, 3000, 256, BF16, 9, masked=True)
    base = linear_cross_entropy_grad(x, weight, targets, w)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(base, linear_cross_entropy_grad(x, weight, targets, w)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = linear_cross_entropy_grad(x, weight, targets, w)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(base, other))


@pytest.mark.parametrize('dtype', [BF16, F32])
def test_graph(dtype):
    """A captured step, replayed on other tokens with other masks."""
    from noise_amd.vocab import linear_cross_entropy, linear_cross_entropy_grad
    x, weight, targets, w = make(500, 1000, 128, dtype, 10)
    leaves = x.clone().requires_grad_(), weight.clone().requires_grad_()

    def step():
        loss = linear_cross_entropy(*leaves, targets, softcap=15.0)
        return (loss, *torch.autograd.grad(loss, leaves, w), *linear_cross_entropy_grad(*leaves, targets, w, softcap=15.0))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(3):
        new = make(500, 1000, 128, dtype, 20 + seed, masked=seed > 0)
        with torch.no_grad():
            for a, b in zip((*leaves, targets, w), new):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip([o.detach().clone() for o in outs], step()):
            assert torch.equal(a, b.detach())


@pytest.mark.parametrize('R', [1, 40, 100])
@pytest.mark.parametrize('dtype', [BF16, F32])
def test_few_rows_captured_and_repeated(dtype, R):
    """The same bits every time, on another stream, and from two graphs replayed in turn on other tokens with other masks."""
    from noise_amd.vocab import linear_cross_entropy, linear_cross_entropy_grad
    V, D = 1500, 203
    sets, graphs = [make(R, V, D, dtype, seed) for seed in (1, 2)], []

    def step(x, weight, targets, w):
        leaves = x.detach().requires_grad_(), weight.detach().requires_grad_()
        loss = linear_cross_entropy(*leaves, targets, softcap=15.0)
        return (loss.detach(), *torch.autograd.grad(loss, leaves, w), *linear_cross_entropy_grad(x, weight, targets, w, softcap=15.0))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [step(*s) for s in sets]
    torch.cuda.synchronize()
    for s, o in zip(sets, other):
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(o, step(*s)))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(*s)
        graphs.append((graph, outs))
    for seed in range(3):
        for s, (graph, outs) in zip(sets, graphs):
            for a, b in zip(s, make(R, V, D, dtype, 30 + seed, masked=seed > 0)):
                a.copy_(b)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip([o.clone() for o in outs], step(*s)):
                assert torch.equal(a, b)


def test_gradients_asked_for_one_by_one():
    from noise_amd.vocab import linear_cross_entropy
    x, weight, targets, w = make(300, 900, 128, BF16, 11)
    both = [x.detach().requires_grad_(), weight.detach().requires_grad_()]
    every = torch.autograd.grad(linear_cross_entropy(*both, targets), both, w)
    for i in range(2):
        leaves = [t.detach().requires_grad_(i == j) for j, t in enumerate((x, weight))]
        assert torch.equal(torch.autograd.grad(linear_cross_entropy(*leaves, targets), leaves[i], w)[0], every[i])


@pytest.mark.parametrize('dtype', [BF16, F32])
def test_few_gradients_asked_for_one_by_one(dtype):
    from noise_amd.vocab import linear_cross_entropy
    for R in (1, 33, 70):
        x, weight, targets, w = make(R, 900, 127, dtype, 11, masked=R > 1)
        both = [x.detach().requires_grad_(), weight.detach().requires_grad_()]
        every = torch.autograd.grad(linear_cross_entropy(*both, targets), both, w)
        for i in range(2):
            leaves = [t.detach().requires_grad_(i == j) for j, t in enumerate((x, weight))]
            assert torch.equal(torch.autograd.grad(linear_cross_entropy(*leaves, targets), leaves[i], w)[0], every[i])


def test_differences():
    """The gradients along a direction against a difference quotient (fp32; step 2^-8: off by the second differences and the
    losses' roundings over the step)."""
    from noise_amd.vocab import linear_cross_entropy, linear_cross_entropy_grad
    x, weight, targets, w = make(20, 50, 32, F32, 12)
    _, dx, dw = linear_cross_entropy_grad(x, weight, targets, w, softcap=15.0)
    value = lambda a, b: (linear_cross_entropy(a, b, targets, softcap=15.0).double() * w.double()).sum().item()
    g = torch.Generator(DEV).manual_seed(1)
    h = 2.0 ** -8
    for i, d in enumerate((dx, dw)):
        along = torch.randn(d.shape, device=DEV, generator=g)
        step = lambda s: value(x + s * along, weight) if i == 0 else value(x, weight + s * along)
        quotient, exact = (step(h) - step(-h)) / (2 * h), (d.double() * along).sum().item()
        size = w.sum().item()
        assert abs(quotient - exact) <= size * (200 * F / h + 100 * h * h), (i, quotient, exact)


def test_no_rows():
    from noise_amd.vocab import linear_cross_entropy, linear_cross_entropy_grad
    x, weight, targets, w = make(0, 30, 16, F32)
    loss, dx, dw = linear_cross_entropy_grad(x, weight, targets, w)
    assert loss.shape == (0,) and dx.shape == (0, 16) and not dw.any()
    leaf = weight.detach().requires_grad_()
    assert not torch.autograd.grad(linear_cross_entropy(x, leaf, targets).sum(), leaf)[0].any()


def test_compiled():
    from noise_amd.vocab import linear_cross_entropy, linear_cross_entropy_grad
    x, weight, targets, w = make(100, 300, 64, BF16, 13)

    def step(x, weight):
        return linear_cross_entropy(x, weight, targets, softcap=15)
    a, b = ([t.detach().requires_grad_() for t in (x, weight)] for _ in range(2))
    la, lb = step(*a), torch.compile(step, fullgraph=True)(*b)
    assert torch.equal(la, lb)
    for p, q in zip(torch.autograd.grad(la, a, w), torch.autograd.grad(lb, b, w)):
        assert torch.equal(p, q)
    both = lambda x, weight: linear_cross_entropy_grad(x, weight, targets, w)
    for p, q in zip(both(x, weight), torch.compile(both, fullgraph=True)(x, weight)):
        assert torch.equal(p, q)
