"""distill_loss and distill_loss_grad against the 64-bit definition.

Bounds: z, the teacher's t and their exponents are fp32 values of size up to A = max |z| + log V, each with a few roundings
(2^-24 each: cap, quotient, shift, exponent), so a loss is off by at most about 16 2^-24 tau^2 (A + sum p |log p|) and a
gradient by 2^-24 (16 + 8 A) tau (q_v + p_v) |cap'| plus the cap's own 8 roundings and, in bf16, half a step of the result."""
import math

import pytest
import torch

from oracle import distill as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda', 0)
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
F = 2.0 ** -24


def make(R, V, W, K, dtype, seed, index=torch.int64, scale=3.0):
    g = torch.Generator(DEV).manual_seed(seed)
    x = scale * torch.randn(R, W, device=DEV, generator=g)
    t, i = (x[:, :V] + torch.randn(R, V, device=DEV, generator=g)).topk(K, -1)
    return x.to(dtype), t.to(dtype), i.to(index), torch.rand(R, device=DEV, generator=g)


def check_all(x, t, i, w, vocab, tau, cap):
    from noise_amd.distill import distill_loss, distill_loss_grad
    loss, grad = distill_loss_grad(x, t, i, w, vocab=vocab, temperature=tau, softcap=cap)
    assert loss.dtype == torch.float32 and grad.dtype == x.dtype and grad.shape == x.shape
    want, want_grad = oracle.distill(x, t, i, vocab, tau, cap, w)
    A = (x[:, :vocab].double().abs().clamp(max=cap or 1e30).amax(-1) / tau + math.log(vocab) +
         t.double().nan_to_num(neginf=0).abs().amax(-1) / tau)
    off = (loss.double() - want).abs()
    assert (off <= 16 * F * tau ** 2 * A).all(), (off / (F * tau ** 2 * A)).max()
    z = x[:, :vocab].double()
    slope = 1.0
    if cap:
        z, slope = cap * torch.tanh(z / cap), 1 - torch.tanh(z / cap) ** 2
    qv = torch.softmax(z / tau, -1)
    g = want_grad[:, :vocab].abs()
    wt = 1 if w is None else w.double()[:, None]
    parts = (g + 2 * qv * slope * tau * wt)                       # >= (q + p) |cap'| tau weight
    bound = HALF[x.dtype] * g + F * (16 + 8 * A)[:, None] * parts
    if cap:
        bound = bound + 8 * F * (g / slope.clamp(min=1e-30)).nan_to_num(0, 0, 0).clamp(max=tau) * wt
    off = (grad[:, :vocab].double() - want_grad[:, :vocab]).abs()
    assert (off <= bound + 1e-37).all(), (off - bound).max()
    assert (grad[:, vocab:] == 0).all()
    assert torch.equal(distill_loss(x, t, i, vocab=vocab, temperature=tau, softcap=cap), loss)
    leaf = x.detach().requires_grad_()
    by = distill_loss(leaf, t, i, vocab=vocab, temperature=tau, softcap=cap)
    assert torch.equal(torch.autograd.grad(by, leaf, torch.ones_like(by) if w is None else w)[0], grad)
    return loss, grad


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('V', [1, 2, 7, 63, 64, 65, 257, 1000, 2049, 4096, 4097, 8191, 16384, 20011, 65536, 100001, 200003, 250000])
def test_vocabularies(V, dtype):
    for W, K, tau, cap in ((V, min(V, 5), 1.0, None), (V + 1, min(V, 64), 2.0, 15.0), (V + 47, 1, 0.7, None)):
        print(V, W, K, tau, cap, dtype, flush=True)
        check_all(*make(6, V, W, K, dtype, V), V, tau, cap)


@pytest.mark.parametrize('K', [1, 2, 63, 64, 65, 129, 300, 1000])
def test_entries(K):
    for index in (torch.int32, torch.int64):
        check_all(*make(9, 1200, 1201, K, torch.float32, K, index), 1200, 1.5, 15.0)


def test_entries_left_out():
    """Indices of -1, past the vocabulary and far out, logits of -inf, whole rows of them; the same index twice."""
    x, t, i, w = make(8, 500, 512, 20, torch.float32, 1)
    i[0] = -1
    i[1, 3:] = -1
    i[2, :] = 500
    i[3, ::2] = 2 ** 40
    t[4, 5:9] = -math.inf
    t[5] = -math.inf
    i[6, :10] = i[6, 10]
    i[7] = 499
    loss, grad = check_all(x, t, i, w, 500, 2.0, None)
    for r in (0, 2, 5):
        assert loss[r] == 0 and (grad[r] == 0).all()
    check_all(x.bfloat16(), t.bfloat16(), i, None, 500, 1.0, 15.0)


def test_extreme_logits():
    """The type's lowest value and -inf beside ordinary logits, a lone peak, equal logits."""
    x, t, i, w = make(5, 300, 300, 8, torch.float32, 2)
    x[0, 100:200] = torch.finfo(torch.float32).min
    x[1, 100:200] = -math.inf
    for r in (0, 1):
        i[r] = torch.arange(8, device=DEV)
    x[2] = -100.0
    x[2, 7] = 100.0
    x[3] = 0.0
    check_all(x, t, i, w, 300, 1.0, None)
    from noise_amd.distill import distill_loss_grad
    x[1, 0] = -math.inf      # the teacher wants what the student rules out
    loss, _ = distill_loss_grad(x, t, i)
    assert loss[1] == math.inf and torch.isfinite(loss[[0, 2, 3, 4]]).all()
    x[4, 9] = math.nan
    t[3, 0] = math.nan
    loss, _ = distill_loss_grad(x, t, i)
    assert torch.isnan(loss[[3, 4]]).all() and torch.isfinite(loss[[0, 2]]).all()


@pytest.mark.parametrize('cap', [None, 15.0])
@pytest.mark.parametrize('dtype,V', [(torch.float32, 300), (torch.float32, 100001), (torch.bfloat16, 300),
                                     (torch.bfloat16, 200003)])
def test_infinities_in_rows_of_any_width(V, dtype, cap):
    """-inf (a value of -softcap under the cap, nothing without it) over the first half of a row, everywhere but at one place
    or the last one, and in the whole row; NaN beside -inf at the row's start, or at its end, in a row that is finite elsewhere;
    inf under the cap.

    Bounds: a sum over the vocabulary has at most V / 1024 + 16 terms in turn (a thread's) and 10 levels, so log s is off by
    (V / 1024 + 26) 2^-24 beside the loss's 16 A 2^-24. In a gradient the cap's slope 1 - t^2 is off by less than 24 2^-24 (8
    roundings of t, twice, and those of the product) of the parts q + p that it multiplies."""
    from noise_amd.distill import distill_loss_grad
    tau, K = 2.0, 10
    x, t, i, w = make(8, V, V + 1, K, dtype, 30)
    half = V // 2 // 64 * 64
    x[0, :half] = -math.inf
    x[1, :V] = -math.inf
    x[1, half + 5] = 1.5
    x[2, :V] = -math.inf
    x[2, V - 1] = -2.5
    x[3, ::2] = -math.inf
    x[4, :V] = -math.inf
    x[5, :128] = -math.inf
    x[5, 70] = math.nan            # (in a thread's first elements, one without any of the row's last ones)
    x[6, V - 1] = math.nan
    where = torch.arange(half, half + 2 * K, 2, device=DEV) + 1
    i[0], i[1], i[2], i[3] = where, half + 5, V - 1, where    # (finite logits, so that a loss without the cap is)
    if cap:
        i[0, :3], i[1, 1:4], i[2, 1:4] = 0, 7, 8
        x[7, 9] = math.inf
    loss, grad = distill_loss_grad(x, t, i, w, vocab=V, temperature=tau, softcap=cap)
    assert torch.isnan(loss[5:7]).all() and torch.isnan(grad[5:7, :V]).all()
    rows = [0, 1, 2, 3, 7] + ([4] if cap else [])
    want, want_grad = oracle.distill(x[rows], t[rows], i[rows], V, tau, cap, w[rows])
    z = x[rows, :V].double()
    z = z if cap is None else cap * torch.tanh(z / cap)
    A = (z.abs().masked_fill(z == -math.inf, 0).amax(-1) + t[rows].double().abs().amax(-1)) / tau + math.log(V)
    off = (loss[rows].double() - want).abs()
    assert (off <= F * tau ** 2 * (16 * A + V / 1024 + 26)).all(), off
    parts = torch.softmax(z / tau, -1).scatter_add_(1, i[rows], torch.softmax(t[rows].double() / tau, -1))
    g = want_grad[:, :V]
    bound = HALF[dtype] * g.abs() + F * (40 + 8 * A + V / 1024 + 26)[:, None] * tau * w[rows].double()[:, None] * parts
    off = (grad[rows, :V].double() - g).abs()
    assert (off <= bound + 1e-37).all(), (off - bound).amax(-1)
    if cap is None:
        assert torch.isnan(loss[4])     # a row of nothing but -inf has no softmax


def test_agreement():
    """A student equal to the teacher over the whole vocabulary: no loss, no gradient (to the roundings)."""
    x, _, _, _ = make(4, 64, 64, 1, torch.float32, 3)
    i = torch.arange(64, device=DEV).expand(4, 64)
    loss, grad = check_all(x, x.clone(), i, None, 64, 1.5, None)
    assert loss.abs().max() < 1e-4 and grad.abs().max() < 1e-6


def test_shapes_and_strides():
    from noise_amd.distill import distill_loss, distill_loss_grad
    x, t, i, w = make(12, 200, 209, 6, torch.bfloat16, 4)
    want = check_all(x, t, i, w, 200, 1.0, None)
    shaped = distill_loss_grad(x.view(3, 4, 209), t.view(3, 4, 6), i.view(3, 4, 6), w.view(3, 4), vocab=200)
    assert torch.equal(shaped[0].view(-1), want[0]) and torch.equal(shaped[1].view(12, 209), want[1])
    for view in (torch.randn(12, 300, device=DEV).bfloat16()[:, 5:214], torch.randn(209, 12, device=DEV).bfloat16().t(),
                 torch.randn(1, 209, device=DEV).bfloat16().expand(12, 209)):
        got = distill_loss_grad(view, t, i, w, vocab=200)
        same = distill_loss_grad(view.contiguous(), t, i, w, vocab=200)
        assert torch.equal(got[0], same[0]) and torch.equal(got[1], same[1])
    assert distill_loss(x[:0], t[:0], i[:0]).shape == (0,)
    leaf = x.detach().requires_grad_()
    distill_loss(leaf, t, i).mean().backward()      # an expanded upstream gradient
    ones = distill_loss_grad(x, t, i, torch.full((12,), 1 / 12, device=DEV))[1]
    assert torch.equal(leaf.grad, ones)


def test_gradients_against_differences():
    x, t, i, w = make(3, 90, 90, 10, torch.float32, 5)
    from noise_amd.distill import distill_loss_grad
    _, grad = distill_loss_grad(x, t, i, w, temperature=1.7, softcap=15.0)
    d = grad.double()
    at = lambda step: (oracle.distill(x.double() + step * d, t, i, 90, 1.7, 15.0)[0] * w.double()).sum()
    h = 1e-4 / d.abs().max()
    slope = (at(h) - at(-h)) / (2 * h)
    assert abs(slope - d.square().sum()) <= 1e-5 * d.square().sum()


def test_repeats_graphs_and_the_operator():
    from noise_amd.distill import distill_loss_grad
    x, t, i, w = make(50, 3000, 3001, 30, torch.bfloat16, 6)
    step = lambda: distill_loss_grad(x, t, i, w, temperature=2.0, softcap=15.0)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        x.mul_(-0.7)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    leaf = x.detach().requires_grad_()
    loss = torch.ops.noise_amd.distill_loss(leaf, t, i, 3001, 2.0, 15.0)
    assert torch.equal(loss, step()[0]) and torch.equal(torch.autograd.grad(loss, leaf, w)[0], step()[1])
