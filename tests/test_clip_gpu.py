"""clip_gradients against 64 bits.

Bounds: squares and sums are in fp64, so the norm is off by its rounding to fp32 (2^-24) and the factor, rounded to fp32, by as much
again; a clipped value has one more rounding in fp32, and in bf16 half a step of its own."""
import math

import pytest
import torch

from oracle import training as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda', 0)
BF16, F32 = torch.bfloat16, torch.float32
F = 2.0 ** -24


def make(sizes, types, seed=0, scale=0.01, offset=0):
    g = torch.Generator(DEV).manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        t = torch.randn(n + offset, device=DEV, generator=g).mul_(scale).to(types[i % len(types)])
        out.append(t[offset:])
    return out


def check(gradients, max_norm):
    from noise_amd.clip import clip_gradients
    want, clipped = oracle.clip(gradients, max_norm)
    before = [g.clone() for g in gradients]
    norm = clip_gradients(gradients, max_norm)
    assert norm.dtype == F32 and norm.shape == () and abs(norm.item() - want) <= 2 * F * want
    for g, b, c in zip(gradients, before, clipped):
        if want + 1e-6 <= max_norm:
            assert torch.equal(g, b)
            continue
        step = F if g.dtype == F32 else 2.0 ** -8 * (1 + 2 ** -10)
        assert ((g.double() - c).abs() <= (step + 3 * F) * c.abs() + 1e-45).all()
    return norm


SIZES = [1, 2, 3, 5, 8, 31, 255, 4096, 16383, 16384, 16385, 100003]


@pytest.mark.parametrize('offset', [0, 1, 2, 3, 7])
@pytest.mark.parametrize('types', [(F32,), (BF16,), (F32, BF16)])
def test_sizes(types, offset):
    for n in SIZES:
        check(make([n], types, n, offset=offset), 0.005 * math.sqrt(n))
    check(make(SIZES, types, 1, offset=offset), 1.0)
    check(make(SIZES, types, 1, offset=offset), 1e9)


@pytest.mark.parametrize('count', [1, 2, 191, 192, 193, 384, 385, 1000])
def test_counts(count):
    """Tables of one launch, of several, and empty tensors between."""
    sizes = [(i * 7919) % 3001 if i % 5 else 0 for i in range(count)]
    gradients = make(sizes, (F32, BF16), count)
    if sum(sizes):
        check(gradients, 0.003 * math.sqrt(sum(sizes)))
    before = [g.clone() for g in gradients]
    check(gradients, math.inf)
    assert all(torch.equal(a, b) for a, b in zip(gradients, before))


def test_large():
    """Past 2^32 bytes in one tensor; more units than workgroups."""
    g = make([2 ** 30 + 2 ** 28 + 5, 77], (F32, BF16), 3)
    want = math.sqrt(sum(float(torch.linalg.vector_norm(t, dtype=torch.float64)) ** 2 for t in g))
    last, first = g[0][-5:].double(), g[0][:5].double()
    from noise_amd.clip import clip_gradients
    norm = clip_gradients(g, 1.0)
    assert abs(norm.item() - want) <= 2 * F * want
    factor = 1.0 / (want + 1e-6)
    for a, b in ((g[0][-5:], last), (g[0][:5], first)):
        assert ((a.double() - b * factor).abs() <= 4 * F * (b * factor).abs()).all()
    left = float(torch.linalg.vector_norm(g[0], dtype=torch.float64))
    assert abs(left - 1.0) <= 1e-4


def test_values():
    """Norms past fp32's range of squares; zeros; NaN and infinities."""
    from noise_amd.clip import clip_gradients
    check([torch.full((1000,), 1e30, device=DEV)], 1.0)
    check([torch.full((1000,), 1e-30, device=DEV)], 1e-29)
    check([torch.zeros(50, device=DEV), torch.zeros(3, device=DEV, dtype=BF16)], 1.0)
    check([torch.ones(50, device=DEV)], 0.0)
    g = make([100, 200], (F32, BF16), 4)
    g[0][3] = float('nan')
    assert math.isnan(clip_gradients(g, 1.0).item()) and all(bool(t.isnan().all()) for t in g)
    g = make([100, 200], (F32, BF16), 4)
    g[1][3] = float('inf')
    assert clip_gradients(g, 1.0).item() == math.inf
    assert bool((g[0] == 0).all()) and math.isnan(g[1][3].item()) and int((g[1] == 0).sum()) == 199
    g = make([100], (F32,), 4)
    g[0][3] = float('inf')
    before = g[0].clone()
    assert clip_gradients(g, math.inf).item() == math.inf and torch.equal(g[0], before)


def test_layouts_and_repetition():
    """Transposed and permuted gradients; the same bits every time."""
    a = torch.randn(30, 50, device=DEV).t()
    b = torch.randn(4, 5, 6, device=DEV).permute(2, 0, 1).to(BF16)
    results = []
    for _ in range(3):
        g = [a.clone(memory_format=torch.preserve_format), b.clone(memory_format=torch.preserve_format)]
        results.append((check(g, 3.0), *g))
    for r in results[1:]:
        assert all(torch.equal(x, y) for x, y in zip(results[0], r))


def test_graph():
    """Captured and replayed on new values, with two captured graphs in turn."""
    from noise_amd.clip import clip_gradients
    sets = [make([5000, 70001, 3], (F32, BF16), s) for s in (1, 2)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        clip_gradients([g.clone() for g in sets[0]], 1.0)
    torch.cuda.synchronize()
    graphs = []
    for g in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norm = clip_gradients(g, 1.0)
        graphs.append((graph, norm))
    for seed in range(3):
        for (graph, norm), g in zip(graphs, sets):
            new = make([5000, 70001, 3], (F32, BF16), 10 + seed)
            for t, v in zip(g, new):
                t.copy_(v)
            graph.replay()
            assert norm.item() == clip_gradients(new, 1.0).item()
            assert all(torch.equal(t, v) for t, v in zip(g, new))


def test_eggroll_step_clips():
    """Eggroll.step's bound: the update is the one without it, scaled as its norm asks."""
    from noise_amd.eggroll import Eggroll
    from noise_amd.model import make_model
    tokens = torch.randint(0, 4096, (1, 257), generator=torch.Generator().manual_seed(0)).to(DEV)
    x, y = tokens[:, :-1], tokens[:, 1:]
    seen = []
    for max_norm in (None, 1e30, 1e-3):
        es = Eggroll(make_model(DEV, 0), pairs=4)
        es.step(x, y, torch.optim.SGD(es.params.values(), lr=0.0), 0, max_norm=max_norm)
        seen.append([p.grad.clone() for p in es.params.values()])
    assert all(torch.equal(a, b) for a, b in zip(seen[0], seen[1]))
    norm, want = oracle.clip(seen[0], 1e-3)
    assert norm > 1e-3
    for g, w in zip(seen[2], want):
        assert ((g.double() - w).abs() <= 4 * F * w.abs() + 1e-45).all()


def test_factors_past_fp32():
    """Norms so far above the bound that the factor has no normal fp32 value: the values are as near as with any other (the 64-bit
    factor's parts, one rounding to 24 bits and the product's); the norm, past fp32's range, is stored as infinite."""
    from noise_amd.clip import clip_gradients
    g = torch.Generator(DEV).manual_seed(5)
    for types, scale, max_norm in (((F32,), 1e38, 1.0), ((BF16, F32), 1e38, 3.0), ((F32,), 1e38, 1e-30), ((F32, BF16), 1e10, 1e-30),
                                   ((F32,), 3e38, 1e-38)):
        gradients = [((torch.rand(n, device=DEV, generator=g) + 0.1) * scale).to(types[i % len(types)]) for i, n in enumerate((1000, 70001, 3))]
        want, clipped = oracle.clip(gradients, max_norm)
        norm = clip_gradients(gradients, max_norm)
        assert norm.item() == math.inf if want > 3.5e38 else abs(norm.item() - want) <= 2 * F * want
        for a, b in zip(gradients, clipped):
            step = F if a.dtype == F32 else 2.0 ** -8 * (1 + 2 ** -10)
            least = 2.0 ** -150 if a.dtype == F32 else 2.0 ** -134   # half the smallest values' step
            assert ((a.double() - b).abs() <= (step + 3 * F) * b.abs() + 2 * least).all(), (types, scale, max_norm)
