"""sink_attention_decode and qk_norm_rotary_append: new tokens against a cache.

The output's bound is sink_attention's: the weights are rounded to bf16 once and the result once (2^-8 each); parts of a
split row are joined in fp32."""
import math

import pytest
import torch

from oracle import sinks as oracle
from tests.test_sink_attention_gpu import DEV, MORE, U, check

pytestmark = pytest.mark.gpu


def caches(B, S, H, Hk, D, T, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    return [torch.randn(*s, device=DEV, generator=g).bfloat16() for s in ((B, T, H, D), (B, S, Hk, D), (B, S, Hk, D))]


def check_decode(q, k, v, start, window, sinks):
    from noise_amd.sinks import sink_attention_decode
    out = sink_attention_decode(q, k, v, start, window, sinks)
    want, weight = oracle.decode(q, k, v, start, window, sinks)
    check(out, want, U * (weight + want.abs()), 'out')
    return out


def spoil(k, v, start, T, window, sinks):
    """NaN, infinities and the lowest value in every slot that no token of the call sees."""
    D, bad = k.shape[3], torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(torch.bfloat16).min], device=DEV)
    j = torch.arange(k.shape[1], device=DEV)
    for b in range(k.shape[0]):
        seen = torch.zeros_like(j, dtype=torch.bool)
        for t in range(T):
            seen |= oracle.visible(int(start[b]) + t, j, window, sinks)
        for c in (k, v):
            c[b, ~seen] = bad.repeat(D // 4).bfloat16()


@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('H,Hk', [(1, 1), (8, 8), (8, 2), (12, 1), (32, 2)])
@pytest.mark.parametrize('T', [1, 3, 16])
def test_heads_and_positions(H, Hk, T, D):
    S = 700
    for window, sinks in ((10 ** 9, 0), (100, 4), (63, 64), (0, 0), (5, 130)):
        start = torch.tensor([0, S - T, -T, 317, 64, 5, S + 20, -2], device=DEV, dtype=torch.int32)
        print(H, Hk, T, D, window, sinks, flush=True)
        q, k, v = caches(8, S, H, Hk, D, T, 1)
        spoil(k, v, start, T, window, sinks)
        out = check_decode(q, k, v, start, window, sinks)
        assert (out[2] == 0).all()


@pytest.mark.parametrize('S', [1, 2, 31, 32, 33, 64, 65, 127, 129, 500])
def test_small_caches(S):
    for D, T in ((64, 1), (128, 2)):
        q, k, v = caches(3, S, 4, 2, D, T, S)
        start = torch.tensor([S - 1, S // 2, 0], device=DEV)
        check_decode(q, k, v, start, 17, 3)
        check_decode(q, k, v, start, S, 0)


@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('B', [1, 5, 40])
def test_long_caches(B, D):
    """Rows long enough to be split, among short and idle ones."""
    S = 9000
    q, k, v = caches(B, S, 4, 1, D, 1, B)
    start = torch.tensor([(S - 1, 4000, -1, 7, 8191)[b % 5] for b in range(B)], device=DEV, dtype=torch.int64)
    for window, sinks in ((10 ** 12, 0), (5000, 4), (1024, 300)):
        spoiled = k.clone(), v.clone()
        spoil(*spoiled, start, 1, window, sinks)
        check_decode(q, *spoiled, start, window, sinks)


def test_huge_positions_and_masks():
    q, k, v = caches(4, 100, 2, 2, 64, 2, 3)
    start = torch.tensor([2 ** 62, -2 ** 62, 2 ** 31, 99], device=DEV)
    for window, sinks in ((2 ** 40, 2 ** 40), (3, 2 ** 40), (2 ** 40, 1), (3, 0)):
        check_decode(q, k, v, start, window, sinks)
    far = torch.tensor([2 ** 63 - 1, -2 ** 63, 2 ** 63 - 2, 99], device=DEV)
    assert (check_decode(q, k, v, far.clamp(-1000, 1000), 3, 5) == check_decode(q, k, v, start, 3, 5))[[0, 3]].all()
    from noise_amd.sinks import sink_attention_decode
    assert torch.equal(sink_attention_decode(q, k, v, far, 3, 5), sink_attention_decode(q, k, v, start, 3, 5))


def test_strided_caches():
    g = torch.Generator(DEV).manual_seed(2)
    both = torch.randn(2, 3, 2, 300, 64, device=DEV, generator=g).bfloat16()   # [batch, head, k / v, slot, dim]
    k, v = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    q = torch.randn(2, 2, 6, 65, device=DEV, generator=g).bfloat16()[..., 1:]
    check_decode(q, k, v, torch.tensor([298, 100], device=DEV), 70, 9)


def test_offsets_past_32_bits():
    """A cache whose last slots lie more than 2^32 bytes (and 2^31 elements) from its start."""
    from noise_amd.sinks import sink_attention_decode
    S, Hk, D = 2_300_000, 8, 128
    k = torch.zeros(1, S, Hk, D, device=DEV, dtype=torch.bfloat16)
    v = torch.zeros(1, S, Hk, D, device=DEV, dtype=torch.bfloat16)
    g = torch.Generator(DEV).manual_seed(1)
    for c in (k, v):
        c[:, :4] = torch.randn(1, 4, Hk, D, device=DEV, generator=g).bfloat16()
        c[:, S - 3000:] = torch.randn(1, 3000, Hk, D, device=DEV, generator=g).bfloat16()
    q = torch.randn(1, 1, 16, D, device=DEV, generator=g).bfloat16()
    out = sink_attention_decode(q, k, v, torch.tensor([S - 1], device=DEV), 2999, 4)
    cut = [torch.cat([c[:, :4], c[:, S - 3000:]], 1) for c in (k, v)]
    want, weight = oracle.decode(q, *cut, torch.tensor([3003], device=DEV), 2999, 4)
    check(out, want, U * (weight + want.abs()), 'out')


def test_captured_decode():
    """One captured step replayed while the positions move on, against eager calls; two graphs share no workspace."""
    from noise_amd.sinks import sink_attention_decode
    S = 6000
    q, k, v = caches(2, S, 8, 2, 64, 1, 9)
    start = torch.tensor([10, 4000], device=DEV)
    step = lambda window: sink_attention_decode(q, k, v, start, window, 4)
    step(2000), step(100)
    torch.cuda.synchronize()
    graphs = []
    for window in (2000, 100):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(window)
        graphs.append((graph, out, window))
    for _ in range(4):
        start += 321
        q.mul_(-1)
        for graph, out, window in graphs:
            graph.replay()
        want = [step(window) for _, _, window in graphs]
        torch.cuda.synchronize()
        assert all(torch.equal(out, w) for (_, out, _), w in zip(graphs, want))


def tables(n, D):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    return a.cos().float().to(DEV), a.sin().float().to(DEV)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('D', [64, 128])
def test_append(D, dtype):
    """The cache takes k' and v at the tokens' positions and keeps every other slot; tokens past the cache or the tables
    and idle sequences write nothing and get zeros."""
    from noise_amd.sinks import qk_norm_rotary, qk_norm_rotary_append
    g = torch.Generator(DEV).manual_seed(D)
    for T, S, L in ((1, 9, 9), (5, 40, 40), (7, 64, 33), (3, 20, 50)):
        B, H, Hk = 6, 4, 2
        q, k, v, kc, vc = (torch.randn(*s, device=DEV, generator=g).to(dtype) for s in
                           ((B, T, H, D), (B, T, Hk, D), (B, T, Hk, D), (B, S, Hk, D), (B, S, Hk, D)))
        v[0, 0, 0, :2] = torch.tensor([math.nan, -math.inf], device=DEV)
        w = torch.randn(2, D, device=DEV, generator=g)
        cos, sin = tables(L, D)
        start = torch.tensor([0, S - T, -T, S - 1, 2 ** 40, -1], device=DEV)
        wk, wv = kc.clone(), vc.clone()
        got = qk_norm_rotary_append(q, k, v, cos, sin, kc, vc, start, w[0], w[1])
        want, keys = qk_norm_rotary(q, k, cos, sin, w[0], w[1], start=start)
        for b in range(B):
            for t in range(T):
                p = int(start[b]) + t
                if 0 <= p < min(S, L):
                    wk[b, p], wv[b, p] = keys[b, t], v[b, t]
                else:
                    want[b, t] = 0
        assert torch.equal(got, want) and torch.equal(kc, wk)
        assert torch.equal(vc.view(torch.uint8), wv.view(torch.uint8))


def test_append_into_strided_caches():
    from noise_amd.sinks import qk_norm_rotary, qk_norm_rotary_append
    g = torch.Generator(DEV).manual_seed(3)
    B, T, H, Hk, D, S = 2, 3, 4, 2, 64, 30
    both = torch.full((B, Hk, 2, S, D), 7.0, device=DEV, dtype=torch.bfloat16)
    qkv = torch.randn(B, T, H + 2 * Hk, D, device=DEV, generator=g).bfloat16()
    q, k, v = qkv.split([H, Hk, Hk], 2)
    cos, sin = tables(S, D)
    start = torch.tensor([4, 20], device=DEV, dtype=torch.int32)
    kc, vc = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    got = qk_norm_rotary_append(q, k, v, cos, sin, kc, vc, start)
    want, keys = qk_norm_rotary(q, k, cos, sin, start=start)
    assert torch.equal(got, want)
    for b in range(B):
        at = slice(int(start[b]), int(start[b]) + T)
        assert torch.equal(kc[b, at], keys[b]) and torch.equal(vc[b, at], v[b])
        rest = torch.ones(S, dtype=torch.bool, device=DEV)
        rest[at] = False
        assert (kc[b, rest] == 7).all() and (vc[b, rest] == 7).all()


@pytest.mark.parametrize('D,H,Hk', [(64, 8, 8), (128, 8, 2)])
def test_a_conversation(D, H, Hk):
    """A prompt, then tokens one by one and some at once: the rows agree with one sink_attention over everything, within
    the roundings of both."""
    from noise_amd.sinks import qk_norm_rotary, qk_norm_rotary_append, sink_attention, sink_attention_decode
    g = torch.Generator(DEV).manual_seed(1)
    B, T, P, window, sinks = 2, 230, 200, 64, 4
    q, k, v = (torch.randn(B, T, h, D, device=DEV, generator=g).bfloat16() for h in (H, Hk, Hk))
    cos, sin = tables(T, D)
    whole = sink_attention(*qk_norm_rotary(q, k, cos, sin), v, window, sinks)
    kc, vc = (torch.full((B, T, Hk, D), math.nan, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    cut = lambda a, n: [t[:, a:a + n] for t in (q, k, v)]
    start = torch.zeros(B, device=DEV, dtype=torch.int32)
    first = qk_norm_rotary_append(*cut(0, P), cos, sin, kc, vc, start)
    rows = [sink_attention(first, kc[:, :P], vc[:, :P], window, sinks)]
    at = P
    for n in (1, 1, 5, 1, 16, 6):
        start.fill_(at)
        new = qk_norm_rotary_append(*cut(at, n), cos, sin, kc, vc, start)
        rows.append(sink_attention_decode(new, kc, vc, start, window, sinks))
        at += n
    rows = torch.cat(rows, 1).double()
    assert at == T
    want, weight = oracle.attend(*qk_norm_rotary(q, k, cos, sin), v, window, sinks)
    bound = MORE * U * (weight + want.abs())
    assert ((rows - want).abs() <= bound).all() and ((whole.double() - want).abs() <= bound).all()


def test_views_with_odd_strides_of_single_elements():
    """A batch of one, one token and one head, cut out of buffers whose pitch is no multiple of 16 B: the bits of their copies."""
    from noise_amd.sinks import qk_norm_rotary, qk_norm_rotary_append, sink_attention, sink_attention_decode
    g = torch.Generator(DEV).manual_seed(6)
    cos, sin = tables(70, 64)
    for B, T, H in ((1, 70, 2), (2, 1, 2), (2, 70, 1), (1, 1, 1)):
        strides = (T * H * 64 + (5 if B == 1 else 0), H * 64 + (9 if T == 1 else 0), 64 + (3 if H == 1 else 0), 1)
        if H == 1:
            strides = (T * 72, 72, 67, 1) if B > 1 else (T * 72 + 5, 72, 67, 1)
        if T == 1:
            strides = (strides[0] if B == 1 else 256, 73, strides[2], 1)
        x = [torch.randn(20000, device=DEV, generator=g).bfloat16().as_strided((B, T, H, 64), strides) for _ in range(4)]
        caches = [torch.zeros(40000, device=DEV, dtype=torch.bfloat16).as_strided((B, 70, H, 64), (70 * H * 72 + (5 if B == 1 else 0),
                  H * 72, 67 if H == 1 else 72, 1)) for _ in range(2)]
        start = torch.zeros(B, device=DEV, dtype=torch.int32)

        def run(q, k, v, dout, kc, vc):
            q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
            normed = qk_norm_rotary(q, k, cos, sin)
            out = sink_attention(q, k, v, 20, 2)
            grads = [*torch.autograd.grad(normed, (q, k), (dout, dout)), *torch.autograd.grad(out, (q, k, v), dout)]
            with torch.no_grad():
                new = qk_norm_rotary_append(q, k, v, cos, sin, kc, vc, start)
                return [*normed, out, *grads, new, kc, vc, sink_attention_decode(q[:, -1:], kc, vc, start + T - 1, 20, 2)]

        for got, want in zip(run(*x, *caches), run(*(t.clone(memory_format=torch.contiguous_format) for t in x),
                                                   *(torch.zeros(B, 70, H, 64, device=DEV, dtype=torch.bfloat16) for _ in range(2)))):
            assert torch.equal(got, want)


def test_compiled_calls():
    """The calls themselves in compiled functions without a graph break, a training step, a prompt and a serving step: the eager
    bits."""
    from noise_amd.distill import distill_loss, distill_loss_grad
    from noise_amd.sinks import qk_norm_rotary, qk_norm_rotary_append, sink_attention, sink_attention_decode
    g = torch.Generator(DEV).manual_seed(7)
    q, k, v = (torch.randn(2, 64, h, 64, device=DEV, generator=g).bfloat16() for h in (4, 2, 2))
    cos, sin = tables(100, 64)
    t, i = torch.randn(2, 64, 4, 3, device=DEV, generator=g), torch.randint(0, 64, (2, 64, 4, 3), device=DEV, generator=g)
    start = torch.full((2,), 64, device=DEV)

    def train(q, k, v, w):
        q, k = qk_norm_rotary(q, k, cos, sin, w)
        return distill_loss(sink_attention(q, k, v, 20, 2), t, i, softcap=15.0)

    def serve(q, k, v, kc, vc):
        first = qk_norm_rotary_append(q, k, v, cos, sin, kc, vc, start - 64)
        out = sink_attention(first, kc[:, :64], vc[:, :64], 20, 2)
        new = qk_norm_rotary_append(q[:, :1], k[:, :1], v[:, :1], cos, sin, kc, vc, start)
        return out, sink_attention_decode(new, kc, vc, start, 20, 2), *distill_loss_grad(out, t, i, None, 60, 2.0)

    results = []
    for wrap in (lambda f: f, lambda f: torch.compile(f, backend='aot_eager', fullgraph=True)):
        leaves = [x.detach().requires_grad_() for x in (q, k, v, torch.ones(64, device=DEV))]
        loss = wrap(train)(*leaves)
        caches = [torch.zeros(2, 100, 2, 64, device=DEV, dtype=torch.bfloat16) for _ in range(2)]
        results.append((loss, *torch.autograd.grad(loss.sum(), leaves), *wrap(serve)(q, k, v, *caches), *caches))
    assert all(torch.equal(x, y) for x, y in zip(*results))


@pytest.mark.parametrize('D', [64, 128])
def test_captured_serving_step(D):
    """A step as it is served, new tokens into the cache, attention and the positions moved on, captured once and replayed with
    new tokens, beside eager steps on caches of their own; one sequence is idle, one runs past its cache."""
    from noise_amd.sinks import qk_norm_rotary_append, sink_attention_decode
    g = torch.Generator(DEV).manual_seed(8)
    B, T, H, Hk, S = 4, 2, 8, 2, 1100
    new = lambda: [torch.randn(B, T, h, D, device=DEV, generator=g).bfloat16() for h in (H, Hk, Hk)]
    cos, sin = tables(S, D)
    q, k, v = new()
    both = torch.randn(2, B, S, 2, Hk, D, device=DEV, generator=g).bfloat16()     # keys and values side by side
    begin = torch.tensor([0, 1000, -10 ** 6, S - 5], device=DEV)
    starts = [begin.clone(), begin.clone()]

    def step(n):
        kc, vc = both[n, :, :, 0], both[n, :, :, 1]
        out = sink_attention_decode(qk_norm_rotary_append(q, k, v, cos, sin, kc, vc, starts[n]), kc, vc, starts[n], 700, 4)
        starts[n] += T
        return out

    both[1] = both[0]
    step(0)
    both[0] = both[1]
    starts[0].copy_(begin)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(0)
    for _ in range(6):
        for t, x in zip((q, k, v), new()):
            t.copy_(x)
        want = step(1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(both[0], both[1]) and torch.equal(*starts)
        assert (out[2] == 0).all() and bool(torch.isfinite(out).all())
