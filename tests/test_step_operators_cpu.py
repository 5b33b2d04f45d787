"""What the calls of noise_amd.residual, noise_amd.vocab and noise_amd.clip do around their kernels, without a GPU: what they refuse,
what would have been launched, the C entry points' checks, the header's structs and the 64-bit definitions."""
import ctypes
import math
import subprocess
from array import array
from pathlib import Path

import pytest
import torch
from torch.autograd import forward_ad

from noise_amd import _lib, clip, residual, vocab
from oracle import training as oracle

BF16, F32 = torch.bfloat16, torch.float32
ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture
def launches(monkeypatch):
    """The entry points' names and arguments, in order"""
    made = []
    for module in (residual, vocab, clip):
        monkeypatch.setattr(module, '_call', lambda name, device, *args: made.append((name, args)))
    return made


def operands():
    t = dict(x=torch.randn(2, 5, 24), y=torch.randn(2, 5, 24).to(BF16), x0=torch.randn(2, 5, 24), scale=torch.tensor(0.9),
             x0_scale=torch.tensor([0.1]), gate=torch.rand(24), y_weight=torch.rand(24), weight=torch.rand(24))
    t.update(head=torch.randn(30, 24), targets=torch.randint(30, (2, 5)), token_weight=torch.rand(2, 5))
    t.update(g0=torch.randn(7, 3), g1=torch.randn(9).to(BF16))
    return t


NORM = ('x', 'y', 'x0', 'scale', 'x0_scale', 'gate', 'y_weight', 'weight')
CALLS = {   # call -> its tensors that may be differentiated, the call, its torch.ops form
    'residual_norm': (
        NORM, lambda t: residual.residual_norm(*(t[n] for n in NORM), norm_y=True),
        lambda t: torch.ops.noise_amd.residual_norm(*(t[n] for n in NORM), True, None, 1e-6)),
    'linear_cross_entropy': (
        ('x', 'head'), lambda t: vocab.linear_cross_entropy(t['x'], t['head'], t['targets'], softcap=15),
        lambda t: torch.ops.noise_amd.linear_cross_entropy(t['x'], t['head'], t['targets'], 30, 15.0)),
    'linear_cross_entropy_grad': (
        ('x', 'head', 'token_weight'),
        lambda t: vocab.linear_cross_entropy_grad(t['x'], t['head'], t['targets'], t['token_weight'], vocab=29),
        lambda t: torch.ops.noise_amd.linear_cross_entropy_grad(t['x'], t['head'], t['targets'], t['token_weight'], 29, None)),
    'clip_gradients': (
        ('g0', 'g1'), lambda t: clip.clip_gradients([t['g0'], t['g1']], 1),
        lambda t: torch.ops.noise_amd.clip_gradients([t['g0'], t['g1']], 1.0)),
}


@pytest.mark.parametrize('name', CALLS)
def test_forward_mode_is_refused(name, launches):
    tensors, call, operator = CALLS[name]
    for which in tensors:
        t = operands()
        with forward_ad.dual_level():
            t[which] = forward_ad.make_dual(t[which], torch.ones_like(t[which]))
            for f in (call, operator):
                with pytest.raises(NotImplementedError, match='forward.mode'):
                    f(t)
                with torch.no_grad(), pytest.raises(NotImplementedError, match='forward.mode'):
                    f(t)
        assert not launches
    with forward_ad.dual_level():
        call(operands())
    assert len(launches) == 1


@pytest.mark.parametrize('name', ['residual_norm', 'linear_cross_entropy'])
def test_derivatives_are_taken_once(name, launches):
    tensors, call, _ = CALLS[name]
    t = operands()
    out = call({**t, tensors[0]: t[tensors[0]].requires_grad_()})
    outs = out if isinstance(out, tuple) else (out,)
    up = [torch.ones_like(o).requires_grad_() for o in outs]
    grad, = torch.autograd.grad(outs, t[tensors[0]], up, create_graph=True)
    assert len(launches) == 2
    with pytest.raises(RuntimeError, match='once_differentiable'):
        grad.sum().backward()


@pytest.mark.parametrize('grad', [True, False])
@pytest.mark.parametrize('name', CALLS)
def test_compiled_callers_trace_the_calls(name, grad, launches):
    """fullgraph: the same launches as the eager call makes, the gradients clipped where it clips them."""
    tensors, call, _ = CALLS[name]
    differentiable = name in ('residual_norm', 'linear_cross_entropy')
    made = []
    for f in (call, torch.compile(call, backend='aot_eager', fullgraph=True)):
        torch.manual_seed(0)
        t = operands()
        leaf = t[tensors[0]].requires_grad_(grad and differentiable)
        before = t['g0']._version
        outs = f(t)
        outs = outs if isinstance(outs, tuple) else (outs,)
        if grad and differentiable:
            assert torch.autograd.grad(outs, leaf, [torch.ones_like(o) for o in outs])[0].shape == leaf.shape
        assert t['g0']._version > before or name != 'clip_gradients'
        made.append([(o.shape, o.dtype) for o in outs] +
                    [(n, [a is None if a is None or isinstance(a, int) and a > 2 ** 32 else a for a in args]) for n, args in launches])
        launches.clear()
    if name == 'linear_cross_entropy' and not grad:
        # (the operator leaves what a backward pass would need)
        drop = lambda m: [x if x[0] != 'noise_vocab_loss' else (x[0], x[1][:3] + x[1][4:]) for x in m]
        made = [drop(m) for m in made]
    assert made[0] == made[1] and len(made[0]) > len(outs)


def refused(f, match, launches):
    with pytest.raises(ValueError, match=match):
        f()
    assert not launches


def test_residual_norm_refuses(launches):
    f = residual.residual_norm
    x, y = torch.randn(2, 5, 24), torch.randn(2, 5, 24).to(BF16)
    half = torch.randn(2, 5, 24).half()
    for call, match in ((lambda: f(half, half), 'bfloat16 or float32'), (lambda: f(x, half), 'h has the type'),
                        (lambda: f(y, x), 'h has the type'), (lambda: f(x, y, dtype=F32), 'h has the type'),
                        (lambda: f(y, dtype=F32), 'h has the type'), (lambda: f(x, y[:1]), 'y must be'),
                        (lambda: f(x, y, x[:, :4]), 'x0 must be'), (lambda: f(x, y, y), 'one type'),
                        (lambda: f(x, gate=x[0, 0]), 'without y'), (lambda: f(x, norm_y=True), 'without y'),
                        (lambda: f(x, y, y_weight=x[0, 0]), 'norm_y'), (lambda: f(x, y, x0_scale=x[0, 0, 0]), 'without x0'),
                        (lambda: f(x, y, scale=x[0, 0]), 'one value'), (lambda: f(x, y, scale=2.0), 'a tensor'),
                        (lambda: f(x, y, weight=x[0]), 'weight must be'), (lambda: f(x, y, weight=torch.ones(24, dtype=torch.int32)), 'weight'),
                        (lambda: f(x, y, gate=x[:, 0]), 'gate must be'), (lambda: f(x, y, gate=x[:1]), 'gate must be'),
                        (lambda: f(x, y, gate=x[None]), 'gate must be'), (lambda: f(x, y, gate=x[0, 0, 0]), 'gate must be'),
                        (lambda: f(x, y, gate=x[0, 0].half()), 'gate must be'), (lambda: f(x[..., :0]), 'dim must be'),
                        (lambda: f(torch.zeros(2, 8193)), 'dim must be'), (lambda: f(torch.zeros(())), 'x')):
        refused(call, match, launches)


def test_residual_norm_takes(monkeypatch):
    """Gates in the shapes that the documentation names, with as many rows sharing one as it says."""
    x = torch.randn(3, 4, 5, 24)
    y = torch.randn(3, 4, 5, 24)
    seen = []
    monkeypatch.setattr(residual, '_call', lambda name, device, at, *args: seen.append(list((ctypes.c_int64 * 18).from_address(at))))
    for shape, rows in (((24,), 60), ((1, 24), 60), ((1, 1, 1, 24), 60), ((3, 1, 1, 24), 20), ((3, 4, 1, 24), 5), ((3, 4, 5, 24), 1)):
        residual.residual_norm(x, y, gate=torch.rand(shape))
        assert seen.pop()[11:14] == [60, rows, 24]
    # rows at one distance are taken where they are, others are copied
    wide = torch.randn(3, 4, 5, 40)[..., 3:27]
    residual.residual_norm(wide, y)
    assert seen[-1][0] == wide.data_ptr() and seen[-1][3:5] == [40, 24]
    turned = torch.randn(5, 4, 3, 24).transpose(0, 2)
    residual.residual_norm(turned, y)
    assert seen[-1][0] != turned.data_ptr() and seen[-1][3] == 24
    one = torch.randn(24).expand(3, 4, 5, 24)
    residual.residual_norm(one, y)
    assert seen[-1][0] == one.data_ptr() and seen[-1][3] == 0


def test_linear_cross_entropy_refuses(launches):
    x, w, t = torch.randn(6, 24), torch.randn(30, 24), torch.zeros(6, dtype=torch.int64)
    for f in (vocab.linear_cross_entropy, vocab.linear_cross_entropy_grad):
        for call, match in ((lambda: f(x.half(), w.half(), t), 'bfloat16 or float32'), (lambda: f(x, w.to(BF16), t), 'of its type'),
                            (lambda: f(x, w[:, :23], t), 'weight'), (lambda: f(x, w[None], t), 'weight'),
                            (lambda: f(x, w, t[:5]), 'targets must be'), (lambda: f(x, w, t.float()), 'targets must be'),
                            (lambda: f(x, w, t.short()), 'targets must be'), (lambda: f(x, w, t, vocab=31), 'vocab must be'),
                            (lambda: f(x, w, t, vocab=0), 'vocab must be'), (lambda: f(x, w, t, vocab=-1), 'vocab must be'),
                            (lambda: f(x, w, t, softcap=0.0), 'softcap'), (lambda: f(x, w, t, softcap=-1.0), 'softcap'),
                            (lambda: f(x, w, t, softcap=math.nan), 'softcap'), (lambda: f(x[:, :0], w[:, :0], t), 'dim must be'),
                            (lambda: f(x, w.to('meta'), t), 'tensors on'), (lambda: f(x, w, t.to('meta')), 'tensors on')):
            refused(call, match, launches)
    refused(lambda: vocab.linear_cross_entropy_grad(x, w, t, torch.ones(5)), 'token weights', launches)
    refused(lambda: vocab.linear_cross_entropy_grad(x, w, t, torch.ones(6, device='meta')), 'token weights', launches)


def test_clip_gradients_refuses(launches):
    a, b = torch.randn(5, 4), torch.randn(3)
    for call, match in ((lambda: clip.clip_gradients([], 1.0), 'no gradients'), (lambda: clip.clip_gradients([None], 1.0), 'no gradients'),
                        (lambda: clip.clip_gradients([a], -1.0), 'max_norm'), (lambda: clip.clip_gradients([a], math.nan), 'max_norm'),
                        (lambda: clip.clip_gradients([a, b.half()], 1.0), 'bfloat16 or float32'),
                        (lambda: clip.clip_gradients([a, b.to('meta')], 1.0), 'gradients on'),
                        (lambda: clip.clip_gradients([a[:, :2]], 1.0), 'gaps'), (lambda: clip.clip_gradients([b.expand(4, 3)], 1.0), 'gaps'),
                        (lambda: clip.clip_gradients([a.requires_grad_()], 1.0), 'not differentiable')):
        refused(call, match, launches)
    with torch.no_grad():
        clip.clip_gradients([a, None, b, torch.randn(0)], 1.0)
    assert launches[0][1][1] == 3


def test_clip_raises_the_gradients_versions(launches):
    """A graph that holds a gradient as it was must not run backwards on what was clipped; a norm alone changes nothing."""
    for max_norm, more in ((1.0, 1), (math.inf, 0)):
        g = torch.randn(5)
        before = g._version
        clip.clip_gradients([g], max_norm)
        assert g._version == before + more


def gradients(*entries):
    return array('q', [v for e in entries for v in e])


def test_clip_entry_point_refuses():
    lib = _lib.lib()
    need = lib.noise_clip_workspace_bytes(2)

    def call(table, count, max_norm=1.0, norm=16, work=16, size=need):
        return lib.noise_clip_gradients(None if table is None else table.buffer_info()[0], count, max_norm, norm, work, size, None)
    good = gradients((4096, 10, 1), (8192, 10, 0))
    for args, match in (((None, 2), 'table'), ((good, -1), 'table'), ((good, 2, -1.0), 'max_norm'), ((good, 2, math.nan), 'max_norm'),
                        ((good, 2, 1.0, None), 'norm'), ((good, 2, 1.0, 18), 'norm'), ((good, 2, 1.0, 16, None), 'workspace'),
                        ((good, 2, 1.0, 16, 16, need - 1), 'workspace'), ((gradients((4096, 10, 2)), 1), 'type'),
                        ((gradients((4096, -1, 1)), 1), 'elements'), ((gradients((0, 10, 1)), 1), 'NULL'),
                        ((gradients((4098, 10, 1)), 1), 'aligned'), ((gradients((4097, 10, 0)), 1), 'aligned'),
                        ((gradients((4096, 10, 1), (4096, 10, 1)), 2), 'share memory'),
                        ((gradients((4096, 10, 1), (4132, 10, 1)), 2), 'share memory'),
                        ((gradients((8192, 10, 1), (4096, 1025, 1)), 2), 'share memory'),
                        ((gradients((8192, 10, 1), (4096, 10, 0), (4114, 10, 0)), 3, 1.0, 16, 16, need), 'share memory')):
        assert call(*args) == -1 and match in lib.noise_last_error().decode(), (match, lib.noise_last_error())


def test_residual_entry_points_refuse():
    lib = _lib.lib()
    base = dict(x=4096, y=8192, x0=0, sx=24, sy=24, s0=0, scale=0, x0_scale=0, gate=0, wy=0, w=0, rows=4, gate_rows=4, dim=24,
                x_type=1, y_type=0, gate_type=1, norm_y=0)

    def call(out=4096, h=4096, eps=1e-6, **change):
        t = array('q', {**base, **change}.values())
        return lib.noise_residual_norm(t.buffer_info()[0], out, h, eps, None)
    for change, match in ((dict(dim=0), 'dim'), (dict(dim=8193), 'dim'), (dict(rows=-1), 'rows'), (dict(x_type=0, y_type=1), 'types'),
                          (dict(x_type=2), 'types'), (dict(eps=-1.0), 'eps'), (dict(eps=math.nan), 'eps'), (dict(x=0), 'x NULL'),
                          (dict(x=4098), 'aligned'), (dict(y=0, gate=16), 'without y'), (dict(y=0, norm_y=1), 'without y'),
                          (dict(wy=16), 'without the norm'), (dict(x0_scale=16), 'without x0'), (dict(scale=18), 'aligned'),
                          (dict(gate=16, gate_type=2), 'gate type'), (dict(gate=16, gate_rows=3), 'gate_rows'),
                          (dict(gate=16, gate_rows=0), 'gate_rows'), (dict(out=None), 'output'), (dict(h=4097), 'output')):
        assert call(**change) == -1 and match in lib.noise_last_error().decode(), (change, lib.noise_last_error())
    assert call(rows=0) == 0

    def backward(grads, work=None, size=0, **change):
        t, g = array('q', {**base, **change}.values()), array('q', grads)
        return lib.noise_residual_norm_bwd(t.buffer_info()[0], 4096, 4096, g.buffer_info()[0], 1e-6, work, size, None)
    for grads, match in (((0, 0, 16, 0, 0, 0, 0, 0), 'absent'), ((0, 0, 0, 0, 16, 0, 0, 0), 'absent'), ((0, 0, 0, 0, 0, 16, 0, 0), 'absent'),
                         ((0, 0, 0, 0, 0, 0, 16, 0), 'absent'), ((18, 0, 0, 0, 0, 0, 0, 0), 'aligned'),
                         ((0, 0, 0, 16, 0, 0, 0, 0), 'workspace'), ((0, 0, 0, 0, 0, 0, 0, 16), 'workspace')):
        assert backward(grads) == -1 and match in lib.noise_last_error().decode(), (grads, lib.noise_last_error())
    assert backward((0, 0, 0, 0, 0, 0, 0, 16), 16, lib.noise_residual_norm_bwd_workspace_bytes(4, 4, 24) - 1) == -1
    assert backward((0, 0, 0, 0, 0, 0, 0, 16), rows=0) == 0


def test_vocab_entry_points_refuse():
    lib = _lib.lib()
    base = dict(x=4096, xs=24, w=4096, ws=24, t=4096, wide=1, rows=4, dim=24, vocab=30, type=1)
    table = lambda **change: array('q', {**base, **change}.values())

    def loss(softcap=0.0, loss=16, work=16, size=1 << 40, **change):
        t = table(**change)
        return lib.noise_vocab_loss(t.buffer_info()[0], softcap, loss, None, work, size, None)
    for change, match in ((dict(type=2), 'type'), (dict(rows=-1), 'rows'), (dict(rows=2 ** 30 + 1), 'rows'), (dict(dim=0), 'dim'),
                          (dict(dim=65537), 'dim'), (dict(vocab=0), 'vocab'), (dict(vocab=2 ** 22 + 1), 'vocab'), (dict(softcap=-1.0), 'softcap'),
                          (dict(softcap=math.nan), 'softcap'), (dict(x=0), 'NULL'), (dict(w=4098), 'aligned'), (dict(t=4100), 'aligned'),
                          (dict(loss=None), 'loss'), (dict(work=None), 'workspace'), (dict(size=0), 'workspace'),
                          (dict(work=24), 'workspace')):
        for rows in (4, 100):   # (few rows have a kernel of their own)
            assert loss(**{'rows': rows, **change}) == -1 and match in lib.noise_last_error().decode(), (change, lib.noise_last_error())
    assert loss(rows=0) == 0

    def grad(lse=None, loss=16, width=30, size=1 << 40, weight=None, dw=16):
        t = table()
        return lib.noise_vocab_grad(t.buffer_info()[0], 0.0, weight, lse, loss, 16, dw, width, 16, size, None)
    for change, match in ((dict(lse=16), 'either'), (dict(loss=None), 'either'), (dict(width=29), 'width'), (dict(weight=18), 'aligned'),
                          (dict(dw=18), 'aligned'), (dict(size=100), 'workspace')):
        assert grad(**change) == -1 and match in lib.noise_last_error().decode(), (change, lib.noise_last_error())
    bad = table(dim=0)
    assert lib.noise_vocab_workspace_bytes(bad.buffer_info()[0], 1) == -1
    # the products' buffers stay within their bounds whatever the sizes: dZ takes at most 2 GiB, the joined sums 256 MiB each
    for rows, dim, V, kind in ((2 ** 20, 512, 4096, 0), (8192, 2048, 131072, 0), (8192, 2048, 131072, 1), (100000, 64, 50, 1)):
        t = table(rows=rows, dim=dim, vocab=V, type=kind)
        parts = 2 if kind else 1
        operands = 2 * parts * (rows + 256 + V) * (dim + 64) + 40 * rows
        need = lib.noise_vocab_workspace_bytes(t.buffer_info()[0], 1)
        assert 0 < need <= operands + 2 ** 31 + 2 ** 29 + 4 * V * (dim + 64) + 8 * 2 ** 31 // 256 + 2 ** 22


def test_vocab_entry_points_refuse_negative_strides():
    lib = _lib.lib()
    for change in (dict(xs=-24), dict(ws=-24)):
        table = array('q', {**dict(x=4096, xs=24, w=4096, ws=24, t=4096, wide=1, rows=4, dim=24, vocab=30, type=1), **change}.values())
        at = table.buffer_info()[0]
        assert lib.noise_vocab_loss(at, 0.0, 16, None, 16, 1 << 40, None) == -1
        assert 'stride' in lib.noise_last_error().decode()
        assert lib.noise_vocab_grad(at, 0.0, None, None, 16, 16, 16, 30, 16, 1 << 40, None) == -1
        assert lib.noise_vocab_workspace_bytes(at, 1) == -1


def test_workspace_queries_refuse():
    lib = _lib.lib()
    for query, bad in ((lib.noise_clip_workspace_bytes, ((0,), (-1,), (2 ** 24 + 1,))),
                       (lib.noise_residual_norm_bwd_workspace_bytes, ((0, 1, 8), (4, 0, 8), (4, 3, 8), (4, 4, 0), (4, 4, 8193), (-4, 4, 8))),
                       (lib.noise_vocab_workspace_bytes, ((None, 1),))):
        for args in bad:
            assert query(*args) == -1 and lib.noise_last_error(), (query, args)
    good = gradients((4096, 10, 1))
    assert lib.noise_clip_gradients(good.buffer_info()[0], 0, 1.0, 16, 16, 1 << 20, None) == -1


def test_struct_layouts_match_the_header(tmp_path):
    """The tables of 64-bit words that the Python layer packs have the C structs' sizes and orders."""
    fields = {'noise_gradient_t': 'ptr numel type', 'noise_residual_grads_t': 'dx dy dx0 dscale dx0_scale dgate dy_weight dweight',
              'noise_residual_t': 'x y x0 x_stride y_stride x0_stride scale x0_scale gate y_weight weight rows gate_rows dim x_type '
                                  'y_type gate_type norm_y',
              'noise_vocab_t': 'x x_stride weight weight_stride targets targets_wide rows dim vocab type'}
    source = tmp_path / 'layout.c'
    checks = ''.join(f'_Static_assert(sizeof({t}) == {8 * len(f.split())}, "{t}");\n' +
                     ''.join(f'_Static_assert(offsetof({t}, {n}) == {8 * i}, "{t}.{n}");\n' for i, n in enumerate(f.split()))
                     for t, f in fields.items())
    source.write_text(f'#include <stddef.h>\n#include "{ROOT}/include/noise_amd.h"\n{checks}')
    subprocess.run(['gcc', '-c', str(source), '-o', str(tmp_path / 'layout.o')], check=True)


def test_definitions():
    """The oracle's formulas against independent ones: gradients by difference quotients (fp64, step 1e-6: off by 1e-9)."""
    g = torch.Generator().manual_seed(0)
    randn = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    t = dict(x=randn(3, 6), y=randn(3, 6), x0=randn(3, 6), scale=randn(()), x0_scale=randn(()), gate=randn(6), y_weight=randn(6),
             weight=randn(6))
    out, h = oracle.residual(**t, norm_y=True, eps=1e-6)
    for r in range(3):
        ry = 1 / math.sqrt(sum(v * v for v in t['y'][r].tolist()) / 6 + 1e-6)
        row = [t['scale'] * (t['x'][r, c] + t['gate'][c] * t['y'][r, c] * ry * t['y_weight'][c]) + t['x0_scale'] * t['x0'][r, c]
               for c in range(6)]
        r2 = 1 / math.sqrt(sum(float(v) ** 2 for v in row) / 6 + 1e-6)
        for c in range(6):
            assert abs(out[r, c] - row[c]) < 1e-12 and abs(h[r, c] - row[c] * r2 * t['weight'][c]) < 1e-12
    x, w, targets, tw = randn(4, 5), randn(7, 5), torch.tensor([2, -1, 6, 9]), torch.rand(4, generator=g)
    loss, dx, dw = oracle.linear_cross_entropy(x, w, targets, 7, 3.0, tw)
    z = 3 * torch.tanh(x @ w.t() / 3)
    assert abs(loss[0] - (torch.log(z[0].exp().sum()) - z[0, 2])) < 1e-12 and loss[1] == loss[3] == 0
    value = lambda x, w: (oracle.linear_cross_entropy(x, w, targets, 7, 3.0)[0] * tw).sum()
    for a, d, f in ((x, dx, lambda e: value(x + e, w)), (w, dw, lambda e: value(x, w + e))):
        e = randn(*a.shape)
        assert abs((f(1e-6 * e) - f(-1e-6 * e)) / 2e-6 - (d * e).sum()) < 1e-8
    norm, clipped = oracle.clip([torch.tensor([3.0]), torch.tensor([4.0])], 1.0)
    assert norm == 5.0 and abs(clipped[0].item() - 3 / (5 + 1e-6)) < 1e-12


def test_compiled_gradients_in_one_call_of_leaves(launches):
    """linear_cross_entropy_grad's results are plain tensors for operands that require a gradient, compiled as well, and the steps
    around it go on from them."""
    def step(t):
        loss, dx, dw = vocab.linear_cross_entropy_grad(t['x'], t['head'], t['targets'], t['token_weight'])
        return loss, dx, dw, clip.clip_gradients([dw], 1.0)
    made = []
    for f in (step, torch.compile(step, backend='aot_eager', fullgraph=True)):
        t = operands()
        hidden = t['x'].requires_grad_() * 2
        outs = f({**t, 'x': hidden, 'head': t['head'].requires_grad_(), 'token_weight': t['token_weight'].requires_grad_()})
        assert not any(o.requires_grad for o in outs)
        hidden.backward(outs[1])
        assert torch.equal(t['x'].grad, 2 * outs[1]) or torch.isnan(outs[1]).any()
        made.append([n for n, _ in launches])
        launches.clear()
    assert made[0] == made[1] == ['noise_vocab_grad', 'noise_clip_gradients']


def test_vocab_workspaces_of_the_largest_vocabularies():
    """What the documents bound: dZ by 2 GiB, or by 256 tokens' (fp32 of more than 2^21 entries: 4 GiB); few tokens' logits in fp32, and
    their dZ twice, by rows and by entries, in as many parts as it has (of up to 32 bf16 tokens two, of 64 one; fp32 by rows takes the
    logits' place)."""
    lib = _lib.lib()

    def need(rows, V, kind, grad=1, dim=64):
        t = array('q', (4096, dim, 4096, dim, 4096, 1, rows, dim, V, kind))
        return lib.noise_vocab_workspace_bytes(t.buffer_info()[0], grad)
    for V in (2 ** 22, 2 ** 21 + 1, 2 ** 20, 131072):
        up = (V + 255) // 256 * 256
        for kind, size in ((0, 2), (1, 4)):
            for rows in (65, 200, 257, 1000, 5000):
                operands = size * (rows + 256 + V) * 128 + 40 * (rows + 256)
                partial = 8 * (V + 127) // 128 * (rows + 256)
                few = 4 * rows * (V + 32) + 8 * rows * (V // 16 + 1) if rows * V <= 2 ** 28 else 0
                dz = max(2 ** 31, 256 * up * size)
                assert 0 < need(rows, V, kind) <= operands + partial + few + dz + 2 ** 29 + 4 * V * 64 + 2 ** 22, (rows, V, kind)
            for rows in (1, 16, 17, 32, 33, 64):
                held, entries = (16, 32) if rows <= 16 else (32, 32) if rows <= 32 else (64, 64)
                parts = 2 if kind == 0 and rows <= 32 else 1
                if kind == 1:
                    entries = held
                logits, dz, dzt = 4 * held * (V + 32), 0 if kind else 2 * parts * held * (V + 32), size * parts * entries * (V + 32)
                assert 0 < need(rows, V, kind) <= logits + dz + dzt + 8 * rows * (V // 16 + 1) + 2 ** 24, (rows, V, kind)
