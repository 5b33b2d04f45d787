"""What the calls of noise_amd.sinks and noise_amd.distill do around their kernels, without a GPU: the launches are left out, and
what would have been launched is kept."""
import ctypes
import math

import pytest
import torch
from torch.autograd import forward_ad

from noise_amd import _lib, distill, sinks

BF16 = torch.bfloat16


@pytest.fixture
def launches(monkeypatch):
    """The entry points' names and arguments, in order"""
    made = []
    for module in (sinks, distill):
        monkeypatch.setattr(module, '_call', lambda name, device, *args: made.append((name, args)))
    return made


def operands(B=2, T=5, H=4, Hk=2, D=64, S=9):
    """A call's tensors by name"""
    t = {n: torch.randn(B, T, h, D).to(BF16) for n, h in (('q', H), ('k', Hk), ('v', Hk))}
    t.update({n: torch.zeros(B, S, Hk, D, dtype=BF16) for n in ('k_cache', 'v_cache')}, start=torch.zeros(B, dtype=torch.int64))
    t.update({n: torch.rand(S, D // 2) for n in ('cos', 'sin')}, q_weight=torch.rand(D), k_weight=torch.rand(D))
    t.update(logits=torch.randn(3, 10), teacher=torch.randn(3, 4), index=torch.zeros(3, 4, dtype=torch.int64),
             weight=torch.rand(3))
    return t


CALLS = {   # call -> its tensors that may be differentiated, the call, its torch.ops form
    'qk_norm_rotary': (
        ('q', 'k', 'q_weight', 'k_weight'),
        lambda t: sinks.qk_norm_rotary(t['q'], t['k'], t['cos'], t['sin'], t['q_weight'], t['k_weight']),
        lambda t: torch.ops.noise_amd.qk_norm_rotary(t['q'], t['k'], t['cos'], t['sin'], t['q_weight'], t['k_weight'], None,
                                                     1e-6)),
    'qk_norm_rotary_append': (
        ('q', 'k', 'v', 'k_cache', 'v_cache', 'q_weight', 'k_weight'),
        lambda t: sinks.qk_norm_rotary_append(t['q'], t['k'], t['v'], t['cos'], t['sin'], t['k_cache'], t['v_cache'],
                                              t['start'], t['q_weight'], t['k_weight']),
        lambda t: torch.ops.noise_amd.qk_norm_rotary_append(t['q'], t['k'], t['v'], t['cos'], t['sin'], t['k_cache'],
                                                            t['v_cache'], t['start'], t['q_weight'], t['k_weight'], 1e-6)),
    'sink_attention': (
        ('q', 'k', 'v'), lambda t: sinks.sink_attention(t['q'], t['k'], t['v'], 3, 1),
        lambda t: torch.ops.noise_amd.sink_attention(t['q'], t['k'], t['v'], 3, 1, None)),
    'sink_attention_decode': (
        ('q', 'k_cache', 'v_cache'), lambda t: sinks.sink_attention_decode(t['q'], t['k_cache'], t['v_cache'], t['start'], 3, 1),
        lambda t: torch.ops.noise_amd.sink_attention_decode(t['q'], t['k_cache'], t['v_cache'], t['start'], 3, 1)),
    'distill_loss': (
        ('logits', 'teacher'), lambda t: distill.distill_loss(t['logits'], t['teacher'], t['index']),
        lambda t: torch.ops.noise_amd.distill_loss(t['logits'], t['teacher'], t['index'], 10, 1.0, None)),
    'distill_loss_grad': (
        ('logits', 'teacher', 'weight'),
        lambda t: distill.distill_loss_grad(t['logits'], t['teacher'], t['index'], t['weight']),
        lambda t: torch.ops.noise_amd.distill_loss_grad(t['logits'], t['teacher'], t['index'], t['weight'], 10, 1.0, None)),
}


@pytest.mark.parametrize('name', CALLS)
def test_forward_mode_is_refused(name, launches):
    """A tangent on any tensor is refused with and without gradients, by the call and by the operator; without tangents the call
    goes through inside a forward-mode level."""
    tensors, call, operator = CALLS[name]
    for which in tensors:
        for also in (None, tensors[0]):
            t = operands()
            if also is not None and 'cache' not in which and name in ('qk_norm_rotary', 'sink_attention', 'distill_loss'):
                t[also].requires_grad_()
            with forward_ad.dual_level():
                t[which] = forward_ad.make_dual(t[which], torch.ones_like(t[which]))
                for f in (call, operator):
                    with pytest.raises(NotImplementedError, match='forward.mode'):
                        f(t)
                    with torch.no_grad(), pytest.raises(NotImplementedError, match='forward.mode'):
                        f(t)
            # (an autograd function refuses its tangents after its forward pass)
            assert also is not None or not launches
            launches.clear()
    with forward_ad.dual_level():
        call(operands())
    assert len(launches) == 1


@pytest.mark.parametrize('name', CALLS)
def test_forward_mode_transforms_are_refused(name, launches):
    """torch.func.jvp gives no derivatives of 0 either."""
    tensors, call, operator = CALLS[name]
    for which in tensors:
        for f in (call, operator):
            t = operands()
            with pytest.raises((NotImplementedError, RuntimeError)):
                torch.func.jvp(lambda x: f({**t, which: x}), (t[which],), (torch.ones_like(t[which]),))
            assert not launches


@pytest.mark.parametrize('name,grads', [('qk_norm_rotary', 2), ('sink_attention', 1), ('distill_loss', 1)])
def test_tangents_of_upstream_gradients_are_refused(name, grads, launches):
    t = operands()
    tensors, call, _ = CALLS[name]
    out = call({**t, tensors[0]: t[tensors[0]].requires_grad_()})
    outs = out if isinstance(out, tuple) else (out,)
    with forward_ad.dual_level():
        up = [forward_ad.make_dual(torch.ones_like(o), torch.ones_like(o)) for o in outs]
        with pytest.raises(NotImplementedError, match='forward.mode'):
            torch.autograd.grad(outs, t[tensors[0]], up)
    assert len(outs) == grads and len(launches) == 1


def test_append_raises_the_caches_versions(launches):
    """A graph that holds a cache as it was must not run backwards on what was written over it; views of a cache count, and
    caches made in inference mode have no version."""
    for of in (lambda c: c, lambda c: c[:, 2:]):
        t = operands()
        for n in ('k_cache', 'v_cache'):
            held = torch.ones_like(t[n], requires_grad=True) * t[n]
            before = t[n]._version
            CALLS['qk_norm_rotary_append'][1]({**t, 'k_cache': of(t['k_cache']), 'v_cache': of(t['v_cache'])})
            assert t[n]._version == before + 1
            with pytest.raises(RuntimeError, match='modified by an inplace operation'):
                held.float().sum().backward()
    with torch.inference_mode():
        CALLS['qk_norm_rotary_append'][1](operands())
    assert len(launches) == 5


@pytest.mark.parametrize('name', ['qk_norm_rotary_append', 'sink_attention_decode'])
def test_calls_without_a_derivative_refuse_to_drop_one(name, launches):
    """A tensor that requires a gradient, a leaf or not, is refused while gradients are recorded, nothing launched; under
    no_grad it is a tensor like others. The operator's backward pass is refused."""
    tensors, call, operator = CALLS[name]
    for which in tensors:
        for of in (lambda x: x, lambda x: x * 1):
            t = operands()
            t[which] = of(t[which].requires_grad_())
            with pytest.raises(ValueError, match='not differentiable'):
                call(t)
            assert not launches
            with torch.no_grad():
                assert not call(t).requires_grad
            out = operator(t)
            with pytest.raises(RuntimeError, match='no autograd formula'):
                out.float().sum().backward()
            assert len(launches) == 2
            launches.clear()


def append_into(k_cache, v_cache):
    B, S, Hk, D = k_cache.shape
    t = operands(B=B, Hk=Hk, H=Hk, D=D)
    return sinks.qk_norm_rotary_append(t['q'], t['k'], t['v'], t['cos'], t['sin'], k_cache, v_cache, t['start'])


def test_caches_that_share_slots_are_refused(launches):
    """Of one another and of their own sequences, slots and heads."""
    buf = torch.zeros(2, 12, 2, 64, dtype=BF16)
    flat = torch.zeros(5000, dtype=BF16)
    other = torch.zeros_like(buf)
    for k, v in ((buf[:, :8], buf[:, 1:9]), (buf[:, 4:], buf[:, :8]), (buf[:, :7], buf[:, 5:]),
                 (buf[:, :, :1], buf[:, :, :1].clone().set_(buf[:, :, :1])),
                 (buf[:1], buf.as_strided((1, 12, 2, 64), (80, 128, 64, 1), 12 * 128 - 128)),
                 (flat.as_strided((2, 8, 2, 64), (1024, 128, 64, 1)), flat.as_strided((2, 8, 2, 64), (1024, 64, 512, 1), 1024))):
        for a, b in ((k, v), (v, k)):
            with pytest.raises(ValueError, match='same memory'):
                append_into(a, b)
    for c in (flat.as_strided((2, 8, 2, 64), (512, 128, 64, 1)), flat.as_strided((2, 8, 2, 64), (1024, 64, 64, 1)),
              flat.as_strided((2, 8, 2, 64), (2048, 128, 56, 1)), flat.as_strided((1, 8, 2, 64), (0, 128, 120, 1))):
        for a, b in ((c, other[:c.shape[0], :8]), (other[:c.shape[0], :8], c)):
            with pytest.raises(ValueError, match='overlap'):
                append_into(a, b)
    assert not launches


def test_caches_side_by_side_are_taken(launches):
    """Keys and values next to each other per slot, per head, per sequence and one after the other; sequences of one."""
    flat = torch.zeros(2 * 9 * 2 * 2 * 64, dtype=BF16)
    slot, head = flat.view(2, 9, 2, 2, 64), flat.view(2, 9, 2, 128)
    rows = flat.view(2, 2, 2, 9, 64)
    pairs = [(slot[:, :, 0], slot[:, :, 1]), (slot[:, :, :, 0], slot[:, :, :, 1]), (head[..., :64], head[..., 64:]),
             (rows[:, :, 0].transpose(1, 2), rows[:, :, 1].transpose(1, 2)), (rows[:, 0].transpose(1, 2), rows[:, 1].transpose(1, 2)),
             tuple(flat.view(2, 2, 9, 2, 64)), tuple(flat.view(2, 2, 9, 2, 64).unbind(1)),
             (flat.view(4, 9, 2, 64)[:1], flat.view(4, 9, 2, 64)[1:2]), (flat.view(4, 9, 128)[:, :, None, :64][:1], slot[1:, :, :1, 0]),
             (flat.as_strided((1, 9, 1, 64), (8, 64, 24, 1)), flat.as_strided((1, 9, 1, 64), (16, 64, 40, 1), 9 * 64))]
    for n, (k, v) in enumerate([*pairs, *((v, k) for k, v in pairs)], 1):
        append_into(k, v)
        assert len(launches) == n
    empty = torch.zeros(0, 9, 2, 64, dtype=BF16)
    append_into(empty, empty.clone())


def test_caches_that_share_memory_against_enumeration(launches):
    """Of random layouts, those in which an element belongs to two slots are refused; others with sequences, slots and heads
    inside one another, in any order, are taken."""
    import random
    rng = random.Random(0)
    taken = refused = 0
    for _ in range(600):
        shape = (rng.randint(1, 3), rng.randint(1, 4), rng.randint(1, 2))
        strides, end = [0, 0, 0], 64
        for d in rng.sample(range(3), 3):
            strides[d] = end + 8 * rng.choice([0, 0, 1, 8, 30]) - 8 * rng.choice([0] * 9 + [1])
            end = strides[d] * (shape[d] - 1) + end
        flat = torch.zeros(3 * end + 5000, dtype=BF16)
        at = [8 * rng.randint(0, end // 4) for _ in range(2)]
        k, v = (flat.as_strided((*shape, 64), (*strides, 1), a) for a in at)
        own = [{a + sum(i * s for i, s in zip((b, t, h), strides)) + d for b in range(shape[0]) for t in range(shape[1])
                for h in range(shape[2]) for d in range(64)} for a in at]
        meets = len(own[0]) < k.numel() or not own[0].isdisjoint(own[1])
        try:
            append_into(k, v)
            assert not meets, (shape, strides, at)
            taken += 1
        except ValueError:
            assert meets, (shape, strides, at)
            refused += 1
    assert taken > 50 and refused > 50


@pytest.mark.parametrize('scale', [0.0, -0.125, math.nan, math.inf, -math.inf, 1e-40, 1e38])
def test_entry_points_refuse_a_scale_that_is_not_positive(scale):
    """Hidden keys are -inf before the scale is applied: 0 would make them NaN and a negative one inf. (No sequences: a scale that
    is taken launches nothing.)"""
    lib = _lib.lib()
    heads = ctypes.byref(_lib.Heads(16, 5 * 128, 128, 64, 2))
    forward = lambda x: lib.noise_sink_attention_fwd(*[heads] * 4, None, None, None, 0, 0, 5, 64, 3, 0, x, None)
    decode = lambda x: lib.noise_sink_decode(*[heads] * 4, 16, 0, 0, 1, 9, 64, 3, 0, x, None, 0, None)
    backward = lambda x: lib.noise_sink_attention_bwd(*[heads] * 6, 16, *[heads] * 3, None, 0, 0, 5, 64, 3, 0, x, None, 0, None)
    for call in (forward, decode, backward):
        assert call(scale) == -1 and 'scale' in lib.noise_last_error().decode()
        assert call(0.125) == 0


def odd(B, T, H, D=64, dtype=BF16):
    """A [B, T, H, D] view with a pitch that is no multiple of 16 B in every dimension of one element"""
    unit = 16 // torch.empty(0, dtype=dtype).element_size()
    h = D if H > 1 else D + 3
    t = H * D if T > 1 else H * D + 1 + unit
    b = T * H * D if B > 1 else T * H * D + 5
    return torch.randn(2 * B * T * H * D + 64).to(dtype).as_strided((B, T, H, D), (b, t, h, 1))


@pytest.mark.parametrize('dtype', [BF16, torch.float32])
@pytest.mark.parametrize('B,T,H', [(1, 7, 4), (2, 1, 4), (2, 7, 1), (1, 1, 4), (1, 7, 1), (2, 1, 1), (1, 1, 1)])
def test_strides_of_single_elements_do_not_matter(B, T, H, dtype, monkeypatch):
    """Views whose only odd strides are those of dimensions with one element are taken as they are (torch calls them contiguous),
    their outputs and caches too: every stride that reaches an entry point is a multiple of 16 B."""
    unit = 16 // torch.empty(0, dtype=dtype).element_size()
    checked = []

    def call(name, device, *args):
        at = args[0]
        for n in range({'noise_qk_norm_rotary': 4 if args[3] is None else 6, 'noise_qk_norm_rotary_bwd': 6, 'noise_sink_attention_fwd': 4,
                        'noise_sink_attention_bwd': 9, 'noise_sink_decode': 4}[name]):
            t = _lib.Heads.from_address(at + n * sinks._HEADS)
            assert t.ptr % 16 == 0 and not any(s % unit for s in (t.s_b, t.s_t, t.s_h)), (name, n, t.s_b, t.s_t, t.s_h)
            checked.append((t.ptr, t.heads))

    monkeypatch.setattr(sinks, '_call', call)
    x = lambda: odd(B, T, H, dtype=dtype)
    pointers = lambda: {p for p, _ in checked}
    cos = sin = torch.rand(9, 32)
    start = torch.zeros(B, dtype=torch.int32)
    q, k, v = (x().requires_grad_() for _ in range(3))
    for n, s in enumerate((B, T, H)):
        assert s > 1 or q.stride(n) % unit
    torch.autograd.grad(sinks.qk_norm_rotary(q, k, cos, sin), (q, k), (x(), x()))
    assert {q.data_ptr(), k.data_ptr()} <= pointers()
    with torch.no_grad():
        caches = odd(B, 9, H, dtype=dtype), odd(B, 9, H, dtype=dtype)
        sinks.qk_norm_rotary_append(q, k, v, cos, sin, *caches, start)
        assert {c.data_ptr() for c in caches} <= pointers()
        one = odd(B, 1, H, dtype=dtype)
        sinks.qk_norm_rotary_append(q[:, :1], k[:, :1], v[:, :1], cos, sin, one, odd(B, 1, H, dtype=dtype), start)
        assert one.data_ptr() in pointers()
    if dtype == BF16:
        torch.autograd.grad(sinks.sink_attention(q, k, v, 3, 1), (q, k, v), x())
        assert v.data_ptr() in pointers()
        with torch.no_grad():
            sinks.sink_attention_decode(q, *caches, start, 3)


@pytest.mark.parametrize('grad', [True, False])
@pytest.mark.parametrize('name', CALLS)
def test_compiled_callers_trace_the_calls(name, grad, launches):
    """fullgraph, as the framework's other calls: the same launches as the eager call makes, the caches written where it does."""
    tensors, call, _ = CALLS[name]
    differentiable = name in ('qk_norm_rotary', 'sink_attention', 'distill_loss')
    made = []
    for f in (call, torch.compile(call, backend='aot_eager', fullgraph=True)):
        torch.manual_seed(0)
        t = operands()
        if grad and differentiable:
            t[tensors[0]].requires_grad_()
        before = t['k_cache']._version
        outs = f(t)
        outs = outs if isinstance(outs, tuple) else (outs,)
        if grad and differentiable:
            assert torch.autograd.grad(outs, t[tensors[0]], [torch.ones_like(o) for o in outs])[0].shape == t[tensors[0]].shape
        assert t['k_cache']._version > before or name != 'qk_norm_rotary_append'
        # (which pointers are given, and every number)
        made.append([(o.shape, o.dtype) for o in outs] +
                    [(n, [a is None if a is None or isinstance(a, int) and a > 2 ** 32 else a for a in args]) for n, args in launches])
        launches.clear()
    assert made[0] == made[1] and len(made[0]) > len(outs)


def test_compiled_callers_may_give_whole_numbers(launches):
    t = operands()
    torch.compile(lambda t: distill.distill_loss(t['logits'], t['teacher'], t['index'], temperature=2, softcap=15),
                  backend='aot_eager', fullgraph=True)(t)
    torch.compile(lambda t: distill.distill_loss_grad(t['logits'], t['teacher'], t['index'], vocab=9, temperature=2, softcap=15),
                  backend='aot_eager', fullgraph=True)(t)
    torch.compile(lambda t: sinks.sink_attention(t['q'], t['k'], t['v'], 10 ** 30, 10 ** 30), backend='aot_eager',
                  fullgraph=True)(t)
    torch.compile(lambda t: sinks.qk_norm_rotary(t['q'], t['k'], t['cos'], t['sin'], eps=1), backend='aot_eager',
                  fullgraph=True)(t)
    assert len(launches) == 4
