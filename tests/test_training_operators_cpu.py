"""Refusals of the training and serving operators (noise_amd.sinks, noise_amd.distill), their C entry points' argument checks and
the shapes of their torch.library registrations, without a GPU; and the 64-bit oracles against plain dense attention."""
import ctypes
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from noise_amd import _lib, distill, sinks
from oracle import distill as distill_oracle
from oracle import sinks as oracle

BF16 = torch.bfloat16


def qkv(B=2, T=5, H=4, Hk=2, D=64, dtype=BF16):
    return [torch.zeros(B, T, h, D, dtype=dtype) for h in (H, Hk, Hk)]


def test_attention_refusals():
    q, k, v = qkv()
    for args, words in (((q[0], k, v, 3), 'batch, token, head, dim'), ((q, k[:1], v, 3), 'one batch'),
                        ((q, k, v[:, :4], 3), 'one shape'), ((q, k[:, :4], v[:, :4], 3), 'length of q'),
                        ((q[:, :, :3], k, v, 3), 'no multiple'), ((q, k, v, -1), 'negative'), ((q, k, v, 3, -1), 'negative'),
                        ((*qkv(D=32), 3), '64 or 128'), ((*qkv(dtype=torch.float32), 3), 'bfloat16'),
                        ((q.half(), k, v, 3), 'bfloat16'), ((q, k, v, 3, 0, torch.zeros(3, dtype=torch.int32)), 'lengths'),
                        ((q, k, v, 3, 0, torch.zeros(2)), 'lengths'), ((q, k, v, 3), 'on a GPU')):
        with pytest.raises(ValueError, match=words):
            sinks.sink_attention(*args)


def test_decode_refusals():
    q, k, v = qkv(T=9)
    q = q[:, :1]
    start = torch.zeros(2, dtype=torch.int32)
    wide = torch.zeros(2, 9, 2, 65, dtype=BF16)[..., 1:]
    for args, words in (((q, k, v[:, :8], start, 3), 'one shape'), ((q, k[:, :0], v[:, :0], start, 3), 'capacity'),
                        ((torch.zeros(2, 17, 4, 64, dtype=BF16), k, v, start, 3), 'at most 16'),
                        ((q, k, v, start[:1], 3), 'start'), ((q, k, v, start.float(), 3), 'start'),
                        ((q, k, v, start, -3), 'negative'), ((q, wide, wide, start, 3), 'cache rows'),
                        ((q.float(), k, v, start, 3), 'bfloat16'), ((q, k, v, start, 3), 'on a GPU')):
        with pytest.raises(ValueError, match=words):
            sinks.sink_attention_decode(*args)


def test_norm_refusals():
    q, k, v = qkv()
    cos = sin = torch.zeros(5, 32)
    start = torch.zeros(2, dtype=torch.int64)
    for args, words in (((q, k[:, :4], cos, sin), 'one length'), ((q, k.float(), cos, sin), 'one length and type'),
                        ((q.half(), k.half(), cos, sin), 'bfloat16 or float32'), ((q, k, cos[:4], sin[:4]), 'positions'),
                        ((q, k, cos[:, :30], sin), 'cos and sin'), ((q, k, cos, sin, torch.zeros(32)), 'weights'),
                        ((q, k, cos, sin, None, None, start[:1]), 'start'), ((q, k, cos, sin), 'on a GPU')):
        with pytest.raises(ValueError, match=words):
            sinks.qk_norm_rotary(*args)
    cache = torch.zeros(2, 9, 2, 64, dtype=BF16)
    odd = torch.zeros(2, 9, 2, 65, dtype=BF16)[..., 1:]
    for args, words in (((q, k, v[:, :4], cos, sin, cache, cache, start), "k's shape"),
                        ((q, k, v.float(), cos, sin, cache, cache, start), "k's shape"),
                        ((q, k, v, cos, sin, cache[:, :, :1], cache, start), 'caches must be'),
                        ((q, k, v, cos, sin, cache, cache[:, :8], start), 'caches must be'),
                        ((q, k, v, cos, sin, cache, cache.float(), start), 'caches must be'),
                        ((q, k, v, cos, sin, odd, cache, start), 'cache rows'),
                        ((q, k, v, cos, sin, cache, cache, None), 'start is required'),
                        ((q, k, v, cos, sin, cache[:1].expand(2, 9, 2, 64), cache, start), 'broadcast'),
                        ((q, k, v, cos, sin, cache, cache, start), 'same memory'),
                        ((q, k, v, cos, sin, cache, cache.clone(), start), 'on a GPU')):
        with pytest.raises(ValueError, match=words):
            sinks.qk_norm_rotary_append(*args)


def test_distill_refusals():
    x, t, i = torch.zeros(3, 10), torch.zeros(3, 4), torch.zeros(3, 4, dtype=torch.int64)
    for args, more, words in (((x.half(), t, i), {}, 'bfloat16 or float32'), ((x, t[:2], i), {}, 'entries'),
                              ((x, t, i[:, :3]), {}, 'entries'), ((x, t[:, :0], i[:, :0]), {}, 'entries'),
                              ((x, t.repeat(1, 257), i.repeat(1, 257)), {}, 'at most 1024'), ((x, t, i.float()), {}, 'int32 or int64'), ((x, t.double(), i), {}, 'teacher logits'),
                              ((x, t, i), dict(vocab=11), 'vocab'), ((x, t, i), dict(vocab=0), 'vocab'),
                              ((x, t, i), dict(temperature=0.0), 'temperature'),
                              ((x, t, i), dict(temperature=math.nan), 'temperature'), ((x, t, i), dict(temperature=math.inf), 'temperature'),
                              ((x, t, i), dict(softcap=0.0), 'softcap'), ((x, t, i), dict(softcap=-1.0), 'softcap'),
                              ((x, t, i), {}, 'on a GPU')):
        with pytest.raises(ValueError, match=words):
            distill.distill_loss(*args, **more)
    with pytest.raises(ValueError, match='weights'):
        distill.distill_loss_grad(x, t, i, torch.zeros(2))


def test_entry_points_refuse():
    lib = _lib.lib()
    rows = lambda ptr=16, s=64, heads=2: _lib.Heads(ptr, 5 * s * heads, s * heads, s, heads)
    H = lambda **more: ctypes.byref(rows(**more))
    err = lambda: lib.noise_last_error().decode()
    fwd = lambda q=H(), k=H(), v=H(), o=H(), rest=None, B=1, T=5, D=64, W=3, n=0: lib.noise_sink_attention_fwd(
        q, k, v, o, rest, None, None, 0, B, T, D, W, n, 0.1, None)
    def refused(st, words):
        assert st == -1 and words in err(), (st, err())

    refused(fwd(D=96), 'head_dim')
    refused(fwd(W=-1), 'window')
    refused(fwd(n=-1), 'sinks')
    refused(fwd(q=H(ptr=8)), 'aligned')
    refused(fwd(k=H(s=68)), 'multiples of 8')
    refused(fwd(o=H(heads=3)), 'heads')
    refused(fwd(q=H(heads=3), o=H(heads=3)), 'key heads')
    refused(fwd(v=None), 'missing')
    refused(fwd(rest=H()), 'go together')
    refused(fwd(T=-1), 'tokens')
    refused(fwd(T=1 << 40), 'tokens')
    refused(fwd(B=1 << 50, T=1 << 29), 'too many')
    assert fwd(B=0) == 0 and fwd(T=0) == 0
    h = [H() for _ in range(9)]
    bwd = lambda ws, size: lib.noise_sink_attention_bwd(*h[:6], 16, *h[6:9], None, 0, 1, 5, 64, 3, 0, 0.1, ws, size, None)
    refused(bwd(16, 8), 'workspace')
    refused(bwd(None, 1 << 40), 'workspace')
    refused(lib.noise_sink_attention_bwd_workspace_bytes(1, 5, 3, 2, 64, 3, 0), 'key heads')
    # first tokens all over a long sequence do not cut its lists into ever more parts
    for sinks in (0, 4, 1000, 16384):
        assert 0 < lib.noise_sink_attention_bwd_workspace_bytes(8, 16384, 64, 64, 128, 0, sinks) < 1 << 30
        assert 0 < lib.noise_sink_attention_bwd_workspace_bytes(1, 1 << 22, 8, 1, 64, 100, sinks) < 1 << 30
    dec = lambda T=1, start=16, S=9, ws=None: lib.noise_sink_decode(*h[:4], start, 0, 1, T, S, 64, 3, 0, 0.1, ws, 0, None)
    refused(dec(T=17), '16')
    refused(dec(start=None), 'start')
    refused(dec(start=2), 'start')
    two, w = (_lib.Heads * 2)(rows(), rows()), (ctypes.c_void_p * 2)(None, None)
    norm = lambda D=64, kind=0, T=5, table=5, cap=0, v=None, w=w, x=two, eps=0.1: lib.noise_qk_norm_rotary(
        x, two, w, v, v, 16, 16, table, None, 0, 1, T, cap, D, kind, eps, None)
    refused(norm(D=32), 'head_dim')
    refused(norm(kind=2), 'type')
    refused(norm(table=4), 'tables')
    refused(norm(cap=3), 'cache')
    refused(norm(v=H()), 'cache')
    refused(norm(eps=-1.0), 'eps')
    refused(norm(x=(_lib.Heads * 2)(rows(heads=3), rows())), 'heads')
    refused(norm(w=(ctypes.c_void_p * 2)(4, None)), 'aligned')
    nb = lambda ws, size: lib.noise_qk_norm_rotary_bwd(two, two, two, (ctypes.c_void_p * 2)(16, None),
                                                       (ctypes.c_void_p * 2)(16, None), 16, 16, 5, None, 0, 1, 5, 64, 0,
                                                       0.1, ws, size, None)
    refused(nb(None, 0), 'workspace')
    dist = lambda rows=2, vocab=9, K=3, tau=1.0, cap=0.0, grad=16, width=9, gs=9, x=16: lib.noise_distill(
        x, 1, rows, vocab, 9, 16, 1, 16, 1, K, None, tau, cap, 16, grad, width, gs, None)
    for st in (dist(vocab=0), dist(K=0), dist(K=1025), dist(tau=0.0), dist(cap=-1.0), dist(width=8), dist(gs=8), dist(x=2), dist(x=None)):
        assert st == -1
    assert dist(rows=0) == 0


def test_fake_shapes():
    with FakeTensorMode():
        q, k, v = qkv()
        out, rest, lse = torch.ops.noise_amd.sink_attention(q, k, v, 3, 1, None)
        assert out.shape == rest.shape == q.shape and lse.shape == (2, 4, 5) and lse.dtype == torch.float32
        start = torch.zeros(2, dtype=torch.int64)
        assert torch.ops.noise_amd.sink_attention_decode(q[:, :1], k, v, start, 3, 1).shape == (2, 1, 4, 64)
        a, b = torch.ops.noise_amd.qk_norm_rotary(q, k, torch.zeros(5, 32), torch.zeros(5, 32), None, None, None, 1e-6)
        assert a.shape == q.shape and b.shape == k.shape
        x, t, i = torch.zeros(3, 10), torch.zeros(3, 4), torch.zeros(3, 4, dtype=torch.int64)
        assert torch.ops.noise_amd.distill_loss(x, t, i, 10, 1.0, None).shape == (3,)
        loss, grad = torch.ops.noise_amd.distill_loss_grad(x, t, i, None, 10, 1.0, 15.0)
        assert loss.shape == (3,) and grad.shape == (3, 10)


def test_oracles():
    """The 64-bit oracles against each other, torch's own differentiation and the model's windowed attention."""
    g = torch.Generator().manual_seed(0)
    q, k, v, dout = (torch.randn(2, 30, h, 64, generator=g, dtype=torch.float64, requires_grad=True) for h in (4, 2, 2, 4))
    from oracle import model as om
    want = om.attention(q.detach(), *(t.detach().repeat_interleave(2, 2) for t in (k, v)), 7)
    assert torch.allclose(oracle.attend(q, k, v, 7, 0)[0].float(), want, atol=1e-5)
    out, _ = oracle.attend(q, k, v, 7, 3, torch.tensor([30, 11]))
    grads, slack = oracle.attend_grads(q, k, v, dout, 7, 3, torch.tensor([30, 11]))
    for mine, auto in zip(grads, torch.autograd.grad((out * dout).sum(), (q, k, v))):
        assert torch.allclose(mine, auto, atol=1e-12)
    assert all((s >= 0).all() for s in slack)
    last, _ = oracle.decode(q[:, 10:11], k, v, torch.tensor([10, 10]), 7, 3)
    assert torch.allclose(last, out[:, 10:11], atol=1e-12)
    x = torch.randn(3, 12, generator=g, dtype=torch.float64, requires_grad=True)
    t, i = torch.randn(3, 4, generator=g), torch.tensor([[1, 1, 5, -1], [0, 2, 3, 11], [-1, 12, -1, -1]])
    loss, grad = distill_oracle.distill(x, t, i, 12, 2.0, 15.0)
    auto, = torch.autograd.grad(loss.sum(), x)
    assert torch.allclose(grad, auto, atol=1e-12) and loss[2] == 0 and (grad[2] == 0).all()


def test_tensor_tables_match_the_header(tmp_path):
    """noise_heads_t as a C compiler lays it out, as ctypes mirrors it and as the calls pack it: five 64-bit numbers."""
    import shutil
    import subprocess
    from pathlib import Path
    root = Path(__file__).resolve().parents[1]
    q = torch.zeros(3, 5, 7, 64, dtype=BF16)[:, :, 1:]
    w = torch.zeros(64)
    table, at = sinks._table(q, q[:, 2:], pointers=(None, w))
    assert ctypes.sizeof(_lib.Heads) == sinks._HEADS == 40
    for i, t in enumerate((q, q[:, 2:])):
        h = _lib.Heads.from_address(at + i * sinks._HEADS)
        assert (h.ptr, h.s_b, h.s_t, h.s_h, h.heads) == (t.data_ptr(), *t.stride()[:3], 6)
    assert list((ctypes.c_int64 * 2).from_address(at + 2 * sinks._HEADS)) == [0, w.data_ptr()] and len(table) == 12
    gcc = shutil.which('gcc')
    if gcc is None:
        pytest.skip('gcc not available')
    fields = [n for n, _ in _lib.Heads._fields_]
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "noise_amd.h"', 'int main(void) {',
             '    printf("%zu", sizeof(noise_heads_t));']
    lines += [f'    printf(" %zu", offsetof(noise_heads_t, {n}));' for n in fields]
    (tmp_path / 'layout.c').write_text('\n'.join([*lines, '    return 0;', '}']) + '\n')
    subprocess.run([gcc, '-std=c99', '-I', str(root / 'include'), str(tmp_path / 'layout.c'), '-o', str(tmp_path / 'layout')],
                   check=True)
    out = subprocess.run([str(tmp_path / 'layout')], capture_output=True, text=True, check=True).stdout.split()
    assert list(map(int, out)) == [40, *(getattr(_lib.Heads, n).offset for n in fields)]
