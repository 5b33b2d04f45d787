"""The ends of a training step with exact gradients, as cases that a timing program can run.

  norm   residual_norm: a block's output through its norm and gate onto the scaled residual stream, and the norm that the next
         block reads; alone (serving) or with its gradients
  head   linear_cross_entropy and linear_cross_entropy_grad: the losses of hidden states against a vocabulary, alone (an
         evaluation), through autograd, or with the gradients in one call
  clip   clip_gradients: the norm of all gradients, and the gradients scaled to a bound on it

`run` computes them in elementary torch operations, or through noise_amd where `own` is true.
"""
import math

import torch

own = False

DEV = 'cuda'
F32, F64 = torch.float32, torch.float64
DTYPES = {'bf16': torch.bfloat16, 'fp32': torch.float32}
EPS = torch.finfo(F32).eps
UNIT = 1e-6       # beside the norm in the clipping quotient
DECAY = 0.999     # of the clipping bound, from pass to pass


def listed():
    return [
        # one new token of four conversations between two blocks of the model: the call itself is what counts
        dict(name='norm-token', kind='norm', grad=False, batch=4, length=1, dim=512, x='bf16', y='bf16', post=False,
             gate='none', mix=True, weights=False),
        # the model's block entry in training under autocast: fp32 residual stream, bf16 branches, both mixing scalars
        dict(name='norm-model', kind='norm', grad=True, batch=8, length=2048, dim=512, x='fp32', y='bf16', post=False,
             gate='none', mix=True, weights=False),
        # documents of an odd length and width in fp32, norms on both sides, a gate for each sequence
        dict(name='norm-ragged', kind='norm', grad=True, batch=3, length=1111, dim=1001, x='fp32', y='fp32', post=True,
             gate='sequence', mix=False, weights=True),
        # a wide model in bf16, norms on both sides, a learned gate for each channel
        dict(name='norm-wide', kind='norm', grad=True, batch=4, length=2048, dim=4096, x='bf16', y='bf16', post=True,
             gate='channel', mix=False, weights=True),
        # log probabilities of one next token of four conversations over a wide vocabulary: the weight's bytes are what counts
        dict(name='head-token', kind='head', grad='none', rows=4, vocab=65536, width=65536, dim=2048, dtype='bf16',
             softcap=0.0, masked=False),
        # the model's head on 8 of its sequences, loss and gradients in one call
        dict(name='head-model', kind='head', grad='direct', rows=16384, vocab=4096, width=4096, dim=512, dtype='bf16',
             softcap=15.0, masked=False),
        # the same with the model's fp32 head, through autograd
        dict(name='head-fp32', kind='head', grad='backward', rows=16384, vocab=4096, width=4096, dim=512, dtype='fp32',
             softcap=15.0, masked=False),
        # odd numbers of rows and tokens, a width that ends inside tiles, prompts masked out, through autograd
        dict(name='head-ragged', kind='head', grad='backward', rows=3333, vocab=50021, width=50048, dim=776,
             dtype='bf16', softcap=0.0, masked=True),
        # a wide vocabulary, loss and gradients in one call
        dict(name='head-wide', kind='head', grad='direct', rows=8192, vocab=131072, width=131072, dim=2048,
             dtype='bf16', softcap=0.0, masked=False),
        # the gradients of one block
        dict(name='clip-least', kind='clip', count=6, elements=2 ** 20, dtypes='fp32', offset=0),
        # the model's 60 parameters, fp32
        dict(name='clip-model', kind='clip', count=60, elements=37750000, dtypes='fp32', offset=0),
        # a large model's gradients in flat buckets, fp32 and bf16, at odd offsets
        dict(name='clip-wide', kind='clip', count=300, elements=10 ** 9, dtypes='mixed', offset=1),
    ]


def _log(rng, low, high):
    """A whole number from low .. high, spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(['norm', 'norm', 'head', 'head', 'head', 'clip', 'clip'])
    if kind == 'norm':
        x, y = rng.choice([('bf16', 'bf16'), ('fp32', 'bf16'), ('fp32', 'fp32')])
        dim = rng.choice([64 * rng.randint(1, 128), 8 * rng.randint(2, 1024), rng.randint(16, 8192)])
        case = dict(kind=kind, grad=rng.random() < 0.7, batch=_log(rng, 1, 16), length=_log(rng, 1, 4096), dim=dim, x=x, y=y,
                    post=rng.random() < 0.5, gate=rng.choice(['none', 'channel', 'sequence', 'token']),
                    mix=rng.random() < 0.5, weights=rng.random() < 0.6)
        case['length'] = max(1, min(case['length'], 2 ** 25 // (case['batch'] * dim)))
        return case
    if kind == 'head':
        grad = rng.choice(['none', 'backward', 'direct'])
        vocab, dim = _log(rng, 50, 131072), rng.choice([64 * rng.randint(1, 64), 8 * rng.randint(4, 512), _log(rng, 33, 4096)])
        rows = min(_log(rng, 1, 16384), 2 ** 28 // vocab, 2 ** 39 // (vocab * dim))
        return dict(kind=kind, grad=grad, rows=max(1, rows), vocab=vocab, width=vocab + rng.choice([0, 0, 1, 27]), dim=dim,
                    dtype=rng.choice(['bf16', 'bf16', 'fp32']), softcap=rng.choice([0.0, 15.0]), masked=rng.random() < 0.4)
    count = _log(rng, 1, 500)
    return dict(kind=kind, count=count, elements=_log(rng, 100 * count, 10 ** 9), dtypes=rng.choice(['fp32', 'bf16', 'mixed']),
                offset=rng.choice([0, 0, 1, 3]))


# --- inputs ---


def _masked(case):
    """Which rows of a head case have no target: with masked, the first third of each 100 rows (a prompt)."""
    return [case['masked'] and r % 100 < 33 for r in range(case['rows'])]


def _sizes(case):
    """The tensors' numbers of elements: a large one in eight, others a sixteenth of it, a few vectors."""
    parts = [(16, 1, 1, 1, 2, 4, 1, 0.01)[i % 8] for i in range(case['count'])]
    return [max(1, int(case['elements'] * p / sum(parts))) for p in parts]


def _places(case):
    """(type, offset in that type's flat buffer, elements) of each tensor, and the buffers' sizes."""
    ends, places = {}, []
    for i, n in enumerate(_sizes(case)):
        dt = ('fp32', 'bf16')[i // 2 % 2] if case['dtypes'] == 'mixed' else case['dtypes']
        at = ends.get(dt, 0)
        if not case['offset']:
            at = -(-at // 64) * 64
        places.append((dt, at + case['offset'], n))
        ends[dt] = at + case['offset'] + n
    return places, ends


def _gradients(case):
    """Whether each tensor of a case has its own memory (few of them) or is a view of its type's flat buffer."""
    return case['count'] <= 60 and not case['offset']


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    randn = lambda *s, dtype=F32: torch.randn(*s, device=DEV, generator=g).to(dtype)
    s = dict(case=dict(case), kind=case['kind'])
    if case['kind'] == 'norm':
        B, T, D = case['batch'], case['length'], case['dim']
        xt, yt = DTYPES[case['x']], DTYPES[case['y']]
        x = randn(B, T, D)
        s.update(x=x.to(xt), y=randn(B, T, D, dtype=yt), x0=None, scale=None, x0_scale=None, gate=None, y_weight=None,
                 weight=None)
        if case['mix']:
            s.update(x0=randn(B, T, D, dtype=xt), scale=0.9 + 0.05 * randn(()), x0_scale=0.1 + 0.02 * randn(()))
        if case['gate'] != 'none':
            shape = dict(channel=(D,), sequence=(B, 1, D), token=(B, T, D))[case['gate']]
            s['gate'] = (0.5 + 0.2 * randn(*shape)).to(F32 if case['gate'] == 'channel' else yt)
        if case['weights']:
            s.update(weight=1 + 0.2 * randn(D))
            if case['post']:
                s.update(y_weight=1 + 0.2 * randn(D))
        if case['grad']:
            # upstream gradients that go along with the residual stream, as a loss's do
            s.update(dx=(randn(B, T, D) + 0.1 * x).to(xt), dh=(randn(B, T, D) + 0.1 * x).to(yt))
        return s
    if case['kind'] == 'head':
        R, V, W, D = (case[n] for n in ('rows', 'vocab', 'width', 'dim'))
        dt = DTYPES[case['dtype']]
        weight = randn(W, D).mul_(2 / math.sqrt(D))
        targets = torch.randint(V, (R,), device=DEV, generator=g)
        # hidden states after their norm, which know something of their targets
        row = weight[targets]
        x = randn(R, D) + 2 * row / row.norm(dim=-1, keepdim=True)
        targets[torch.tensor(_masked(case), device=DEV)] = -100
        s.update(x=x.to(dt), weight=weight.to(dt), targets=targets, vocab=V, softcap=case['softcap'] or None)
        if case['grad'] != 'none':
            s['token_weight'] = torch.rand(R, device=DEV, generator=g) / R
        return s
    places, ends = _places(case)
    if _gradients(case):
        s['gradients'] = [randn(n, dtype=DTYPES[dt]).mul_(0.01) for dt, _, n in places]
        s['buffers'] = s['gradients']
    else:
        flat = {dt: randn(n, dtype=DTYPES[dt]).mul_(0.01) for dt, n in ends.items()}
        s['gradients'] = [flat[dt][at:at + n] for dt, at, n in places]
        s['buffers'] = [flat[dt] for dt in sorted(flat)]
    # below the norm on the first pass; falling, so that gradients that were clipped are clipped again
    s['bound'] = 0.007 * math.sqrt(sum(_sizes(case)))
    return s


# --- one pass ---


def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from noise_amd import clip, residual, vocab
    case = s['case']
    if s['kind'] == 'norm':
        names = [n for n in ('x', 'y', 'x0', 'scale', 'x0_scale', 'gate', 'y_weight', 'weight') if s[n] is not None]
        leaves = {n: s[n].detach().requires_grad_(case['grad']) for n in names}
        outs = residual.residual_norm(**leaves, norm_y=case['post'])
        if not case['grad']:
            return outs
        return (*outs, *torch.autograd.grad(outs, list(leaves.values()), (s['dx'], s['dh'])))
    if s['kind'] == 'head':
        more = dict(vocab=s['vocab'], softcap=s['softcap'])
        if case['grad'] == 'none':
            return vocab.linear_cross_entropy(s['x'], s['weight'], s['targets'], **more)
        if case['grad'] == 'direct':
            return vocab.linear_cross_entropy_grad(s['x'], s['weight'], s['targets'], s['token_weight'], **more)
        leaves = [s['x'].detach().requires_grad_(), s['weight'].detach().requires_grad_()]
        loss = vocab.linear_cross_entropy(*leaves, s['targets'], **more)
        return (loss, *torch.autograd.grad(loss, leaves, s['token_weight']))
    bound, s['bound'] = s['bound'], s['bound'] * DECAY
    return clip.clip_gradients(s['gradients'], bound), s['buffers']


def _run_plain(s):
    if s['kind'] == 'norm':
        return _norm_plain(s)
    if s['kind'] == 'head':
        return _head_plain(s)
    bound, s['bound'] = s['bound'], s['bound'] * DECAY
    norm = torch.stack([g.to(F64).square().sum() for g in s['gradients']]).sum().sqrt()
    factor = (bound / (norm + UNIT)).clamp(max=1.0).float()
    [g.copy_(g.float() * factor) for g in s['gradients']]
    return norm.float(), s['buffers']


def _norm_plain(s):
    case, D = s['case'], s['case']['dim']
    there = lambda n: s[n] is not None
    x, y = s['x'].float(), s['y'].float()
    if case['post']:
        ry = torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)
        ny = y * ry
        b = ny * s['y_weight'] if there('y_weight') else ny
    else:
        b = y
    gate = s['gate'].float() if there('gate') else None
    inner = x + (b if gate is None else gate * b)
    out = inner * s['scale'] if there('scale') else inner
    if there('x0'):
        out = out + s['x0_scale'] * s['x0'].float()
    r = torch.rsqrt(out.square().mean(-1, keepdim=True) + EPS)
    n = out * r
    h = n * s['weight'] if there('weight') else n
    outs = out.to(s['x'].dtype), h.to(s['y'].dtype)
    if not case['grad']:
        return outs
    dh = s['dh'].float()
    u = dh * s['weight'] if there('weight') else dh
    G = s['dx'].float() + r * (u - n * (u * n).mean(-1, keepdim=True))
    U = G * s['scale'] if there('scale') else G
    grads = [U.to(s['x'].dtype)]
    db = U if gate is None else U * gate
    if case['post']:
        e = db * s['y_weight'] if there('y_weight') else db
        grads.append((ry * (e - ny * (e * ny).mean(-1, keepdim=True))).to(s['y'].dtype))
    else:
        grads.append(db.to(s['y'].dtype))
    if there('x0'):
        grads += [(s['x0_scale'] * G).to(s['x'].dtype), (G * inner).sum(dtype=F64).float(),
                  (G * s['x0'].float()).sum(dtype=F64).float()]
    if gate is not None:
        over = dict(channel=(0, 1), sequence=(1,), token=())[case['gate']]
        dg = U * b
        grads.append((dg.sum(over, keepdim=case['gate'] == 'sequence') if over else dg).to(s['gate'].dtype))
    if there('y_weight'):
        grads.append((db * ny).sum((0, 1)))
    if there('weight'):
        grads.append((dh * n).sum((0, 1)))
    return (*outs, *grads)


def _head_plain(s):
    case, V, cap = s['case'], s['vocab'], s['softcap']
    x, w = s['x'].float(), s['weight'][:V].float()
    used = (s['targets'] >= 0) & (s['targets'] < V)
    at = torch.where(used, s['targets'], 0)[:, None]
    z = x @ w.t()
    th = None
    if cap is not None:
        th = torch.tanh(z / cap)
        z = cap * th
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    loss = torch.where(used, (top + total.log() - z.gather(1, at))[:, 0], 0.0)
    if case['grad'] == 'none':
        return loss
    weight = torch.where(used, s['token_weight'], 0.0)[:, None]
    d = e.div_(total).mul_(weight).scatter_add_(1, at, -weight)
    if th is not None:
        d.mul_(1 - th * th)
    dw = torch.zeros(s['weight'].shape, dtype=s['weight'].dtype, device=DEV)
    dw[:V] = d.t() @ x
    return loss, (d @ w).to(s['x'].dtype), dw


# --- what a pass cannot do without ---


def work(case):
    size = lambda n: 2 if case[n] == 'bf16' else 4
    if case['kind'] == 'norm':
        n, grad = case['batch'] * case['length'] * case['dim'], case['grad']
        per = 2 * size('x') + 2 * size('y') + (size('x') if case['mix'] else 0)
        flops = 10 + (4 if case['post'] else 0)
        if grad:
            per += 2 * size('x') + 2 * size('y') + (size('x') if case['mix'] else 0)
            flops += 16 + (8 if case['post'] else 0)
        if case['gate'] == 'token':
            per += size('y') * (2 if grad else 1)
        return dict(bytes=per * n + 4 * case['dim'], flops=flops * n)
    if case['kind'] == 'head':
        R, V, D = case['rows'], case['vocab'], case['dim']
        grad = case['grad'] != 'none'
        live = R - sum(_masked(case))
        return dict(bytes=(R + V) * D * size('dtype') * (2 if grad else 1) + 12 * R, flops=(6 if grad else 2) * live * V * D)
    n = sum((4 if dt == 'fp32' else 2) * n for dt, _, n in _places(case)[0])
    return dict(bytes=2 * n + 4, flops=3 * sum(_sizes(case)))


# --- the same results in 64 bits ---


def exact(case, seed):
    s = prepare(case, seed)
    return dict(norm=_norm64, head=_head64, clip=_clip64)[case['kind']](s, case)


def _rms64(x, w):
    u = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
    return u if w is None else u * w


def _norm64(s, case):
    """By differentiating the definition."""
    names = [n for n in ('x', 'y', 'x0', 'scale', 'x0_scale', 'gate', 'y_weight', 'weight') if s[n] is not None]
    t = {n: s[n].double().requires_grad_(case['grad']) for n in names}
    b = _rms64(t['y'], t.get('y_weight')) if case['post'] else t['y']
    x = t.get('scale', 1.0) * (t['x'] + t.get('gate', 1.0) * b)
    if case['mix']:
        x = x + t['x0_scale'] * t['x0']
    outs = x, _rms64(x, t.get('weight'))
    if not case['grad']:
        return outs
    return (*(o.detach() for o in outs), *torch.autograd.grad(outs, [t[n] for n in names], (s['dx'].double(), s['dh'].double())))


def _head64(s, case):
    """At most 2^28 logits at a time."""
    V, R = s['vocab'], case['rows']
    grad = case['grad'] != 'none'
    w = s['weight'][:V].double()
    losses, dx = torch.zeros(R, dtype=F64, device=DEV), torch.zeros(s['x'].shape, dtype=F64, device=DEV)
    dw = torch.zeros(s['weight'].shape, dtype=F64, device=DEV)
    live = torch.tensor([r for r, out in enumerate(_masked(case)) if not out], device=DEV, dtype=torch.long)
    for rows in live.split(max(1, 2 ** 28 // V)):
        x, t = s['x'][rows].double(), s['targets'][rows]
        raw = torch.mm(x, w.t())
        z = raw if s['softcap'] is None else torch.tanh(raw / s['softcap']) * s['softcap']
        log_p = torch.log_softmax(z, -1)
        losses[rows] = torch.nn.functional.nll_loss(log_p, t, reduction='none')
        if grad:
            p = log_p.exp_()
            p[torch.arange(len(rows), device=DEV), t] -= 1
            p *= s['token_weight'][rows].double()[:, None]
            if s['softcap'] is not None:
                p *= 1 - (z / s['softcap']) ** 2
            dx[rows] = torch.mm(p, w)
            dw[:V] += torch.mm(p.t(), x)
    return (losses, dx, dw) if grad else losses


def _clip64(s, case):
    norm = math.sqrt(sum(float(torch.linalg.vector_norm(g.double())) ** 2 for g in s['gradients']))
    places = _places(case)[0]
    factor = min(1.0, s['bound'] / (norm + UNIT))
    done = [b.double() for b in s['buffers']]
    if _gradients(case):
        done = [b * factor for b in done]
    else:
        kinds = sorted({dt for dt, _, _ in places})
        for dt, at, n in places:
            done[kinds.index(dt)][at:at + n] *= factor
    return torch.tensor(norm, dtype=F64), done
