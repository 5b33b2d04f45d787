"""The operators of a distilled student with long-context attention, as cases that a timing program can run.

  norm     qk_norm_rotary with its gradients: the queries and keys of a training step
  append   qk_norm_rotary_append: the same for new tokens, whose keys and values go into a cache
  attend   sink_attention: a window and the first tokens; the output alone (a prompt) or with the gradients
  decode   sink_attention_decode: one or a few new tokens against the cache
  distill  distill_loss and distill_loss_grad: the loss against a teacher's top logits, alone or with its gradient

`run` computes them in elementary torch operations, or through noise_amd where `own` is true.
"""
import math

import torch

own = False

DEV = 'cuda'
F32, F64 = torch.float32, torch.float64
DTYPES = {'bf16': torch.bfloat16, 'fp32': torch.float32}
EPS = torch.finfo(F32).eps


def listed():
    return [
        # the model's own layer in training: 8 heads of 64, a batch of its sequences
        dict(name='norm-model', kind='norm', batch=8, length=2048, heads=8, kv_heads=8, dim=64, dtype='bf16',
             weights=True),
        # documents of an odd length with shared key heads, fp32 activations
        dict(name='norm-ragged', kind='norm', batch=3, length=1111, heads=16, kv_heads=4, dim=128, dtype='fp32',
             weights=True),
        # one new token of a few conversations: the call itself is what counts
        dict(name='append-token', kind='append', batch=4, length=1, heads=8, kv_heads=8, dim=64, capacity=2048,
             dtype='bf16', weights=False, idle=False),
        # a batch of prompts into their cache
        dict(name='append-prompt', kind='append', batch=16, length=1500, heads=32, kv_heads=8, dim=128, capacity=2048,
             dtype='bf16', weights=True, idle=False),
        # one long prompt, shared key heads, a short window and four first tokens
        dict(name='attend-prompt', kind='attend', grad=False, batch=1, length=16384, heads=16, kv_heads=4, dim=128,
             window=2048, sinks=4, ragged=False),
        # the model's half-window layer in training
        dict(name='attend-model', kind='attend', grad=True, batch=8, length=2048, heads=8, kv_heads=8, dim=64,
             window=1024, sinks=4, ragged=False),
        # a padded batch of documents in training, shared key heads, a window that ends inside tiles
        dict(name='attend-ragged', kind='attend', grad=True, batch=5, length=1777, heads=8, kv_heads=2, dim=128,
             window=300, sinks=70, ragged=True),
        # one new token of one conversation with the model's heads
        dict(name='decode-least', kind='decode', batch=1, length=1, heads=8, kv_heads=8, dim=64, capacity=2048,
             window=1024, sinks=4, idle=False),
        # a full serving batch deep in its caches
        dict(name='decode-batch', kind='decode', batch=64, length=1, heads=32, kv_heads=8, dim=128, capacity=16384,
             window=4096, sinks=4, idle=False),
        # a small batch, an odd vocabulary, few entries: the loss of an evaluation
        dict(name='distill-least', kind='distill', grad=False, rows=100, vocab=4000, width=4001, entries=17,
             dtype='bf16', temperature=1.0, softcap=0.0, ragged=True),
        # the model's soft-capped logits of 8 sequences, in fp32, loss and gradient
        dict(name='distill-model', kind='distill', grad=True, rows=16384, vocab=4096, width=4096, entries=64,
             dtype='fp32', temperature=2.0, softcap=15.0, ragged=False),
        # a wide vocabulary in bf16, loss and gradient
        dict(name='distill-wide', kind='distill', grad=True, rows=4096, vocab=65536, width=65536, entries=100,
             dtype='bf16', temperature=1.5, softcap=0.0, ragged=True),
    ]


def _log(rng, low, high):
    """A whole number from low .. high, spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8])
    return dict(heads=kv * rng.choice([1, 2, 4]), kv_heads=kv, dim=rng.choice([64, 128]))


def draw(rng):
    kind = rng.choice(['norm', 'append', 'attend', 'attend', 'attend', 'decode', 'decode', 'distill', 'distill'])
    if kind == 'norm':
        case = dict(kind=kind, batch=_log(rng, 1, 16), length=_log(rng, 1, 4096), **_heads(rng),
                    dtype=rng.choice(['bf16', 'bf16', 'fp32']), weights=rng.random() < 0.7)
        per = case['batch'] * (case['heads'] + case['kv_heads']) * case['dim']
        case['length'] = max(1, min(case['length'], 2 ** 25 // per))
        return case
    if kind == 'append':
        case = dict(kind=kind, batch=_log(rng, 1, 64), length=rng.choice([1, 1, rng.randint(2, 9), _log(rng, 10, 2000)]),
                    **_heads(rng), capacity=0, dtype=rng.choice(['bf16', 'bf16', 'fp32']), weights=rng.random() < 0.7,
                    idle=rng.random() < 0.3)
        per = case['batch'] * (case['heads'] + 2 * case['kv_heads']) * case['dim']
        case['length'] = max(1, min(case['length'], 2 ** 27 // per))
        case['capacity'] = case['length'] + rng.randint(0, 1000)
        return case
    if kind == 'attend':
        grad = rng.random() < 0.6
        least = rng.choice([1, 40, 200])
        case = dict(kind=kind, grad=grad, batch=_log(rng, 1, 8), length=_log(rng, least, 4096 if grad else 16384),
                    **_heads(rng), window=0, sinks=0, ragged=rng.random() < 0.4)
        rows = case['batch'] * case['heads']
        case['length'] = min(case['length'], math.isqrt(2 ** (30 if grad else 32) // rows))
        case['window'] = min(_log(rng, 1, 4096), 2 ** (27 if grad else 29) // (rows * case['length']))
        case['sinks'] = rng.choice([0, 1, 4, _log(rng, 1, 300)])
        return case
    if kind == 'decode':
        case = dict(kind=kind, batch=_log(rng, 1, 128), length=rng.choice([1, 1, 1, rng.randint(2, 8)]), **_heads(rng),
                    capacity=_log(rng, 8, 32768), window=_log(rng, 1, 16384), sinks=rng.choice([0, 1, 4, rng.randint(2, 99)]),
                    idle=rng.random() < 0.3)
        per = case['batch'] * case['kv_heads'] * case['dim']
        case['capacity'] = max(8, min(case['capacity'], 2 ** 30 // per))
        return case
    vocab = _log(rng, 50, 100000)
    rows = max(1, min(_log(rng, 1, 16384), 2 ** 26 // vocab))
    return dict(kind=kind, grad=rng.random() < 0.7, rows=rows, vocab=vocab, width=vocab + rng.choice([0, 0, 1, 47]),
                entries=_log(rng, 1, min(128, vocab)), dtype=rng.choice(['bf16', 'fp32']),
                temperature=rng.choice([1.0, 0.7, 2.0, 3.5]), softcap=rng.choice([0.0, 15.0]),
                ragged=rng.random() < 0.5)


# --- inputs ---


def _starts(case):
    """Positions of each sequence's first new token: caches filled to between three quarters and all of what they take,
    and, with idle sequences, some that hold nothing and take no token (their positions are negative)."""
    room = max(0, case['capacity'] - case['length'])
    starts = [room - (b * 37) % (room // 4 + 1) for b in range(case['batch'])]
    if case['idle']:
        starts[2::3] = [-case['length']] * len(starts[2::3])
    return starts


def _prompt_starts(case):
    """As _starts, for tokens that are appended: anywhere in the cache."""
    room = max(0, case['capacity'] - case['length'])
    starts = [(b * 97) % (room + 1) for b in range(case['batch'])]
    if case['idle']:
        starts[2::3] = [-case['length']] * len(starts[2::3])
    return starts


def _lengths(case):
    """Lengths of a padded batch: all, one token, two thirds, none, and so on."""
    T = case['length']
    return [(T, max(1, 2 * T // 3), 1, 0, T - T // 7)[b % 5] for b in range(case['batch'])]


def _used(case):
    """Teacher entries in use per row: all, or fewer in some rows (none in a few)."""
    K = case['entries']
    return [0 if r % 50 == 49 else max(1, K - r % 5) if r % 2 else K for r in range(case['rows'])]


def _tables(length, dim):
    """cos and sin [length, dim / 2] in fp32, of angles in 64 bits."""
    inv = 10000.0 ** (-torch.arange(0, dim, 2, device=DEV, dtype=F64) / dim)
    angle = torch.arange(length, device=DEV, dtype=F64)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    randn = lambda *s, dtype=F32: torch.randn(*s, device=DEV, generator=g).to(dtype)
    kind = case['kind']
    s = dict(case=dict(case), kind=kind)
    if kind == 'distill':
        R, V, W, K = case['rows'], case['vocab'], case['width'], case['entries']
        dt = DTYPES[case['dtype']]
        logits = randn(R, W).mul_(3)
        values, index = (logits[:, :V] + randn(R, V)).topk(K, -1)      # a teacher that agrees in part
        used = torch.tensor(_used(case), device=DEV) if case['ragged'] else torch.full((R,), K, device=DEV)
        index[torch.arange(K, device=DEV) >= used[:, None]] = -1
        s.update(logits=logits.to(dt), teacher=values.to(dt), index=index.int(),
                 weight=torch.rand(R, device=DEV, generator=g) / R, vocab=V, temperature=case['temperature'],
                 softcap=case['softcap'] or None)
        return s
    B, T, H, Hk, D = (case[n] for n in ('batch', 'length', 'heads', 'kv_heads', 'dim'))
    if kind in ('norm', 'append'):
        dt = DTYPES[case['dtype']]
        s.update(q=randn(B, T, H, D, dtype=dt), k=randn(B, T, Hk, D, dtype=dt), qw=None, kw=None)
        if case['weights']:
            s.update(qw=1 + 0.2 * randn(D), kw=1 + 0.2 * randn(D))
        if kind == 'norm':
            s['cos'], s['sin'] = _tables(T, D)
            s.update(dq=randn(B, T, H, D, dtype=dt), dk=randn(B, T, Hk, D, dtype=dt))
        else:
            s['cos'], s['sin'] = _tables(case['capacity'], D)
            s.update(v=randn(B, T, Hk, D, dtype=dt), k_cache=randn(B, case['capacity'], Hk, D, dtype=dt),
                     v_cache=randn(B, case['capacity'], Hk, D, dtype=dt),
                     start=torch.tensor(_prompt_starts(case), device=DEV, dtype=torch.int32))
        return s
    # queries and keys as they leave the head norm; queries share a direction that the first keys answer to
    shared = randn(Hk, D)
    unit = lambda t: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + EPS)
    S = T if kind == 'attend' else case['capacity']
    q = unit(randn(B, T, H, D) + 0.5 * shared.repeat_interleave(H // Hk, 0))
    k = randn(B, S, Hk, D)
    k[:, :case['sinks']] += shared
    bf = torch.bfloat16
    q, k, v = q.to(bf), unit(k).to(bf), randn(B, S, Hk, D, dtype=bf)
    s.update(q=q, window=case['window'], sinks=case['sinks'])
    if kind == 'attend':
        s.update(k=k, v=v, lengths=None)
        if case['ragged']:
            s['lengths'] = torch.tensor(_lengths(case), device=DEV, dtype=torch.int32)
        if case['grad']:
            s['dout'] = randn(B, T, H, D, dtype=bf)
    else:
        s.update(k_cache=k, v_cache=v, start=torch.tensor(_starts(case), device=DEV, dtype=torch.int32))
    return s


# --- one pass ---


def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from noise_amd import distill, sinks
    kind, case = s['kind'], s['case']
    if kind == 'norm':
        leaves = [s['q'], s['k']] + ([s['qw'], s['kw']] if case['weights'] else [])
        leaves = [t.detach().requires_grad_() for t in leaves]
        q, k = sinks.qk_norm_rotary(leaves[0], leaves[1], s['cos'], s['sin'], *leaves[2:])
        return (q, k, *torch.autograd.grad((q, k), leaves, (s['dq'], s['dk'])))
    if kind == 'append':
        q = sinks.qk_norm_rotary_append(s['q'], s['k'], s['v'], s['cos'], s['sin'], s['k_cache'], s['v_cache'],
                                        s['start'], s['qw'], s['kw'])
        return q, s['k_cache'], s['v_cache']
    if kind == 'attend':
        if not case['grad']:
            return sinks.sink_attention(s['q'], s['k'], s['v'], s['window'], s['sinks'], s['lengths'])
        leaves = [s[n].detach().requires_grad_() for n in ('q', 'k', 'v')]
        out = sinks.sink_attention(*leaves, s['window'], s['sinks'], s['lengths'])
        return (out, *torch.autograd.grad(out, leaves, s['dout']))
    if kind == 'decode':
        return sinks.sink_attention_decode(s['q'], s['k_cache'], s['v_cache'], s['start'], s['window'], s['sinks'])
    args = (s['logits'], s['teacher'], s['index'])
    more = dict(vocab=s['vocab'], temperature=s['temperature'], softcap=s['softcap'])
    if case['grad']:
        return distill.distill_loss_grad(*args, s['weight'], **more)
    return distill.distill_loss(*args, **more)


def _run_plain(s):
    kind, case = s['kind'], s['case']
    if kind == 'norm':
        pos = torch.arange(case['length'], device=DEV).expand(case['batch'], -1)
        q, dq, dqw = _norm_plain(s['q'], s['qw'], s['cos'], s['sin'], pos, s['dq'])
        k, dk, dkw = _norm_plain(s['k'], s['kw'], s['cos'], s['sin'], pos, s['dk'])
        return (q, k, dq, dk, dqw, dkw) if case['weights'] else (q, k, dq, dk)
    if kind == 'append':
        pos = s['start'].long()[:, None] + torch.arange(case['length'], device=DEV)
        q = _norm_plain(s['q'], s['qw'], s['cos'], s['sin'], pos)
        k = _norm_plain(s['k'], s['kw'], s['cos'], s['sin'], pos)
        if case['idle']:
            b, t = torch.where((pos >= 0) & (pos < case['capacity']))
        else:
            b, t = (i.reshape(-1) for i in torch.meshgrid(*(torch.arange(n, device=DEV) for n in pos.shape), indexing='ij'))
        s['k_cache'][b, pos[b, t]] = k[b, t]
        s['v_cache'][b, pos[b, t]] = s['v'][b, t]
        return q, s['k_cache'], s['v_cache']
    if kind == 'attend':
        return _attend_plain(s['q'], s['k'], s['v'], s['window'], s['sinks'], s['lengths'], s.get('dout'))
    if kind == 'decode':
        return _decode_plain(s)
    return _distill_plain(s)


def _norm_plain(x, w, cos, sin, pos, dy=None):
    """The rotated norm of x [B, T, heads, D] at positions pos [B, T]; with dy also the gradients of x and w."""
    h = x.shape[-1] // 2
    there = ((pos >= 0) & (pos < cos.shape[0]))[..., None, None]
    at = pos.clamp(0, cos.shape[0] - 1)
    c, sn = cos[at][:, :, None], sin[at][:, :, None]
    f = x.float()
    r = torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS)
    n = f * r
    u = n if w is None else n * w
    y = torch.cat([u[..., :h] * c + u[..., h:] * sn, u[..., h:] * c - u[..., :h] * sn], -1)
    y = torch.where(there, y, torch.zeros_like(y)).to(x.dtype)
    if dy is None:
        return y
    d = dy.float()
    du = torch.cat([d[..., :h] * c - d[..., h:] * sn, d[..., :h] * sn + d[..., h:] * c], -1)
    dw = None if w is None else (du * n).sum((0, 1, 2))
    gr = du if w is None else du * w
    dx = r * (gr - n * (gr * n).mean(-1, keepdim=True))
    return y, dx.to(x.dtype), dw


def _attend_plain(q, k, v, window, sinks, lengths, dout):
    """One sequence and at most 1024 queries at a time, in fp32."""
    B, T, H, D = q.shape
    Hk = k.shape[2]
    G, scale = H // Hk, D ** -0.5
    out = torch.zeros_like(q)
    if dout is not None:
        grads = [torch.zeros(t.shape, dtype=F32, device=DEV) for t in (q, k, v)]
    j = torch.arange(T, device=DEV)
    for b in range(B):
        kt, vt = (x[b].float().transpose(0, 1).contiguous() for x in (k, v))       # [Hk, T, D]
        kT = kt.transpose(1, 2).contiguous()
        for t0 in range(0, T, 1024):
            n = min(1024, T - t0)
            i, hi = j[t0:t0 + n, None], t0 + n
            seen = (j[:hi] <= i) & ((i - j[:hi] <= window) | (j[:hi] < sinks))
            if lengths is not None:
                seen = seen & (j[:hi] < lengths[b]) & (i < lengths[b])
            rows = lambda x: x[b, t0:hi].float().view(n, Hk, G, D).permute(1, 2, 0, 3).reshape(Hk, G * n, D)
            back = lambda x: x.view(Hk, G, n, D).permute(2, 0, 1, 3).reshape(n, H, D)
            qs = rows(q)
            sc = (torch.bmm(qs, kT[:, :, :hi].contiguous()) * scale).view(Hk * G, n, hi)
            sc.masked_fill_(~seen, -math.inf)
            top = sc.amax(-1, keepdim=True).clamp(min=torch.finfo(F32).min)
            p = torch.exp(sc - top)
            total = p.sum(-1, keepdim=True)
            p = (p / torch.where(total > 0, total, torch.ones_like(total))).view(Hk, G * n, hi)
            o = torch.bmm(p, vt[:, :hi].contiguous())
            out[b, t0:hi] = back(o).to(q.dtype)
            if dout is not None:
                do = rows(dout)
                delta = (do * o).sum(-1, keepdim=True)
                ds = p * (torch.bmm(do, vt[:, :hi].transpose(1, 2).contiguous()) - delta) * scale
                grads[0][b, t0:hi] = back(torch.bmm(ds, kt[:, :hi].contiguous()))
                grads[1][b, :hi] += torch.bmm(ds.transpose(1, 2).contiguous(), qs).transpose(0, 1)
                grads[2][b, :hi] += torch.bmm(p.transpose(1, 2).contiguous(), do).transpose(0, 1)
    if dout is None:
        return out
    return (out, *(x.to(q.dtype) for x in grads))


def _decode_plain(s):
    q, start, window, sinks = s['q'], s['start'].long(), s['window'], s['sinks']
    B, T, H, D = q.shape
    S, Hk = s['k_cache'].shape[1:3]
    G = H // Hk
    j = torch.arange(S, device=DEV)
    i = start[:, None] + torch.arange(T, device=DEV)
    seen = (j <= i[..., None]) & ((i[..., None] - j <= window) | (j < sinks))           # [B, T, S]
    qs = q.float().view(B, T, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B * Hk, G * T, D)
    kT = s['k_cache'].float().permute(0, 2, 3, 1).reshape(B * Hk, D, S).contiguous()
    vs = s['v_cache'].float().permute(0, 2, 1, 3).reshape(B * Hk, S, D).contiguous()
    sc = (torch.bmm(qs, kT) * D ** -0.5).view(B, Hk * G, T, S).masked_fill_(~seen[:, None], -math.inf)
    top = sc.amax(-1, keepdim=True).clamp(min=torch.finfo(F32).min)
    p = torch.exp(sc - top)
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total > 0, total, torch.ones_like(total))).view(B * Hk, G * T, S)
    return torch.bmm(p, vs).view(B, Hk, G, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, H, D).to(q.dtype)


def _distill_plain(s):
    case, tau, cap = s['case'], s['temperature'], s['softcap']
    V, K, index = s['vocab'], case['entries'], s['index'].long()
    raw = s['logits'][:, :V].float()
    th = None if cap is None else torch.tanh(raw / cap)
    z = (raw if cap is None else cap * th) / tau
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    used = (index >= 0) & (index < V)
    t = (s['teacher'].float() / tau).masked_fill(~used, -math.inf)
    t = t - t.amax(-1, keepdim=True).clamp(min=torch.finfo(F32).min)
    p = torch.exp(t)
    mass = p.sum(-1, keepdim=True)
    some = mass > 0
    mass = torch.where(some, mass, torch.ones_like(mass))
    p = p / mass
    at = index.clamp(0, V - 1)
    terms = p * (t - mass.log() - (z.gather(1, at) - top - total.log()))
    loss = tau * tau * torch.where(p > 0, terms, torch.zeros_like(terms)).sum(-1)
    if not case['grad']:
        return loss
    d = torch.where(some, e / total, torch.zeros_like(e))
    d.scatter_add_(1, at, -p)
    d *= tau * s['weight'][:, None]
    if cap is not None:
        d *= 1 - th * th
    grad = torch.zeros(s['logits'].shape, dtype=s['logits'].dtype, device=DEV)
    grad[:, :V] = d
    return loss, grad


# --- what a pass cannot do without ---


def _pairs(length, window, sinks):
    """Visible (query, key) pairs of one head over a sequence of this length."""
    return sum(min(i + 1, window + 1 + min(sinks, max(0, i - window))) for i in range(length))


def _visible(case):
    """Keys that the new tokens of each sequence see between them, and (query, key) pairs, summed over sequences."""
    keys = pairs = 0
    for start in _starts(case):
        seen = set()
        low = None
        for t in range(case['length']):
            i = start + t
            if i < 0:
                continue
            first, last = max(0, i - case['window']), min(i, case['capacity'] - 1)
            sunk = min(case['sinks'], first)
            low = first if low is None else low
            pairs += last - first + 1 + sunk
            seen = (min(case['sinks'], low), low, last)
        if seen:
            keys += seen[0] + seen[2] - seen[1] + 1
    return keys, pairs


def work(case):
    kind = case['kind']
    if kind == 'distill':
        size = 2 if case['dtype'] == 'bf16' else 4
        R, V, K = case['rows'], case['vocab'], case['entries']
        step = case['grad']
        return dict(bytes=R * V * size + (R * case['width'] * size + 4 * R if step else 0) + R * (K * (size + 4) + 4),
                    flops=R * V * (8 if step else 4))
    B, T, H, Hk, D = (case[n] for n in ('batch', 'length', 'heads', 'kv_heads', 'dim'))
    if kind == 'norm':
        size, n = (2 if case['dtype'] == 'bf16' else 4), B * T * (H + Hk) * D
        return dict(bytes=4 * n * size + 4 * T * D, flops=24 * n)
    if kind == 'append':
        size = 2 if case['dtype'] == 'bf16' else 4
        rows = B * T * D
        return dict(bytes=size * rows * (2 * H + 4 * Hk) + 4 * T * D, flops=8 * rows * (H + Hk))
    if kind == 'attend':
        lengths = _lengths(case) if case['ragged'] else [T] * B
        pairs = H * sum(_pairs(n, case['window'], case['sinks']) for n in lengths)
        n = B * T * D * 2
        if case['grad']:
            return dict(bytes=n * (4 * H + 4 * Hk), flops=14 * D * pairs)
        return dict(bytes=n * (2 * H + 2 * Hk), flops=4 * D * pairs)
    keys, pairs = _visible(case)
    return dict(bytes=2 * D * (2 * B * T * H + 2 * keys * Hk), flops=4 * D * H * pairs)


# --- the same results in 64 bits ---


def exact(case, seed):
    s = prepare(case, seed)
    kind = case['kind']
    if kind == 'norm':
        leaves = [t.double().requires_grad_() for t in (s['q'], s['k'], s['qw'], s['kw']) if t is not None]
        weights = leaves[2:] or [None, None]
        at = torch.arange(case['length'], device=DEV)[None].expand(case['batch'], -1)
        outs = [_norm64(x, w, s, at) for x, w in zip(leaves, weights)]
        return (*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves, (s['dq'].double(), s['dk'].double())))
    if kind == 'append':
        at = s['start'].long()[:, None] + torch.arange(case['length'], device=DEV)
        q, k = _norm64(s['q'].double(), s['qw'], s, at), _norm64(s['k'].double(), s['kw'], s, at)
        kc, vc = s['k_cache'].double(), s['v_cache'].double()
        for b, first in enumerate(_prompt_starts(case)):
            if first >= 0:
                kc[b, first:first + case['length']] = k[b]
                vc[b, first:first + case['length']] = s['v'][b].double()
        return q, kc, vc
    if kind == 'attend':
        return _attend64(s, case)
    if kind == 'decode':
        return _decode64(s, case)
    return _distill64(s, case)


def _norm64(x, w, s, at):
    u = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
    if w is not None:
        u = u * w.double()
    inside = (at >= 0) & (at < len(s['cos']))
    at = torch.where(inside, at, 0)
    turn = torch.complex(s['cos'].double(), -s['sin'].double())[at][:, :, None]
    first, second = u.chunk(2, -1)
    y = torch.view_as_real(torch.complex(first, second) * turn)
    return torch.cat([y[..., 0], y[..., 1]], -1) * inside[..., None, None]


def _attend64(s, case):
    """One head of one sequence at a time; gradients by differentiating the definition."""
    T, H, D = case['length'], case['heads'], case['dim']
    G = H // case['kv_heads']
    lengths = _lengths(case) if case['ragged'] else [T] * case['batch']
    results = [torch.zeros(s['q'].shape, dtype=F64, device=DEV)]
    if case['grad']:
        results += [torch.zeros(s[n].shape, dtype=F64, device=DEV) for n in ('q', 'k', 'v')]
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        at = torch.arange(n, device=DEV)
        age = at[:, None] - at[None, :]
        hidden = (age < 0) | ((age > case['window']) & (at >= case['sinks'])[None, :])
        for h in range(H):
            leaves = [s['q'][b, :n, h].double(), s['k'][b, :n, h // G].double(), s['v'][b, :n, h // G].double()]
            if case['grad']:
                leaves = [x.requires_grad_() for x in leaves]
            q, k, v = leaves
            o = torch.softmax((q @ k.t() / math.sqrt(D)).masked_fill(hidden, -math.inf), -1) @ v
            results[0][b, :n, h] = o.detach()
            if case['grad']:
                dq, dk, dv = torch.autograd.grad(o, leaves, s['dout'][b, :n, h].double())
                results[1][b, :n, h] = dq
                results[2][b, :n, h // G] += dk
                results[3][b, :n, h // G] += dv
    return tuple(results) if case['grad'] else results[0]


def _decode64(s, case):
    """One token of one sequence at a time, over the keys that it sees."""
    H, Hk, D = case['heads'], case['kv_heads'], case['dim']
    out = torch.zeros(s['q'].shape, dtype=F64, device=DEV)
    for b, start in enumerate(_starts(case)):
        for t in range(case['length']):
            at = start + t
            if at < 0:
                continue
            first = max(0, at - case['window'])
            keys = torch.tensor([*range(min(case['sinks'], first)), *range(first, min(at + 1, case['capacity']))],
                                device=DEV)
            k, v = s['k_cache'][b, keys].double(), s['v_cache'][b, keys].double()
            q = s['q'][b, t].double().view(Hk, H // Hk, D)
            score = torch.matmul(q, k.permute(1, 2, 0).contiguous()) / math.sqrt(D)
            out[b, t] = torch.matmul(torch.softmax(score, -1), v.transpose(0, 1).contiguous()).reshape(H, D)
    return out


def _distill64(s, case):
    """At most 2^26 logits at a time."""
    tau, V, K = case['temperature'], case['vocab'], case['entries']
    losses, grad = [], torch.zeros(s['logits'].shape, dtype=F64, device=DEV) if case['grad'] else None
    step = max(1, 2 ** 26 // V)
    for r in range(0, case['rows'], step):
        x = s['logits'][r:r + step, :V].double()
        if case['grad']:
            x.requires_grad_()
        z = x if s['softcap'] is None else s['softcap'] * torch.tanh(x / s['softcap'])
        index = s['index'][r:r + step].long()
        used = index >= 0
        some = used.any(-1, keepdim=True)
        t = torch.where(used | ~some, s['teacher'][r:r + step].double() / tau, -math.inf)
        log_p = torch.log_softmax(t, -1)
        log_q = torch.log_softmax(z / tau, -1).gather(1, index.clamp(min=0))
        terms = torch.where(used, log_p.exp() * (torch.where(used, log_p, 0) - log_q), 0)
        loss = tau ** 2 * terms.sum(-1)
        losses.append(loss.detach())
        if case['grad']:
            grad[r:r + step, :V], = torch.autograd.grad((loss * s['weight'][r:r + step].double()).sum(), x)
    losses = torch.cat(losses)
    return (losses, grad) if case['grad'] else losses
