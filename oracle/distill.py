"""The distillation loss in 64 bits, from its definition, one row at a time."""
import math

import torch


def distill(logits, teacher, index, vocab, temperature=1.0, softcap=None, weight=None):
    """(loss [rows], gradient of sum weight * loss [rows, width]) of 2-D logits; a gradient of an entry that stands more
    than once adds up."""
    rows, width = logits.shape
    x = logits[:, :vocab].double()
    th = None if softcap is None else torch.tanh(x / softcap)
    z = (x if softcap is None else softcap * th) / temperature
    log_q = torch.log_softmax(z, -1)
    loss = torch.zeros(rows, dtype=torch.float64, device=logits.device)
    grad = torch.zeros(rows, width, dtype=torch.float64, device=logits.device)
    for r in range(rows):
        t = teacher[r].double() / temperature
        used = (index[r] >= 0) & (index[r] < vocab) & ~(t == -math.inf)
        if not bool(used.any()):
            continue
        log_p = torch.log_softmax(t[used], -1)
        p, i = log_p.exp(), index[r][used].long()
        terms = torch.where(p > 0, p * (log_p - log_q[r, i]), torch.zeros_like(p))
        loss[r] = temperature ** 2 * terms.sum()
        d = log_q[r].exp().index_add(0, i, -p) * temperature
        if softcap is not None:
            d = d * (1 - th[r] ** 2)
        grad[r, :vocab] = d * (1.0 if weight is None else weight[r].double())
    return loss, grad
