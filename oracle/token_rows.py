"""CPU oracle of the operators over rows of logits -- TEST INFRASTRUCTURE ONLY.

Float64 torch on the CPU, written from the definitions:
  * ``logp``: log softmax(x / temperature)[label], 0 where a row does not count;
  * ``dlogits``: coef / temperature (onehot(label) - softmax(x / temperature));
  * ``policy``: loss and coef = d loss / d logp of the clipped policy loss;
  * ``preference``: loss, sequence sums and coef of the preference loss.

Pinned by tests/test_oracle_operators.py: float64 autograd of the losses'
expressions, central differences, closed forms and planted mistakes.
"""

import torch

IGNORE = -100


def counted(labels, mask=None):
    keep = labels != IGNORE
    return keep if mask is None else keep & (mask != 0)


def logp(x, labels, temperature=1.0, keep=None):
    """[rows] of x [rows, V]."""
    x = x.double() / temperature
    keep = counted(labels) if keep is None else keep
    out = torch.zeros(labels.shape, dtype=torch.float64)
    for r in keep.nonzero().flatten().tolist():
        lab = int(labels[r])
        if not 0 <= lab < x.shape[1]:
            out[r] = float("nan")
            continue
        m = x[r].max()
        if m == -float("inf"):
            out[r] = float("nan")
            continue
        out[r] = (x[r, lab] - m) - torch.log(torch.exp(x[r] - m).sum())
    return out


def softmax(x, temperature=1.0):
    x = x.double() / temperature
    e = torch.exp(x - x.max(1, keepdim=True).values)
    return e / e.sum(1, keepdim=True)


def dlogits(x, labels, coef, temperature=1.0, keep=None):
    keep = counted(labels) if keep is None else keep
    out = torch.zeros(x.shape, dtype=torch.float64)
    rows = keep.nonzero().flatten()
    if rows.numel():
        p = -softmax(x[rows], temperature)
        lab = labels[rows]
        bad = (lab < 0) | (lab >= x.shape[1])
        p[torch.arange(rows.numel()), lab.clamp(0, x.shape[1] - 1)] += 1.0
        p[bad] = float("nan")
        out[rows] = p * (coef.double()[rows] / temperature)[:, None]
    return out


def policy(lp, labels, old, adv, ref=None, mask=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0,
           denom=None):
    """(loss, coef) from logp lp, all [rows] float64."""
    keep = counted(labels, mask)
    w = keep.double() if mask is None or mask.dtype != torch.float32 else \
        torch.where(keep, mask.double(), 0.0)
    D = float(denom) if denom is not None else float(w.sum())
    coef = torch.zeros_like(lp)
    if D == 0.0:
        return torch.zeros((), dtype=torch.float64), coef
    total = torch.zeros((), dtype=torch.float64)
    i = keep.nonzero().flatten()
    r = torch.exp(lp[i] - old.double()[i])
    a = adv.double()[i]
    low, high = 1 - clip_low, 1 + clip_high
    cut = torch.clamp(r, low, high)
    term = -torch.minimum(r * a, cut * a)
    held = torch.where(a >= 0, r > high, r < low)
    g = torch.where(held, torch.zeros_like(r), -r * a)
    if kl_coef:
        d = ref.double()[i] - lp[i]
        term = term + kl_coef * (torch.expm1(d) - d)
        g = g - kl_coef * torch.expm1(d)
    total = (w[i] * term).sum() / D
    coef[i] = w[i] * g / D
    return total, coef


def preference(lp, labels, seqs, ref=None, beta=0.1, eps=0.0, average=False):
    """(loss, seq [2 N], coef [rows]); seqs: the rows of each sequence."""
    n = len(seqs) // 2
    count = torch.tensor([max(int((labels[s] != IGNORE).sum()), 1) for s in seqs],
                         dtype=torch.float64)
    share = 1.0 / count if average else torch.ones_like(count)
    seq = torch.stack([lp[s].sum() for s in seqs]) * share
    h = beta * (seq - (ref.double() if ref is not None else 0.0))
    d = h[:n] - h[n:]
    sp = torch.nn.functional.softplus
    loss = ((1 - eps) * sp(-d) + eps * sp(d)).mean()
    g = beta / n * (eps * torch.sigmoid(d) - (1 - eps) * torch.sigmoid(-d))
    coef = torch.zeros_like(lp)
    for i in range(n):
        coef[seqs[i]] = g[i] * share[i]
        coef[seqs[n + i]] = -g[i] * share[n + i]
    return loss, seq, coef
