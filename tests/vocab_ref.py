"""The operators on a model's vocabulary at 64 bits, with bounds for what 32-bit arithmetic and one rounding at the end may lose."""
import math

import numpy as np
import torch

F64 = torch.float64


def embedding(idx, table, scale):
    idx, w = idx.reshape(-1).long().cpu(), table.detach().to(F64).cpu()
    out = torch.zeros(idx.numel(), w.shape[1], dtype=F64)
    for n, i in enumerate(idx.tolist()):
        if 0 <= i < w.shape[0]:
            out[n] = w[i] * scale
    return out


def embedding_grad(idx, dout, vocab, scale, pad=None):
    """(gradient, bound of the error before the last rounding): a sum of m numbers in 32 bits is off by m 2^-24 times the sum of their sizes, the factor by 2^-24 more."""
    idx, dy = idx.reshape(-1).long().cpu(), dout.detach().to(F64).cpu().reshape(idx.numel(), -1)
    live = (idx >= 0) & (idx < vocab)
    if pad is not None:
        live &= idx != pad
    grad, size = torch.zeros(vocab, dy.shape[1], dtype=F64), torch.zeros(vocab, dy.shape[1], dtype=F64)
    grad.index_add_(0, idx[live], dy[live])
    size.index_add_(0, idx[live], dy[live].abs())
    count = torch.zeros(vocab, dtype=F64).index_add_(0, idx[live], torch.ones(int(live.sum()), dtype=F64))
    return grad * scale, size * abs(scale) * (count + 2)[:, None] * 2.0 ** -24


def rounding(want, dtype):
    """Half a step of the type, or of its smallest numbers."""
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return want.abs() * (torch.finfo(dtype).eps / 2) * (1 + 2.0 ** -10) + tiny


def distillation(z, t, idx, temperature, reduction, up=None):
    """(loss, its bound, gradient, its bound before the last rounding).

    2^x of x = (z - max) log2(e) / T comes with a relative error of 2^-22 from the exponential and of ln 2 |x| 4 2^-24 from x (difference, factor, product and the
    factor's own rounding); a sum of V of them in 512 threads adds at most V / 512 + 24 roundings of 2^-24, and its terms' errors weighted with q, under which
    |x| is on average at most log2(V) + 2."""
    z, t, idx = z.detach().to(F64).cpu(), t.detach().to(F64).cpu(), idx.cpu()
    N, V = z.shape
    there = (idx >= 0) & (idx < V) & (t != -math.inf)
    has = there.any(1)
    j = idx.long().clamp(0, V - 1)
    log_q = torch.log_softmax(z / temperature, 1)
    a = torch.where(there, t / temperature, torch.full_like(t, -math.inf))
    a = torch.where(has[:, None], a, torch.zeros_like(a))
    log_p = torch.log_softmax(a, 1)
    p = torch.where(there, log_p.exp(), torch.zeros_like(log_p))
    lq = log_q.gather(1, j)
    used = p > 0
    terms = torch.where(used, p * (torch.where(used, log_p, torch.zeros_like(p)) - torch.where(used, lq, torch.zeros_like(p))), torch.zeros_like(p))
    rows = temperature ** 2 * terms.sum(1)
    u = 2.0 ** -22
    x = ((z - z.amax(1, keepdim=True)) / temperature / math.log(2)).abs()
    xt = torch.where(used, ((a - a.amax(1, keepdim=True)) / temperature / math.log(2)).abs(), torch.zeros_like(a))
    rel_s = (math.log2(V) + 3 + (V / 512 + 24) / 4) * u
    rel_q = x * u + u + rel_s
    rel_p = xt * u + u + (math.log2(p.shape[1]) + 3 + (p.shape[1] / 512 + 24) / 4) * u
    share = 1.0 / max(int(has.sum()), 1) if reduction == "mean" else 1.0
    g = torch.ones(N, dtype=F64) if up is None else up.detach().to(F64).cpu().expand(N)
    w = (temperature * share * g * has)[:, None]
    q = log_q.exp()
    grad = (q - torch.zeros_like(q).scatter_add_(1, j, p)) * w
    bound = (torch.where(q > 0, q * rel_q, torch.zeros_like(q)) + torch.zeros_like(q).scatter_add_(1, j, p * rel_p)) * w.abs() + grad.abs() * 4 * 2.0 ** -24
    # a term of the loss: p's own error, and absolute errors of both logarithms (x and the logarithm of the sum)
    finite = torch.where(used & torch.isfinite(terms), (log_p - lq).abs(), torch.zeros_like(p))
    near = torch.where(torch.isfinite(x.gather(1, j)), x.gather(1, j), torch.zeros_like(p))
    lost = temperature ** 2 * (p * (rel_p * finite + rel_p + near * u + rel_s + 8 * u * (1 + finite))).sum(1)
    # (by definition, whatever the student's logits are there)
    grad, bound = (torch.where(has[:, None], v, torch.zeros_like(v)) for v in (grad, bound))
    if reduction == "none":
        return rows, lost + rows.abs() * 2.0 ** -20, grad, bound
    return rows.sum() * share, lost.sum() * share + rows.abs().sum() * share * 2.0 ** -20, grad, bound


def sample(z, u, tau, k, p, low):
    """(tokens, log probabilities), row by row."""
    z = z.detach().to(F64).cpu().numpy()
    n, V = z.shape

    def column(x, kind):
        return (x.detach().cpu().to(F64).numpy() if torch.is_tensor(x) else np.full(n, float(x))).astype(kind)
    u, tau, k, p, low = column(u, float), column(tau, float), column(k, int), column(p, float), column(low, float)
    tokens, logs = [], []
    for r in range(n):
        x = np.where(np.isnan(z[r]), -np.inf, z[r])
        top = x.max()
        if top == -np.inf:
            tokens.append(-1)
            logs.append(-math.inf)
            continue
        if not tau[r] > 0:
            tokens.append(int(np.argmax(x)))
            logs.append(0.0)
            continue
        with np.errstate(invalid="ignore"):
            y = np.where(x == top, 0.0, np.where(x == -np.inf, -np.inf, (x - top) / tau[r]))
        e = np.exp(y)
        order = np.argsort(-x, kind="stable")
        if k[r] > 0:
            order = order[:k[r]]
        if p[r] < 1:
            c = np.cumsum(e[order])
            stay = (c - e[order]) < p[r] * c[-1]
            stay[0] = True
            order = order[stay]
        stay = np.sort(order[e[order] >= min(low[r], 1.0)])
        stay = stay[e[stay] > 0]
        c = np.cumsum(e[stay])
        at = min(int(np.searchsorted(c, max(u[r], 0.0) * c[-1], side="right")), len(stay) - 1)
        tokens.append(int(stay[at]))
        logs.append(y[stay[at]] - math.log(c[-1]))
    return torch.tensor(tokens), torch.tensor(logs, dtype=F64)
