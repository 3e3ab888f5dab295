"""The distillation loss, its gradient and the selection of top logits in 64 bits, from their definitions, position by position
over [positions, classes]; with the error bounds of an fp32 evaluation."""
import math

import torch


def loss_and_gradient(z, values, indices, lse, T, weight=1.0):
    """z [P, V], values / indices [P, k], lse [P] or None (any float type): (loss [P], gradient of the sum [P, V], counted [P],
    error bound of the loss [P], error bound of the gradient [P, V] before it is rounded to its type)."""
    z, values = z.double(), values.double()
    P, V = z.shape
    loss, grad = torch.zeros(P, dtype=torch.float64), torch.zeros(P, V, dtype=torch.float64)
    lerr, gerr = torch.zeros(P, dtype=torch.float64), torch.zeros(P, V, dtype=torch.float64)
    counted = torch.zeros(P, dtype=torch.bool)
    for i in range(P):
        valid = (indices[i] >= 0) & (indices[i] < V)
        if not bool(valid.any()):
            continue
        counted[i] = True
        at, t = indices[i][valid].long(), values[i][valid] / T
        logq = torch.log_softmax(z[i] / T, 0)
        if lse is None:
            m = t.max()
            p = torch.softmax(t, 0) if m > -math.inf else torch.zeros_like(t)
        else:
            p = torch.exp(t - lse[i].double())
        kept = torch.zeros(V, dtype=torch.bool)
        kept[at] = True
        r = 1.0 - float(p.sum()) if lse is not None else 0.0
        if r <= 2.0 ** -20 or bool(kept.all()):
            r = 0.0
        pc = torch.zeros(V, dtype=torch.float64).index_add_(0, at, p)
        on = p > 0
        row = float((p[on] * (p[on].log() - logq[at][on])).sum())
        q = logq.exp()
        M = float(p.sum()) + r
        g = M * q - pc
        # An fp32 evaluation: the arguments of exp and log carry a handful of roundings, each 2^-24 of a magnitude of at most
        # a few times max |logit| / T (in base 2: 1.45 times that); exp2 and log2 are good to 2^-23; sums over V terms of one sign
        # are pairwise or short.  u bounds what that does to one exp or log, relative to exp and absolute to log.
        big = max([float(x[torch.isfinite(x)].abs().max()) if bool(torch.isfinite(x).any()) else 0.0 for x in (z[i] / T, t)])
        u = 2.0 ** -21 * (8 + 3 * big)
        slope = 0.0
        ge = M * q + pc
        if r > 0:
            outside = ~kept
            log_rest = float(torch.logsumexp(logq[outside], 0))
            row += r * (math.log(r) - log_rest)
            share = torch.where(outside, torch.exp(logq - log_rest), torch.zeros((), dtype=torch.float64))
            g = g - r * share
            ge = ge + (1 + r) * share            # r itself is off by u
            slope = abs(math.log(r) - log_rest) + 1
        loss[i] = T * T * weight * row
        grad[i] = T * weight * g
        lerr[i] = T * T * abs(weight) * u * (3 + slope)
        gerr[i] = T * abs(weight) * u * ge + 2.0 ** -126
    return loss, grad, counted, lerr, gerr


def top(z, k):
    """Values and classes of the k greatest of each row of z [P, V]: NaN first, then by value, ties by class."""
    order = []
    for row in z.double().tolist():
        key = [(0 if math.isnan(v) else 1, 0.0 if math.isnan(v) else -v, c) for c, v in enumerate(row)]
        order.append([e[2] for e in sorted(key)[:k]])
    idx = torch.tensor(order, dtype=torch.int64)
    return torch.gather(z, 1, idx), idx.to(torch.int32)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def cancellation_bounds(z, values, indices, lse, T):
    """Error bounds of an fp32 evaluation that lets nothing cancel, of the loss [P] and of the gradient [P, V] before it is rounded to its
    type, for positions without repeated entries.

    Every probability is known to E = 2^-24 (12 B + n + 16), relative, B = max(|z|, |t|) / T + |lse|: 1 / T, the difference of two
    logits, log2(e) / T and the products round the argument of exp2 (four roundings of at most 2 B; three of |t| / T + |lse| for the teacher), exp2,
    quotients and reciprocals are good to 2^-23, and a sum has at most n = min(V, 128) additions one after the other, or 256 of
    planes with more.  The loss is sum D(p, q) + D(r, R), D = p log(p / q) - p + q: dD/dp = log(p / q), dD/dq = 1 - p / q, and r = 1 - sum p is off by
    E of 1.  Where r counts as 0, R (renormalised) and mass - 1 (a given lse) are added as they are."""
    z, values = z.double(), values.double()
    loss, grad, counted, _, _ = loss_and_gradient(z, values, indices, lse, T)
    lerr, gerr = torch.zeros_like(loss), torch.zeros_like(grad)
    V = z.shape[1]
    for i in torch.nonzero(counted).flatten().tolist():
        valid = (indices[i] >= 0) & (indices[i] < V)
        at, t = indices[i][valid].long(), values[i][valid] / T
        assert at.unique().numel() == at.numel()
        logq = torch.log_softmax(z[i] / T, 0)
        logp = torch.log_softmax(t, 0) if lse is None else t - lse[i].double()
        E = 2.0 ** -24 * (12 * (max(float(z[i].abs().max()) / T, float(t.abs().max())) + (0.0 if lse is None else abs(float(lse[i])))) + (256 if V > 128 else V) + 16)
        p, q = logp.exp(), logq.exp()
        parts = float((p * (logp - logq[at]).abs() + (q[at] - p).abs()).sum())
        outside = torch.ones(V, dtype=torch.bool)
        outside[at] = False
        R, r = float(q[outside].sum()), 0.0 if lse is None else 1.0 - float(p.sum())
        ge = q.clone()
        ge[at] += p
        if r > 2.0 ** -20 and R > 0:
            parts += abs(math.log(r / R)) + abs(R - r)
            ge[outside] += q[outside] * (r + 1) / R
        else:
            parts += R + (0.0 if lse is None else 1.0)
        lerr[i] = T * T * E * parts + 2.0 ** -21 * abs(float(loss[i]))
        gerr[i] = T * E * ge + 2.0 ** -126
    return lerr, gerr
