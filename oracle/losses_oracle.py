"""The losses on scores and gate logits row by row in 64-bit numpy, from their definitions, with the magnitudes that bounds on rounding are made of."""
import numpy as np


def top_logits(z, k, temperature):
    """values [N, k], columns [N, k], logsumexp [N] of z [N, V]; NaN first, then by value, of equal ones the lowest column"""
    values, columns, lse = [], [], []
    for row in np.asarray(z, np.float64):
        order = sorted(range(len(row)), key=lambda c: (not np.isnan(row[c]), 0.0 if np.isnan(row[c]) else -row[c], c))[:k]
        values.append(row[order])
        columns.append(order)
        if np.isnan(row).any():
            lse.append(np.nan)
        else:
            m = row.max()
            lse.append(m if np.isinf(m) else m / temperature + np.log(np.exp((row - m) / temperature).sum()))
    return np.array(values), np.array(columns), np.array(lse)


def distillation(z, values, columns, lse=None, temperature=1.0, mask=None, weight=1.0, reduction="mean", upstream=None):
    """-> (loss, gradient [N, V], loss_size, gradient_size): the sizes are sums of the magnitudes of the terms that cancel in each value"""
    z, values = np.asarray(z, np.float64), np.asarray(values, np.float64)
    n, cols = z.shape
    kept = np.ones(n, bool) if mask is None else np.asarray(mask, bool)
    losses, grad, loss_size, grad_size = np.zeros(n), np.zeros((n, cols)), np.zeros(n), np.zeros((n, cols))
    count = int(kept.sum())
    for r in range(n):
        cs = np.asarray(columns[r])
        scale = weight * temperature * {"mean": 1.0 / max(count, 1)}.get(reduction, 1.0)
        if not kept[r] or (cs < 0).all():
            continue
        if (cs >= cols).any():
            losses[r], grad[r] = np.nan, np.nan
            continue
        with np.errstate(all="ignore"):
            log_q = (z[r] - z[r].max()) / temperature                 # (z / temperature first is off by half a step of itself: 2^-9 at 3e13)
            log_q = log_q - np.log(np.exp(log_q).sum())
        entries = [(values[r, j] / temperature, cs[j]) for j in range(len(cs)) if cs[j] >= 0]
        t = np.array([e[0] for e in entries])
        if lse is None:
            if np.isinf(t.max()) and t.max() < 0:
                continue
            p = np.exp(t - t.max()) / np.exp(t - t.max()).sum()
        else:
            p = np.exp(t - lse[r])
        listed = np.zeros(cols, bool)
        target = np.zeros(cols)
        loss = size = 0.0
        for pj, tj, (_, c) in zip(p, t, entries):
            listed[c] = True
            target[c] += pj
            if pj > 0:
                loss += pj * (np.log(pj) - log_q[c])
                size += pj * (abs(np.log(pj)) + abs(log_q[c]) + 1)
        rest = 0.0 if lse is None or listed.all() else max(0.0, 1.0 - p.sum())
        mass = p.sum() + rest
        q = np.exp(log_q)
        g, gs = mass * q - target, mass * q + target
        if rest > 0:
            others = log_q[~listed]
            m = others.max()
            log_rest = m + np.log(np.exp(others - m).sum()) if m > -np.inf else -np.inf
            loss += rest * (np.log(rest) - log_rest)
            size += rest * (abs(np.log(rest)) + abs(log_rest) + 1)
            if m > -np.inf:
                share = np.where(listed, 0.0, np.exp(np.where(listed, -np.inf, log_q - log_rest)))
                g, gs = g - rest * share, gs + rest * share
            else:
                g[~listed] = 0
        up = 1.0 if upstream is None else float(np.asarray(upstream).reshape(-1)[r if np.ndim(upstream) else 0])
        losses[r], loss_size[r] = loss * scale * temperature, size * abs(scale) * temperature
        grad[r], grad_size[r] = g * scale * up, gs * abs(scale * up)
    if reduction == "none":
        return losses, grad, loss_size, grad_size
    return losses.sum(), grad, loss_size.sum(), grad_size


def balance(z, k, mask=None, weight=1.0):
    """-> (loss, counts [E], gradient [N, E], gradient_size)"""
    z = np.asarray(z, np.float64)
    n, experts = z.shape
    kept = [r for r in range(n) if (mask is None or mask[r]) and not (z[r] == -np.inf).all()]
    counts, sums, probs = np.zeros(experts, np.int64), np.zeros(experts), {}
    for r in kept:
        p = np.exp(z[r] - z[r].max())
        probs[r] = p / p.sum()
        sums += probs[r]
        for c in sorted(range(experts), key=lambda c: (-z[r, c], c))[:k]:
            counts[c] += z[r, c] > -np.inf
    w = weight * experts * counts / (k * max(len(kept), 1) ** 2)
    grad, size = np.zeros(z.shape), np.zeros(z.shape)
    for r in kept:
        mean = (w * probs[r]).sum()
        grad[r], size[r] = probs[r] * (w - mean), probs[r] * (np.abs(w) + np.abs(w * probs[r]).sum())
    return (w * sums).sum(), counts, grad, size
