"""Definitions, in 64 bits and numpy, of what a training step keeps: activations in 8 bits, a LogicLayer's gradients at what they stand for, and the cross
entropy of group sums."""
import numpy as np

GROUP = 128


def codes(x):
    """x: a flat array -> (codes, lowest value and step of every group of 128); NaN in both where a group is not finite"""
    x = np.asarray(x, dtype=np.float64)
    n = len(x)
    groups = -(-n // GROUP)
    out, scales = np.zeros(n, dtype=np.uint8), np.zeros((groups, 2))
    for g in range(groups):
        part = x[g * GROUP:(g + 1) * GROUP]
        low, high = part.min(), part.max()
        with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
            size = high - low
            if not np.isfinite(size * 255.0):
                scales[g] = np.nan
                continue
        if size > 0:
            out[g * GROUP:(g + 1) * GROUP] = np.rint((part - low) * 255.0 / size).astype(np.uint8)
        scales[g] = low, size / 255.0
    return out, scales


def coded(x):
    """what the codes of a flat array stand for"""
    q, scales = codes(x)
    at = np.arange(len(q)) // GROUP
    return scales[at, 0] + q * scales[at, 1]


def gates(a, b):
    """the values of the 16 gates of a and b, and their derivatives"""
    f = np.array([[(i >> 3) & 1, (i >> 2) & 1, (i >> 1) & 1, i & 1] for i in range(16)], dtype=np.float64)     # f00, f01, f10, f11
    f00, f01, f10, f11 = (f[:, k].reshape(16, *([1] * np.ndim(a))) for k in range(4))
    value = f00 * (1 - a) * (1 - b) + f01 * (1 - a) * b + f10 * a * (1 - b) + f11 * a * b
    return value, (f10 - f00) * (1 - b) + (f11 - f01) * b, (f01 - f00) * (1 - a) + (f11 - f10) * a


def softmax(z):
    e = np.exp(z - z.max(-1, keepdims=True))
    return e / e.sum(-1, keepdims=True)


def layer(x, a, b, logits, upstream):
    """x [in, batch], upstream [out, batch] -> y, gradients of x and of the logits at the coded x, and the sums of the magnitudes these are made of"""
    x, upstream, p = np.asarray(x, dtype=np.float64), np.asarray(upstream, dtype=np.float64), softmax(np.asarray(logits, dtype=np.float64))
    y = (p.T[:, :, None] * gates(x[a], x[b])[0]).sum(0)
    kept = coded(x.reshape(-1)).reshape(x.shape)
    value, da, db = gates(kept[a], kept[b])
    da, db = (p.T[:, :, None] * da).sum(0) * upstream, (p.T[:, :, None] * db).sum(0) * upstream
    gx, mx = np.zeros_like(x), np.zeros_like(x)
    for i, part in ((a, da), (b, db)):
        np.add.at(gx, i, part)
        np.add.at(mx, i, np.abs(upstream))
    gp = (value * upstream).sum(2).T
    size = np.abs(upstream).sum(1, keepdims=True)
    return y, gx, p * (gp - (p * gp).sum(1, keepdims=True)), mx, np.broadcast_to(size, p.shape)


def group_cross_entropy(x, targets, k, tau=1.0, smoothing=0.0, weight=1.0, reduction="mean", upstream=None):
    """x [rows, features] -> loss and its gradient w.r.t. x (for `upstream`, 1 if None).  In 80 bits, with the target apart from the others: 64-bit kernels
    are held to this, and 1 - p of a p near 1 has few digits."""
    x = np.asarray(x, dtype=np.longdouble)
    rows, features = x.shape
    targets = np.asarray(targets)
    scores = x.reshape(rows, k, -1).sum(2) / np.longdouble(tau)
    keep, at, row = targets >= 0, np.clip(targets, 0, k - 1), np.arange(rows)
    with np.errstate(all="ignore"):
        top = scores.max(1)
        e = np.exp(scores - top[:, None])
        of_target = e[row, at]
        e[row, at] = 0
        others = e.sum(1)
        total = others + of_target
        margin = top - scores[row, at]
        log_total = np.where(margin == 0, np.log1p(others), np.log(total))
        loss = margin + log_total
        if smoothing:
            loss = (1 - smoothing) * loss + smoothing * (log_total + (top[:, None] - scores).mean(1))
        loss = loss * weight
        grad = e / total[:, None] - np.longdouble(smoothing) / k
        grad[row, at] = np.longdouble(smoothing) - np.longdouble(smoothing) / k - others / total
        grad = grad * (weight / np.longdouble(tau))
    bad = targets >= k
    loss[bad], grad[bad] = np.nan, np.nan
    loss[~keep], grad[~keep] = 0, 0
    if reduction == "mean":
        grad = grad / max(int(keep.sum()), 1)
    up = np.ones(1) if upstream is None else np.asarray(upstream, dtype=np.longdouble).reshape(-1)
    grad = np.repeat(grad * up[:, None], features // k, axis=1)
    grad[~keep] = 0
    if reduction == "none":
        return loss, grad
    return loss.sum() / (max(int(keep.sum()), 1) if reduction == "mean" else 1), grad
