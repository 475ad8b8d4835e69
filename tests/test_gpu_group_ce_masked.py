"""Cross entropy of group sums on the GPU where classes are masked with finite values, against its definition in 64 bits (oracle/keep_oracle.py).

Bounds, per class and relative to the row's highest score alone.  With d = log2(e) times a class's distance from the highest, the argument of its 32-bit exponential is
off by at most (2 d + 2 `held`) 2^-24 powers of two: the roundings of its score and of the difference from the highest.  `held` is the distance from the highest up to
which a kernel may hold scores in 32 bits relative to another value: 128 where it has a row's scores in 32 bits, else 0.  The exponential is off by 2 steps more, and
what becomes of it -- the factor, the product, the rounding -- by 6: (ln 2 (2 d + 2 held) + 8) 2^-24 of itself in all, and the instruction for 2^x gives 0 for results
under 2^-126.  A total is off by its classes' parts, a gradient by its class's and the total's.  A loss is the margin, off by the two scores that it is a difference of,
and the logarithm of the total, or of 1 + the others where the target is the highest.  2^-53 for float64, whose scores are off by the additions of their features too.
Half a step of the type on top."""
import math
import threading

import numpy as np
import pytest
import torch

import convlogic_amd as C
from oracle import keep_oracle as K
from tests.gpu_util import DEV

pytestmark = pytest.mark.gpu

LN2 = 0.6932


def host(t):
    return t.detach().double().cpu().numpy()


def masked(rows, k, group, dtype, value, seed=0):
    """features with masked classes -- by the row: none, the first one, the first half and every third one, all but one -- and which ones are not"""
    g = torch.Generator().manual_seed(seed)
    x = torch.rand(rows, k, group, generator=g, dtype=torch.float64) + torch.randn(rows, k, 1, generator=g, dtype=torch.float64) * (3.0 / group)
    row, c = torch.arange(rows)[:, None] % 4, torch.arange(k)[None, :]
    free = torch.ones(rows, k, dtype=torch.bool)
    free &= ~((row == 1) & (c == 0))
    free &= ~((row == 2) & ((c < k // 2) | (c % 3 == 0)) & (c != k - 1))
    free &= ~((row == 3) & (c != 7 * torch.arange(rows)[:, None] % k))
    x = torch.where(free[:, :, None], x, value)
    return x.view(rows, k * group).to(dtype), free


def targets(free, seed=0):
    """a class that is not masked"""
    score = torch.rand(free.shape, generator=torch.Generator().manual_seed(seed + 1))
    return torch.where(free, score, -1.0).argmax(1)


def held_of(x, k, layout):
    """where scores are in 32 bits: rows of up to 64 features to a class, by a workgroup each, but for the few short ones"""
    rows, features = x.shape
    in_lds = layout == "rows" and x.dtype != torch.float64 and features <= 64 * k and k * 4 <= 144 << 10
    return 128 if in_lds and (rows > 64 or features * x.element_size() <= 64 << 10) and not (rows <= 128 and features <= 64) else 0


def check(x, t, k, layout, tau, smoothing=0.0, reduction="none", upstream=None):
    rows, group, held = x.shape[0], x.shape[1] // k, held_of(x, k, layout)
    leaf = (x.to(DEV) if layout == "rows" else x.to(DEV).t().contiguous().t()).requires_grad_(True)
    loss = C.group_cross_entropy(leaf, t.to(DEV), k, tau=tau, label_smoothing=smoothing, reduction=reduction)
    up = torch.rand(rows, dtype=loss.dtype, generator=torch.Generator().manual_seed(5)) if reduction == "none" else upstream
    want, want_grad = K.group_cross_entropy(host(x), t.numpy(), k, tau, smoothing, 1.0, reduction, None if up is None else up.numpy())
    want, want_grad = np.asarray(want, dtype=np.float64), np.asarray(want_grad, dtype=np.float64)
    double = x.dtype == torch.float64
    unit, at = 2.0 ** -53 if double else 2.0 ** -24, np.arange(rows)
    with np.errstate(all="ignore"):
        parts = host(x).reshape(rows, k, group)
        scores = parts.sum(2) / tau
        top = scores.max(1, keepdims=True)
        d = (top - scores) * 1.442696
        off = LN2 * (2 * d + 2 * held) + 8
        if double:                                                    # (as many roundings as additions, and those of the scale, of two classes)
            sums = np.abs(parts).sum(2) / tau * (group + 8)
            off = off + sums + sums[at, scores.argmax(1)][:, None]
        p = np.exp(scores - top)
        p = p / p.sum(1, keepdims=True)
        each = np.where(p > 0, p * off * unit, 0.0) + 2.0 ** -126
        total = each.sum(1)
        target = t.numpy()
        but = np.where(np.arange(k) == target[:, None], 0.0, each).sum(1)      # (not total less the target's: a loss near 0 has a bound near 0)
        d_t = d[at, target]
        margin = np.where(held > 0, LN2 * (2 * held + d_t), 2.0 ** -20 * (1 + d_t)) * unit
        if double:
            margin = (LN2 * d_t * 2 + sums[at, target] + sums[at, scores.argmax(1)] + 8) * unit
        bound = np.where((d_t == 0) & (smoothing == 0), but, total + margin)
        if smoothing:
            bound = bound + smoothing * (LN2 * held * unit + LN2 * d.mean(1) * (k + 8) * 2.0 ** -53)
    half = torch.finfo(loss.dtype).eps / 2
    if reduction == "mean":
        bound = bound.mean()
    error = np.abs(host(loss) - want)
    assert (error <= bound + 4 * half * np.abs(want)).all(), (host(loss), want, error - bound)
    got, = torch.autograd.grad(loss, leaf, None if up is None else up.to(DEV))
    size = np.ones((rows, 1)) / tau / (rows if reduction == "mean" else 1) * (1.0 if up is None else np.abs(up.numpy().reshape(-1, 1)))
    limit = each + p * total[:, None] + smoothing / k * 8 * unit
    limit[at, target] = but + (1 - p[at, target]).clip(0) * total + smoothing * 8 * unit
    eps, tiny = torch.finfo(x.dtype).eps / 2, torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    error = np.abs(host(got) - want_grad)
    limit = np.repeat(size * limit, group, 1) + (eps * 1.001) * np.abs(want_grad) + tiny
    assert (error <= limit).all(), (error - limit).max()


VALUES = [-1e4, -65504.0, -1e9, "lowest"]


def cases(dtype):
    for value in VALUES:
        if value == "lowest":
            yield torch.finfo(dtype).min
        elif value >= torch.finfo(dtype).min:
            yield value


# rows in pieces of their classes; samples in columns, one or several to a lane, classes whole or in slices
PIECES = [("rows", 40, 2100, 8), ("rows", 3, 40000, 1), ("rows", 7, 5001, 5), ("columns", 33, 10, 4), ("columns", 5, 700, 1), ("columns", 300, 64, 2), ("columns", 1030, 1500, 2),
          ("columns", 64, 10, 2048), ("columns", 257, 5, 513)]


@pytest.mark.parametrize("layout,rows,k,group", PIECES + [("rows", 130, 37000, 2), ("columns", 12, 30000, 1)])
def test_classes_in_pieces(layout, rows, k, group):
    for value in cases(torch.float32):
        x, free = masked(rows, k, group, torch.float32, value)
        check(x, targets(free), k, layout, 0.3 * group ** 0.5)


@pytest.mark.parametrize("dtype,layout,rows,k,group", [(d, *size) for d in (torch.float64, torch.bfloat16, torch.float16) for size in PIECES + [("rows", 40, 4200, 8)]
                                                       if d == torch.float64 or size[0] == "columns" or size[2] * size[3] > 32768])      # (shorter rows go whole)
def test_classes_in_pieces_of_other_types(dtype, layout, rows, k, group):
    for value in cases(dtype):
        x, free = masked(rows, k, group, dtype, value)
        check(x, targets(free), k, layout, 0.3 * group ** 0.5)


@pytest.mark.parametrize("layout,rows,k,group", PIECES)
def test_classes_in_pieces_with_smoothing_and_masked_targets(layout, rows, k, group):
    for value in cases(torch.float32):
        x, free = masked(rows, k, group, torch.float32, value)
        t = targets(free)
        tau = 0.3 * group ** 0.5 + 0.7                                # (losses stay in float32's range: the smoothing's part of the masks is their mean)
        check(x, t, k, layout, tau * group, smoothing=0.1)
        check(x, t, k, layout, tau, reduction="mean", upstream=torch.tensor(3.0))
        if value >= -1e9:
            check(x, torch.where(torch.arange(rows) % 8 >= 4, t, 0), k, layout, tau)


# a workgroup for a row: scores in 32 bits of groups up to 64 features, else in 64
WHOLE = [(129, 10, 1), (200, 1000, 1), (1100, 300, 4), (130, 12, 5), (70, 300, 64), (65, 2000, 16), (150, 9, 100), (130, 30000, 1)]


@pytest.mark.parametrize("rows,k,group", WHOLE)
def test_whole_rows(rows, k, group):
    for value in cases(torch.float32):
        x, free = masked(rows, k, group, torch.float32, value)
        check(x, targets(free), k, "rows", 0.3 * group ** 0.5)


@pytest.mark.parametrize("dtype", [torch.float64, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k,group", WHOLE[:-1] + [(40, 2100, 8), (7, 5001, 5)])
def test_whole_rows_of_other_types(rows, k, group, dtype):
    for value in cases(dtype):
        x, free = masked(rows, k, group, dtype, value)
        check(x, targets(free), k, "rows", 0.3 * group ** 0.5)


@pytest.mark.parametrize("rows,k,group", WHOLE)
def test_whole_rows_with_masked_targets(rows, k, group):
    for value in cases(torch.float32):
        x, free = masked(rows, k, group, torch.float32, value)
        t = targets(free)
        check(x, t, k, "rows", group ** 0.5, reduction="mean", upstream=torch.tensor(3.0))
        if value >= -1e9:
            check(x, torch.where(torch.arange(rows) % 8 >= 4, t, 0), k, "rows", group ** 0.5)


@pytest.mark.parametrize("level", [-1e6, 1e4, 1e9, 1e30])
@pytest.mark.parametrize("first", [0.0, -math.inf])
def test_whole_rows_far_from_zero_and_from_their_first_class(first, level):
    # (steps of 32 bits at these levels: the scores differ by them, and by hundreds)
    step = abs(level) * 2.0 ** -20 if abs(level) > 1e5 else 0.25
    x = (level + step * torch.randint(0, 8, (200, 50), generator=torch.Generator().manual_seed(0)).double()).float()
    x[:, 0] = first if first else x[:, 1]
    t = torch.randint(1, 50, (200,), generator=torch.Generator().manual_seed(1))
    leaf = x.to(DEV).requires_grad_(True)
    tau = step / 0.75
    loss = C.group_cross_entropy(leaf, t.to(DEV), 50, tau=tau, reduction="none")
    grad, = torch.autograd.grad(loss.sum(), leaf)
    want, want_grad = K.group_cross_entropy(host(x), t.numpy(), 50, tau, 0.0, 1.0, "none")
    # distances up to 8 powers of two from the highest
    bound = (LN2 * (2 * 8 + 2 * 128) + 8) * 2.0 ** -24
    assert (np.abs(host(loss) - want) <= bound * 3 * (1 + want)).all() and (np.abs(host(grad) * tau - want_grad * tau) <= 3 * bound).all()


@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("layout,rows,k", [("rows", 200, 50), ("rows", 20, 50), ("rows", 3, 40000), ("columns", 20, 50), ("columns", 1030, 1500)])
def test_rows_of_the_lowest_or_highest_value(layout, rows, k, sign):
    # the classes that are not -inf are alike: each has the same probability
    x = torch.full((rows, k), sign * torch.finfo(torch.float32).max)
    x[:, 0] = -math.inf
    t = torch.full((rows,), k - 1)
    leaf = (x.to(DEV) if layout == "rows" else x.to(DEV).t().contiguous().t()).requires_grad_(True)
    loss = C.group_cross_entropy(leaf, t.to(DEV), k, reduction="none")
    grad, = torch.autograd.grad(loss.sum(), leaf)
    want = torch.full((rows, k), 1 / (k - 1), dtype=torch.float64)
    want[:, 0], want[:, -1] = 0, 1 / (k - 1) - 1
    assert np.abs(host(loss) - math.log(k - 1)).max() <= 4 * 2.0 ** -24 * math.log(k - 1)
    assert (np.abs(host(grad) - want.numpy()) <= 8 * 2.0 ** -24 * np.abs(want.numpy())).all()

@pytest.mark.parametrize("rows,k,group", WHOLE)
def test_whole_rows_with_smoothing(rows, k, group):
    for value in cases(torch.float32):
        x, free = masked(rows, k, group, torch.float32, value)
        check(x, targets(free), k, "rows", (0.3 * group ** 0.5 + 0.7) * group, smoothing=0.1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,k,group", WHOLE)
def test_whole_rows_with_targets_of_the_lowest_value(rows, k, group, dtype):
    # the loss of a target at the lowest value, in float32's range after tau; in powers of two its score is beyond it
    x, free = masked(rows, k, group, dtype, torch.finfo(dtype).min)
    check(x, torch.where(torch.arange(rows) % 8 >= 4, targets(free), 0), k, "rows", 1.2 * group)


# 2^31 - 1 features, as many as a row may have
@pytest.mark.parametrize("layout,rows", [("rows", 1), ("columns", 2)])
def test_as_many_classes_as_there_may_be(layout, rows):
    k = (1 << 31) - 1
    x = torch.zeros((rows, k) if layout == "rows" else (k, rows), dtype=torch.bfloat16, device=DEV)
    leaf = (x if layout == "rows" else x.t())
    leaf[-1, -1] = 20.0
    leaf.requires_grad_(True)
    t = torch.full((rows,), k - 1, device=DEV)
    loss = C.group_cross_entropy(leaf, t, k, reduction="none")
    grad, = torch.autograd.grad(loss.sum(), leaf)
    others = (k - 1) * math.exp(-20.0)
    step = (LN2 * 2 * 29 + 8) * 2.0 ** -24
    assert abs(float(loss[-1].detach()) - math.log1p(others)) <= step * (1 + math.log1p(others))
    assert abs(float(grad[-1, -1]) + others / (1 + others)) <= 2.0 ** -8
    each = math.exp(-20.0) / (1 + others)
    assert abs(float(grad[-1, 0]) - each) <= (2.0 ** -8 + 2 * step) * each
    row = grad[-1]
    assert int((row != row[0]).sum()) == 1                            # (all are written)
    if rows > 1:
        assert abs(float(loss[0].detach()) - math.log(k)) <= step * math.log(k) and int((grad[0] != grad[0, 0]).sum()) == 1


def test_a_class_of_as_many_features_as_there_may_be():
    features = (1 << 31) - 1
    x = torch.zeros(1, features, dtype=torch.bfloat16, device=DEV).requires_grad_(True)
    loss = C.group_cross_entropy(x, torch.zeros(1, dtype=torch.int64, device=DEV), 1)
    assert loss == 0
    grad, = torch.autograd.grad(loss, x, torch.tensor(3.0, device=DEV))
    assert int((grad != 0).sum()) == 0


def test_two_threads_at_once():
    sizes, t = (36000, 13000), torch.zeros(130, dtype=torch.int64, device=DEV)
    x = {k: masked(130, k, 1, torch.float32, -1e9)[0].to(DEV) for k in sizes}
    want = {k: C.group_cross_entropy(x[k], t, k, reduction="none") for k in sizes}
    torch.cuda.synchronize()
    failed = []

    def calls(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                got = [C.group_cross_entropy(x[k], t, k, reduction="none") for _ in range(50)]
                torch.cuda.current_stream().synchronize()
            if not all(torch.equal(v, want[k]) for v in got):
                failed.append(k)
        except RuntimeError as e:
            failed.append(e)
    threads = [threading.Thread(target=calls, args=(k,)) for k in sizes]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not failed


@pytest.mark.parametrize("smoothing", [0.0, 0.1])
@pytest.mark.parametrize("layout,rows,k,group", [("rows", 200, 50, 1), ("rows", 200, 50, 6), ("rows", 150, 30, 80), ("rows", 5, 3000, 8), ("columns", 1030, 400, 2)])
def test_infinite_and_nan_classes_in_every_place(layout, rows, k, group, smoothing):
    # a class of each row, at another place in each, is not finite; the target is that class, or another one
    x, _ = masked(rows, k, group, torch.float32, 0.0)
    row = torch.arange(rows)
    at, t = 7 * row % k, torch.where(row % 2 == 0, 7 * row % k, (7 * row + 1 + row % (k - 1)) % k)
    x[row, at * group + row % group] = torch.tensor([-math.inf, math.inf, math.nan])[row // 2 % 3]
    leaf = (x.to(DEV) if layout == "rows" else x.to(DEV).t().contiguous().t()).requires_grad_(True)
    loss = C.group_cross_entropy(leaf, t.to(DEV), k, tau=group ** 0.5, label_smoothing=smoothing, reduction="none")
    grad, = torch.autograd.grad(loss.sum(), leaf)
    want, want_grad = K.group_cross_entropy(host(x), t.numpy(), k, group ** 0.5, smoothing, 1.0, "none")
    loss, grad, want, want_grad = host(loss), host(grad), np.asarray(want, dtype=np.float64), np.asarray(want_grad, dtype=np.float64)
    nan = (row // 2 % 3 != 0).numpy()
    assert np.isnan(loss[nan]).all() and np.isnan(want[nan]).all()
    # (the target's gradient alone could be finite: of +inf elsewhere, all are NaN)
    assert np.isnan(grad[nan]).any(1).all() and (np.isnan(grad) == np.isnan(want_grad)).all()
    step = (LN2 * (2 * 40 + 2 * 128) + 8) * 2.0 ** -24               # (distances up to 40 powers of two)
    assert np.allclose(loss[~nan], want[~nan], rtol=step, atol=step)
    assert np.allclose(grad[~nan] * group ** 0.5, want_grad[~nan] * group ** 0.5, rtol=0, atol=2 * step)
