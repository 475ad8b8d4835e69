"""Cross entropy of group sums on the CPU: against its definition and torch's cross entropy of a GroupSum, and what is refused."""
import math

import numpy as np
import pytest
import torch

import convlogic_amd as C
from oracle import keep_oracle as K


def features(rows, k, group, dtype=torch.float64, seed=0):
    return torch.rand(rows, k * group, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dtype)


def labels(rows, k, seed=0):
    return torch.randint(0, k, (rows,), generator=torch.Generator().manual_seed(seed + 1))


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("smoothing", [0.0, 0.2, 1.0])
@pytest.mark.parametrize("rows,k,group", [(1, 1, 1), (5, 3, 1), (7, 10, 6), (4, 2, 33)])
def test_against_the_definition(rows, k, group, smoothing, reduction):
    x, t = features(rows, k, group).requires_grad_(True), labels(rows, k)
    if rows > 4:
        t[2] = -100
    loss = C.group_cross_entropy(x, t, k, tau=0.7, label_smoothing=smoothing, weight=1.5, reduction=reduction)
    up = torch.rand(rows, dtype=torch.float64) if reduction == "none" else None
    grad, = torch.autograd.grad(loss, x, up)
    want, want_grad = K.group_cross_entropy(x.detach().numpy(), t.numpy(), k, 0.7, smoothing, 1.5, reduction, None if up is None else up.numpy())
    want, want_grad = np.asarray(want, dtype=np.float64), np.asarray(want_grad, dtype=np.float64)
    assert np.allclose(loss.detach().numpy(), want, rtol=1e-12, atol=1e-14) and np.allclose(grad.numpy(), want_grad, rtol=1e-11, atol=1e-14)
    # (and the definition is that of the modules)
    ref = x.detach().requires_grad_(True)
    other = 1.5 * torch.nn.functional.cross_entropy(C.GroupSum(k, 0.7)(ref), t, label_smoothing=smoothing, reduction=reduction)
    ref_grad, = torch.autograd.grad(other, ref, up)
    assert torch.allclose(loss, other, rtol=1e-10) and torch.allclose(grad, ref_grad, rtol=1e-9, atol=1e-13)


def test_gradient_against_differences():
    x, t = features(6, 4, 3).requires_grad_(True), labels(6, 4)
    for smoothing in (0.0, 0.1):
        assert torch.autograd.gradcheck(lambda x: C.group_cross_entropy(x, t, 4, tau=0.5, label_smoothing=smoothing), x)


def test_rows_that_do_not_count():
    x, t = features(4, 3, 2), torch.tensor([0, -1, 2, -100])
    x[1], x[3, 0] = math.nan, math.inf
    x.requires_grad_(True)
    loss = C.group_cross_entropy(x, t, 3)
    loss.backward()
    assert torch.isfinite(loss) and (x.grad[[1, 3]] == 0).all() and torch.isfinite(x.grad).all()
    none = C.group_cross_entropy(x, torch.full((4,), -1), 3)
    assert none == 0
    assert C.group_cross_entropy(features(4, 3, 2)[:0], t[:0], 3) == 0
    assert C.group_cross_entropy(features(4, 3, 2)[:0], t[:0], 3, reduction="none").shape == (0,)


def test_a_target_that_is_no_class():
    x, t = features(4, 3, 2).requires_grad_(True), torch.tensor([0, 3, 2, 1])
    loss = C.group_cross_entropy(x, t, 3, reduction="none")
    loss.sum().backward()
    assert loss.isnan().tolist() == [False, True, False, False] and x.grad.isnan().all(1).tolist() == [False, True, False, False]


def test_types_and_leading_dimensions():
    x, t = features(12, 5, 2), labels(12, 5)
    want = C.group_cross_entropy(x, t, 5, reduction="none")
    for dtype, kind in [(torch.float32, torch.float32), (torch.float16, torch.float32), (torch.bfloat16, torch.float32), (torch.float64, torch.float64)]:
        leaf = x.to(dtype).view(3, 4, 10).requires_grad_(True)
        loss = C.group_cross_entropy(leaf, t.int().view(3, 4), 5, reduction="none")
        assert loss.dtype == kind and loss.shape == (3, 4)
        loss.sum().backward()
        assert leaf.grad.dtype == dtype
        assert torch.allclose(loss.double().view(-1), want, rtol=20 * torch.finfo(dtype).eps)
    assert C.group_cross_entropy(x[0], t[0], 5).shape == ()


def test_refusals():
    x, t = features(4, 3, 2), labels(4, 3)
    for bad, error, match in [
            (dict(x=x.int()), RuntimeError, "float32, float64"), (dict(x=[1.0]), RuntimeError, "float32, float64"),
            (dict(targets=t.float()), RuntimeError, "int32 or int64"), (dict(targets=t[:3]), RuntimeError, "int32 or int64"),
            (dict(targets=[0, 1, 2, 0]), RuntimeError, "int32 or int64"), (dict(targets=t.to("meta")), RuntimeError, "one device"),
            (dict(k=4), ValueError, "divisor"), (dict(k=0), ValueError, "divisor"), (dict(tau=0.0), ValueError, "tau"), (dict(tau=-1.0), ValueError, "tau"),
            (dict(tau=math.inf), ValueError, "tau"), (dict(label_smoothing=-0.1), ValueError, "between 0 and 1"), (dict(label_smoothing=1.1), ValueError, "between 0 and 1"),
            (dict(label_smoothing=math.nan), ValueError, "label_smoothing"), (dict(weight=math.inf), ValueError, "weight"), (dict(reduction="max"), ValueError, "reduction")]:
        with pytest.raises(error, match=match):
            C.group_cross_entropy(**{**dict(x=x, targets=t, k=3), **bad})
    with pytest.raises(RuntimeError, match="columns"):
        C.group_cross_entropy(torch.ones(4, 0), t, 1)


@pytest.mark.parametrize("value", [-1e4, -1e9, torch.finfo(torch.float32).min])
@pytest.mark.parametrize("k,group,smoothing", [(10, 1, 0.0), (7, 5, 0.1)])
def test_classes_masked_with_finite_values(k, group, smoothing, value):
    x, t = features(8, k, group), labels(8, k)
    x[::2, :group] = value
    t[::2] = t[::2].clamp(min=1)
    x = x.float().requires_grad_(True)
    loss = C.group_cross_entropy(x, t, k, tau=float(group), label_smoothing=smoothing, reduction="none")
    grad, = torch.autograd.grad(loss.sum(), x)
    want, want_grad = K.group_cross_entropy(x.detach().numpy(), t.numpy(), k, float(group), smoothing, 1.0, "none")
    # (scores and exponentials in 64 bits: the rounding to float32 is what is left)
    assert np.allclose(loss.detach().numpy(), np.asarray(want, dtype=np.float64), rtol=2.0 ** -24 * 1.01, atol=1e-12)
    assert np.allclose(grad.numpy(), np.asarray(want_grad, dtype=np.float64), rtol=2.0 ** -24 * 1.01, atol=1e-12)
