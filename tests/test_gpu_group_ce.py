"""Cross entropy of group sums on the GPU against its definition in 64 bits (oracle/keep_oracle.py).

Bounds.  Scores are 64-bit sums.  The argument of a 32-bit exponential, in powers of two, is off by the rounding of the score relative to the row's pivot and to its
highest, U 2^-24 each with U = log2(e) times the largest of these differences, and by that of their difference; the exponential by 2 steps, and what becomes of it --
the factor, the product, the rounding -- by 6 more.  So an exponential is within (3 U + 8) 2^-24 of itself.  A gradient is w / tau times its probability and a part
of the smoothing, of the target the others' probabilities; a loss is the margin, off by the two roundings that it is a difference of, and the logarithm of 1 + the
others, off by their part of it.  2^-53 for float64.  Half a step of the type on top.  The instruction for 2^x gives 0 for results under 2^-126, so that much of an
exponential may be missing."""
import math

import numpy as np
import pytest
import torch

import convlogic_amd as C
from oracle import keep_oracle as K
from tests.gpu_util import DEV

pytestmark = pytest.mark.gpu

NAN, INF = math.nan, math.inf
TYPES = [torch.float32, torch.bfloat16, torch.float16, torch.float64]


def features(rows, k, group, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.rand(rows, k, group, generator=g, dtype=torch.float64) + torch.randn(rows, k, 1, generator=g, dtype=torch.float64) * (2.0 / group)
    return (x * scale).view(rows, k * group).to(dtype)


def labels(rows, k, seed=0, masked=False):
    g = torch.Generator().manual_seed(seed + 1)
    t = torch.randint(0, k, (rows,), generator=g)
    return torch.where(torch.rand(rows, generator=g) < 0.3, -100, t) if masked else t


def on_gpu(x, layout):
    x = x.to(DEV)
    return x if layout == "rows" else x.t().contiguous().t()


def host(t):
    return t.detach().double().cpu().numpy()


def check(x, t, k, layout, tau=1.0, smoothing=0.0, weight=1.0, reduction="mean", grad=True, upstream=None):
    leaf = on_gpu(x, layout).requires_grad_(grad)
    loss = C.group_cross_entropy(leaf, t.to(DEV), k, tau=tau, label_smoothing=smoothing, weight=weight, reduction=reduction)
    assert loss.dtype == (torch.float64 if x.dtype == torch.float64 else torch.float32)
    rows, group = x.shape[0], x.shape[1] // k
    up = None
    if reduction == "none":
        up = torch.rand(rows, dtype=loss.dtype) if upstream is None else upstream
    elif upstream is not None:
        up = torch.tensor(upstream, dtype=loss.dtype)
    want, want_grad = K.group_cross_entropy(host(x), t.numpy(), k, tau, smoothing, weight, reduction, None if up is None else up.numpy())
    # the sizes that the bounds are relative to
    count = max(int((t >= 0).sum()), 1) if reduction == "mean" else 1
    scores = host(x).reshape(rows, k, group).sum(2) / tau
    near = min(group, 64)
    pivot = host(x)[:, :near].sum(1, keepdims=True) * (group / near / tau)
    top = scores.max(1, keepdims=True)
    u = 1.4427 * np.max([np.abs(scores - top).max(1), np.abs(scores - pivot).max(1), np.abs(top - pivot)[:, 0]], axis=0)
    unit = 2.0 ** -53 if x.dtype == torch.float64 else 2.0 ** -24
    if x.dtype == torch.float64:                                      # (the sums themselves: as many roundings as additions, at most one for every feature)
        u = u + np.abs(host(x)).reshape(rows, k, group).sum(2).max(1) / tau * (group + 8)
    step = (3 * u + 8) * unit
    p = np.exp(scores - top)
    p /= p.sum(1, keepdims=True)
    inside = np.clip(t.numpy(), 0, k - 1)
    at = np.arange(rows)
    others = (p.sum(1) - p[at, inside]).clip(0) if k > 1 else np.zeros(rows)
    is_top = scores[at, inside] == top[:, 0]
    loss_rows, _ = K.group_cross_entropy(host(x), t.numpy(), k, tau, smoothing, 1.0, "none")
    size = np.where(is_top & (smoothing == 0), np.minimum(loss_rows, 1.0), 1.0 + np.abs(loss_rows)) * abs(weight)
    bound = step * np.where(t.numpy() >= 0, size, 0)
    half = torch.finfo(loss.dtype).eps / 2
    if reduction != "none":
        bound = bound.sum() / count
    assert (np.abs(host(loss) - want) <= bound + 2 * half * np.abs(want)).all(), (np.abs(host(loss) - want) - bound).max()
    if not grad:
        return
    got, = torch.autograd.grad(loss, leaf, None if up is None else up.to(DEV))
    assert got.dtype == x.dtype and got.shape == x.shape and (layout == "rows" or x.shape[0] == 1 or x.shape[1] == 1 or got.t().is_contiguous())
    mass = p + smoothing / k
    mass[at, inside] = others + smoothing
    mass = mass * np.where(t.numpy() >= 0, 1, 0)[:, None] * abs(weight) / tau / count
    if up is not None:
        mass = mass * np.abs(up.numpy().reshape(-1, 1))
    eps, tiny = torch.finfo(x.dtype).eps / 2, torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    error = np.abs(host(got) - want_grad)
    scale = mass / np.maximum(p + smoothing / k, 2.0 ** -1000)        # of an exponential over the total, in the gradient
    scale[at, inside] = 0
    limit = np.repeat(step[:, None] * mass + 2.0 ** -126 * scale, group, 1) + (eps * 1.001) * np.abs(want_grad) + tiny
    assert (error <= limit).all(), (error - limit).max()


SIZES = [(1, 1, 1), (3, 2, 1), (100, 10, 1), (5, 7, 3), (33, 10, 4), (64, 12, 8), (2, 5, 100), (130, 9, 5), (17, 100, 2), (200, 30, 64), (1500, 10, 7),
         (3, 3, 2100), (129, 10, 1000), (257, 2, 515)]


@pytest.mark.parametrize("layout", ["rows", "columns"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k,group", SIZES)
def test_mean_and_gradient(rows, k, group, dtype, layout):
    check(features(rows, k, group, dtype), labels(rows, k), k, layout, tau=0.1 * group ** 0.5 + 0.2)


@pytest.mark.parametrize("layout", ["rows", "columns"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("smoothing", [0.0, 0.1, 1.0])
@pytest.mark.parametrize("rows,k,group", [(100, 10, 1), (70, 33, 6), (5, 300, 200), (40, 4, 2000), (1030, 3, 2)])
def test_reductions_smoothing_and_masks(rows, k, group, smoothing, reduction, layout):
    for masked, grad in [(False, True), (True, True), (True, False)]:
        check(features(rows, k, group), labels(rows, k, masked=masked), k, layout, tau=0.3 * group ** 0.5, smoothing=smoothing, weight=0.7, reduction=reduction, grad=grad)


@pytest.mark.parametrize("layout", ["rows", "columns"])
@pytest.mark.parametrize("rows,k,group", [(130, 30000, 1), (3, 40000, 1), (2, 50001, 5), (130, 37000, 2), (1, 4, 30000), (300, 20000, 1)])
def test_many_classes_and_long_groups(rows, k, group, layout):
    check(features(rows, k, group, scale=3.0), labels(rows, k), k, layout, tau=0.3 * group ** 0.5)


def test_double_rows_beyond_lds():
    check(features(130, 20000, 1, torch.float64), labels(130, 20000), 20000, "rows")


@pytest.mark.parametrize("layout", ["rows", "columns"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rows_at_any_address(dtype, layout):
    x, t = features(60, 11, 5, dtype), labels(60, 11)
    if layout == "rows":
        wide = torch.zeros(60, 55 + 4, dtype=dtype, device=DEV)
        wide[:, 3:58] = x.to(DEV)
        leaf = wide[:, 3:58].requires_grad_(True)
    else:
        flat = torch.zeros(60 * 55 + 1, dtype=dtype, device=DEV)
        flat[1:] = x.t().contiguous().to(DEV).view(-1)
        leaf = flat[1:].view(55, 60).t().requires_grad_(True)
    loss = C.group_cross_entropy(leaf, t.to(DEV), 11)
    other = x.to(DEV).requires_grad_(True)
    want = C.group_cross_entropy(other, t.to(DEV), 11)
    assert abs(float(loss - want)) <= 2e-6 * abs(float(want))
    g, w = torch.autograd.grad(loss, leaf)[0], torch.autograd.grad(want, other)[0]
    assert torch.allclose(g.float(), w.float(), rtol=2 * torch.finfo(dtype).eps, atol=1e-7)
    spread = x.to(DEV).repeat_interleave(2, 1)[:, ::2].requires_grad_(True)      # (strides that the kernels do not read)
    assert torch.equal(C.group_cross_entropy(spread, t.to(DEV), 11), want)


@pytest.mark.parametrize("layout", ["rows", "columns"])
@pytest.mark.parametrize("rows,k,group", [(20, 8, 1), (20, 8, 20), (3, 9, 3000), (140, 8, 4)])
@pytest.mark.parametrize("upstream", [1.0, 0.5, -3.0, 0.0])
def test_other_upstream_gradients(upstream, rows, k, group, layout):
    for reduction in ("mean", "sum"):
        check(features(rows, k, group), labels(rows, k, masked=True), k, layout, tau=group ** 0.5, reduction=reduction, upstream=upstream)


@pytest.mark.parametrize("layout", ["rows", "columns"])
@pytest.mark.parametrize("rows,k,group", [(20, 8, 1), (20, 8, 20), (3, 9, 3000), (2, 3000, 9)])
def test_rows_that_do_not_count_and_targets_that_are_no_class(rows, k, group, layout):
    x, t = features(rows, k, group), labels(rows, k)
    x[0], t[0] = NAN, -1
    t[1] = k
    leaf = on_gpu(x, layout).requires_grad_(True)
    loss = C.group_cross_entropy(leaf, t.to(DEV), k, reduction="none")
    assert loss[0] == 0 and loss[1].isnan() and loss[2:].isfinite().all()
    grad, = torch.autograd.grad(loss.sum(), leaf)
    assert (grad[0] == 0).all() and grad[1].isnan().all() and grad[2:].isfinite().all()
    t[1] = -5
    leaf = on_gpu(x, layout).requires_grad_(True)
    loss = C.group_cross_entropy(leaf, t.to(DEV), k)
    grad, = torch.autograd.grad(loss, leaf)
    assert loss.isfinite() and (grad[:2] == 0).all() and grad.isfinite().all()
    none = C.group_cross_entropy(leaf, torch.full((rows,), -1, device=DEV), k)
    assert none == 0 and (torch.autograd.grad(none, leaf)[0] == 0).all()


@pytest.mark.parametrize("layout", ["rows", "columns"])
@pytest.mark.parametrize("group", [1, 6, 3000])
def test_infinite_and_nan_features(group, layout):
    k = 5
    for value, at, target in [(-INF, 1, 2), (-INF, 2, 2), (INF, 1, 2), (INF, 2, 2), (NAN, 1, 2), (NAN, 2, 2), (-INF, 0, 2), (INF, 0, 2)]:
        x = features(4, k, group)
        x[1, at * group] = value
        t = torch.full((4,), target)
        leaf = on_gpu(x, layout).requires_grad_(True)
        loss = C.group_cross_entropy(leaf, t.to(DEV), k, tau=group ** 0.5, reduction="none")
        grad, = torch.autograd.grad(loss.sum(), leaf)
        ref = x.double().requires_grad_(True)
        want = torch.nn.functional.cross_entropy(ref.view(4, k, group).sum(2) / group ** 0.5, t, reduction="none")
        want_grad, = torch.autograd.grad(want.sum(), ref)
        assert torch.allclose(loss.cpu().double(), want.detach(), rtol=1e-5, equal_nan=True), (value, at)
        assert torch.allclose(grad.cpu().double(), want_grad, rtol=1e-4, atol=1e-6, equal_nan=True), (value, at)
    x = features(4, k, group)
    x[1] = -INF
    loss = C.group_cross_entropy(on_gpu(x, layout), torch.full((4,), 1, device=DEV), k, reduction="none")
    assert loss.isnan().tolist() == [False, True, False, False]


@pytest.mark.parametrize("layout", ["rows", "columns"])
def test_scores_far_apart_and_far_from_zero(layout):
    # a loss near 0 keeps its digits, one of hundreds is the margin; levels far from 0 are taken off in 64 bits
    for gap in (5.0, 20.0, 60.0, 500.0):
        for level in (0.0, 1000.0):
            x = torch.zeros(6, 4 * 10, dtype=torch.float32) + level
            x[:, 10:20] += gap / 8
            t = torch.tensor([1, 1, 1, 0, 2, 3])
            got = C.group_cross_entropy(on_gpu(x, layout), t.to(DEV), 4, tau=1.25, reduction="none").cpu().double()
            d = 10 * np.float64((x[0, 10] - x[0, 0]).double()) / 1.25
            small = math.log1p(3 * math.exp(-d))
            want = torch.tensor([small] * 3 + [small + d] * 3)
            assert torch.allclose(got, want, rtol=(6 * 1.4427 * d + 20) * 2.0 ** -24, atol=1e-44), (gap, level)


def test_half_gradients_of_scaled_losses():
    x, t = features(300, 50, 4, torch.float16), labels(300, 50)
    for upstream in (1.0, 4096.0):
        check(x, t, 50, "rows", weight=256.0, upstream=upstream)
        check(x, t, 50, "columns", weight=256.0, upstream=upstream)


def test_int32_targets_and_shapes():
    x, t = features(24, 6, 5).to(DEV), labels(24, 6).to(DEV)
    want = C.group_cross_entropy(x, t, 6, reduction="none")
    assert torch.equal(C.group_cross_entropy(x, t.int(), 6, reduction="none"), want)
    assert torch.equal(C.group_cross_entropy(x.view(2, 3, 4, 30), t.view(2, 3, 4), 6, reduction="none").view(-1), want)
    assert torch.equal(C.group_cross_entropy(x, t.repeat_interleave(2)[::2], 6, reduction="none"), want)
    assert torch.equal(C.group_cross_entropy(x[3], t[3], 6), want[3])
    for reduction, shape in (("none", (0,)), ("mean", ()), ("sum", ())):
        empty = x[:0].requires_grad_(True)
        loss = C.group_cross_entropy(empty, t[:0], 6, reduction=reduction)
        assert loss.shape == shape and (loss == 0).all()
        loss.sum().backward()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["rows", "columns"])
@pytest.mark.parametrize("group", [2, 3, 5, 6, 7, 9, 13, 15, 17, 31, 33, 61, 63, 65, 127, 255, 513])
def test_groups_of_every_kind(group, layout, dtype):
    check(features(150, 5, group, dtype), labels(150, 5), 5, layout, tau=0.3 * group ** 0.5)
    check(features(4, 600, group, dtype), labels(4, 600), 600, layout, tau=0.3 * group ** 0.5, reduction="none")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [63, 64, 65, 128, 129, 191, 256, 257, 300, 511, 700, 1025])
def test_columns_of_every_width(rows, dtype):
    check(features(rows, 6, 20, dtype), labels(rows, 6, masked=True), 6, "columns", tau=1.5)
    check(features(rows, 770, 2, dtype), labels(rows, 770, masked=True), 770, "columns", tau=0.5, reduction="none")


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("layout,rows,k,group", [
    ("rows", 128, 64, 1), ("rows", 129, 64, 1), ("rows", 128, 13, 5), ("rows", 64, 300, 60), ("rows", 65, 300, 60), ("rows", 64, 250, 64),                # one workgroup, pieces, whole rows
    ("rows", 70, 512, 1), ("rows", 70, 513, 1), ("rows", 70, 1024, 8), ("rows", 70, 1025, 8), ("rows", 1024, 512, 8), ("rows", 1024, 1025, 4),            # threads
    ("columns", 3, 2, 65536), ("columns", 17, 3, 20001), ("columns", 64, 10, 2048), ("columns", 70, 256, 130), ("columns", 70, 257, 130),                 # slices
    ("columns", 16, 140, 3), ("columns", 17, 140, 3), ("columns", 64, 128, 2), ("columns", 65, 128, 2), ("columns", 1030, 1500, 2), ("rows", 20, 2000, 64)])  # joins
def test_borders_of_the_shapes(layout, rows, k, group, reduction):
    check(features(rows, k, group), labels(rows, k, masked=True), k, layout, tau=0.3 * group ** 0.5, smoothing=0.1, reduction=reduction)
    check(features(rows, k, group), labels(rows, k), k, layout, tau=0.3 * group ** 0.5, reduction=reduction, grad=False)


@pytest.mark.parametrize("bits", [None, 8])
def test_a_topology_without_its_group_sum(bits):
    torch.manual_seed(0)
    net = C.ConvLogicCifarModel(k_param=4, checkpoint_bits=bits).to(DEV)
    x, t = (torch.rand(20, 3, 32, 32, device=DEV) > 0.5).float(), torch.randint(0, 10, (20,), device=DEV)
    loss = C.group_cross_entropy(net.network[:-1](x), t, k=10, tau=20.0, label_smoothing=0.1)
    other = torch.nn.functional.cross_entropy(net(x), t, label_smoothing=0.1)
    assert abs(float(loss - other)) <= 1e-5 * float(other)
    got, want = (torch.autograd.grad(v, list(net.parameters())) for v in (loss, other))
    # (with codes the layers of the end keep their inputs' codes, its trees those of the first layer's input alone)
    assert all((u - v).norm() <= (1e-4 if bits is None else 0.05) * v.norm() + 1e-9 for u, v in zip(got, want))


def test_features_of_more_than_2_to_the_31_elements():
    rows, k, group = 70000, 32768, 1
    x = torch.zeros(rows, k, device=DEV, dtype=torch.bfloat16)
    x[-1, 7] = 5.0
    t = torch.zeros(rows, dtype=torch.int64, device=DEV)
    t[-1] = 7
    for leaf in (x.requires_grad_(True), x.detach().t().contiguous().t().requires_grad_(True)):
        loss = C.group_cross_entropy(leaf, t, k, reduction="none")
        grad, = torch.autograd.grad(loss.sum(), leaf)
        assert abs(float(loss[0].detach()) - math.log(k)) <= 1e-5 and abs(float(loss[-1].detach()) - math.log1p((k - 1) * math.exp(-5))) <= 1e-5
        p = 1 / (1 + (k - 1) * math.exp(-5))
        assert abs(float(grad[-1, 7]) - (p - 1)) <= 2.0 ** -8 and abs(float(grad[-1, -1]) - p * math.exp(-5)) <= 2.0 ** -8 * p * math.exp(-5)
        assert abs(float(grad[-2, 0]) - (1 / k - 1)) <= 2.0 ** -8 and abs(float(grad[-2, -1]) - 1 / k) <= 2.0 ** -8 / k
        del grad, loss


def test_many_rows():
    check(features(70001, 3, 1), labels(70001, 3, masked=True), 3, "rows")
    check(features(70001, 3, 2), labels(70001, 3, masked=True), 3, "columns", smoothing=0.1)


def test_refusals():
    x, t = features(4, 3, 2).to(DEV), labels(4, 3)
    with pytest.raises(RuntimeError, match="one device"):
        C.group_cross_entropy(x, t, 3)
    leaf = x.clone().requires_grad_(True)
    loss = C.group_cross_entropy(leaf, t.to(DEV), 3)
    grad, = torch.autograd.grad(loss, leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        grad.sum().backward()
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda x: C.group_cross_entropy(x, t.to(DEV), 3), (x,))


@pytest.mark.parametrize("layout", ["rows", "columns"])
@pytest.mark.parametrize("rows,k,group", [(40, 10, 1), (40, 10, 50), (3, 4, 3000), (130, 20000, 1)])
def test_retained_graphs_streams_and_recordings(rows, k, group, layout):
    x, t = on_gpu(features(rows, k, group), layout), labels(rows, k).to(DEV)
    leaf = x.clone().requires_grad_(True) if layout == "rows" else x.t().clone().t().requires_grad_(True)
    loss = C.group_cross_entropy(leaf, t, k)
    first, = torch.autograd.grad(loss, leaf, retain_graph=True)
    kept = first.clone()
    first.zero_()                                                     # (its receiver may do so)
    second, = torch.autograd.grad(loss, leaf, retain_graph=True)
    third, = torch.autograd.grad(2 * loss, leaf)
    close = dict(rtol=1e-5, atol=1e-9)                                # (a pass of its own, and the one with the sums)
    assert torch.allclose(second, kept, **close) and torch.allclose(third, 2 * kept, **close)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = C.group_cross_entropy(leaf, t, k)
        fourth, = torch.autograd.grad(other, leaf)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, loss) and torch.equal(fourth, kept)
    del loss, other
    for factor in (1.0, 0.5):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = C.group_cross_entropy(leaf, t, k)
            grad, = torch.autograd.grad(out * factor if factor != 1.0 else out, leaf)
        for seed in range(3):
            with torch.no_grad():
                leaf.copy_(features(rows, k, group, seed=seed).to(DEV))
            grad.zero_()
            graph.replay()
            want = C.group_cross_entropy(leaf, t, k)
            want_grad, = torch.autograd.grad(want * factor if factor != 1.0 else want, leaf)
            assert torch.equal(out, want) and torch.equal(grad, want_grad)
            torch.cuda.synchronize()
            del want


def test_the_loss_of_a_network():
    # a run of the operators together: layers that keep codes, the loss of what the last one puts out, against the modules and torch's loss
    torch.manual_seed(0)
    net = torch.nn.Sequential(*(C.LogicLayer(a, b, implementation="cuda", checkpoint_bits=8) for a, b in [(64, 128), (128, 64), (64, 40)])).to(DEV)
    x, t = torch.rand(150, 64, device=DEV), torch.randint(0, 10, (150,), device=DEV)
    loss = C.group_cross_entropy(net(x), t, 10, tau=1.3)
    got = torch.autograd.grad(loss, list(net.parameters()))
    other = torch.nn.functional.cross_entropy(C.GroupSum(10, 1.3)(net(x)), t)
    want = torch.autograd.grad(other, list(net.parameters()))
    assert abs(float(loss - other)) <= 1e-5 * float(other)
    # (float32 gradients of the loss that differ in their last places, through three layers of products of magnitude 2)
    assert all((u - v).norm() <= 1e-4 * v.norm() for u, v in zip(got, want))
    del loss, other                                                   # (no eager graph of the parameters may live while a step is recorded)
    step = C.GraphedStep(lambda x, t: C.group_cross_entropy(net(x), t, 10, tau=1.3), (x, t), net.parameters())
    for seed in range(3):
        x = torch.rand(150, 64, device=DEV)
        value = float(step(x, t))
        grads = [p.grad.clone() for p in net.parameters()]
        eager = C.group_cross_entropy(net(x), t, 10, tau=1.3)
        ref = torch.autograd.grad(eager, list(net.parameters()))
        assert value == float(eager.detach()) and all(torch.equal(u, v) for u, v in zip(grads, ref))
        del eager, ref


def test_the_loss_of_a_topology():
    torch.manual_seed(0)
    net = C.ConvLogicMnistModel(k_param=4, checkpoint_bits=8).to(DEV)
    x, t = (torch.rand(16, 1, 28, 28, device=DEV) > 0.5).float(), torch.randint(0, 10, (16,), device=DEV)
    loss = C.group_cross_entropy(net(x), t, 10)
    other = torch.nn.functional.cross_entropy(net(x), t)
    assert abs(float(loss - other)) <= 1e-5 * float(other)
    got, want = (torch.autograd.grad(v, list(net.parameters())) for v in (loss, other))
    assert all((u - v).norm() <= 1e-4 * v.norm() + 1e-9 for u, v in zip(got, want))
