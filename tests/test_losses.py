"""Losses on scores and gate logits without a GPU: the plain forms of CPU tensors against the 64-bit definitions and against differences, the refusals of the
public functions and of the C entry points."""
import math

import numpy as np
import pytest
import torch

import convlogic_amd as C
from convlogic_amd.hip import _lib
from oracle import losses_oracle as L

NAN, INF = math.nan, math.inf


def scores(rows, cols, dtype=torch.float32, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, cols, generator=g) * scale).to(dtype)


# The plain forms work in 64 bits and round once: half a step of the result's type, and some 2^-50 of the terms that cancel.
def close(got, want, size, name):
    got_64 = got.detach().double().numpy()
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    bound = half * np.abs(want) * (1 + 2.0 ** -20) + 2.0 ** -45 * np.asarray(size) + tiny
    assert np.array_equal(np.isnan(got_64), np.isnan(want)), name
    bad = ~(np.isnan(want) | (np.abs(got_64 - want) <= bound) | (got_64 == want))
    assert not bad.any(), (name, np.abs(got_64 - want)[bad].max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,cols,k", [(1, 1, 1), (3, 10, 4), (5, 33, 33), (4, 200, 17)])
def test_top_logits(dtype, rows, cols, k):
    z = scores(rows, cols, dtype)
    z[0, 0] = z[0, cols - 1]                                          # (a tie where there are two columns)
    got = C.top_logits(z, k, temperature=2.0)
    values, columns, lse = L.top_logits(z.double().numpy(), k, 2.0)
    assert np.array_equal(got.indices.numpy(), columns) and np.array_equal(got.values.double().numpy(), values)
    assert got.values.dtype == dtype and got.logsumexp.dtype == (torch.float64 if dtype == torch.float64 else torch.float32)
    assert np.allclose(got.logsumexp.double().numpy(), lse, rtol=2.0 ** -23, atol=2.0 ** -23)


def test_top_logits_orders_nan_infinities_and_zeros():
    z = torch.tensor([[0.0, -0.0, INF, NAN, -INF, 1.0, NAN, INF], [-INF] * 8])
    got = C.top_logits(z, 8)
    assert got.indices.tolist() == [[3, 6, 2, 7, 5, 0, 1, 4], list(range(8))]
    assert got.logsumexp[0].isnan() and got.logsumexp[1] == -INF
    assert not C.top_logits(torch.randn(3, 4, requires_grad=True), 2).values.requires_grad
    assert C.top_logits(torch.randn(2, 3, 7), 2).values.shape == (2, 3, 2) and C.top_logits(torch.randn(7), 2).logsumexp.shape == ()


def distill_case(seed, rows=6, cols=23, k=5, rest=False, dtype=torch.float32):
    z, t = scores(rows, cols, dtype, seed), scores(rows, cols, torch.float32, seed + 100)
    top = C.top_logits(t, k, temperature=1.5)
    return z, top.values, top.indices, top.logsumexp if rest else None


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_distillation(dtype, rest, reduction):
    z, values, columns, lse = distill_case(1, rest=rest, dtype=dtype)
    if not rest:
        columns[0, 2:], columns[1] = -1, -1                           # a short row and one without entries
    mask = torch.tensor([True, True, False, True, True, True])
    z[2] = torch.tensor([NAN, INF, -INF] + [0.0] * 20).to(dtype)
    z[4, 7] = -INF if int((columns[4] == 7).sum()) == 0 else z[4, 7]
    z.requires_grad_(True)
    loss = C.distillation_loss(z, values, columns, lse, temperature=1.5, mask=mask, weight=0.7, reduction=reduction)
    up = torch.rand(6, dtype=loss.dtype) if reduction == "none" else torch.tensor(3.0, dtype=loss.dtype)
    grad, = torch.autograd.grad(loss, z, up)
    want = L.distillation(z.detach().double().numpy(), values.double().numpy(), columns.numpy(), None if lse is None else lse.double().numpy(), 1.5,
                          mask.numpy(), 0.7, reduction, up.double().numpy())
    close(loss, want[0], want[2], "loss")
    close(grad, want[1], want[3], "grad")
    assert (grad[2] == 0).all() and grad.dtype == dtype and (rest or (grad[1] == 0).all())


@pytest.mark.parametrize("rest", [False, True])
def test_distillation_gradient_against_differences(rest):
    z, values, columns, lse = distill_case(5, 3, 11, 4, rest)
    z = z.double().requires_grad_(True)
    assert torch.autograd.gradcheck(lambda x: C.distillation_loss(x, values.double(), columns, lse, temperature=1.5, reduction="none"), (z,))


def test_distillation_special_rows():
    z, values, columns, lse = distill_case(7, 4, 9, 3)
    # a teacher that lists every column, in order: the same with its logsumexp, there is nothing else
    every = C.top_logits(scores(4, 9, torch.float64, 9), 9)
    a = C.distillation_loss(z.double(), every.values, every.indices)
    b = C.distillation_loss(z.double(), every.values, every.indices, every.logsumexp)
    assert abs(float(a - b)) <= 1e-12 * abs(float(a))
    # a teacher of itself
    own = C.top_logits(z.double(), 3)
    assert abs(float(C.distillation_loss(z.double(), own.values, own.indices, own.logsumexp))) <= 1e-12
    # a column listed twice counts twice
    twice, t = torch.tensor([[2, 2, 5]] * 4), torch.zeros(4, 3)
    x = z.double().requires_grad_(True)
    want = L.distillation(z.double().numpy(), t.numpy(), twice.numpy())
    loss = C.distillation_loss(x, t, twice)
    close(loss, want[0], want[2], "loss")
    close(torch.autograd.grad(loss, x)[0], want[1], want[3], "grad")
    # a column behind the last: that row alone is NaN, unless its mask is off
    columns[1, 0] = 9
    loss = C.distillation_loss(x, values, columns, reduction="none")
    assert loss.isnan().tolist() == [False, True, False, False]
    assert torch.autograd.grad(loss.sum(), x)[0].isnan().any(1).tolist() == [False, True, False, False]
    keep = torch.tensor([True, False, True, True])
    assert C.distillation_loss(x, values, columns, mask=keep).isfinite()
    # no row at all
    assert C.distillation_loss(x, values, columns, mask=torch.zeros(4, dtype=torch.bool)) == 0
    empty = C.distillation_loss(z[:0], values[:0], columns[:0])
    assert empty == 0 and C.distillation_loss(z[:0], values[:0], columns[:0], reduction="none").shape == (0,)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
@pytest.mark.parametrize("rows,experts,k", [(1, 1, 1), (9, 16, 1), (20, 7, 3), (12, 5, 5)])
def test_balance(dtype, rows, experts, k):
    z = scores(rows, experts, dtype, 3)
    z[0, 0] = -INF
    mask = torch.arange(rows) % 4 != 1
    z.requires_grad_(True)
    loss, counts = C.balance_loss(z, k, mask=mask, weight=0.5)
    grad, = torch.autograd.grad(loss, z)
    want = L.balance(z.detach().double().numpy(), k, mask.numpy(), 0.5)
    assert counts.tolist() == want[1].tolist() and not counts.requires_grad
    close(loss, want[0], want[0], "loss")
    close(grad, want[2], want[3], "grad")


def test_balance_by_differences_and_without_rows():
    z = scores(6, 5, torch.float64, 4).requires_grad_(True)
    assert torch.autograd.gradcheck(lambda x: C.balance_loss(x, 2).loss, (z,))
    none = C.balance_loss(z, 2, mask=torch.zeros(6, dtype=torch.bool))
    assert none.loss == 0 and none.counts.tolist() == [0] * 5 and (torch.autograd.grad(none.loss, z)[0] == 0).all()
    assert C.balance_loss(torch.zeros(8, 4), 4).loss == 1              # every expert has its share
    assert C.balance_loss(torch.zeros(2, 3, 4)).counts.tolist() == [6, 0, 0, 0]


def test_gate_balance_of_a_network():
    model = C.ConvLogicMnistModel(k_param=2, implementation="python")
    tensors = list(model.parameters())
    with torch.no_grad():
        for p in tensors:
            p.add_(torch.randn(p.shape))
    loss, counts = C.gate_balance(model, weight=2.0)
    parts = [C.balance_loss(p) for p in tensors]
    assert torch.allclose(loss, 2 * torch.stack([a.loss for a in parts]).mean(), rtol=1e-6) and torch.equal(counts, torch.stack([a.counts for a in parts]))
    assert counts.sum(1).tolist() == [p.numel() // 16 for p in tensors]
    loss.backward()
    assert all(p.grad is not None and p.grad.shape == p.shape for p in tensors)
    layer = C.LogicLayer(8, 12, implementation="python")
    assert C.gate_balance(layer).counts.shape == (1, 16) and C.gate_balance([layer.weights]).loss == C.gate_balance(layer).loss


def test_refusals():
    z, values, columns, lse = distill_case(1)
    lse = torch.zeros(6)
    cases = [
        (RuntimeError, lambda: C.top_logits(z.int(), 2)), (RuntimeError, lambda: C.top_logits([1.0], 1)), (ValueError, lambda: C.top_logits(z, 0)),
        (ValueError, lambda: C.top_logits(z, 24)), (ValueError, lambda: C.top_logits(torch.zeros(1, 2000), 1025)),
        (ValueError, lambda: C.top_logits(z, 2, temperature=0)), (ValueError, lambda: C.top_logits(z, 2, temperature=NAN)),
        (RuntimeError, lambda: C.top_logits(torch.zeros(()), 1)), (RuntimeError, lambda: C.top_logits(torch.zeros(3, 0), 1)),
        (RuntimeError, lambda: C.distillation_loss(z.long(), values, columns)), (RuntimeError, lambda: C.distillation_loss(z, values.int(), columns)),
        (RuntimeError, lambda: C.distillation_loss(z, values[:3], columns[:3])), (RuntimeError, lambda: C.distillation_loss(z, values, columns[:, :2])),
        (RuntimeError, lambda: C.distillation_loss(z, values, columns.float())), (RuntimeError, lambda: C.distillation_loss(z, values, columns, lse[:2])),
        (RuntimeError, lambda: C.distillation_loss(z, values, columns, lse.int())), (RuntimeError, lambda: C.distillation_loss(z, values[:, :0], columns[:, :0])),
        (RuntimeError, lambda: C.distillation_loss(z, values, columns, mask=torch.ones(6))),
        (RuntimeError, lambda: C.distillation_loss(z, values, columns, mask=torch.ones(5, dtype=torch.bool))),
        (RuntimeError, lambda: C.distillation_loss(z, values.clone().requires_grad_(True), columns)),
        (ValueError, lambda: C.distillation_loss(z, torch.zeros(6, 1025), torch.zeros(6, 1025, dtype=torch.long))),
        (ValueError, lambda: C.distillation_loss(z, values, columns, temperature=-1)), (ValueError, lambda: C.distillation_loss(z, values, columns, weight=INF)),
        (ValueError, lambda: C.distillation_loss(z, values, columns, reduction="batchmean")),
        (RuntimeError, lambda: C.distillation_loss(z.to("meta"), values.to("meta"), columns.to("meta"))),
        (RuntimeError, lambda: C.balance_loss(z.long())), (ValueError, lambda: C.balance_loss(z, 0)), (ValueError, lambda: C.balance_loss(z, 24)),
        (ValueError, lambda: C.balance_loss(torch.zeros(2, 1025))), (RuntimeError, lambda: C.balance_loss(z, mask=torch.ones(6))),
        (ValueError, lambda: C.balance_loss(z, weight=NAN)), (ValueError, lambda: C.gate_balance([])), (ValueError, lambda: C.gate_balance(torch.nn.Linear(2, 2))),
        (RuntimeError, lambda: C.gate_balance([z])), (RuntimeError, lambda: C.gate_balance([torch.zeros(2, 16), torch.zeros(2, 16).double()])),
    ]
    for i, (kind, call) in enumerate(cases):
        with pytest.raises(kind):
            call()
            print("not refused:", i)


def test_the_c_entry_points_refuse_before_they_launch():
    # (in a thread of its own: the message of the last error is a thread's, and others look at the main one's)
    from concurrent.futures import ThreadPoolExecutor
    with ThreadPoolExecutor(1) as pool:
        pool.submit(refused_by_the_c_entry_points).result()


def refused_by_the_c_entry_points():
    lib = _lib.load()
    p = 4096                                                          # never read: every call is refused on the host
    top = [0, p, 8, 2, 8, 3, 1.0, p, p, p, None, None]
    for at, value in [(0, 7), (2, -1), (3, -1), (3, 1 << 31), (4, 0), (4, 1 << 31), (5, 0), (5, 9), (5, 1025), (6, 0.0), (6, NAN), (1, None), (7, None), (8, None)]:
        args = list(top)
        args[at] = value
        assert lib.clg_top_logits(*args) == -1 and b"clg_top_logits" in lib.clg_last_error(), (at, value)
    assert lib.clg_top_logits(0, None, 8, 0, 8, 3, 1.0, None, None, None, None, None) == 0
    assert lib.clg_top_logits_scratch_bytes(0, 2, 8, 3) == 0 and lib.clg_top_logits_scratch_bytes(0, 2, 1 << 20, 3) > 0
    assert lib.clg_top_logits(0, p, 1 << 20, 2, 1 << 20, 3, 1.0, p, p, p, None, None) == -1 and b"scratch" in lib.clg_last_error()
    forward = [0, p, 8, p, 0, p, 64, p, 0, p, 2, 8, 3, 1.0, 1.0, 2, p, p, p, p, None]
    for at, value in [(0, 9), (1, None), (2, -8), (3, None), (4, 9), (5, None), (6, 16), (8, 9), (10, -1), (10, 1 << 31), (11, 0), (11, 1 << 31), (12, 0), (12, 1025),
                      (13, 0.0), (13, INF), (15, 3), (15, 0), (16, None), (17, None), (18, None), (19, None)]:
        args = list(forward)
        args[at] = value
        assert lib.clg_distill_forward(*args) == -1 and b"clg_distill_forward" in lib.clg_last_error(), (at, value)
        if at not in (15, 16, 18, 19) and not (at == 17):
            assert lib.clg_distill_backward(*args) == -1 and b"clg_distill_backward" in lib.clg_last_error(), (at, value)
    for at in (16, 17):
        args = list(forward)
        args[at] = None
        assert lib.clg_distill_backward(*args) == -1
    import ctypes
    one = (ctypes.c_void_p * 1)(p)
    rows, stride, bad = (ctypes.c_int64 * 1)(4), (ctypes.c_int64 * 1)(16), (ctypes.c_int64 * 1)(-1)
    balance = [0, 1, one, rows, stride, 16, 1, None, 1.0, p, p, p, p, None]
    for at, value in [(0, 5), (1, 0), (1, 17), (2, None), (3, None), (3, bad), (4, bad), (5, 0), (5, 1025), (6, 0), (6, 17), (9, None), (10, None), (11, None),
                      (12, None), (2, (ctypes.c_void_p * 1)(None))]:
        args = list(balance)
        args[at] = value
        assert lib.clg_balance_forward(*args) == -1 and b"clg_balance_forward" in lib.clg_last_error(), (at, value)
    two = [0, 2, (ctypes.c_void_p * 2)(p, p), (ctypes.c_int64 * 2)(4, 4), (ctypes.c_int64 * 2)(16, 16), 16, 1, p, 1.0, p, p, p, p, None]
    assert lib.clg_balance_forward(*two) == -1 and b"mask" in lib.clg_last_error()
    backward = [0, 1, one, rows, stride, 16, None, p, p, one, None]
    for at, value in [(0, 5), (1, 0), (7, None), (8, None), (9, None), (9, (ctypes.c_void_p * 1)(None))]:
        args = list(backward)
        args[at] = value
        assert lib.clg_balance_backward(*args) == -1 and b"clg_balance_backward" in lib.clg_last_error(), (at, value)
    assert lib.clg_balance_scratch_bytes(0, 0) == 0 and lib.clg_balance_scratch_bytes(0, 16) > 0 and lib.clg_distill_scratch_bytes(-1) == 0


def test_distillation_of_close_logits_at_a_low_temperature():
    # logits of 30 that differ in their last bits, over 1e-12: their differences count, not what is left of 3e13.  Probabilities in 50 digits
    from decimal import Decimal, localcontext
    z = 30.0 - 2.0 ** -48 * torch.tensor([[4.0, 1.0, 0.0, 7.0, 3.0]], dtype=torch.float64)
    with localcontext() as context:
        context.prec = 50
        e = [(Decimal(float(x)) / Decimal(1e-12) - Decimal(30.0) / Decimal(1e-12)).exp() for x in z[0]]
        want = [float(x / sum(e)) for x in e]
    leaf = z.requires_grad_(True)
    C.distillation_loss(leaf, torch.zeros(1, 1), torch.tensor([[2]]), temperature=1e-12, weight=1e12, reduction="sum").backward()
    want[2] -= 1.0
    assert np.abs(leaf.grad[0].numpy() - np.array(want)).max() <= 16 * 2.0 ** -53


def test_distillation_from_close_values_at_a_low_temperature():
    # float64 values of 30 that differ in their last bits, over 1e-12: their differences count.  The teacher's probabilities in 50 digits, an undecided student
    from decimal import Decimal, localcontext
    values = 30.0 - 2.0 ** -48 * torch.tensor([[4.0, 1.0, 0.0, 7.0, 3.0]], dtype=torch.float64)
    with localcontext() as context:
        context.prec = 50
        e = [((Decimal(float(v)) - 30) / Decimal(1e-12)).exp() for v in values[0]]
        p = [x / sum(e) for x in e]
        want = float(sum(x * x.ln() for x in p) + Decimal(10).ln())
    loss = C.distillation_loss(torch.zeros(1, 10, dtype=torch.float64), values, torch.arange(5)[None], temperature=1e-12, weight=1e24, reduction="sum")
    assert abs(float(loss) - want) <= 2.0 ** -46 * (want + 10)


@pytest.mark.parametrize("times", [255, 256, 257, 512, 1024])
def test_distillation_of_a_column_listed_many_times(times):
    z = scores(2, 3, torch.float64, 2).requires_grad_(True)
    columns = torch.full((2, times), 1)
    columns[1, -1] = 2
    values, lse = torch.full((2, times), -8.0, dtype=torch.float64), torch.zeros(2, dtype=torch.float64)
    loss = C.distillation_loss(z, values, columns, lse)
    grad, = torch.autograd.grad(loss, z)
    want = L.distillation(z.detach().numpy(), values.numpy(), columns.numpy(), lse.numpy())
    close(loss, want[0], want[2], "loss")
    close(grad, want[1], want[3], "grad")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
def test_distillation_of_a_student_with_nothing_beside_the_listed_columns(dtype):
    # the teacher has mass elsewhere: the loss is inf, the gradient is that of the listed columns; a row that lists every column; an ordinary one
    z = scores(4, 4, dtype, 1)
    z[0, 1:], z[1, 0], z[1, 3] = -INF, -INF, -INF
    columns = torch.tensor([[0, -1, -1, -1], [2, 1, -1, -1], [3, 0, 1, 2], [1, 2, -1, -1]])
    values, lse = torch.zeros(4, 4), torch.full((4,), 1.5)
    leaf = z.requires_grad_(True)
    loss = C.distillation_loss(leaf, values, columns, lse, reduction="none")
    grad, = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
    want = L.distillation(z.detach().double().numpy(), values.numpy(), columns.numpy(), lse.numpy(), reduction="none")
    assert loss.tolist()[:2] == [INF, INF] and want[0].tolist()[:2] == [INF, INF] and loss[2:].isfinite().all()
    close(loss[2:], want[0][2:], want[2][2:], "loss")
    close(grad, want[1], want[3], "grad")


def test_gate_balance_refuses_a_bare_tensor():
    # (its rows would each be a layer of one neuron)
    for logits in (torch.zeros(12, 16), torch.nn.Parameter(torch.zeros(3, 7, 16))):
        with pytest.raises(RuntimeError, match="sequence"):
            C.gate_balance(logits)
    assert C.gate_balance([torch.zeros(12, 16)]).counts.tolist() == [[12] + [0] * 15] and C.gate_balance(iter([torch.zeros(12, 16)])).loss == 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_distillation_of_a_listed_logit_far_above_the_others(dtype):
    # the gradient of the columns that are not listed goes by their differences among themselves: T (M q_v - p_r q_v / q_r), here -T p_r times their softmax
    z = scores(2, 9, dtype, 3)
    z[:, 4] = torch.tensor([1e30, torch.finfo(dtype).max / 4], dtype=dtype)     # (as float32 the second would be inf)
    leaf = z.requires_grad_(True)
    columns, values, lse = torch.tensor([[4, 0], [4, 0]]), torch.tensor([[1.0, 0.5], [1.0, 0.5]]), torch.full((2,), 2.0)
    grad, = torch.autograd.grad(C.distillation_loss(leaf, values, columns, lse, temperature=1.5, reduction="sum", weight=1e-3), leaf)
    others = [1, 2, 3, 5, 6, 7, 8]
    rest = 1.0 - (values.double() / 1.5 - 2.0).exp().sum(1, keepdim=True)
    want = -1.5e-3 * rest * torch.softmax(z.detach()[:, others].double() / 1.5, 1)
    assert (grad[:, others].double() - want).abs().max() <= torch.finfo(dtype).eps * want.abs().max()
