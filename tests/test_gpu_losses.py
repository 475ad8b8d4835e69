"""The kernels of the losses on scores and gate logits against their definitions in 64 bits (oracle/losses_oracle.py).

Bounds.  An exponential of a float32 argument x = (z - max) / temperature * log2(e) is off by the two roundings of x, 2 |x| 2^-24 relative, and by its
own 2 steps; the terms that matter have |x| <= X = log2(e) (max - min) / temperature, and what is further down than 2^-126 may vanish.  A sum of n such
terms in at most 160 additions in a row (128 elements of a thread, a tree over the workgroup, tiles) is off by 160 steps more.  So values are within
(2 X + 170) 2^-24 of the sum of the magnitudes they are made of, and half a step of the type they are rounded to; 2^-53 in place of 2^-24 for float64."""
import math

import numpy as np
import pytest
import torch

import convlogic_amd as C
from oracle import losses_oracle as L
from tests.gpu_util import DEV, set_knobs

pytestmark = pytest.mark.gpu

NAN, INF = math.nan, math.inf
TYPES = [torch.float32, torch.bfloat16, torch.float16, torch.float64]


def scores(rows, cols, dtype=torch.float32, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, cols, generator=g) * scale).to(dtype).to(DEV)


def spread(z, temperature=1.0):
    finite = z.detach()[torch.isfinite(z)].double()
    return min(1.4427 * float(finite.max() - finite.min()) / temperature if finite.numel() else 0.0, 150.0)


def close(got, want, size, z, name, temperature=1.0, steps=170):
    unit = 2.0 ** -53 if z.dtype == torch.float64 else 2.0 ** -24
    half = torch.finfo(got.dtype).eps / 2
    least = torch.finfo(got.dtype).smallest_normal * (1 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps)
    g = got.detach().double().cpu().numpy()
    bound = (2 * spread(z, temperature) + steps) * unit * np.asarray(size) + half * np.abs(want) * (1 + 2.0 ** -10) + least
    assert g.shape == np.shape(want), name
    assert np.array_equal(np.isnan(g), np.isnan(want)), name
    with np.errstate(invalid="ignore"):
        bad = ~(np.isnan(want) | (np.abs(g - want) <= bound) | (g == want))
    assert not bad.any(), (name, int(bad.sum()), np.abs(g - want)[bad].max(), np.broadcast_to(bound, g.shape)[bad].min())


def host(t):
    return None if t is None else t.detach().double().cpu().numpy()


# ---- top logits ----------------------------------------------------------------------------------
def check_top(z, k, temperature=1.0):
    got = C.top_logits(z, k, temperature=temperature)
    flat = z.detach().double().cpu().reshape(-1, z.shape[-1])
    values, columns, lse = [], [], []
    for row in flat:                                                  # (as the oracle, with a sort that takes long rows)
        order = np.lexsort((np.arange(len(row)), -row.nan_to_num(nan=INF, posinf=INF, neginf=-INF).numpy(), ~row.isnan().numpy()))[:k]
        columns.append(order)
        values.append(row.numpy()[order])
        lse.append(float(torch.logsumexp(row / temperature, 0)) if not row.isnan().any() else NAN)
    indices = got.indices.cpu().reshape(-1, k).numpy()
    assert np.array_equal(indices, np.array(columns)), (indices, columns)
    assert np.array_equal(got.values.double().cpu().reshape(-1, k).numpy(), np.array(values), equal_nan=True)
    assert got.values.dtype == z.dtype and got.values.shape == (*z.shape[:-1], k) and got.logsumexp.shape == z.shape[:-1]
    want = np.array(lse).reshape(got.logsumexp.shape)
    # max / temperature + log(sum) is rounded twice in 64 bits, half a step each, and so is what it is compared with: of float64 results, 4 half steps in all,
    # 3 beside the one that close() allows.  (Off by one step in 600 values near 3e13, of which the exact value was 0.59 and 0.41 away.)
    more = 3 / 170 * np.abs(np.nan_to_num(want, posinf=0, neginf=0)) if z.dtype == torch.float64 else 0
    close(got.logsumexp, want, 1 + more, z, "logsumexp", temperature)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [1, 2, 7, 8, 9, 10, 63, 64, 65, 128, 129, 255, 257, 511, 512, 513, 1000, 1025, 2047, 2049, 4097, 8191, 8193])
def test_top_logits(dtype, cols):
    for k in sorted({1, min(3, cols), min(cols, 40), min(cols, 300)}):
        check_top(scores(3, cols, dtype, cols + k), k, 1.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [16385, 32767, 32768, 32769, 65535, 65537, 131071, 131072, 131073, 200003])
def test_top_logits_of_long_rows(dtype, cols):
    for k in (1, 64, 257):
        check_top(scores(2, cols, dtype, cols + k), k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols,k", [(10, 10), (700, 700), (700, 5), (5000, 64), (5000, 1024), (40000, 20), (140000, 100), (300000, 1024)])
def test_top_logits_of_rows_that_are_hard_to_sort(dtype, cols, k):
    up = torch.linspace(-50, 50, cols, dtype=torch.float64)
    few = torch.randint(0, 3, (cols,), generator=torch.Generator().manual_seed(1)).double()
    rows = [up, up.flip(0), torch.zeros(cols, dtype=torch.float64), few, torch.full((cols,), -INF, dtype=torch.float64)]
    block = torch.randn(cols, generator=torch.Generator().manual_seed(2)).double()
    start = cols // 3
    block[start:start + 2 * k] += 100                                 # the highest next to one another
    rows.append(block)
    low = torch.full((cols,), float(torch.finfo(dtype).min), dtype=torch.float64)
    low[-1] = 0
    rows.append(low)
    check_top(torch.stack(rows).to(dtype).to(DEV), k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [9, 600, 70000, 150000])
def test_top_logits_orders_nan_infinities_and_zeros(dtype, cols):
    z = scores(4, cols, dtype, cols)
    z[0, 1], z[0, cols - 1], z[0, 4], z[0, cols // 2] = NAN, NAN, INF, -INF
    z[1] = -z[1].abs()
    z[1, cols - 2], z[1, 3] = -0.0, 0.0
    z[2] = -INF
    z[2, cols - 3] = -7.0
    z[3, 2], z[3, 6] = INF, INF
    check_top(z, 9)


def test_top_logits_of_views_streams_and_graphs():
    z = scores(40, 333, torch.float32, 1)
    for view in (z[:, 5:300], z[::3, ::2], z.t(), z.view(4, 10, 333), z.view(4, 10, 333).transpose(0, 1), z[0], z[:1].expand(5, -1)):
        check_top(view, 7)
    assert C.top_logits(z[:0], 4).values.shape == (0, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = C.top_logits(z, 7)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = C.top_logits(z, 7)
    for i in range(3):
        want = C.top_logits(z, 7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(recorded, want)) and (i or all(torch.equal(a, b) for a, b in zip(other, want)))
        z.copy_(scores(40, 333, torch.float32, 7 + i))


# ---- distillation --------------------------------------------------------------------------------
def teacher(rows, cols, k, rest, seed, temperature):
    t = C.top_logits(scores(rows, cols, torch.float32, seed + 1000), k, temperature=temperature)
    return t.values, t.indices, t.logsumexp if rest else None


def check_distill(z, values, columns, lse, temperature=1.0, mask=None, weight=1.0, reduction="mean", upstream=None):
    leaf = z.detach().requires_grad_(True)
    kw = dict(temperature=temperature, mask=mask, weight=weight, reduction=reduction)
    loss = C.distillation_loss(leaf, values, columns, lse, **kw)
    alone = C.distillation_loss(z.detach(), values, columns, lse, **kw)
    assert torch.equal(loss, alone) or bool(loss.isnan().any())
    grad, = torch.autograd.grad(loss, leaf, upstream)
    flat = (lambda t: None if t is None else t.reshape(-1, t.shape[-1]))
    want = L.distillation(host(flat(z)), host(flat(values)), flat(columns).cpu().numpy(), None if lse is None else host(lse.reshape(-1)), temperature,
                          None if mask is None else mask.reshape(-1).cpu().numpy(), weight, reduction,
                          None if upstream is None else host(upstream.reshape(-1)) if reduction == "none" else host(upstream))
    close(loss, np.reshape(want[0], loss.shape), np.reshape(want[2], loss.shape), z, "loss", temperature)
    close(grad, np.reshape(want[1], grad.shape), np.reshape(want[3], grad.shape), z, "grad", temperature)
    assert grad.dtype == z.dtype
    return loss, grad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("cols", [1, 2, 7, 8, 9, 10, 33, 64, 127, 255, 256, 257, 511, 513, 1000, 2047, 2049, 4100, 8191, 8193])
def test_distillation(dtype, rest, cols):
    for k in sorted({1, min(4, cols), min(33, cols), min(300, cols)}):
        z = scores(3, cols, dtype, cols)
        check_distill(z, *teacher(3, cols, k, rest, k, 2.0), temperature=2.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("cols", [16385, 32768, 32769, 65535, 65536, 65537, 131071, 131072, 131073, 200003])
def test_distillation_over_long_rows(dtype, rest, cols):
    z = scores(2, cols, dtype, cols)
    check_distill(z, *teacher(2, cols, 64, rest, 3, 1.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("cols", [10, 301, 9000])
def test_distillation_of_padded_rows(dtype, reduction, cols):
    z = scores(7, cols, dtype, 5)
    values, columns, _ = teacher(7, cols, 6, False, 5, 1.5)
    columns[0, 3:], columns[1], columns[2, 0] = -1, -5, -1            # short rows, one without entries
    mask = torch.tensor([True, True, True, False, True, False, True], device=DEV)
    z[3], z[5, 0], z[1, 2] = NAN, INF, NAN                            # rows that do not count
    up = torch.rand(7, device=DEV).to(torch.float64 if dtype == torch.float64 else torch.float32)
    up = up if reduction == "none" else up[0]
    _, grad = check_distill(z, values, columns, None, 1.5, mask, 0.3, reduction, up)
    assert (grad[[1, 3, 5]] == 0).all()
    none = C.distillation_loss(z, values, columns, mask=torch.zeros_like(mask), reduction=reduction)
    assert (none == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [12, 700, 70000, 140000])
def test_distillation_of_special_values(dtype, cols):
    # columns that the student masks, by -inf and by the type's lowest value; a row that is lowest everywhere; all scores far below zero
    z = scores(5, cols, dtype, 6)
    values, columns, lse = teacher(5, cols, 5, True, 6, 1.0)
    for r in range(5):
        free = [c for c in range(8) if c not in columns[r].tolist()]
        z[r, free[0]] = -INF
        z[r, free[1]] = torch.finfo(dtype).min
    z[3] = torch.finfo(dtype).min
    z[4] -= 500.0
    for r in (slice(0, 3), slice(3, 4), slice(4, 5)):
        for l in (None, lse[r]):
            check_distill(z[r], values[r], columns[r], l)
    # the teacher has mass where the student has none
    x = scores(2, cols, dtype, 7)
    x[1, columns[1, 0]] = -INF
    loss = C.distillation_loss(x, values[:2], columns[:2], reduction="none")
    assert loss[0].isfinite() and loss[1] == INF
    # a student that has nothing but the listed columns
    y = torch.full((1, cols), -INF, dtype=dtype, device=DEV)
    y[0, columns[0]] = 1.0
    assert C.distillation_loss(y, values[:1], columns[:1]).isfinite() and C.distillation_loss(y, values[:1], columns[:1], lse[:1]) == INF
    # NaN and +inf of the student, NaN of the teacher, a column behind the last: their own rows
    x = scores(5, cols, dtype, 8).requires_grad_(True)
    v, c = values.clone(), columns.clone()
    with torch.no_grad():
        x[0, [i for i in range(8) if i not in c[0].tolist()][0]] = NAN
        x[1, 3] = INF
    v[2, 1] = NAN
    c[3, 4] = cols
    for l in (None, lse):
        loss = C.distillation_loss(x, v, c, l, reduction="none")
        grad, = torch.autograd.grad(loss.sum(), x)
        assert loss.isnan().tolist() == [True, True, True, True, False]
        assert grad.isnan().any(1).tolist() == [True, True, True, True, False]
    # teacher's values of -inf are no mass
    v = values.clone()
    v[0, 2], v[1] = -INF, -INF
    check_distill(scores(5, cols, dtype, 9), v, columns, None)
    check_distill(scores(5, cols, dtype, 9), v, columns, lse)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols,k", [(3, 3), (40, 7), (40, 100), (3000, 700), (70000, 1024), (140000, 50)])
def test_distillation_of_columns_listed_twice(dtype, cols, k):
    g = torch.Generator().manual_seed(k)
    columns = torch.randint(0, cols, (4, k), generator=g).to(DEV)
    columns[:, k // 2] = columns[:, 0]
    columns[1] = columns[1, 0]
    values = torch.randn(4, k, generator=g).to(DEV)
    check_distill(scores(4, cols, dtype, 3), values, columns, None)
    check_distill(scores(4, cols, dtype, 3), values, columns, torch.logsumexp(values, 1) + 1.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_distillation_of_every_type_shape_and_layout_of_its_arguments(dtype):
    z = scores(6, 50, dtype, 1)
    values, columns, lse = teacher(6, 50, 4, True, 1, 1.0)
    want = check_distill(z, values, columns, lse)
    for c in (columns.int(), columns.t().contiguous().t()):
        got = check_distill(z, values, c, lse)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for t in TYPES:
        check_distill(z, values.to(t), columns, None)
        check_distill(z, values.to(t), columns, lse.to(t))
    wide = scores(12, 60, dtype, 2)
    for view in (wide[::2, 3:53], wide[:6, :50], wide[:6, ::1][:, 10:], wide[6:, 5:55], wide[:1, :50].expand(6, -1)):
        check_distill(view, values, columns, lse)
    strided = scores(50, 6, dtype, 3).t()
    check_distill(strided, values, columns, lse)
    three = (z.view(2, 3, 50), values.view(2, 3, 4), columns.view(2, 3, 4), lse.view(2, 3))
    for reduction in ("mean", "none"):
        check_distill(*three, reduction=reduction, upstream=torch.ones(2, 3, device=DEV, dtype=lse.dtype if dtype != torch.float64 else dtype) if reduction == "none" else None)
    check_distill(three[0].transpose(0, 1), three[1].transpose(0, 1), three[2].transpose(0, 1), three[3].transpose(0, 1))
    check_distill(z[0], values[0], columns[0], lse[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [10, 3000])
@pytest.mark.parametrize("masked", [False, True])
def test_distillation_under_other_upstream_gradients_and_retained_graphs(dtype, cols, masked):
    z = scores(5, cols, dtype, 2).requires_grad_(True)
    values, columns, lse = teacher(5, cols, 4, True, 2, 1.0)
    mask = torch.tensor([True, False, True, True, True], device=DEV) if masked else None
    call = lambda: C.distillation_loss(z, values, columns, lse, mask=mask)
    one, = torch.autograd.grad(call(), z)
    half, = torch.autograd.grad(0.5 * call(), z)
    assert torch.equal(half.double() * 2, one.double()) or dtype == torch.float16      # (powers of two are exact but for subnormal halves)
    loss = call()
    first, = torch.autograd.grad(loss, z, retain_graph=True)
    keep = first.clone()
    first.mul_(7)                                                     # the receiver's to change
    second, = torch.autograd.grad(loss, z, torch.full_like(loss, 0.5), retain_graph=True)
    third, = torch.autograd.grad(loss, z)
    assert torch.equal(keep, one) and torch.equal(second, half) and torch.equal(third, one) and torch.equal(first, keep * 7)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(loss, z)
    z.grad = None
    call().backward()
    call().backward()
    assert torch.equal(z.grad, one + one)
    zero, = torch.autograd.grad(call() * 0.0, z)
    assert (zero == 0).all()
    with torch.no_grad():
        assert not call().requires_grad
    # a second differentiation is refused, not answered with zero
    g, = torch.autograd.grad(call(), z, create_graph=True)
    assert torch.equal(g, one)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        g.double().sum().backward()
    # logits that change between the passes
    x = z.detach().clone().requires_grad_(True)
    y = x * 1
    loss = C.distillation_loss(y, values, columns, lse)
    y.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    again = torch.utils.checkpoint.checkpoint(lambda t: C.distillation_loss(t, values, columns, lse, mask=mask), z, use_reentrant=False)
    assert torch.equal(torch.autograd.grad(again, z)[0], one)


def test_distillation_of_many_rows():
    # more rows than workgroups of the pass that looks at another upstream gradient
    z = scores(5000, 17, torch.float32, 4)
    t = teacher(5000, 17, 3, True, 4, 1.0)
    check_distill(z, *t)
    check_distill(z, *t, mask=torch.arange(5000, device=DEV) % 3 > 0, upstream=torch.tensor(0.3, device=DEV))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("cols,k", [(9, 3), (100, 20), (250, 64), (251, 65), (900, 5), (2047, 7)])
def test_distillation_of_rows_that_share_a_wavefront(monkeypatch, dtype, rest, cols, k):
    # the last wavefront not full; some rows without entries, masked, with other rows' special values beside them
    set_knobs(monkeypatch, CLG_DISTILL_LANES=16)
    rows = 2050
    z = scores(rows, cols, dtype, cols)
    values, columns, lse = teacher(rows, cols, k, rest, k, 1.5)
    mask = torch.arange(rows, device=DEV) % 5 != 2
    z[2] = NAN
    z[9] -= 300.0
    if not rest:
        columns[4] = -1
        columns[5, 1:] = -1
    columns[13, 0] = columns[13, -1]
    check_distill(z, values, columns, lse, 1.5, mask, 0.5, "mean", torch.tensor(3.0, device=DEV, dtype=torch.float64 if dtype == torch.float64 else torch.float32))
    x = z[:2049].clone().requires_grad_(True)
    columns[8, 0] = cols
    loss = C.distillation_loss(x, values[:2049], columns[:2049], None if lse is None else lse[:2049], mask=mask[:2049], reduction="none")
    grad, = torch.autograd.grad(loss.sum(), x)
    assert loss.isnan().nonzero().tolist() == [[8]] and grad.isnan().any(1).nonzero().tolist() == [[8]]


@pytest.mark.parametrize("past", [0, 1 << 20])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_through_and_past_the_caches(monkeypatch, dtype, past):
    # the accesses that large tensors get, on small ones
    set_knobs(monkeypatch, CLG_STREAM_MB=past)
    for cols in (64, 100, 1024, 1027, 20000, 40000, 66000, 140000):
        z = scores(3, cols, dtype, cols)
        check_top(z, 20)
        check_distill(z, *teacher(3, cols, 20, True, 1, 1.0))
    z = scores(2100, 128, dtype, 1)
    check_distill(z, *teacher(2100, 128, 9, True, 1, 1.0))
    for experts in (16, 60, 256):
        check_balance(scores(70, experts, dtype, experts), 2)


def test_rows_beyond_two_to_the_31_elements_and_threads():
    # element 2^31 and more: the last rows as the same rows alone
    rows, cols = 16500, 131072
    z = torch.empty(rows, cols, dtype=torch.bfloat16, device=DEV)
    z.normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    answers = C.top_logits(z, 5)
    some = [0, 8000, rows - 2, rows - 1]
    check_top(z[some], 5)
    for got, want in zip(answers, C.top_logits(z[some], 5)):
        assert torch.equal(got[some], want)
    leaf = z.requires_grad_(True)
    loss = C.distillation_loss(leaf, *answers, reduction="none")
    grad, = torch.autograd.grad(loss.sum(), leaf)
    alone = z.detach()[some].requires_grad_(True)
    of_alone = C.distillation_loss(alone, *(t[some] for t in answers), reduction="none")
    assert torch.equal(loss[some], of_alone) and torch.equal(grad[some], torch.autograd.grad(of_alone.sum(), alone)[0])
    del z, leaf, grad, loss
    # more rows than 2^32 threads have, of any of the teams that a row can get
    rows = (1 << 28) + 6
    z = (torch.arange(2 * rows, device=DEV, dtype=torch.int32) % 7).view(rows, 2).half()
    values, columns = torch.zeros(rows, 1, dtype=torch.float16, device=DEV), torch.ones(rows, 1, dtype=torch.int32, device=DEV)
    loss = C.distillation_loss(z, values, columns, reduction="none")
    total = C.distillation_loss(z, values, columns, reduction="sum")
    want = torch.nn.functional.softplus(torch.arange(-6, 7, device=DEV).double())      # log(1 + e^(z0 - z1))
    for part in (slice(0, 1000), slice(rows // 2, rows // 2 + 1000), slice(rows - 1000, rows)):
        d = (z[part, 0] - z[part, 1]).long() + 6
        assert (loss[part].double() - want[d]).abs().max() <= 2.0 ** -24 * 400
    assert abs(float(total) - float(loss.double().sum())) <= 1e-6 * float(total)
    top = C.top_logits(z[: (1 << 25) + 70], 1)                        # (64 threads to a row)
    assert torch.equal(top.values[-1000:, 0], z[(1 << 25) - 930:(1 << 25) + 70].max(1).values)


@pytest.mark.parametrize("rows", [15, 16, 17, 1023, 16385, 70000, 200001])
def test_the_mean_over_many_masked_rows(rows):
    z = scores(rows, 3, torch.float32, 1)
    values, columns, _ = teacher(rows, 3, 1, False, 1, 1.0)
    kept = torch.rand(rows + 3, device=DEV)[3:] < 0.6
    each = C.distillation_loss(z, values, columns, reduction="none").double()
    for mask in (kept, torch.ones_like(kept), torch.zeros_like(kept)):
        n = max(int(mask.sum()), 1)
        for reduction, want in (("mean", each[mask].sum() / n), ("sum", each[mask].sum())):
            assert abs(float(C.distillation_loss(z, values, columns, mask=mask, reduction=reduction)) - float(want)) <= 2.0 ** -22 * float(want)


def test_what_autograd_offers_around_the_losses():
    z = scores(8, 300, torch.float32, 1).requires_grad_(True)
    t = teacher(8, 300, 5, True, 1, 1.0)
    call = lambda x: C.distillation_loss(x, *t) + C.balance_loss(x, 3).loss
    want, = torch.autograd.grad(call(z), z)
    moved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda s: moved.append(1) or s.cpu(), lambda s: s.to(DEV)):
        got, = torch.autograd.grad(call(z), z)
        half, = torch.autograd.grad(0.5 * call(z), z)
    assert moved and torch.equal(got, want) and torch.equal(half * 2, want)
    for one in (lambda x: C.distillation_loss(x, *(s[0] for s in t)), lambda x: C.balance_loss(x, 3).loss, lambda x: C.top_logits(x, 3).values):
        with pytest.raises(RuntimeError):
            torch.func.vmap(one)(z.detach())
    with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError):
        call(torch.autograd.forward_ad.make_dual(z.detach(), torch.ones_like(z)))


# ---- balance -------------------------------------------------------------------------------------
def check_balance(z, k, mask=None, weight=1.0):
    leaf = z.detach().requires_grad_(True)
    loss, counts = C.balance_loss(leaf, k, mask=mask, weight=weight)
    grad, = torch.autograd.grad(loss, leaf)
    flat = z.reshape(-1, z.shape[-1])
    want = L.balance(host(flat), k, None if mask is None else mask.reshape(-1).cpu().numpy(), weight)
    assert counts.cpu().tolist() == want[1].tolist() and counts.dtype == torch.int64
    close(loss, want[0], abs(want[0]), z, "loss")
    close(grad, np.reshape(want[2], grad.shape), np.reshape(want[3], grad.shape), z, "grad")
    return loss, counts, grad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("experts", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 60, 64, 65, 128, 130, 200, 256, 257, 512, 600, 1023, 1024])
def test_balance(dtype, experts):
    for rows, k in ((1, 1), (37, min(3, experts)), (130, min(8, experts))):
        check_balance(scores(rows, experts, dtype, experts), k, None, 0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("experts,k", [(4, 4), (16, 1), (16, 16), (60, 33), (300, 5)])
def test_balance_of_padded_and_masked_rows(dtype, experts, k):
    z = scores(200, experts, dtype, 3)
    z[5], z[6] = -INF, NAN                                            # no row at all; one that the mask leaves out
    z[7, 1:] = -INF                                                   # one expert left
    z[8] = torch.finfo(dtype).min
    z[9, 0] = torch.finfo(dtype).min
    z[10] = 0.0                                                       # ties
    z[11] = scores(1, experts, dtype, 4).round()
    mask = torch.arange(200, device=DEV) % 5 != 1
    _, _, grad = check_balance(z, k, mask)
    assert (grad[5] == 0).all() and (grad[6] == 0).all()
    nothing = C.balance_loss(z.requires_grad_(True), k, mask=torch.zeros_like(mask))
    assert nothing.loss == 0 and (nothing.counts == 0).all() and (torch.autograd.grad(nothing.loss, z)[0] == 0).all()
    assert C.balance_loss(z, k).loss.isnan()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("experts,k", [(1, 1), (8, 1), (20, 3), (300, 5)])
def test_balance_counts_a_nan_as_the_maximum(dtype, experts, k):
    # a NaN at each expert in turn, alone, behind and in front of +inf, and between experts of -inf; rows of NaN: counts are integers, those of the plain form
    z = scores(4 * experts + 1, experts, dtype, 11)
    for e in range(experts):
        z[4 * e:4 * e + 4, e] = NAN
        z[4 * e + 1, e - 1] = INF
        z[4 * e + 2, e // 2] = INF
        z[4 * e + 3] = torch.where(z[4 * e + 3].isnan(), z[4 * e + 3], -INF)
    z[-1] = NAN
    for rows in (slice(None), slice(0, 1), slice(0, 4), slice(-1, None)):
        assert torch.equal(C.balance_loss(z[rows], k).counts.cpu(), C.balance_loss(z[rows].cpu(), k).counts)


@pytest.mark.parametrize("rows,experts,k,dtype", [(40000, 16, 1, torch.float32), (9000, 64, 8, torch.bfloat16), (20011, 5, 2, torch.float32)])
def test_balance_of_many_rows(rows, experts, k, dtype):
    z = scores(rows, experts, dtype, 8)
    p = torch.softmax(z.double(), 1)
    chosen = torch.zeros_like(p).scatter_(1, torch.sort(z.double(), dim=1, descending=True, stable=True).indices[:, :k], 1.0)
    w = chosen.sum(0) * experts / (k * float(rows) ** 2)
    leaf = z.requires_grad_(True)
    loss, counts = C.balance_loss(leaf, k)
    grad, = torch.autograd.grad(loss, leaf)
    mean = (p * w).sum(1, keepdim=True)
    assert torch.equal(counts, chosen.sum(0).long())
    close(loss, float((w * p.sum(0)).sum()), float((w * p.sum(0)).sum()), z, "loss", steps=600)      # (rows / 1024 workgroups * lanes: 160 in a row at most)
    close(grad, (p * (w - mean)).cpu().numpy(), (p * (w + mean)).cpu().numpy(), z, "grad")
    again = C.balance_loss(leaf, k)
    assert torch.equal(again.loss, loss) and torch.equal(torch.autograd.grad(again.loss * 2, leaf)[0].double(), 2 * grad.double())


def test_balance_of_views_and_shapes():
    z = scores(60, 48, torch.float32, 1)
    for view in (z[:, 4:36], z[::2, ::3], z.t(), z.view(3, 20, 48), z.view(3, 20, 48).transpose(0, 1), z[0], z[:1].expand(7, -1)):
        check_balance(view, 2)
    check_balance(z.view(3, 20, 48), 2, torch.rand(3, 20, device=DEV) < 0.7)
    empty = C.balance_loss(z[:0])
    assert empty.loss == 0 and (empty.counts == 0).all()
    leaf = z.clone().requires_grad_(True)
    loss = C.balance_loss(leaf, 2).loss
    one, = torch.autograd.grad(loss, leaf, retain_graph=True)
    assert torch.equal(torch.autograd.grad(loss, leaf)[0], one)
    g, = torch.autograd.grad(C.balance_loss(leaf, 2).loss, leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        g.sum().backward()


def huge(dtype, cols, base, seed=0):
    # rows of a value, and of it with neighbours a few steps of the type away; of values of every size up to it
    g = torch.Generator().manual_seed(seed)
    step = abs(base) * torch.finfo(dtype).eps * (2 if dtype == torch.float64 else 1)
    near = base - step * torch.randint(0, 9, (2, cols), generator=g).double()
    sizes = torch.tensor([-1.0, -0.3, 1e-3, 0.5, 0.9, 1.0], dtype=torch.float64) * abs(base)
    mixed = sizes[torch.randint(0, 6, (2, cols), generator=g)]
    one = torch.randn(1, cols, generator=g).double()
    one[0, cols // 2] = base
    return torch.cat([torch.full((1, cols), base, dtype=torch.float64), near, mixed, one]).to(dtype).to(DEV)


# (losses, about |base| temperature weight, and logsumexps, |base| / temperature, within float32)
HUGE = [(torch.float32, 1e10, 1.0), (torch.float32, -1e20, 1.0), (torch.float32, -1e38, 1.0), (torch.float32, 1e30, 1e5), (torch.float32, -30.0, 1e-12),
        (torch.float32, 1e6, 1e-25), (torch.bfloat16, -1e10, 1.0), (torch.bfloat16, -1e38, 1.0), (torch.bfloat16, 7.0, 1e-10), (torch.float16, -6e4, 1e-6),
        (torch.float16, 20.0, 1e-15), (torch.float64, -1e20, 1.0), (torch.float64, 30.0, 1e-12)]


@pytest.mark.parametrize("dtype,base,temperature", HUGE)
@pytest.mark.parametrize("cols", [5, 600, 9000, 140000])
def test_logits_far_beyond_what_an_exponential_takes(dtype, base, temperature, cols):
    z = huge(dtype, cols, base)
    check_top(z, min(cols, 4), temperature)
    values, columns, lse = teacher(len(z), cols, min(cols, 4), cols < 9000, 3, 1.0)
    if lse is not None and cols > 5:
        lse += math.log(2.0)                                          # (half of its answers are elsewhere)
    check_distill(z, (values.double() * temperature).float(), columns, lse, temperature, weight=max(1.0, 1.0 / temperature))
    if cols <= 1024:
        check_balance(z, 3)


@pytest.mark.parametrize("dtype", TYPES)
def test_gate_balance(dtype):
    sizes = [7, 1, 300, 0, 64, 5000, 16, 33, 2, 90, 11, 5, 8, 70, 129, 31, 40, 3]    # more than one launch takes
    tensors = [scores(n, 16, dtype, n).requires_grad_(n != 64) for n in sizes]
    loss, counts = C.gate_balance(tensors, weight=3.0)
    wanted = [t for t in tensors if t.requires_grad]
    grads = iter(torch.autograd.grad(loss, wanted))
    total = 0.0
    for t, c in zip(tensors, counts):
        want = L.balance(host(t), 1, None, 3.0 / len(tensors))
        total += want[0]
        assert c.cpu().tolist() == want[1].tolist()
        if t.requires_grad:
            close(next(grads), want[2], want[3], t, "grad")
    close(loss, np.array(total), np.array(total), tensors[5], "loss", steps=300)


# ---- together ------------------------------------------------------------------------------------
def networks():
    torch.manual_seed(11)
    big, small = C.ConvLogicMnistModel(k_param=6).to(DEV).eval(), C.ConvLogicMnistModel(k_param=2).to(DEV)
    with torch.no_grad():
        for p in [*big.parameters(), *small.parameters()]:
            p.add_(torch.randn(p.shape, device=DEV))
    x = (torch.rand(40, 1, 28, 28, device=DEV) < 0.5).float()
    return big, small, x


def test_a_student_learns_from_a_teachers_answers():
    # answers of a larger network, the student's loss against them, the balance of its gates: gradients of the whole against the plain forms' in float64
    big, small, x = networks()
    with torch.no_grad():
        answers = C.top_logits(big(x), 4, temperature=2.0)
    params = list(small.parameters())
    scores_ = small(x)
    loss = C.distillation_loss(scores_, *answers, temperature=2.0) + C.gate_balance(small, weight=0.1).loss
    got = torch.autograd.grad(loss, [scores_, *params])
    again = small(x)
    plain = scores_.detach().cpu().double().requires_grad_(True)
    cpu = [p.detach().cpu().double().requires_grad_(True) for p in params]
    host_loss = C.distillation_loss(plain, *(t.cpu() for t in answers), temperature=2.0)
    host_balance = C.gate_balance(cpu, weight=0.1).loss
    assert abs(float(host_loss + host_balance) - float(loss)) <= 1e-5 * abs(float(loss))
    of_scores, = torch.autograd.grad(host_loss, plain)
    assert (got[0].cpu().double() - of_scores).abs().max() <= 1e-5 * of_scores.abs().max()
    through = torch.autograd.grad(again, params, of_scores.float().to(DEV))
    for g, a, b in zip(got[1:], through, torch.autograd.grad(host_balance, cpu)):
        want = a.double().cpu() + b
        assert (g.double().cpu() - want).abs().max() <= 1e-4 * want.abs().max() + 1e-9


def test_the_step_replays_from_a_graph():
    big, small, x = networks()
    with torch.no_grad():
        answers = C.top_logits(big(x), 4, temperature=2.0)
    mask = torch.arange(40, device=DEV) % 4 != 3

    def loss_of(x, values, columns, lse, mask):
        return 0.5 * C.distillation_loss(small(x), values, columns, lse, temperature=2.0, mask=mask) + C.gate_balance(small, weight=0.1).loss

    step = C.GraphedStep(loss_of, (x, *answers, mask), small.parameters())
    params = list(small.parameters())
    for i in range(4):
        x = (torch.rand(40, 1, 28, 28, device=DEV) < 0.4 + 0.05 * i).float()
        with torch.no_grad():
            answers = C.top_logits(big(x), 4, temperature=2.0)
        mask = mask.roll(1)
        loss = step(x, *answers, mask).clone()
        got = [p.grad.clone() for p in params]
        torch.cuda.synchronize()
        with torch.enable_grad():
            eager = loss_of(x, *answers, mask)
            want = torch.autograd.grad(eager, params)
        assert torch.equal(loss, eager.detach())
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_recorded_steps_share_nothing():
    z, w = scores(64, 700, torch.bfloat16, 1), scores(64, 700, torch.bfloat16, 2)
    t = teacher(64, 700, 8, True, 1, 1.0)
    steps = [C.GraphedStep(lambda x, m: C.distillation_loss(x, *t, mask=m, weight=c), (s, torch.ones(64, dtype=torch.bool, device=DEV)), [], input_grads=True)
             for s, c in ((z, 1.0), (w, 0.5))]
    for i in range(3):
        m = torch.arange(64, device=DEV) % (i + 2) > 0
        for s in steps:
            s(s.inputs[0].detach().clone(), m)
        torch.cuda.synchronize()
        for s, c in zip(steps, (1.0, 0.5)):
            leaf = s.inputs[0].detach().clone().requires_grad_(True)
            loss = C.distillation_loss(leaf, *t, mask=m, weight=c)
            assert torch.equal(loss, s.loss) and torch.equal(torch.autograd.grad(loss, leaf)[0], s.input_grads[0])


def test_calls_on_another_stream_and_refusals_on_the_gpu():
    z = scores(300, 2000, torch.bfloat16, 1).requires_grad_(True)
    t = teacher(300, 2000, 8, True, 1, 1.0)
    want = torch.autograd.grad(C.distillation_loss(z, *t), z)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = torch.autograd.grad(C.distillation_loss(z, *t), z)[0]
        balanced = C.balance_loss(z, 3) if z.shape[1] <= 1024 else None
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and balanced is None
    for call in (lambda: C.distillation_loss(z, t[0].cpu(), t[1], t[2]), lambda: C.distillation_loss(z, *t, mask=torch.ones(300, dtype=torch.bool)),
                 lambda: C.gate_balance([torch.zeros(2, 16, device=DEV), torch.zeros(2, 16)]), lambda: C.balance_loss(z[:, :9], mask=torch.ones(300, dtype=torch.bool))):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda a: C.top_logits(a, 2).values, z.detach()[:3, :5])


# ---- students that are close to their teacher ----------------------------------------------------
def check_close_student(z, values, columns, lse, temperature):
    """Loss and gradient of each row within what 32 bits in the sum over the columns that are not listed can do, and nothing else.

    That sum s has a relative error d of at most eps = (2 X + 4 + A) 2^-24: X, the mean of |x| = log2(e) (max - z) / temperature over the columns in it, weighted
    with their shares (two roundings of x, of |x| 2^-24 each), 2 steps of the exponential itself, A additions in a row of half a step each: a thread's elements, 11
    to join up to 1024 threads, one for each tile of a row in tiles.  Everything else of a row is in 64 bits, where the terms that cancel are off by 2^-44 of their
    size.  With q_r the share of those columns, p_r the teacher's and M its whole mass:
        loss = T^2 (... + M log(total) - p_r log(s)):  off by T^2 |M q_r - p_r| d, and d^2 of T^2 M q_r
        gradient, listed: T (M q - p), off by T M q q_r d;  others: T q_v / q_r (M q_r - p_r), where M q_r is off by itself times d, the rest by d and
        the error of its own exponential, (2 |x| + 4) 2^-24, and by two products in 32 bits
    and results are rounded once to their type."""
    leaf = z.detach().requires_grad_(True)
    loss = C.distillation_loss(z, values, columns, lse, temperature=temperature, reduction="none")
    grad, = torch.autograd.grad(C.distillation_loss(leaf, values, columns, lse, temperature=temperature, reduction="sum"), leaf)
    args = (host(values), columns.cpu().numpy(), None if lse is None else host(lse), temperature, None, 1.0)
    want_loss, want_grad, size, _ = L.distillation(host(z), *args, "none")
    unit = 2.0 ** -53 if z.dtype == torch.float64 else 2.0 ** -24
    for r, row in enumerate(host(z)):
        listed = np.zeros(len(row), bool)
        listed[columns[r].cpu().numpy()] = True
        x = np.where(listed, -INF, (row - row[~listed].max()) / temperature * math.log2(math.e))
        share = np.exp2(x) / np.exp2(x).sum()
        q = np.exp((row - row.max()) / temperature)
        q /= q.sum()
        q_r = q[~listed].sum()
        t = host(values)[r] / temperature
        p = np.exp(t - host(lse)[r]) if lse is not None else np.exp(t - t.max()) / np.exp(t - t.max()).sum()
        p_r = max(0.0, 1 - p.sum()) if lse is not None else 0.0
        mass = p.sum() + p_r
        x = np.where(listed, 0.0, -x)
        eps = (2 * (share * x).sum() + 4 + min(129, len(row) // 16 + 16) + 11 + len(row) // 16384) * unit
        bound = temperature ** 2 * (abs(mass * q_r - p_r) * eps + mass * q_r * eps ** 2) + 2.0 ** -44 * size[r]
        half = torch.finfo(loss.dtype).eps / 2
        off = abs(float(loss[r]) - want_loss[r])
        assert off <= bound + half * abs(want_loss[r]) * (1 + 2.0 ** -10), ("loss", r, off, bound, want_loss[r])
        own = np.where(listed, mass * q * q_r * eps, share * (abs(mass * q_r - p_r) * (eps + (2 * x + 6) * unit) + mass * q_r * eps))
        half, least = torch.finfo(grad.dtype).eps / 2, torch.finfo(torch.float32).smallest_normal + torch.finfo(grad.dtype).smallest_normal * torch.finfo(grad.dtype).eps
        bound = temperature * (own + 2.0 ** -44 * (mass * q + listed)) + half * np.abs(want_grad[r]) * (1 + 2.0 ** -10) + unit * np.abs(want_grad[r]) + least
        off = np.abs(host(grad)[r] - want_grad[r])
        assert (off <= bound).all(), ("grad", r, (off / bound).max(), np.argmax(off / bound))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("noise", [1e-2, 1e-1])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("cols", [10, 100, 1000, 5000, 40000, 140000])
def test_distillation_of_a_student_close_to_its_teacher(dtype, noise, rest, cols):
    for rows in (1, 4):
        for k in (1, 2, 8):
            for temperature in (1.0, 4.0):
                z = scores(rows, cols, dtype, cols + k)
                own = z.float() + noise * scores(rows, cols, torch.float32, k, 1.0)
                t = C.top_logits(own, k, temperature=temperature)
                check_close_student(z, t.values, t.indices, t.logsumexp if rest else None, temperature)


@pytest.mark.parametrize("lanes", [16, 64])
def test_distillation_of_close_students_that_share_a_wavefront(monkeypatch, lanes):
    set_knobs(monkeypatch, CLG_DISTILL_LANES=lanes)
    for cols in (17, 100, 250, 1000):
        z = scores(9, cols, torch.float32, cols)
        t = C.top_logits(z + 0.01 * scores(9, cols, torch.float32, 1, 1.0), 4, temperature=4.0)
        check_close_student(z, *t, 4.0)
        check_close_student(z, t.values, t.indices, None, 4.0)


def far_values(kind, rows, k, low, high):
    # the two highest equal, one far below, the others in between or far below too
    v = torch.full((rows, k), low, dtype=kind)
    v[:, :2] = high
    return v.to(DEV)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [10, 600, 9000, 140000])
@pytest.mark.parametrize("kind,high,low,temperature", [
    (torch.float32, 3.3e30, -3.3e30, 1.5), (torch.float32, -1e30, -3.3e30, 1.5), (torch.float32, 1e30, 9e29, 1.5), (torch.float32, -3.4028234663852886e38, -INF, 0.9),
    (torch.float32, 3.4028234663852886e38, -3.4028234663852886e38, 0.9), (torch.float32, 30.0, 29.9, 1e-10), (torch.float32, -7.3, -7.4, 1e-10),
    (torch.bfloat16, 3.3895313892515355e38, 1.0, 0.9), (torch.float16, 65504.0, -65504.0, 1e-7), (torch.float64, 1e300, -1e300, 0.9), (torch.float64, -1e100, -1.1e100, 1.5)])
def test_distillation_from_values_far_beyond_what_an_exponential_takes(dtype, cols, kind, high, low, temperature):
    # (differences of the values over the temperature are 0 or beyond 1000, so that each has its probability, 1/2 or 0)
    z = scores(3, cols, dtype, 5)
    columns = torch.arange(4, device=DEV).repeat(3, 1)
    values = far_values(kind, 3, 4, low, high)
    columns[2, 1] = -1                                                # (one of the two alone)
    loss, _ = check_distill(z, values, columns, None, temperature, weight=max(1.0, 1.0 / temperature), reduction="none", upstream=torch.ones(3, device=DEV, dtype=C.distillation_loss(z, values, columns).dtype))
    assert loss.isfinite().all() and (loss[:2] != 0).all()            # (the last is 0 where an all but certain student has the one answer of its teacher)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [10, 600, 9000])
def test_distillation_from_close_values_at_a_low_temperature(dtype, cols):
    # float64 values of 30 that differ in their last bits, over 1e-12; an undecided student.  The teacher's probabilities in 50 digits
    from decimal import Decimal, localcontext
    values = 30.0 - 2.0 ** -48 * torch.tensor([[4.0, 1.0, 0.0, 7.0, 3.0]], dtype=torch.float64)
    with localcontext() as context:
        context.prec = 50
        e = [((Decimal(float(v)) - 30) / Decimal(1e-12)).exp() for v in values[0]]
        p = [x / sum(e) for x in e]
        want = float(sum(x * x.ln() for x in p) + Decimal(cols).ln())
    loss = C.distillation_loss(torch.zeros(1, cols, dtype=dtype, device=DEV), values.to(DEV), torch.arange(5, device=DEV)[None], temperature=1e-12, weight=1e24, reduction="sum")
    # (equal logits: their exponentials are 1 and sums of them whole numbers; the rest is in 64 bits, and T^2 weight is 1 but for 3 roundings)
    assert abs(float(loss) - want) <= torch.finfo(loss.dtype).eps / 2 * want + 2.0 ** -46 * (want + 10)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [10, 600, 9000, 140000])
def test_distillation_of_a_student_with_nothing_beside_the_listed_columns(dtype, cols):
    # the teacher has mass elsewhere: the loss is inf, the gradient is that of the listed columns
    values, columns, lse = teacher(3, cols, 5, True, 1, 1.0)
    z = torch.full((3, cols), -INF, dtype=dtype, device=DEV)
    z.scatter_(1, columns, scores(3, 5, dtype, 2))
    z[2] = scores(1, cols, dtype, 3)[0]
    leaf = z.requires_grad_(True)
    loss = C.distillation_loss(leaf, values, columns, lse, reduction="none")
    grad, = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
    want = L.distillation(host(z), host(values), columns.cpu().numpy(), host(lse), reduction="none")
    assert loss.tolist()[:2] == [INF, INF] and want[0].tolist()[:2] == [INF, INF]
    close(loss[2], want[0][2], want[2][2], z, "loss")
    close(grad, want[1], want[3], z, "grad")


def test_a_recorded_backward_pass_replays_without_its_forward_pass():
    # forward and backward pass in a graph each: the second is replayed again after its gradient was changed by its receiver
    z = scores(12, 300, torch.float32, 1).requires_grad_(True)
    t = teacher(12, 300, 5, True, 1, 1.0)
    want, = torch.autograd.grad(C.distillation_loss(z, *t), z)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    forward, backward = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(forward, stream=stream):
        loss = C.distillation_loss(z, *t)
    up = torch.ones_like(loss)
    with torch.cuda.graph(backward, pool=forward.pool(), stream=stream):
        grad, = torch.autograd.grad(loss, z, up, retain_graph=True)
    for i in range(4):
        if i % 2 == 0:
            forward.replay()
        backward.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad, want), i
        with torch.no_grad():
            grad.mul_(7)                                              # (the receiver's to change)
        torch.cuda.synchronize()


def test_forward_and_backward_passes_in_graphs_of_their_own():
    # as torch.cuda.make_graphed_callables records them
    z = scores(12, 300, torch.float32, 1).requires_grad_(True)
    t = teacher(12, 300, 5, True, 1, 1.0)
    call = torch.cuda.make_graphed_callables(lambda x: C.distillation_loss(x, *t), (z.detach().clone().requires_grad_(True),))
    for i in range(3):
        x = scores(12, 300, torch.float32, 2 + i).requires_grad_(True)
        for factor in (1.0, 0.5):
            loss = call(x)
            got, = torch.autograd.grad(loss * factor, x)
            want, = torch.autograd.grad(C.distillation_loss(x, *t) * factor, x)
            torch.cuda.synchronize()
            assert torch.equal(loss, C.distillation_loss(x, *t)) and torch.equal(got, want)


def overlapping_rows(rows, cols):
    # row r is elements r .. r + cols - 1 of one buffer: many rows in little memory
    base = (torch.arange(rows + cols, device=DEV, dtype=torch.int32) * 7919 % 1009).half()
    return base.as_strided((rows, cols), (1, 1))


@pytest.mark.parametrize("cols,most", [(17, 1 << 25), (2, 1 << 27)])
def test_top_logits_of_more_rows_than_a_launch_has(cols, most):
    # 2^31 threads: 2^25 rows of 64 threads, 2^27 of 16
    rows = most + 70
    z = overlapping_rows(rows, cols)
    got = C.top_logits(z, 1)
    for part in (slice(0, 100), slice(most - 100, most + 70)):
        want = C.top_logits(z[part].cpu(), 1)
        assert torch.equal(got.values[part].cpu(), want.values) and torch.equal(got.indices[part].cpu(), want.indices)
        close(got.logsumexp[part], want.logsumexp.double().numpy(), 1.0 + np.abs(want.logsumexp.double().numpy()) / 128, z[part], "logsumexp")   # (`want` is rounded too)


def test_distillation_of_more_rows_than_a_launch_of_64_lanes_has(monkeypatch):
    set_knobs(monkeypatch, CLG_DISTILL_LANES=64)
    most = 1 << 25
    rows = most + 6
    z = (overlapping_rows(rows, 17) / 128).requires_grad_(True)
    columns = (torch.arange(rows, device=DEV, dtype=torch.int32) % 17)[:, None]
    loss = C.distillation_loss(z, torch.zeros(rows, 1, dtype=torch.float16, device=DEV), columns, reduction="none")
    grad, = torch.autograd.grad(loss, z, torch.ones_like(loss))
    for part in (slice(0, 20), slice(most - 20, most + 6)):
        x = z[part].detach()
        want = L.distillation(host(x), np.zeros((len(x), 1)), columns[part].cpu().numpy(), reduction="none")
        close(loss[part], want[0], want[2], x, "loss")
        close(grad[part], want[1], want[3], x, "grad")


def test_balance_on_two_streams_at_once():
    # several workgroups end the sums of each call, the last of them by a ticket that the launch before resets
    some = [scores(4000, 60, torch.float32, 1), scores(4000, 60, torch.float32, 2)]
    gates = [[scores(n, 16, torch.float32, n + i) for n in (700, 33, 5000)] for i in range(2)]

    def call(i):
        leaf = some[i].detach().requires_grad_(True)
        leaves = [g.detach().requires_grad_(True) for g in gates[i]]
        loss, counts = C.balance_loss(leaf, 4)
        even, of_gates = C.gate_balance(leaves)
        return [loss.detach(), counts, even.detach(), of_gates, *torch.autograd.grad(loss, leaf), *torch.autograd.grad(even, leaves)]

    want = [call(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(i))
    torch.cuda.synchronize()
    for i in range(2):
        for one in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(one, want[i]))
