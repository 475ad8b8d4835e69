"""Activations in 8 bits on the GPU, and the layers that keep them, against their definitions in 64 bits (oracle/keep_oracle.py).

Bounds.  Codes, lowest values and steps are the definition's own; a value is one multiply-add, off by half a step of float32 (of float64), and by half a step of
a 16-bit type.  A gradient is a sum of products of the incoming gradient with a coefficient of a magnitude up to 2 (the sums over the 16 gates of at most |1|, |2|)
times values up to 1: each term is off by the few roundings of its product, of the coefficient (a softmax of 16 and sums over it, 24 steps in all) and of
the value, 32 steps of 2^-24 together, and the sum by as many more as it has additions in a row -- the consumers of an input, or samples."""
import copy
import math

import numpy as np
import pytest
import torch

import convlogic_amd as C
from oracle import keep_oracle as K
from tests.gpu_util import DEV

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float64, torch.float16, torch.bfloat16]


def activations(shape, dtype=torch.float32, seed=0):
    return torch.rand(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dtype)


def host(t):
    return t.detach().double().cpu().numpy()


# ---- codes ---------------------------------------------------------------------------------------
def check(x):
    """x on the CPU; the kernels have its codes and values bit for bit, but for the last place of a sum"""
    kept, want = C.encode_activations(x.to(DEV)), C.encode_activations(x)
    assert torch.equal(kept.codes.cpu(), want.codes)
    assert torch.equal(kept.scales.cpu().nan_to_num(nan=-7.0), want.scales.nan_to_num(nan=-7.0))
    back, plain = kept.decode(), want.decode()
    assert back.shape == x.shape and back.dtype == x.dtype and back.stride() == plain.stride()
    back = back.cpu()
    assert torch.equal(back.isnan(), plain.isnan())
    eps = torch.finfo(x.dtype).eps
    size = want.scales.nan_to_num().abs().double().sum(1).repeat_interleave(128)[:x.numel()] * 256       # of a float32 sum that cancels
    error = (back.double() - plain.double()).nan_to_num().as_strided((x.numel(),), (1,)).abs()
    assert (error <= size * 2.0 ** -23 * (1 if x.dtype != torch.float64 else 2.0 ** -29) + eps * plain.nan_to_num().double().abs().as_strided((x.numel(),), (1,))).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 7, 127, 128, 129, 2047, 2048, 2049, 100003])
def test_codes(dtype, n):
    check(activations((n,), dtype, n))


@pytest.mark.parametrize("dtype", TYPES)
def test_codes_of_wide_and_narrow_groups(dtype):
    g = torch.Generator().manual_seed(1)
    spread = 10.0 ** torch.linspace(-30, 30, 200, dtype=torch.float64) if dtype in (torch.float32, torch.float64, torch.bfloat16) else torch.linspace(1, 60000, 200)
    x = torch.randn(200, 128, generator=g, dtype=torch.float64).clamp(-1, 1) * spread[:, None]
    x[::7] += 3 * spread[::7, None] if dtype != torch.float16 else 0
    check(x.to(dtype))


def test_values_next_to_the_border_of_a_code():
    # halves between two codes, and their neighbours above and below, for several ranges
    rows = []
    for low, high in [(0.0, 1.0), (0.0, 255.0), (0.1, 0.9), (-3.0, 7.0), (0.0, 1e-20), (1e10, 3e10)]:
        t = (low + (torch.arange(126, dtype=torch.float64) * 2 + 0.5) * ((high - low) / 255)).float()
        for u in (t, torch.nextafter(t, torch.tensor(math.inf)), torch.nextafter(t, torch.tensor(-math.inf))):
            rows.append(torch.cat([u, torch.tensor([low, high])]))
    check(torch.cat(rows))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_groups_that_are_not_finite(bad):
    for dtype in TYPES:
        x = activations((700,), dtype)
        x[200] = bad
        x[699] = bad
        check(x)


def test_extreme_values():
    big = torch.finfo(torch.float32).max
    check(torch.tensor([-big, big, 0.0, big / 2, -big / 3]))
    check(torch.tensor([0.0, 1e-45, 0.0, 3e-45]))
    check(torch.tensor([-1.7e308, 1.7e308], dtype=torch.float64))
    check(torch.tensor([0.0, 5e-324, 1e-323], dtype=torch.float64))
    check(torch.full((300,), 0.3))
    check((activations((3000,)) > 0.5).float())
    check(torch.tensor([65504.0, -65504.0, 1.0], dtype=torch.float16))


def test_layouts_and_any_address():
    x = activations((60, 40))
    check(x.t())
    check(x.view(3, 20, 8, 5).permute(3, 0, 1, 2))
    for dtype in TYPES:
        flat = activations((5000,), dtype)
        kept, want = C.encode_activations(flat.to(DEV)[3:]), C.encode_activations(flat[3:])
        assert torch.equal(kept.codes.cpu(), want.codes)
    gaps = x.to(DEV)[:, ::3]
    assert torch.equal(C.encode_activations(gaps).decode(), C.encode_activations(gaps.contiguous()).decode())
    for shape in [(0,), (3, 0), ()]:
        assert C.encode_activations(torch.ones(shape, device=DEV)).decode().shape == shape
    assert C.encode_activations(x.to(DEV).requires_grad_(True)).decode().requires_grad is False


def test_codes_of_another_tensor_are_refused():
    kept = C.encode_activations(activations((300,)).to(DEV))
    for change in (dict(codes=kept.codes[:200]), dict(scales=kept.scales[:1]), dict(scales=kept.scales.double()), dict(dtype=torch.float64),
                   dict(shape=(3000,), stride=(1,)), dict(stride=(2,)), dict(dtype=torch.int32), dict(codes=kept.codes.int())):
        other = copy.copy(kept)
        for name, value in change.items():
            setattr(other, name, value)
        with pytest.raises(RuntimeError):
            other.decode()


def test_codes_on_another_stream_and_in_a_graph():
    x = activations((40, 1000)).to(DEV)
    want = C.encode_activations(x).decode()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = C.encode_activations(x).decode()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = C.encode_activations(x).decode()
    for seed in range(3):
        x.copy_(activations((40, 1000), seed=seed))
        graph.replay()
        assert torch.equal(out, C.encode_activations(x).decode())


# ---- layers --------------------------------------------------------------------------------------
def layer_of(inputs, neurons, seed=0, **kw):
    torch.manual_seed(seed)
    layer = C.LogicLayer(inputs, neurons, implementation="cuda", checkpoint_bits=8, **kw).to(DEV)
    with torch.no_grad():
        layer.weights.mul_(2)
    return layer


def check_layer(layer, batch, sample_major=False, need=(True, True), seed=0):
    inputs, neurons = layer.in_dim, layer.out_dim
    x = activations((inputs, batch), seed=seed)
    up = torch.randn(batch, neurons, generator=torch.Generator().manual_seed(seed + 1))
    leaf = (x.t().contiguous().to(DEV) if sample_major else x.to(DEV).t()).requires_grad_(need[0])
    layer.weights.requires_grad_(need[1])
    y = layer(leaf)
    plain = copy.deepcopy(layer)
    plain.checkpoint_bits = None
    assert torch.equal(y, plain(leaf.detach()))
    wanted = [t for t in (leaf, layer.weights) if t.requires_grad]
    got = list(torch.autograd.grad(y, wanted, up.to(DEV) if sample_major else up.t().contiguous().to(DEV).t()))
    a, b = layer.indices_0.cpu().numpy(), layer.indices_1.cpu().numpy()
    _, gx, gl, mx, ml = K.layer(x.numpy(), a, b, host(layer.weights), up.t().double().numpy())
    if need[0]:
        fan = int(np.bincount(np.concatenate([a, b])).max())
        error = np.abs(host(got.pop(0)).T - gx)
        assert (error <= (32 + fan) * 2.0 ** -24 * 2 * mx).all(), (error - (32 + fan) * 2.0 ** -24 * 2 * mx).max()
    if need[1]:
        # (a gate's sum enters all 16 gradients of its neuron, through the softmax)
        error, bound = np.abs(host(got.pop(0)) - gl), (32 + batch) * 2.0 ** -24 * 4 * ml
        assert (error <= bound).all(), (error - bound).max()


@pytest.mark.parametrize("batch", [1, 2, 3, 4, 5, 15, 16, 17, 63, 64, 65, 100, 127, 128, 129, 255, 256, 257, 333, 512, 515, 1031])
@pytest.mark.parametrize("inputs,neurons", [(50, 37), (64, 32), (11, 90)])
def test_layer(inputs, neurons, batch):
    check_layer(layer_of(inputs, neurons), batch, seed=batch)


@pytest.mark.parametrize("batch", [1, 17, 100, 256, 301])
@pytest.mark.parametrize("need", [(True, False), (False, True)])
def test_layer_of_which_one_gradient_is_wanted(need, batch):
    check_layer(layer_of(40, 33), batch, need=need)
    check_layer(layer_of(40, 20), batch, need=need)


@pytest.mark.parametrize("batch", [150, 191, 192, 193, 300, 383, 384, 385, 400, 511, 513])
@pytest.mark.parametrize("inputs,neurons", [(3, 5), (33, 700), (300, 150)])
def test_layer_with_several_samples_of_a_row_to_a_lane(inputs, neurons, batch):
    check_layer(layer_of(inputs, neurons), batch, seed=batch)


@pytest.mark.parametrize("inputs,neurons,batch", [(2001, 90000, 187), (2001, 90000, 192), (50000, 45000, 377), (2001, 45000, 384), (2001, 33000, 511)])
def test_large_layer_whose_sums_are_ended_apart(inputs, neurons, batch):
    check_layer(layer_of(inputs, neurons), batch, seed=batch)


@pytest.mark.parametrize("batch", [1, 33, 128, 300])
def test_layer_on_samples_in_rows(batch):
    check_layer(layer_of(50, 37), batch, sample_major=True)
    check_layer(layer_of(50, 25), batch, sample_major=True)


def test_layer_with_inputs_that_few_or_all_neurons_read():
    layer = layer_of(20, 300)
    with torch.no_grad():
        layer.indices_0.fill_(3)                                      # input 3 by all, the others by a few, some by none
        layer.indices_1.copy_(torch.arange(300) % 7)                  # (and neurons that read an input twice)
    check_layer(layer, 100)
    check_layer(layer, 5)
    one = layer_of(2, 1)
    check_layer(one, 128)
    check_layer(layer_of(1, 1), 7)


@pytest.mark.parametrize("batch", [3, 16, 60, 128, 130, 192, 250, 280, 333, 384, 450, 600])
def test_layer_with_long_and_empty_lists_of_readers(batch):
    layer = layer_of(40, 300)
    with torch.no_grad():
        layer.indices_0.copy_((torch.arange(300) ** 2) % 11 * 3)      # every third input up to 30 by many, the others by none
        layer.indices_1.copy_(torch.where(torch.arange(300) % 5 == 0, layer.indices_0.cpu(), 3 * (torch.arange(300) % 13)))
    check_layer(layer, batch)
    check_layer(layer, batch, need=(True, False))


@pytest.mark.parametrize("bits", [None, 8])
def test_a_layer_without_samples_is_refused_by_its_forward_pass(bits):
    layer = C.LogicLayer(16, 8, implementation="cuda", checkpoint_bits=bits).to(DEV)
    with pytest.raises(RuntimeError, match="batch must be positive"):
        layer(torch.rand(0, 16, device=DEV))


def test_layer_with_groups_of_one_value_and_gradients_that_are_not_finite():
    layer = layer_of(40, 30)
    x = torch.full((40, 128), 0.25)
    x[3] = 1.0
    leaf = x.to(DEV).t().requires_grad_(True)
    up = torch.ones(128, 30)
    up[5, 2] = math.nan
    gx, gl = torch.autograd.grad(layer(leaf), (leaf, layer.weights), up.to(DEV))
    assert gl[2].isnan().all() and gl.isnan().any(1).sum() == 1
    readers = {int(layer.indices_0[2]), int(layer.indices_1[2])}
    assert set(gx.isnan().any(0).nonzero().flatten().tolist()) == readers and gx.isnan().any(1).nonzero().flatten().tolist() == [5]


@pytest.mark.parametrize("dtype", [torch.float64, torch.float16])
def test_layer_of_other_types(dtype):
    layer = layer_of(30, 41)
    if dtype == torch.float64:
        layer = layer.double()
    x = activations((30, 70), dtype)
    up = torch.randn(70, 41, dtype=torch.float64).to(dtype)
    leaf = x.to(DEV).t().requires_grad_(True)
    gx, gl = torch.autograd.grad(layer(leaf), (leaf, layer.weights), up.to(DEV))
    kept = C.encode_activations(x.to(DEV)).decode().t().requires_grad_(True)
    plain = copy.deepcopy(layer)
    plain.checkpoint_bits = None
    wx, wl = torch.autograd.grad(plain(kept), (kept, plain.weights), up.to(DEV))
    # (the same kernels on the same values; of float64 the fused ones, which add in another order)
    tol = 1e-12 if dtype == torch.float64 else 0
    assert torch.allclose(gx, wx, rtol=tol, atol=tol) and torch.allclose(gl, wl, rtol=tol, atol=tol)


def test_gradient_against_differences():
    layer = layer_of(12, 9)
    x = (activations((12, 200)) > 0.5).float()                        # the codes keep 0 and 1
    up = torch.randn(200, 9, dtype=torch.float64).to(DEV)
    leaf = x.to(DEV).t().requires_grad_(True)
    got, = torch.autograd.grad(layer(leaf), layer.weights, up.float())
    plain = copy.deepcopy(layer).double()
    plain.checkpoint_bits = None
    step = 1e-5
    for j, i in [(0, 0), (4, 9), (8, 15)]:
        values = []
        for sign in (1, -1):
            other = copy.deepcopy(plain)
            with torch.no_grad():
                other.weights[j, i] += sign * step
                values.append(float((other(leaf.detach().double()) * up.float().double()).sum()))
        # (third-order terms of a softmax under 1, 200 samples: step^2 * 200; the float32 sums: (32 + 200) steps of 200 terms)
        assert abs((values[0] - values[1]) / (2 * step) - float(got[j, i])) <= 200 * step ** 2 + 232 * 2.0 ** -24 * 4 * float(up[:, j].abs().sum())


def test_a_step_holds_less():
    held = {}
    for bits in (None, 8):
        torch.manual_seed(0)
        layers = torch.nn.Sequential(*(C.LogicLayer(4000, 4000, implementation="cuda", checkpoint_bits=bits) for _ in range(8))).to(DEV)
        x = torch.rand(4000, 1024, device=DEV).t().requires_grad_(True)
        layers(x).sum().backward()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = layers(x)
        held[bits] = torch.cuda.memory_allocated() - before - y.numel() * 4
        del y
    one = 4000 * 1024
    assert held[None] >= 7 * 4 * one                                  # (x itself is the caller's)
    # (codes and scales, probabilities and coefficients; the allocator hands a tensor of more than 1 MiB, which are the codes alone, up to 1 MiB more than it
    # asks for, when what is left of a block is too little to be split off)
    assert held[8] <= 8 * (one * (1 + 8 / 128) + 4000 * 80 + 8192 + (1 << 20))


def test_an_updated_wiring_is_refused_by_the_backward_pass():
    layer = layer_of(30, 20)
    y = layer(activations((30, 64)).to(DEV).t().requires_grad_(True))
    with torch.no_grad():
        layer.indices_0.copy_(layer.indices_0.flip(0))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_a_layer_on_two_streams_and_through_a_retained_graph():
    layer = layer_of(60, 45)
    x = activations((60, 300)).to(DEV).t().requires_grad_(True)
    y = layer(x)
    first = torch.autograd.grad(y.sum(), (x, layer.weights), retain_graph=True)
    second = torch.autograd.grad(y.sum(), (x, layer.weights))
    assert all(torch.equal(u, v) for u, v in zip(first, second))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = layer(x)
        third = torch.autograd.grad(z.sum(), (x, layer.weights))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(u, v) for u, v in zip(first, third))


def test_a_recorded_step_of_layers():
    torch.manual_seed(0)
    net = torch.nn.Sequential(*(C.LogicLayer(a, b, implementation="cuda", checkpoint_bits=8) for a, b in [(60, 80), (80, 80), (80, 40)]), C.GroupSum(10)).to(DEV)
    x, t = torch.rand(300, 60, device=DEV), torch.randint(0, 10, (300,), device=DEV)
    step = C.GraphedStep(lambda x, t: torch.nn.functional.cross_entropy(net(x), t), (x, t), net.parameters())
    for seed in range(3):
        x, t = activations((300, 60), seed=seed).to(DEV), torch.randint(0, 10, (300,), device=DEV)
        loss = float(step(x, t))
        got = [p.grad.clone() for p in net.parameters()]
        want_loss = torch.nn.functional.cross_entropy(net(x), t)
        want = torch.autograd.grad(want_loss, list(net.parameters()))
        assert loss == float(want_loss) and all(torch.equal(u, v) for u, v in zip(got, want))
        torch.cuda.synchronize()


def test_the_gradient_of_a_layer_cannot_be_differentiated():
    layer = layer_of(12, 9)
    x = activations((12, 20)).to(DEV).t().requires_grad_(True)
    g, = torch.autograd.grad(layer(x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        g.sum().backward()


def test_codes_of_more_than_2_to_the_31_elements():
    n = (1 << 31) + 300
    x = torch.zeros(n, dtype=torch.float16, device=DEV)
    x[-300:] = activations((300,), torch.float16).to(DEV)
    x[5] = 1.0
    back = C.encode_activations(x).decode()
    assert back[5] == 1 and back[:1000].sum() == 1
    assert torch.equal(back[-300:], C.encode_activations(x[(n - 300) // 128 * 128:]).decode()[-300:])


def test_layer_of_more_than_2_to_the_30_elements():
    # 0/1 inputs, which the codes keep, in the last rows and samples alone, so that a few of them can be checked one by one
    inputs, neurons, batch = 66000, 33000, 17000
    layer = layer_of(inputs, neurons)
    with torch.no_grad():                                             # (no input is read once only)
        layer.indices_0[-1], layer.indices_1[-1], layer.indices_0[-2] = inputs - 1, inputs - 2, inputs - 1
        if layer.indices_0[0] == layer.indices_0[1]:
            layer.indices_0[0] += 1
        layer.indices_0[0] = layer.indices_0[1]
    xt = torch.zeros(inputs, batch, device=DEV)
    xt[-2:, -5:] = torch.tensor([[0.0, 1, 0, 1, 1], [1, 1, 0, 0, 1]], device=DEV)
    x = xt.t().requires_grad_(True)
    y = layer(x)
    up = torch.zeros(neurons, batch, device=DEV)
    up[-1, -5:] = torch.tensor([1.0, 2, 3, 4, 5], device=DEV)
    gx, gl = torch.autograd.grad(y, (x, layer.weights), up.t())
    p = torch.softmax(layer.weights[-1].detach().double(), 0).cpu().numpy()
    a, b, g = xt[-1, -5:].cpu().double().numpy(), xt[-2, -5:].cpu().double().numpy(), np.array([1.0, 2, 3, 4, 5])
    value, da, db = K.gates(a, b)
    want = p * ((value * g).sum(1) - (p[:, None] * value * g).sum())
    # (five samples; coefficients and softmax as in the other tests)
    assert np.abs(host(gl[-1]) - want).max() <= 64 * 2.0 ** -24 * 15 and (gl[:-1] == 0).all()
    got = host(gx[-5:, -2:])
    assert np.abs(got[:, 1] - (p[:, None] * da).sum(0) * g).max() <= 64 * 2.0 ** -24 * 10
    assert np.abs(got[:, 0] - (p[:, None] * db).sum(0) * g).max() <= 64 * 2.0 ** -24 * 10
    assert int((gx != 0).sum()) == int((gx[-5:, -2:] != 0).sum())     # (counted: sums of both in float32 differ in the order of their terms)


# ---- blocks and networks -------------------------------------------------------------------------
def block_of(seed=0, **kw):
    torch.manual_seed(seed)
    return C.ConvLogicLayer(5, 12, kernel=3, padding=1, complete=True, implementation="cuda", **kw).to(DEV)


@pytest.mark.parametrize("images,side", [(1, 4), (7, 8), (64, 12)])
@pytest.mark.parametrize("feature_major", [False, True])
def test_block(images, side, feature_major):
    layer, plain = block_of(checkpoint_bits=8), block_of()
    layer.feature_major_output = plain.feature_major_output = feature_major
    x = activations((images, 5, side, side)).to(DEV)
    leaf = x.clone().requires_grad_(True)
    y = layer(leaf)
    assert torch.equal(y, plain(x))
    up = torch.randn_like(y)
    gx, gl = torch.autograd.grad(y, (leaf, layer.weights), up)
    # inputs that the codes keep: all as without them
    kept = C.encode_activations(x).decode().requires_grad_(True)
    again = C.encode_activations(kept.detach()).decode()
    out = layer(kept)
    wx, wl = torch.autograd.grad(out, (kept, layer.weights), up)
    other = plain(kept)
    vx, vl = torch.autograd.grad(other, (kept, plain.weights), up)
    assert torch.equal(out, other)
    assert (again - kept.detach()).abs().max() <= 2.0 ** -23          # (values of codes have these codes, but for the last place of the step)
    assert torch.allclose(wx, vx, rtol=1e-5, atol=1e-5 * float(vx.abs().max())) and torch.allclose(wl, vl, rtol=1e-5, atol=1e-5 * float(vl.abs().max()))
    # and the others as near as half a code moves a gate: products of up to 8 taps through three levels, each derivative at most 2 in a value of magnitude 1
    assert gx.shape == x.shape and (gl - vl).norm() <= 0.05 * vl.norm() and (gx - vx).norm() <= 0.1 * vx.norm()


def test_block_refusals():
    layer = block_of(checkpoint_bits=8)
    with pytest.raises(RuntimeError, match="float32 activations"):
        layer.double()(torch.rand(2, 5, 4, 4, device=DEV, dtype=torch.float64))
    layer.float().eval()
    layer(torch.rand(2, 5, 4, 4, device=DEV))
    with torch.no_grad():
        layer.train()(torch.rand(2, 5, 4, 4, device=DEV))


@pytest.mark.parametrize("make,shape", [(C.ConvLogicMnistModel, (20, 1, 28, 28)), (C.ConvLogicCifarModel, (12, 3, 32, 32))])
def test_networks(make, shape):
    torch.manual_seed(0)
    net = make(k_param=8, checkpoint_bits=8).to(DEV)
    plain = copy.deepcopy(net)
    for m in plain.modules():
        if hasattr(m, "checkpoint_bits"):
            m.checkpoint_bits = None
    x, t = (activations(shape) > 0.5).float().to(DEV), torch.randint(0, 10, shape[:1], device=DEV)
    loss = torch.nn.functional.cross_entropy(net(x), t)
    want = torch.nn.functional.cross_entropy(plain(x), t)
    # (the modules' kernels against those of a whole network in one node)
    assert abs(float(loss - want)) <= 1e-5 * abs(float(want))
    got = torch.autograd.grad(loss, list(net.parameters()))
    ref = torch.autograd.grad(want, list(plain.parameters()))
    # gates that started as wires: what half a code moves is a small part of a gradient
    assert all((u - v).norm() <= 0.05 * v.norm() + 1e-8 for u, v in zip(got, ref))
    net.eval(), plain.eval()
    assert torch.equal(net(x), plain(x))


def test_a_recorded_step_of_a_network():
    torch.manual_seed(0)
    net = C.ConvLogicMnistModel(k_param=4, checkpoint_bits=8).to(DEV)
    x, t = (activations((16, 1, 28, 28)) > 0.5).float().to(DEV), torch.randint(0, 10, (16,), device=DEV)
    step = C.GraphedStep(lambda x, t: C.group_cross_entropy(net(x), t, 10), (x, t), net.parameters())
    for seed in range(3):
        x, t = (activations((16, 1, 28, 28), seed=seed) > 0.5).float().to(DEV), torch.randint(0, 10, (16,), device=DEV)
        value = float(step(x, t))
        grads = [p.grad.clone() for p in net.parameters()]
        loss = C.group_cross_entropy(net(x), t, 10)
        want = torch.autograd.grad(loss, list(net.parameters()))
        assert value == float(loss.detach()) and all(torch.equal(u, v) for u, v in zip(grads, want))
        del loss
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [torch.float64, torch.float16])
def test_an_updated_wiring_of_other_types_is_refused_by_the_backward_pass(dtype):
    layer = layer_of(30, 20)
    if dtype == torch.float64:
        layer = layer.double()
    y = layer(activations((30, 64), dtype).to(DEV).t().requires_grad_(True))
    with torch.no_grad():
        layer.indices_0.copy_(layer.indices_0.flip(0))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
