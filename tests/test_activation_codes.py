"""Activations in 8 bits on the CPU: the codes against their definition, layers that keep them, and what is refused."""
import copy
import math
import pickle

import numpy as np
import pytest
import torch

import convlogic_amd as C
from oracle import keep_oracle as K

TYPES = [torch.float32, torch.float64, torch.float16, torch.bfloat16]


def activations(shape, dtype=torch.float32, seed=0):
    return torch.rand(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dtype)


def check(x):
    kept = C.encode_activations(x)
    flat = x.detach().as_strided((x.numel(),), (1,)) if x.numel() else x.detach().reshape(0)
    codes, scales = K.codes(flat.double().numpy())
    assert np.array_equal(kept.codes.numpy(), codes)
    assert kept.scales.dtype == (torch.float64 if x.dtype == torch.float64 else torch.float32)
    want = torch.from_numpy(scales).to(kept.scales.dtype)
    assert torch.equal(kept.scales, want) or torch.allclose(kept.scales, want, rtol=0, atol=0, equal_nan=True)
    back = kept.decode()
    assert back.shape == x.shape and back.dtype == x.dtype and back.stride() == x.stride() and not back.requires_grad
    # (half a step of the codes, the roundings of step and value, and the type's own)
    half = torch.from_numpy(scales[:, 1].repeat(128)[:x.numel()]) / 2
    error = (back.as_strided((x.numel(),), (1,)).double() - flat.double()).abs()
    size = flat.double().abs() + 255 * 2 * half
    assert (error <= half + size * (2.0 ** -22 + torch.finfo(x.dtype).eps / 2)).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1,), (0,), (3, 0), (), (127,), (128,), (129,), (5, 77), (2, 3, 8, 8)])
def test_codes_are_their_definition(dtype, shape):
    check(activations(shape, dtype))


def test_memory_order_and_gaps():
    x = activations((60, 20))
    check(x.t())
    check(x.view(3, 20, 4, 5).permute(3, 0, 1, 2))
    gaps = x[:, ::2]
    kept = C.encode_activations(gaps)
    assert np.array_equal(kept.codes.numpy(), K.codes(gaps.contiguous().double().numpy().reshape(-1))[0])
    assert kept.decode().shape == gaps.shape


def test_what_is_kept_exactly():
    bits = (activations((1000,)) > 0.5).float()
    assert torch.equal(C.encode_activations(bits).decode(), bits)
    assert torch.equal(C.encode_activations(torch.full((300,), 0.3)).decode(), torch.full((300,), 0.3))
    x = activations((128,))
    back = C.encode_activations(x).decode()
    assert back[x.argmin()] == x.min() and abs(float(back[x.argmax()] - x.max())) <= 2.0 ** -23


def test_a_half_goes_to_the_even_code():
    x = torch.tensor([0.0, 255.0, 0.5, 1.5, 2.5, 253.5])
    assert C.encode_activations(x).codes.tolist() == [0, 255, 0, 2, 2, 254]


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_groups_that_are_not_finite(bad):
    x = activations((300,))
    x[130] = bad
    back = C.encode_activations(x).decode()
    assert back[128:256].isnan().all() and back[:128].isfinite().all() and back[256:].isfinite().all()


def test_extreme_values():
    big = torch.finfo(torch.float32).max
    x = torch.tensor([-big, big, 0.0, big / 2])
    back = C.encode_activations(x).decode()
    assert back.isfinite().all() and (back - x).abs().max() / big < 2 / 500
    tiny = torch.tensor([0.0, 1e-45, 0.0])
    assert (C.encode_activations(tiny).decode() - tiny).abs().max() <= 1e-45
    far = torch.tensor([-1.7e308, 1.7e308], dtype=torch.float64)
    assert C.encode_activations(far).decode().isnan().all()
    assert C.encode_activations(torch.tensor([0.0, 5e-324], dtype=torch.float64)).decode().abs().max() <= 5e-324


def test_refusals():
    with pytest.raises(RuntimeError, match="float32, float64, float16 or bfloat16"):
        C.encode_activations(torch.ones(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="float32, float64, float16 or bfloat16"):
        C.encode_activations([1.0])
    with pytest.raises(RuntimeError, match="dense tensor"):
        C.encode_activations(torch.ones(3).to_sparse())
    with pytest.raises(RuntimeError, match="dense tensor"):
        C.encode_activations(torch.ones(3, device="meta"))
    with pytest.raises(TypeError, match="ActivationCodes"):
        C.decode_activations(torch.ones(3))
    for bits in (4, 16, True, "8", 8.5):
        with pytest.raises(ValueError, match="None or 8"):
            C.LogicLayer(4, 4, implementation="python", checkpoint_bits=bits)
    with pytest.raises(ValueError, match="complete blocks"):
        C.ConvLogicLayer(3, 4, implementation="python", complete=True, checkpoint_bits=8)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda x: C.encode_activations(x).decode(), (torch.rand(4),))


def layer_of(inputs, neurons, seed=0, **kw):
    torch.manual_seed(seed)
    return C.LogicLayer(inputs, neurons, implementation="python", **kw)


@pytest.mark.parametrize("batch", [1, 5, 130])
@pytest.mark.parametrize("inputs,neurons", [(7, 5), (12, 6), (9, 40)])
def test_a_layers_gradients_are_those_at_the_codes(inputs, neurons, batch):
    layer = layer_of(inputs, neurons, checkpoint_bits=8).double()
    x = activations((batch, inputs), torch.float64, 3).requires_grad_(True)
    up = torch.randn(batch, neurons, dtype=torch.float64)
    y = layer(x)
    y.backward(up)
    # (the codes of a sample-major tensor run along the samples' features: the same formulas on a layer of one row per group are compared here)
    kept = C.encode_activations(x).decode().requires_grad_(True)
    plain = layer_of(inputs, neurons).double()
    plain.load_state_dict(layer.state_dict())
    out = plain(kept)
    out.backward(up)
    assert torch.equal(y, plain(x.detach()))
    assert torch.allclose(x.grad, kept.grad, rtol=1e-12) and torch.allclose(layer.weights.grad, plain.weights.grad, rtol=1e-10, atol=1e-15)


def test_gradients_near_differences():
    # of 0/1 inputs, which the codes keep: the gradient w.r.t. the logits is that of the output itself
    layer = layer_of(10, 8, checkpoint_bits=8).double()
    x = (activations((16, 10), torch.float64) > 0.5).double()
    up = torch.randn(16, 8, dtype=torch.float64)
    (layer(x) * up).sum().backward()
    step, got = 1e-6, layer.weights.grad.clone()
    for j, i in [(0, 0), (3, 7), (7, 15)]:
        values = []
        for sign in (1, -1):
            with torch.no_grad():
                layer.weights[j, i] += sign * step
                values.append(float((layer(x) * up).sum()))
                layer.weights[j, i] -= sign * step
        assert abs((values[0] - values[1]) / (2 * step) - float(got[j, i])) <= 1e-7


def test_where_nothing_is_kept():
    layer = layer_of(6, 6, checkpoint_bits=8)
    x = activations((4, 6))
    with torch.no_grad():
        assert not layer(x).requires_grad
    layer.eval()
    assert layer(x).grad_fn is None or "Codes" not in type(layer(x).grad_fn).__name__
    layer.train()
    layer.weights.requires_grad_(False)
    assert not layer(x).requires_grad
    x.requires_grad_(True)
    layer(x).sum().backward()
    assert x.grad is not None and layer.weights.grad is None


def test_the_gradient_cannot_be_differentiated():
    layer = layer_of(6, 6, checkpoint_bits=8)
    x = activations((4, 6)).requires_grad_(True)
    g, = torch.autograd.grad(layer(x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_state_copies_and_pickles():
    layer = layer_of(6, 6, checkpoint_bits=8)
    assert set(layer.state_dict()) == set(layer_of(6, 6).state_dict())
    for other in (copy.deepcopy(layer), pickle.loads(pickle.dumps(layer))):
        assert other.checkpoint_bits == 8
    old = layer_of(6, 6)
    del old.__dict__["checkpoint_bits"]                               # (a layer that was pickled before there was one)
    x = activations((4, 6)).requires_grad_(True)
    old(x).sum().backward()


def test_the_oracle_against_autograd():
    x = activations((9, 130), torch.float64, 5)
    a, b = torch.randint(0, 9, (12,)), torch.randint(0, 9, (12,))
    z, up = torch.randn(12, 16, dtype=torch.float64, requires_grad=True), torch.randn(12, 130, dtype=torch.float64)
    kept = C.encode_activations(x).decode().requires_grad_(True)
    from convlogic_amd.difflogic.functional import bin_op_s
    out = bin_op_s(kept[a].t(), kept[b].t(), torch.softmax(z, -1)).t()
    gx, gz = torch.autograd.grad(out, (kept, z), up)
    _, want_x, want_z, _, _ = K.layer(x.numpy(), a.numpy(), b.numpy(), z.detach().numpy(), up.numpy())
    assert np.allclose(gx.numpy(), want_x, rtol=1e-11, atol=1e-13) and np.allclose(gz.numpy(), want_z, rtol=1e-9, atol=1e-12)


def test_an_updated_wiring_is_refused_by_the_backward_pass():
    layer = layer_of(6, 9, checkpoint_bits=8)
    x = activations((20, 6)).requires_grad_(True)
    y = layer(x)
    y.sum().backward(retain_graph=True)
    with torch.no_grad():
        layer.indices_0.copy_(layer.indices_0.flip(0))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_a_replaced_wiring_leaves_the_backward_pass_its_own():
    layer = layer_of(6, 9, checkpoint_bits=8)
    x = activations((20, 6)).requires_grad_(True)
    y = layer(x)
    want = torch.autograd.grad(y.sum(), (x, layer.weights), retain_graph=True)
    layer.indices_0 = layer.indices_0.flip(0)
    got = torch.autograd.grad(y.sum(), (x, layer.weights))
    assert all(torch.equal(u, v) for u, v in zip(got, want))
