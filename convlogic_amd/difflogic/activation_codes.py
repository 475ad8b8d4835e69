"""Activations in 8 bits: what a layer with checkpoint_bits=8 keeps of its input between the forward and the backward pass.

  encode_activations   128 elements, as they lie in memory, share their lowest value and a step -> ActivationCodes
  decode_activations   the tensor that codes stand for

Tensors on the GPU go through HIP kernels (csrc/activation_codes.hip) and raise if the compiled library is missing; tensors on the CPU through plain torch
operations, with the same codes.  No counterpart in the reference."""
import torch
from torch.autograd.function import once_differentiable

from ..hip import _lib

GROUP = 128                                                           # elements that share a scale
_TYPES = (torch.float32, torch.float64, torch.float16, torch.bfloat16)


class ActivationCodes:
    """codes uint8 [n] and scales [ceil(n / 128), 2] -- element i stands for scales[i // 128, 0] + codes[i] * scales[i // 128, 1] -- with the shape, strides
    and dtype of the tensor they were made of."""

    __slots__ = ("codes", "scales", "shape", "stride", "dtype")

    def __init__(self, codes, scales, shape, stride, dtype):
        self.codes, self.scales, self.shape, self.stride, self.dtype = codes, scales, shape, stride, dtype

    @property
    def device(self):
        return self.codes.device

    def nbytes(self):
        return self.codes.numel() + self.scales.numel() * self.scales.element_size()

    def decode(self):
        return decode_activations(self)

    def __repr__(self):
        return f"ActivationCodes({tuple(self.shape)}, {self.dtype}, {self.device})"


def _check(x):
    if not isinstance(x, torch.Tensor) or x.dtype not in _TYPES:
        raise RuntimeError(f"activations must be a float32, float64, float16 or bfloat16 tensor, got {x.dtype if isinstance(x, torch.Tensor) else type(x)}")
    if x.layout != torch.strided or not (x.is_cuda or x.device.type == "cpu"):
        raise RuntimeError(f"activations must be a dense tensor on the GPU or the CPU, got {x.layout} on {x.device}")


def encode_activations(x):
    """The ActivationCodes of a float tensor: an element of a group of 128 with lowest value l and highest h is off by at most (h - l) / 510 and the roundings of
    the step and of its type (by more where the step is no normal number, for ranges under 255 times the smallest one: in the end all are l).  The lowest value is kept, the
    highest but for these roundings; 0 and 1 are exact where a group holds both, or one of them alone.  Groups run through the elements as
    they lie in memory (those of a tensor with gaps as of its contiguous copy).  All elements of a group with a NaN or an infinity become NaN.  A constant for
    autograd, whatever x is."""
    _check(x)
    if _lib.traced():
        raise RuntimeError("encode_activations cannot be traced")
    x = x.detach()
    if not torch.ops.aten.is_non_overlapping_and_dense(x):
        x = x.contiguous()
    codes, scales = _lib.nodes().encode(x) if x.is_cuda else _encode_plain(x)
    return ActivationCodes(codes, scales, x.shape, x.stride(), x.dtype)


def decode_activations(codes):
    """The tensor that codes stand for, with the shape, strides and dtype of the one they were made of."""
    if not isinstance(codes, ActivationCodes):
        raise TypeError(f"ActivationCodes expected, got {type(codes)}")
    if _lib.traced():
        raise RuntimeError("decode_activations cannot be traced")
    if codes.codes.is_cuda:
        return _lib.nodes().decode(codes.codes, codes.scales, codes.shape, codes.stride, codes.dtype)
    return _decode_plain(codes)


def _in_memory(x):
    """the elements of a tensor without gaps, as they lie in memory"""
    return x.as_strided((x.numel(),), (1,))


def _encode_plain(x):
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    n = x.numel()
    if n == 0:
        return torch.empty((0,), dtype=torch.uint8), torch.empty((0, 2), dtype=wide)
    flat = _in_memory(x)
    flat = torch.cat([flat, flat[-1:].expand(-n % GROUP)]).double().view(-1, GROUP)
    low, high = flat.amin(1, keepdim=True), flat.amax(1, keepdim=True)
    size = high - low
    bad = ~(flat.isfinite().all(1, keepdim=True) & (size * 255.0).isfinite())
    codes = torch.where(bad, 0.0, ((flat - low) * 255.0 / torch.where(size > 0, size, 1.0)).round()).to(torch.uint8).view(-1)[:n].clone()
    step = (size / 255.0).to(wide)
    top = (255.0 * step.double() + low).to(wide)
    step = torch.where(top.isfinite(), step, step * (1 - 2.0 ** -23))
    scales = torch.cat([low.to(wide), step], 1)
    return codes, torch.where(bad, float("nan"), scales)


def _decode_plain(codes):
    n = codes.codes.numel()
    groups = torch.arange(n) // GROUP
    low, step = codes.scales[groups].double().unbind(1)
    out = torch.empty_strided(codes.shape, codes.stride, dtype=codes.dtype)
    _in_memory(out).copy_((codes.codes.double() * step + low).to(codes.scales.dtype).to(codes.dtype))
    return out


def check_bits(bits):
    """the checkpoint_bits of a layer: None or 8"""
    if bits not in (None, 8):
        raise ValueError(f"checkpoint_bits must be None or 8, got {bits!r}")
    return bits


class RecomputedFromCodes(torch.autograd.Function):
    """y = evaluate(x, weights, *wiring), with the gradients of that at what the codes of x stand for: x is kept in codes, and the backward pass evaluates
    again, with the wiring of the forward pass (autograd refuses one that was written since)."""

    @staticmethod
    def forward(ctx, x, weights, evaluate, *wiring):
        kept = encode_activations(x)
        ctx.save_for_backward(kept.codes, kept.scales, weights, *wiring)
        ctx.of, ctx.evaluate = (kept.shape, kept.stride, kept.dtype), evaluate
        return evaluate(x.detach(), weights.detach(), *wiring)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        codes, scales, weights, *wiring = ctx.saved_tensors
        x = ActivationCodes(codes, scales, *ctx.of).decode().requires_grad_(ctx.needs_input_grad[0])
        w = weights.detach().requires_grad_(ctx.needs_input_grad[1])
        wanted = [t for t in (x, w) if t.requires_grad]
        with torch.enable_grad():
            grads = list(torch.autograd.grad(ctx.evaluate(x, w, *wiring), wanted, grad_y))
        return (grads.pop(0) if x.requires_grad else None, grads.pop(0) if w.requires_grad else None, None) + (None,) * len(wiring)
