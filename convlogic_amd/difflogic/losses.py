"""Losses on the scores of a network and on the logits of its gates, and what they need of a teacher: its highest logits.

  group_cross_entropy cross entropy of a network's GroupSum, from the features that it sums
  top_logits          the highest logits of each row, their columns and the logsumexp of the row: what a teacher's answers are stored as
  distillation_loss   the loss of a student against such answers
  balance_loss        how evenly rows choose among experts, and how many rows chose each
  gate_balance        the same for the gates of a layer or a whole network, 16 to a neuron

Tensors on the GPU go through HIP kernels (csrc/group_ce.hip, csrc/top_logits.hip, csrc/distill.hip, csrc/balance.hip) and raise if the compiled library is missing;
tensors on the CPU, as networks with implementation="python" have them, through plain torch operations.  No counterpart in the reference."""
import math
from typing import NamedTuple

import torch

from ..hip import _lib

MAX_ENTRIES = 1024                                                    # top logits per row
MAX_EXPERTS = 1024
_TOGETHER = 16                                                        # tensors of one launch

_SCORES = (torch.float32, torch.float64, torch.float16, torch.bfloat16)
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


class TopLogits(NamedTuple):
    values: torch.Tensor
    indices: torch.Tensor
    logsumexp: torch.Tensor


class Balance(NamedTuple):
    loss: torch.Tensor
    counts: torch.Tensor


def _check_scores(t, name):
    if not isinstance(t, torch.Tensor) or t.dtype not in _SCORES:
        raise RuntimeError(f"{name} must be a float32, float64, float16 or bfloat16 tensor, got {t.dtype if isinstance(t, torch.Tensor) else type(t)}")
    if t.dim() < 1 or t.shape[-1] < 1:
        raise RuntimeError(f"{name} must be [..., columns] with a column at least, got {tuple(t.shape)}")
    if t.shape[-1] >= 1 << 31 or t.numel() // t.shape[-1] >= 1 << 31:
        raise RuntimeError(f"{name} of shape {tuple(t.shape)}: 2^31 rows or columns and more are not supported")
    if not (t.is_cuda or t.device.type == "cpu"):
        raise RuntimeError(f"{name} must be on the GPU or the CPU, got {t.device}")


def _check_mask(mask, like):
    if mask is None:
        return
    if mask.dtype != torch.bool or mask.shape != like.shape[:-1] or mask.device != like.device:
        raise RuntimeError(f"mask must be a bool tensor of shape {tuple(like.shape[:-1])} on {like.device}, got {mask.dtype} {tuple(mask.shape)} on {mask.device}")


def _check_number(x, name, positive=False):
    x = float(x)
    if not math.isfinite(x) or (positive and not 1e-30 < x < 1e30):
        raise ValueError(f"{name} must be {'positive and ' if positive else ''}finite, got {x}")
    return x


def _nodes(what):
    if _lib.traced():
        raise RuntimeError(f"{what} cannot be traced")
    return _lib.nodes()


def _wide(t):
    return t if t.dtype == torch.float64 else t.float()


# ---- top logits ----------------------------------------------------------------------------------
def top_logits(logits, k, temperature=1.0):
    """The k highest logits of each row of [..., columns], highest first: values [..., k], indices int64 [..., k] (of equal logits the lowest index
    first; a NaN counts as the maximum), and the logsumexp of the whole row at `temperature`, log sum exp(logits / temperature), in float32 (float64
    of float64 logits).  1 <= k <= 1024.  Constants for autograd, whatever the logits are.

    As a float32 number the logsumexp is off by up to 2^-24 of itself, and so is the logarithm of every probability that is taken relative to it: 10^-6
    at 20, more than the probabilities themselves from about 10^7 on.  Logits that are far from 0 go in less a constant per row, or in float64."""
    _check_scores(logits, "logits")
    k, temperature = int(k), _check_number(temperature, "temperature", positive=True)
    if not 1 <= k <= min(MAX_ENTRIES, logits.shape[-1]):
        raise ValueError(f"k must be between 1 and {min(MAX_ENTRIES, logits.shape[-1])}, got {k}")
    if logits.is_cuda:
        return TopLogits(*_nodes("top_logits").top_logits(logits, k, temperature))
    logits = logits.detach()
    x = _wide(logits)
    columns = torch.sort(x.nan_to_num(nan=math.inf, posinf=math.inf, neginf=-math.inf), dim=-1, descending=True, stable=True).indices
    if bool(x.isnan().any()):                                         # (NaN before +inf, each in the order of the columns)
        is_nan = x.gather(-1, columns).isnan()
        columns = columns.gather(-1, torch.sort(is_nan.to(torch.uint8), dim=-1, descending=True, stable=True).indices)
    columns = columns[..., :k].contiguous()
    return TopLogits(logits.gather(-1, columns), columns, torch.logsumexp(x.double() / temperature, -1).to(x.dtype))


# ---- distillation --------------------------------------------------------------------------------
def distillation_loss(logits, values, indices, logsumexp=None, *, temperature=1.0, mask=None, weight=1.0, reduction="mean"):
    """Kullback-Leibler divergence of a student's answers from those that a teacher's top logits stand for, times weight * temperature^2.

    logits [..., columns] are the student's scores; values and indices [..., k] the teacher's logits and the columns they belong to (int32 or int64), k up
    to 1024.  An index below 0 marks an empty slot; one of `columns` or more makes the loss and gradient of its row NaN; a column that is listed
    twice counts with both values.

    Without `logsumexp` the teacher's probabilities are the softmax of values / temperature.  With it -- [...], of the teacher's whole row at this
    temperature, as top_logits() returns it -- they are exp(values / temperature - logsumexp), and all columns that are not listed are one answer more,
    whose probability is what is left of 1 on both sides.  The logsumexp is taken as it is, with the rounding of its type.

    Rows with mask (bool [...]) False, and rows without an entry, have loss 0 and gradient 0, whatever their logits are.  reduction: "mean" over the rows
    that the mask keeps (0 if it keeps none), "sum", or "none" for a loss per row.  The loss is float32 (float64 of float64 logits), the gradient has the
    type of the logits; the teacher's tensors are constants.

    The gradient is computed along with the loss, for an upstream gradient of 1: a factor that is known goes into `weight`, where it costs nothing
    (another upstream gradient costs a second pass over the logits)."""
    _check_scores(logits, "logits")
    _check_scores(values, "values")
    lead = logits.shape[:-1]
    if values.shape[:-1] != lead or indices.shape != values.shape or indices.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"values and int32 or int64 indices must be {(*lead, 'k')}, got {tuple(values.shape)} and {indices.dtype} {tuple(indices.shape)}")
    if values.shape[-1] > MAX_ENTRIES:
        raise ValueError(f"at most {MAX_ENTRIES} of the teacher's logits per row, got {values.shape[-1]}")
    if logsumexp is not None and (logsumexp.dtype not in _SCORES or logsumexp.shape != lead):
        raise RuntimeError(f"logsumexp must be a float tensor of shape {tuple(lead)}, got {logsumexp.dtype} {tuple(logsumexp.shape)}")
    _lib.check_same_device(logits, values, indices, logsumexp)
    _check_mask(mask, logits)
    if torch.is_grad_enabled() and (values.requires_grad or (logsumexp is not None and logsumexp.requires_grad)):
        raise RuntimeError("the teacher's values are constants of the loss: detach them")
    temperature, weight = _check_number(temperature, "temperature", positive=True), _check_number(weight, "weight")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    if logits.is_cuda:
        return _nodes("distillation_loss").distillation(logits, values, indices, logsumexp, mask, temperature, weight, _REDUCTIONS[reduction])
    return _distillation_plain(logits, values, indices, logsumexp, temperature, mask, weight, reduction)


def _finite_highest(t):
    highest = t.detach().amax(-1, keepdim=True)
    return torch.where(highest.isinf(), 0.0, highest)


def _distillation_plain(logits, values, indices, logsumexp, temperature, mask, weight, reduction):
    cols, lead = logits.shape[-1], logits.shape[:-1]
    there = (indices >= 0) & (indices < cols)
    bad = (indices >= cols).any(-1)
    keep = there.any(-1) | bad
    if mask is not None:
        keep = keep & mask
    # rows that do not count are rows of zeros from here on: no inf or NaN of theirs reaches a gradient
    z = torch.where(keep.unsqueeze(-1), _wide(logits), 0.0).double()
    highest = _finite_highest(z)                                      # (subtracted first: z / temperature would be rounded in steps of its own size)
    x = (z - highest) / temperature
    x = x * torch.where(keep & bad, math.nan, 1.0).unsqueeze(-1)
    at = torch.where(there, indices, 0).long()
    t = torch.where(there, values.double(), -math.inf)
    if logsumexp is None:
        t = (t - _finite_highest(t)) / temperature
        total = t.exp().sum(-1, keepdim=True)
        log_p = t - torch.where(total == 0, 0.0, total.log())
    else:
        log_p = t / temperature - logsumexp.double().unsqueeze(-1)
    p = log_p.exp()
    log_q = torch.log_softmax(x, -1)
    used = there & (p != 0)
    loss = torch.where(used, p * (torch.where(used, log_p, 0.0) - torch.where(used, log_q.gather(-1, at), 0.0)), 0.0).sum(-1)
    if logsumexp is not None:
        listed = torch.zeros(x.shape, dtype=torch.int32).scatter_add_(-1, at, there.to(torch.int32)) > 0
        rest = (1.0 - p.sum(-1)).clamp(min=0.0)
        rest = torch.where(listed.all(-1) | ~keep, 0.0, rest)
        # relative to their own highest; nothing beside the listed columns: a constant -inf less the logarithm of the whole, which keeps its gradient
        others = z.masked_fill(listed, -math.inf)
        none = (others == -math.inf).all(-1)
        others = torch.where(none.unsqueeze(-1), 0.0, others)
        highest_other = _finite_highest(others)
        log_others = torch.logsumexp((others - highest_other) / temperature, -1) + ((highest_other - highest) / temperature).squeeze(-1)
        log_rest = torch.where(none, -math.inf, log_others) - torch.logsumexp(x, -1)
        some = rest != 0
        loss = loss + torch.where(some, torch.special.xlogy(rest, rest) - rest * torch.where(some, log_rest, 0.0), 0.0)
    loss = torch.where(keep, loss, 0.0)
    if bool((keep & bad).any()):
        loss = loss + torch.where(keep & bad, x.sum(-1), 0.0)         # (NaN, also where no entry is left)
    loss = loss * (weight * temperature * temperature)
    if reduction == "none":
        return loss.to(_wide(logits).dtype)
    count = lead.numel() if mask is None else int(mask.sum())
    return (loss.sum() / (max(count, 1) if reduction == "mean" else 1)).to(_wide(logits).dtype)


# ---- cross entropy of group sums -----------------------------------------------------------------
def group_cross_entropy(x, targets, k, tau=1.0, *, label_smoothing=0.0, weight=1.0, reduction="mean"):
    """weight * cross_entropy(GroupSum(k, tau)(x), targets, label_smoothing=...) of x [..., features] in one node, which keeps no probabilities: a class is
    features / k features in a row, its score their sum over tau, and k = features takes x as scores.

    targets int32 or int64 [...]: a row with a negative one does not count -- loss 0 and gradient 0, whatever its features are -- and one of k or more makes
    the loss and gradient of its row NaN.  reduction: "mean" over the rows that count (0 if none does), "sum", or "none" for a loss per row.  Sums over features
    are 64-bit numbers.  The loss is float32 (float64 of float64 features), the gradient has the type of the features, and their layout where x is the
    transposed view that a LogicLayer returns.

    As with distillation_loss, the gradient is computed along with the loss, for an upstream gradient of 1: a factor that is known goes into `weight`."""
    _check_scores(x, "x")
    k, tau, weight = int(k), _check_number(tau, "tau", positive=True), _check_number(weight, "weight")
    label_smoothing = _check_number(label_smoothing, "label_smoothing")
    if not isinstance(targets, torch.Tensor) or targets.dtype not in (torch.int32, torch.int64) or targets.shape != x.shape[:-1]:
        raise RuntimeError(f"targets must be an int32 or int64 tensor of shape {tuple(x.shape[:-1])}, got "
                           + (f"{targets.dtype} {tuple(targets.shape)}" if isinstance(targets, torch.Tensor) else f"{type(targets)}"))
    _lib.check_same_device(x, targets)
    if k < 1 or x.shape[-1] % k:
        raise ValueError(f"k must be a divisor of the {x.shape[-1]} features, got {k}")
    if not 0 <= label_smoothing <= 1:
        raise ValueError(f"label_smoothing must be between 0 and 1, got {label_smoothing}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    if x.is_cuda:
        return _nodes("group_cross_entropy").group_ce(x, targets, k, tau, label_smoothing, weight, _REDUCTIONS[reduction])
    return _group_ce_plain(x, targets, k, tau, label_smoothing, weight, reduction)


def _group_ce_plain(x, targets, k, tau, smoothing, weight, reduction):
    keep, bad = targets >= 0, targets >= k
    # rows that do not count are rows of zeros from here on: no inf or NaN of theirs reaches a gradient
    rows = torch.where(keep.unsqueeze(-1), _wide(x), 0.0).double()
    scores = rows.reshape(*x.shape[:-1], k, x.shape[-1] // k).sum(-1) / tau
    scores = scores * torch.where(bad, math.nan, 1.0).unsqueeze(-1)
    log_p = torch.log_softmax(scores, -1)
    loss = -log_p.gather(-1, torch.where(keep & ~bad, targets, 0).long().unsqueeze(-1)).squeeze(-1)
    if smoothing:
        loss = (1 - smoothing) * loss - smoothing * log_p.mean(-1)
    loss = torch.where(keep, loss, 0.0) * weight
    if reduction == "mean":
        loss = loss / max(int(keep.sum()), 1)
    return (loss if reduction == "none" else loss.sum()).to(_wide(x).dtype)


# ---- balance -------------------------------------------------------------------------------------
def balance_loss(logits, top_k=1, *, mask=None, weight=1.0):
    """How evenly rows choose among experts -> (loss, counts).  Of each row of logits [..., experts] the top_k highest are chosen (of equal ones the
    lowest index; a NaN counts as the maximum; -inf is never chosen); counts int64 [experts] are the rows that chose each expert.  With n rows, their softmax p
    and experts E, loss = weight * E / (top_k n^2) * sum_e counts[e] sum_rows p[e]: weight where every expert has its share, more where few have most.  Its
    gradient goes through the probabilities alone.

    Rows with mask (bool [...]) False and rows of -inf alone do not count and have gradient 0.  Up to 1024 experts."""
    _check_scores(logits, "logits")
    _check_mask(mask, logits)
    top_k, weight = int(top_k), _check_number(weight, "weight")
    if logits.shape[-1] > MAX_EXPERTS:
        raise ValueError(f"at most {MAX_EXPERTS} experts, got {logits.shape[-1]}")
    if not 1 <= top_k <= logits.shape[-1]:
        raise ValueError(f"top_k must be between 1 and the number of experts, {logits.shape[-1]}, got {top_k}")
    if logits.is_cuda:
        loss, counts = _nodes("balance_loss").balance([logits], top_k, mask, weight)
    else:
        loss, counts = _balance_plain([logits], top_k, mask, weight)
    return Balance(loss, counts[0])


def _balance_plain(tensors, top_k, mask, weight):
    losses, counts = [], []
    for t in tensors:
        experts = t.shape[-1]
        rows = t.reshape(-1, experts)
        keep = ~(rows.detach() == -math.inf).all(-1)
        if mask is not None:
            keep = keep & mask.reshape(-1)
        x = rows[keep].double()
        best = x.detach().nan_to_num(nan=math.inf, posinf=math.inf, neginf=-math.inf)
        columns = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, :top_k]
        c = torch.bincount(columns[best.gather(-1, columns) != -math.inf], minlength=experts)
        n = max(x.shape[0], 1)
        losses.append((c.double() * torch.softmax(x, -1).sum(0)).sum() * (weight * experts / (top_k * n * n)))
        counts.append(c)
    return (sum(losses) / len(losses)).to(_wide(tensors[0]).dtype), torch.stack(counts)


def _gate_logits(module):
    from ..convlogic.convlogic_layer import ConvLogicLayer
    from ..convlogic.treelogic_layer import TreeLogicLayer
    from .difflogic import LogicLayer
    return [m.weights for m in module.modules() if isinstance(m, (LogicLayer, ConvLogicLayer, TreeLogicLayer))]


def gate_balance(gates, weight=1.0):
    """How evenly the neurons of each layer choose among the 16 gates -> (loss, counts): weight times the mean over the layers of balance_loss() of
    the layer's logits, with a neuron's most probable gate as its choice, and counts int64 [layers, 16], the neurons whose choice is each gate (what
    a layer evaluates with).  gates: a layer, a network (its LogicLayers, ConvLogicLayers and TreeLogicLayers in the order of modules()), or a
    sequence of logits [..., 16].  Up to 16 layers go in one launch."""
    if isinstance(gates, torch.Tensor):
        raise RuntimeError(f"gate_balance takes a module or a sequence of logits, got a tensor of {tuple(gates.shape)}: [logits] for one layer")
    tensors = _gate_logits(gates) if isinstance(gates, torch.nn.Module) else list(gates)
    weight = _check_number(weight, "weight")
    if not tensors:
        raise ValueError("gate_balance needs a layer with gates at least")
    for t in tensors:
        _check_scores(t, "logits")
        if t.shape[-1] != 16 or t.dtype != tensors[0].dtype or t.device != tensors[0].device:
            raise RuntimeError(f"logits must be [..., 16], of one dtype and on one device, got {tuple(t.shape)} {t.dtype} on {t.device}")
    if not tensors[0].is_cuda:
        return Balance(*_balance_plain(tensors, 1, None, weight))
    nodes = _nodes("gate_balance")
    parts = [tensors[i:i + _TOGETHER] for i in range(0, len(tensors), _TOGETHER)]
    done = [nodes.balance(p, 1, None, weight * len(p) / len(tensors)) for p in parts]
    if len(done) == 1:
        return Balance(*done[0])
    return Balance(torch.stack([loss for loss, _ in done]).sum(), torch.cat([counts for _, counts in done]))
