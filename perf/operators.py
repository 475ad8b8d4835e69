"""What stands between a network's scores, or the logits of its gates, and the number that backward() is called on, as timed cases:

* "top"      the highest scores of a teacher, their columns and the logsumexp of each row (what a teacher's answers are stored as)
* "distill"  the loss of a student against such answers, and with "grad" the gradient w.r.t. the student's scores
* "balance"  how evenly rows choose among experts: the loss, the rows per expert and the gradient w.r.t. the logits
* "gates"    the same for the gates of all layers of a network, 16 per neuron

Sizes are those of this package's networks (10 classes, batches of 100 and 256, LogicLayers of 8000 neurons, the k = 32 and k = 1024 topologies) and
generic ones.  Where `own` is false, `run` computes the same from elementary torch operations in 32 bits."""
import math

import torch

own = False

DEV = "cuda:0"
_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "f64": torch.float64}


def listed():
    return [
        # the scores of a batch of digits, as a network of 10 classes gives them: the smallest call, launches and the host
        dict(name="top_classes", kind="top", dtype="f32", rows=256, cols=10, k=3, temperature=2.0),
        # one answer over a long vocabulary: a single token, an odd length
        dict(name="top_one_row", kind="top", dtype="bf16", rows=1, cols=131071, k=20, temperature=1.0),
        # answers of a teacher for a training set, to be stored
        dict(name="top_answers", kind="top", dtype="bf16", rows=4096, cols=65536, k=64, temperature=1.0),
        # a training step of a small network: forward and gradient on the scores of 100 digits
        dict(name="distill_digits", kind="distill", dtype="f32", rows=100, cols=10, k=4, temperature=2.0, rest=True, masked=False, reduction="mean",
             weight=1.0, grad=True),
        # validation of a student of 1000 classes: the loss alone
        dict(name="distill_validation", kind="distill", dtype="f32", rows=10000, cols=1000, k=10, temperature=4.0, rest=False, masked=False,
             reduction="mean", weight=1.0, grad=False),
        # sequences with padding, an odd vocabulary: rows start at any address of two bytes
        dict(name="distill_ragged", kind="distill", dtype="f16", rows=777, cols=50001, k=17, temperature=1.5, rest=False, masked=True, reduction="sum",
             weight=0.5, grad=True),
        # a training step over a long vocabulary, the largest: 1 GiB of logits
        dict(name="distill_tokens", kind="distill", dtype="bf16", rows=4096, cols=131072, k=64, temperature=1.0, rest=True, masked=False,
             reduction="mean", weight=1.0, grad=True),
        # a router: 64 experts, 8 a token, padded sequences
        dict(name="balance_router", kind="balance", dtype="bf16", rows=65536, cols=64, k=8, masked=True, weight=0.01),
        # few tokens, an odd number of experts
        dict(name="balance_few", kind="balance", dtype="f32", rows=333, cols=60, k=4, masked=False, weight=1.0),
        # many tokens, many experts
        dict(name="balance_many", kind="balance", dtype="f32", rows=131072, cols=256, k=2, masked=False, weight=0.01),
        # the gates of the k = 32 network of digits, in every training step
        dict(name="gates_k32", kind="gates", dtype="f32", topology="mnist", k=32, weight=0.1),
        # the gates of the k = 1024 network of colour images
        dict(name="gates_k1024", kind="gates", dtype="f32", topology="cifar", k=1024, weight=0.1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["top", "top", "distill", "distill", "distill", "distill", "balance", "balance", "gates"])
    if kind == "gates":
        return dict(kind=kind, dtype="f32", topology=rng.choice(["mnist", "cifar"]), k=_log(rng, 8, 512), weight=rng.choice([0.01, 0.1, 1.0]))
    dtype = rng.choice(["f32", "f32", "bf16", "bf16", "f16", "f64"])  # (f16: with the factor that such programs scale their losses by)
    size = {"f32": 4, "f64": 8}.get(dtype, 2)
    if kind == "balance":
        cols = _log(rng, 2, 512)
        rows = _log(rng, 1, 200000)
        while rows * cols * size > 1 << 27:
            rows = -(-rows // 2)
        return dict(kind=kind, dtype=dtype, rows=rows, cols=cols, k=min((cols + 1) // 2, _log(rng, 1, 16)), masked=rng.random() < 0.4,
                    weight=4096.0 if dtype == "f16" else rng.choice([0.01, 1.0]))
    cols = _log(rng, 2, 200000) if rng.random() < 0.7 else rng.choice([128, 1024, 4096, 32768, 131072])
    rows = _log(rng, 1, 20000)
    while rows * cols * size > 1 << (29 if kind == "top" else 30) or rows * cols > 1 << 28:
        rows = -(-rows // 2)
    case = dict(kind=kind, dtype=dtype, rows=rows, cols=cols, k=min(cols, _log(rng, 1, 256)), temperature=rng.choice([1.0, 1.0, 1.5, 2.0, 4.0]))
    if kind == "distill":
        case.update(rest=rng.random() < 0.5, masked=rng.random() < 0.4, reduction=rng.choice(["mean", "mean", "mean", "sum", "none"]),
                    weight=1024.0 if dtype == "f16" else rng.choice([1.0, 1.0, 0.5]), grad=rng.random() < 0.8)
    return case


def _gate_rows(case):
    """neurons of every layer: the seven gates of each block's kernels, then the fully connected layers"""
    k = case["k"]
    if case["topology"] == "mnist":
        return [7 * m * k for m in (1, 3, 9)] + [1280 * k, 640 * k, 320 * k]
    m = 2 if k >= 1024 else 1
    return [7 * c * k for c in (1, 4, 16, 32)] + [m * 1280 * k, m * 640 * k, m * 320 * k]


# ---- preparation ----------------------------------------------------------------------------------
def _normal(shape, g, scale=1.0):
    return torch.randn(shape, generator=g, device=DEV) * scale


def _kept(rows, g):
    """padded sequences: about a quarter of the rows, in runs at the ends of sequences of 64, counts for nothing"""
    at = torch.arange(rows, device=DEV)
    lengths = torch.randint(32, 65, (rows // 64 + 1,), generator=g, device=DEV)
    return at % 64 < lengths[at // 64]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s, kind, dtype = dict(case), case["kind"], _DTYPES[case["dtype"]]
    if kind == "gates":
        # logits of a network in training: every gate started as a wire (logit 5 at gate 3) and has moved since
        s["logits"] = []
        for rows in _gate_rows(case):
            z = _normal((rows, 16), g, 2.0)
            z[:, 3] += 5.0
            s["logits"].append(z)
        return s
    rows, cols, k = case["rows"], case["cols"], case["k"]
    # scores: normal, every row with a level and a spread of its own; experts: some are liked more than others
    z = _normal((rows, cols), g)
    if kind == "balance":
        z += _normal((1, cols), g, 0.5)
    else:
        z.mul_(1.5 + 2.0 * torch.rand((rows, 1), generator=g, device=DEV)).add_(_normal((rows, 1), g, 3.0))
    if kind == "distill":
        # a teacher that agrees with the student up to some noise; some rows store fewer answers (empty slots: column -1)
        z_teacher = z + _normal((rows, cols), g, 0.7)
        values, columns = z_teacher.topk(k, dim=1)
        if case["rest"]:
            s["logsumexp"] = torch.logsumexp(z_teacher / case["temperature"], dim=1)
        else:
            s["logsumexp"] = None
            count = torch.where(torch.rand((rows, 1), generator=g, device=DEV) < 0.1, torch.randint(0, k + 1, (rows, 1), generator=g, device=DEV), k)
            columns = torch.where(torch.arange(k, device=DEV) < count, columns, -1)
        s["values"], s["columns"] = values.to(dtype) if dtype == torch.float64 else values, columns
        if case["rest"] and dtype == torch.float64:
            s["logsumexp"] = s["logsumexp"].double()
        del z_teacher
        s["upstream"] = torch.rand((rows,), generator=g, device=DEV).to(dtype if dtype == torch.float64 else torch.float32)
    s["mask"] = _kept(rows, g) if case.get("masked") else None
    s["logits"] = z.to(dtype)
    return s


# ---- the plain forms ------------------------------------------------------------------------------
def _wide(t):
    return t if t.dtype == torch.float64 else t.float()


def _top(z, k):
    """the k highest of each row, a tie goes to the lower column"""
    if z.dtype == torch.float64:
        columns = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]
    else:
        bits = z.float().view(torch.int32).long()
        order = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))
        cols = z.shape[1]
        order = order * cols + torch.arange(cols - 1, -1, -1, device=z.device)
        columns = cols - 1 - order.topk(k, dim=1).values % cols
    return z.gather(1, columns), columns


def _plain_top(s):
    z = s["logits"]
    values, columns = _top(z, s["k"])
    x = _wide(z)
    highest = x.max(1, keepdim=True).values
    total = ((x - highest) / s["temperature"]).exp().sum(1)
    return [values, columns, total.log() + highest[:, 0] / s["temperature"]]


def _plain_distill(s):
    z, columns, tau = _wide(s["logits"]), s["columns"], s["temperature"]
    rows = z.shape[0]
    there = columns >= 0
    keep = there.any(1) if s["mask"] is None else there.any(1) & s["mask"]
    at = columns.clamp(min=0)
    # the teacher's few values, and the logarithms whose differences the loss is, in 64 bits
    t = s["values"].double().masked_fill(~there, -math.inf) / tau
    if s["rest"]:
        log_p = t - s["logsumexp"].double()[:, None]
    else:
        highest = t.max(1, keepdim=True).values.clamp(min=-1e300)
        log_p = t - highest - (t - highest).exp().sum(1, keepdim=True).clamp(min=1.0).log()
    p = log_p.exp()
    highest = z.max(1, keepdim=True).values
    e = ((z - highest) / tau).exp()
    total = e.sum(1, keepdim=True)
    log_total = total.double().log()
    log_q = (z.gather(1, at) - highest).double() / tau - log_total
    loss = (p * (log_p.masked_fill(p == 0, 0.0) - log_q)).masked_fill(~there, 0.0).sum(1)
    mass = p.sum(1, keepdim=True)
    if s["rest"] and s["k"] < s["cols"]:
        # one more answer: all that is not listed
        rest = (1.0 - mass).clamp(min=0.0)
        others = z.scatter(1, at, -math.inf)
        top = others.max(1, keepdim=True).values
        e_others = ((others - top) / tau).exp()
        sum_others = e_others.sum(1, keepdim=True)
        log_rest = (top - highest).double() / tau + sum_others.double().log() - log_total
        loss = loss + (torch.special.xlogy(rest, rest) - rest * log_rest)[:, 0]
        grad = e * ((mass + rest) / total).to(z.dtype) - e_others * (rest / sum_others).to(z.dtype)
    else:
        grad = e * (mass / total).to(z.dtype)
    grad = grad.scatter_add(1, at, (-p).masked_fill(~there, 0.0).to(z.dtype))
    scale = s["weight"]
    count = rows if s["mask"] is None else s["mask"].sum()
    per_row = torch.where(keep, loss, 0.0) * (tau * tau * scale)
    factor = torch.full((rows, 1), tau * scale, dtype=torch.float64, device=z.device)
    if s["reduction"] == "none":
        out, factor = per_row, factor * s["upstream"].double()[:, None]
    elif s["reduction"] == "sum":
        out = per_row.sum()
    else:
        out, factor = per_row.sum() / count, factor / count
    out = out.to(z.dtype)
    if not s["grad"]:
        return [out]
    return [out, (grad * factor.to(z.dtype)).masked_fill(~keep[:, None], 0.0).to(s["logits"].dtype)]


def _plain_balance(logits, k, mask, weight):
    z = _wide(logits)
    rows, experts = z.shape
    e = (z - z.max(1, keepdim=True).values).exp()
    p = e / e.sum(1, keepdim=True)
    chosen = torch.zeros_like(p, dtype=torch.bool).scatter_(1, _top(logits, k)[1], True)
    n = torch.full((), rows, dtype=torch.float64, device=z.device)
    if mask is not None:
        p, chosen, n = p * mask[:, None], chosen & mask[:, None], mask.sum(dtype=torch.float64)
    counts = chosen.sum(0)
    w = (counts.double() * (weight * experts / k) / (n * n)).to(p.dtype)
    loss = (w * p.sum(0)).sum()
    return loss, counts, (p * (w - (p * w).sum(1, keepdim=True))).to(logits.dtype)


def run(s):
    kind = s["kind"]
    if own:
        return _run_own(s)
    if kind == "top":
        return _plain_top(s)
    if kind == "distill":
        return _plain_distill(s)
    if kind == "balance":
        return list(_plain_balance(s["logits"], s["k"], s["mask"], s["weight"]))
    parts = [_plain_balance(z, 1, None, s["weight"] / len(s["logits"])) for z in s["logits"]]
    return [torch.stack([a for a, _, _ in parts]).sum(), torch.stack([c for _, c, _ in parts]), *(g for _, _, g in parts)]


def _run_own(s):
    import convlogic_amd as C
    kind = s["kind"]
    if kind == "top":
        return list(C.top_logits(s["logits"], s["k"], temperature=s["temperature"]))
    if kind == "gates":
        leaves = [z.detach().requires_grad_(True) for z in s["logits"]]
        loss, counts = C.gate_balance(leaves, weight=s["weight"])
        return [loss.detach(), counts, *torch.autograd.grad(loss, leaves)]
    if kind == "balance":
        z = s["logits"].detach().requires_grad_(True)
        loss, counts = C.balance_loss(z, s["k"], mask=s["mask"], weight=s["weight"])
        return [loss.detach(), counts, *torch.autograd.grad(loss, z)]
    z = s["logits"].detach().requires_grad_(s["grad"])
    loss = C.distillation_loss(z, s["values"], s["columns"], s["logsumexp"], temperature=s["temperature"], mask=s["mask"], weight=s["weight"],
                               reduction=s["reduction"])
    if not s["grad"]:
        return [loss]
    return [loss.detach(), *torch.autograd.grad(loss, z, s["upstream"] if s["reduction"] == "none" else None)]


# ---- the definitions in 64 bits -------------------------------------------------------------------
def _chunks(rows, cols):
    step = max(1, (1 << 25) // cols)
    return [slice(i, min(i + step, rows)) for i in range(0, rows, step)]


def _exact_distill(s):
    z, tau = s["logits"], s["temperature"]
    rows, cols = z.shape
    count = rows if s["mask"] is None else int(s["mask"].sum())
    losses, grads = [], []
    for part in _chunks(rows, cols):
        x = z[part].double().requires_grad_(True)
        columns, t = s["columns"][part], s["values"][part].double() / tau
        there = columns >= 0
        keep = there.any(1)
        if s["mask"] is not None:
            keep = keep & s["mask"][part]
        # (row, slot) pairs that are there, one after the other
        row, slot = there.nonzero(as_tuple=True)
        column = columns[row, slot]
        target = torch.zeros(x.shape, dtype=x.dtype, device=x.device)
        if s["rest"]:
            target[row, column] = (t[row, slot] - s["logsumexp"][part].double()[row]).exp()
        else:
            target[row, column] = torch.softmax(t.masked_fill(~there, -math.inf), 1)[row, slot]
        log_q = torch.log_softmax(x / tau, 1)
        loss = torch.special.xlogy(target, target).sum(1) - (target * log_q).sum(1)
        if s["rest"] and s["k"] < cols:
            listed_here = torch.zeros_like(target, dtype=torch.bool)
            listed_here[row, column] = True
            rest = (1.0 - target.sum(1)).clamp(min=0.0)
            loss = loss + torch.special.xlogy(rest, rest) - rest * torch.logsumexp(log_q.masked_fill(listed_here, -math.inf), 1)
        loss = torch.where(keep, loss, 0.0) * (tau * tau * s["weight"])
        if s["reduction"] == "mean":
            loss = loss / count
        up = s["upstream"][part].double() if s["reduction"] == "none" else torch.ones_like(loss)
        if s["grad"]:
            grads.append(torch.autograd.grad(loss, x, up)[0])
        losses.append(loss.detach())
    loss = torch.cat(losses)
    return [loss if s["reduction"] == "none" else loss.sum()] + ([torch.cat(grads)] if s["grad"] else [])


def _exact_balance(logits, k, mask, weight):
    rows, experts = logits.shape
    keep = torch.ones(rows, dtype=torch.bool, device=logits.device) if mask is None else mask
    n = int(keep.sum())
    x = logits.double()
    counts = torch.bincount(torch.sort(x[keep], dim=1, descending=True, stable=True).indices[:, :k].reshape(-1), minlength=experts)
    leaf = x.requires_grad_(True)
    p = torch.softmax(leaf, 1)
    loss = weight * experts * ((counts.double() / (k * n)) * (p[keep].sum(0) / n)).sum()
    return loss.detach(), counts, torch.autograd.grad(loss, leaf)[0]


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "distill":
        return _exact_distill(s)
    if kind == "balance":
        return list(_exact_balance(s["logits"], s["k"], s["mask"], s["weight"]))
    if kind == "gates":
        parts = [_exact_balance(z, 1, None, s["weight"]) for z in s["logits"]]
        return [sum(a for a, _, _ in parts) / len(parts), torch.stack([c for _, c, _ in parts]), *(g / len(parts) for _, _, g in parts)]
    out = []
    for part in _chunks(*s["logits"].shape):
        x = s["logits"][part].double()
        values, columns = torch.sort(x, dim=1, descending=True, stable=True)
        out.append((values[:, :s["k"]].clone(), columns[:, :s["k"]].clone(), torch.logsumexp(x / s["temperature"], 1)))
    return [torch.cat(parts) for parts in zip(*out)]


# ---- what a pass cannot do without ----------------------------------------------------------------
def work(case):
    size = {"f32": 4, "f64": 8}.get(case["dtype"], 2)
    if case["kind"] == "gates":
        elements = 16 * sum(_gate_rows(case))
        return dict(bytes=2 * size * elements, flops=14 * elements)
    rows, cols, k = case["rows"], case["cols"], case["k"]
    elements = rows * cols
    if case["kind"] == "top":
        return dict(bytes=elements * size + rows * (k * (size + 8) + 4), flops=5 * elements)
    if case["kind"] == "balance":
        return dict(bytes=2 * elements * size + rows * bool(case["masked"]), flops=(14 + k) * elements)
    wide = 8 if case["dtype"] == "f64" else 4
    lists = rows * (k * (wide + 8) + wide * case["rest"] + bool(case["masked"]))
    return dict(bytes=elements * size * (2 if case["grad"] else 1) + lists, flops=(10 if case["grad"] else 5) * elements)
