"""A training step that keeps little between its forward and its backward pass, as timed cases:

* "codes"  activations kept in 8 bits: 128 elements, as they lie in memory, share their lowest value and a step; a pass encodes and decodes
* "layer"  a training step of a LogicLayer that keeps its input like that: the output, and both gradients computed from the codes
* "loss"   softmax cross entropy of group sums, score = sum of a class's features / tau, without keeping the scores; with "grad" the gradient
           w.r.t. the features.  "rows" is a row per sample, "columns" a sample per column, as a LogicLayer leaves its output in memory

Sizes are those of this package's networks (10 classes, batches of 100, 128 and 256, LogicLayers of 8000 and of 131072 inputs, 320 k neurons in front of
the classes) and generic ones.  Where `own` is false, `run` computes the same from elementary torch operations in 32 bits, with the codes and the group
sums in 64."""
import math

import torch

own = False

DEV = "cuda:0"
_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "f64": torch.float64}
_SIZES = {"f32": 4, "f16": 2, "bf16": 2, "f64": 8}
GROUP = 128


def listed():
    return [
        # the input of one LogicLayer of 8000 neurons, 100 images: launches and the host
        dict(name="codes_layer", kind="codes", dtype="f32", shape="100x8000"),
        # 16-bit activations of an odd size: the last group is a part of one, nothing is aligned to anything
        dict(name="codes_ragged", kind="codes", dtype="bf16", shape="777x50001"),
        # what a block of the k = 1024 network of colour images takes, 128 images at once
        dict(name="codes_block", kind="codes", dtype="f32", shape="128x4096x16x16"),
        # a layer of 8000 neurons on 100 images: the smallest step, of latency
        dict(name="layer_small", kind="layer", inputs=8000, neurons=8000, batch=100),
        # the halving layers in front of the classes: every input is read once
        dict(name="layer_halving", kind="layer", inputs=163840, neurons=81920, batch=256),
        # an odd batch: rows of the wiring start at any address, a group of 128 covers parts of two features
        dict(name="layer_ragged", kind="layer", inputs=30001, neurons=60000, batch=333),
        # the first LogicLayer behind the blocks of a large network
        dict(name="layer_large", kind="layer", inputs=131072, neurons=1310720, batch=128),
        # the class sums of 100 digits, one feature to a class: the smallest loss
        dict(name="loss_digits", kind="loss", layout="rows", dtype="f32", rows=100, classes=10, group=1, smoothing=0.0, masked=False, reduction="mean",
             weight=1.0, grad=True),
        # 320 k neurons in front of 10 classes for k = 256, as the last layer leaves them
        dict(name="loss_neurons", kind="loss", layout="columns", dtype="f32", rows=256, classes=10, group=8192, smoothing=0.1, masked=False,
             reduction="mean", weight=1.0, grad=True),
        # validation over 1000 classes with a last batch of odd size: the loss of each row
        dict(name="loss_validation", kind="loss", layout="columns", dtype="f32", rows=1111, classes=1000, group=30, smoothing=0.0, masked=True,
             reduction="none", weight=1.0, grad=False),
        # one sequence over a long, odd vocabulary
        dict(name="loss_few", kind="loss", layout="rows", dtype="f16", rows=7, classes=50001, group=5, smoothing=0.0, masked=False, reduction="sum",
             weight=1024.0, grad=True),
        # a training step over a long vocabulary with padded sequences, the largest: 1 GiB of features
        dict(name="loss_tokens", kind="loss", layout="rows", dtype="bf16", rows=4096, classes=32768, group=4, smoothing=0.0, masked=True,
             reduction="mean", weight=1.0, grad=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["codes", "layer", "layer", "layer", "loss", "loss", "loss", "loss"])
    if kind == "codes":
        return dict(kind=kind, dtype=rng.choice(["f32", "f32", "bf16", "f16", "f64"]), shape=f"{_log(rng, 1, 4096)}x{_log(rng, 1, 16384)}")
    if kind == "layer":
        batch = _log(rng, 1, 2048) if rng.random() < 0.6 else rng.choice([64, 100, 128, 256, 512])
        neurons = _log(rng, 32, 1000000)
        while neurons * batch > 1 << 26:
            neurons = -(-neurons // 2)
        inputs = 2 * neurons if rng.random() < 0.3 else max(2, int(neurons * math.exp(rng.uniform(math.log(0.1), math.log(2.0)))))
        return dict(kind=kind, inputs=inputs, neurons=neurons, batch=batch)
    dtype = rng.choice(["f32", "f32", "f32", "bf16", "f16", "f64"])    # (f16: with the factor that such programs scale their losses by)
    classes, group, rows = _log(rng, 2, 65536), _log(rng, 1, 4096), _log(rng, 1, 8192)
    while rows * classes * group * _SIZES[dtype] > 1 << 30:
        if group > 16:
            group = -(-group // 2)
        elif rows > 16:
            rows = -(-rows // 2)
        else:
            classes = -(-classes // 2)
    return dict(kind=kind, layout=rng.choice(["rows", "columns"]), dtype=dtype, rows=rows, classes=classes, group=group,
                smoothing=rng.choice([0.0, 0.0, 0.1]), masked=rng.random() < 0.4, reduction=rng.choice(["mean", "mean", "mean", "sum", "none"]),
                weight=1024.0 if dtype == "f16" else rng.choice([1.0, 1.0, 0.5]), grad=rng.random() < 0.8)


# ---- preparation ----------------------------------------------------------------------------------
def _normal(shape, g, scale=1.0):
    return torch.randn(shape, generator=g, device=DEV) * scale


def _activations(rows, cols, g):
    """what logic gates put out: between 0 and 1, every row with a mean of its own, and a few rows that do not change (in 32 bits)"""
    x = _normal((rows, cols), g, 1.5).add_(_normal((rows, 1), g, 1.5)).sigmoid_()
    return torch.where(torch.rand((rows, 1), generator=g, device=DEV) < 0.02, x[:, :1], x)


def _shape(case):
    return [int(n) for n in case["shape"].split("x")]


def _tau(case):
    return 1.0 if case["group"] == 1 else 0.1 * math.sqrt(case["group"])


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s, kind = dict(case), case["kind"]
    if kind == "codes":
        shape = _shape(case)
        x = _activations(shape[0], math.prod(shape[1:]), g)
        s["x"] = x.to(_DTYPES[case["dtype"]]).view(shape)
        return s
    if kind == "layer":
        inputs, neurons, batch = case["inputs"], case["neurons"], case["batch"]
        # every input is read about equally often, in an order by chance
        slots = torch.randperm(2 * neurons, generator=g, device=DEV) % inputs
        slots = torch.randperm(inputs, generator=g, device=DEV)[slots]
        s["a"], s["b"] = slots[:neurons].contiguous(), slots[neurons:].contiguous()
        # logits of a network in training: every gate started as a wire (logit 5 at gate 3) and has moved since
        s["logits"] = _normal((neurons, 16), g, 2.0)
        s["logits"][:, 3] += 5.0
        s["x"] = _activations(inputs, batch, g).t()                   # (a sample per column in memory, as the layer in front leaves it)
        s["upstream"] = _normal((neurons, batch), g).t()
        if own:
            import convlogic_amd as C
            layer = C.LogicLayer(inputs, neurons, implementation="cuda", checkpoint_bits=8).to(DEV)
            with torch.no_grad():
                layer.weights.copy_(s["logits"])
                layer.indices_0.copy_(s["a"])
                layer.indices_1.copy_(s["b"])
            s["layer"] = layer
        return s
    rows, classes, group, dtype = case["rows"], case["classes"], case["group"], _DTYPES[case["dtype"]]
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    targets = torch.randint(0, classes, (rows,), generator=g, device=DEV)
    at = torch.arange(rows, device=DEV)
    if group == 1:
        x = _normal((rows, classes), g, 3.0)
        x[at, targets] += 6.0                                         # (a network that mostly knows its classes)
    else:
        x = torch.empty((rows, classes, group), device=DEV)
        for part in _chunks(rows, classes * group):
            x[part] = (_normal((x[part].shape), g, 1.5) + _normal((x[part].shape[0], classes, 1), g, 3.0 / math.sqrt(group))).sigmoid_()
        x[at, targets] = x[at, targets] * 0.7 + 0.3
    x = x.view(rows, classes * group).to(dtype)
    s["x"] = x if case["layout"] == "rows" else x.t().contiguous().t()
    if case["masked"]:
        # padded sequences: about a quarter of the rows, in runs at the ends of sequences of 64, counts for nothing
        lengths = torch.randint(32, 65, (rows // 64 + 1,), generator=g, device=DEV)
        targets = torch.where(at % 64 < lengths[at // 64], targets, -100)
    s["targets"], s["tau"] = targets, _tau(case)
    s["upstream"] = torch.rand((rows,), generator=g, device=DEV).to(wide)
    return s


# ---- the plain forms ------------------------------------------------------------------------------
def _coded(x):
    """x as its codes stand for it, in 32 bits (64 of 64); codes in 64, where values lie next to a border"""
    flat = x.reshape(-1)
    n = flat.numel()
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    groups = -(-n // GROUP)
    padded = torch.empty((groups * GROUP,), dtype=wide, device=x.device)
    padded[:n] = flat
    padded[n:] = padded[n - 1].clone()
    padded = padded.view(groups, GROUP)
    low, high = padded.amin(1, keepdim=True), padded.amax(1, keepdim=True)
    size = high.double() - low.double()
    step = (size / 255.0).to(wide)
    codes = ((padded.double() - low.double()) * 255.0 / torch.where(size > 0, size, 1.0)).round()
    return (codes * step.double() + low.double()).to(wide).view(-1)[:n].view(x.shape)


# coefficients of 1, a, b and a b of the 16 gates; gate i has the truth table (f00, f01, f10, f11) = bits of i, highest first
_GATES = [[(i >> 3) & 1, ((i >> 1) & 1) - ((i >> 3) & 1), ((i >> 2) & 1) - ((i >> 3) & 1),
           ((i >> 3) & 1) - ((i >> 2) & 1) - ((i >> 1) & 1) + (i & 1)] for i in range(16)]


def _plain_layer(s):
    """-> y [batch, neurons], gradient of x [batch, inputs], gradient of the logits"""
    a, b, x, up = s["a"], s["b"], s["x"].t(), s["upstream"].t()
    gates = torch.tensor(_GATES, device=x.device)
    e = (s["logits"] - s["logits"].max(1, keepdim=True).values).exp()
    p = e / e.sum(1, keepdim=True)
    c = (p[:, :, None] * gates).sum(1)[:, :, None]
    xa, xb = x[a], x[b]
    y = c[:, 0] + c[:, 1] * xa + c[:, 2] * xb + c[:, 3] * (xa * xb)
    kept = _coded(x)
    xa, xb = kept[a], kept[b]
    grad_x = torch.zeros_like(x).index_add_(0, a, up * (c[:, 1] + c[:, 3] * xb)).index_add_(0, b, up * (c[:, 2] + c[:, 3] * xa))
    sums = torch.stack([up.sum(1), (up * xa).sum(1), (up * xb).sum(1), (up * xa * xb).sum(1)], 1)
    grad_p = (sums[:, None, :] * gates).sum(2)
    return [y.t(), grad_x.t(), p * (grad_p - (p * grad_p).sum(1, keepdim=True))]


def _plain_loss(s):
    x, targets, classes, eps, tau = s["x"], s["targets"], s["classes"], s["smoothing"], s["tau"]
    rows = x.shape[0]
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    scores = x.view(rows, classes, -1).sum(2, dtype=torch.float64) / tau
    keep = targets >= 0
    at = targets.clamp(min=0)[:, None]
    highest = scores.max(1, keepdim=True).values
    e = (scores - highest).to(wide).exp()
    e_target = e.gather(1, at)
    others = e.scatter(1, at, 0.0).sum(1, keepdim=True)               # (all but the target's: a loss near 0 is exact like that)
    total = others + e_target
    margin = (highest - scores.gather(1, at)).to(wide)
    loss = (margin + torch.where(margin == 0, others.log1p(), total.log()))[:, 0]
    if eps:
        loss = (1.0 - eps) * loss + eps * (total.log()[:, 0] + (highest - scores).mean(1).to(wide))
    count = keep.sum().clamp(min=1)
    loss = torch.where(keep, loss, 0.0) * s["weight"]
    factor = s["upstream"] if s["reduction"] == "none" else torch.ones_like(s["upstream"])
    if s["reduction"] == "mean":
        factor = factor / count
    out = loss if s["reduction"] == "none" else (loss.double() * factor).sum().to(wide)
    if not s["grad"]:
        return [out]
    grad = (e / total).scatter(1, at, -others / total) - eps / classes
    if eps:
        grad = grad.scatter_add(1, at, torch.full_like(others, eps))
    grad = torch.where(keep[:, None], grad * (factor * (s["weight"] / tau))[:, None], 0.0).to(x.dtype)
    group = s["group"]
    if s["layout"] == "columns":
        return [out, grad.t().repeat_interleave(group, 0).t()]
    return [out, grad.repeat_interleave(group, 1)]


def run(s):
    kind = s["kind"]
    if own:
        return _run_own(s)
    if kind == "codes":
        return [_coded(s["x"]).to(s["x"].dtype)]
    return _plain_layer(s) if kind == "layer" else _plain_loss(s)


def _run_own(s):
    import convlogic_amd as C
    if s["kind"] == "codes":
        return [C.encode_activations(s["x"]).decode()]
    if s["kind"] == "layer":
        x = s["x"].detach().requires_grad_(True)
        y = s["layer"](x)
        return [y.detach(), *torch.autograd.grad(y, (x, s["layer"].weights), s["upstream"])]
    x = s["x"].detach().requires_grad_(s["grad"])
    loss = C.group_cross_entropy(x, s["targets"], s["classes"], tau=s["tau"], label_smoothing=s["smoothing"], weight=s["weight"], reduction=s["reduction"])
    if not s["grad"]:
        return [loss]
    return [loss.detach(), *torch.autograd.grad(loss, x, s["upstream"] if s["reduction"] == "none" else None)]


# ---- the definitions in 64 bits -------------------------------------------------------------------
def _chunks(rows, cols):
    step = max(1, (1 << 26) // cols)
    return [slice(i, min(i + step, rows)) for i in range(0, rows, step)]


def _exact_coded(x):
    flat = x.reshape(-1).double()
    n = flat.numel()
    whole = n // GROUP * GROUP
    out = torch.empty_like(flat)
    for begin, end in ((0, whole), (whole, n)):
        if begin == end:
            continue
        t = flat[begin:end].view(-1, min(GROUP, end - begin))
        low = t.min(1, keepdim=True).values
        size = t.max(1, keepdim=True).values - low
        codes = torch.where(size > 0, torch.round((t - low) * 255.0 / size), 0.0)
        out[begin:end] = (low + codes * (size / 255.0)).view(-1)
    return out.view(x.shape)


def _gate_values(a, b):
    """the 16 gates of a and b, [16, ...]"""
    both = a * b
    either = a + b - both
    one_of = a + b - 2 * both
    half = [torch.zeros_like(a), both, a - both, a, b - both, b, one_of, either]
    return torch.stack(half + [1 - h for h in reversed(half)])


def _exact_layer(s):
    a, b = s["a"], s["b"]
    x, up = s["x"].t().double(), s["upstream"].t()
    kept = _exact_coded(s["x"].t())
    grad_x = torch.zeros_like(x)
    y = torch.empty(up.shape, dtype=x.dtype, device=x.device)
    grad_logits = torch.empty(s["logits"].shape, dtype=x.dtype, device=x.device)
    for part in _chunks(up.shape[0], 8 * up.shape[1]):
        logits = s["logits"][part].double().requires_grad_(True)
        p = torch.softmax(logits, 1).t().unsqueeze(2)
        with torch.no_grad():
            y[part] = (p * _gate_values(x[a[part]], x[b[part]])).sum(0)
        xa, xb = kept[a[part]].requires_grad_(True), kept[b[part]].requires_grad_(True)
        ga, gb, grad_logits[part] = torch.autograd.grad((p * _gate_values(xa, xb)).sum(0), (xa, xb, logits), up[part].double())
        grad_x.index_add_(0, a[part], ga).index_add_(0, b[part], gb)
    return [y.t(), grad_x.t(), grad_logits]


def _exact_loss(s):
    targets, classes, eps, tau = s["targets"], s["classes"], s["smoothing"], s["tau"]
    x = s["x"]
    rows = x.shape[0]
    count = max(1, int((targets >= 0).sum()))
    losses = []
    grad = torch.empty(x.shape, dtype=torch.float64, device=x.device) if s["grad"] else None
    if s["grad"] and s["layout"] == "columns":
        grad = torch.empty((x.shape[1], rows), dtype=torch.float64, device=x.device).t()
    for part in _chunks(rows, x.shape[1]):
        scores = (x[part].double().view(-1, classes, s["group"]).sum(2) / tau).requires_grad_(True)
        keep = targets[part] >= 0
        goal = torch.full_like(scores, eps / classes)
        goal.scatter_add_(1, targets[part].clamp(min=0)[:, None], torch.full((scores.shape[0], 1), 1.0 - eps, dtype=goal.dtype, device=goal.device))
        loss = torch.where(keep, -(goal * torch.log_softmax(scores, 1)).sum(1), 0.0) * s["weight"]
        if s["reduction"] == "mean":
            loss = loss / count
        up = s["upstream"][part].double() if s["reduction"] == "none" else torch.ones_like(loss)
        if s["grad"]:
            g = torch.autograd.grad(loss, scores, up)[0] / tau
            grad[part] = g.unsqueeze(2).expand(-1, -1, s["group"]).reshape(g.shape[0], -1)
        losses.append(loss.detach())
    loss = torch.cat(losses)
    return [loss if s["reduction"] == "none" else loss.sum()] + ([grad] if s["grad"] else [])


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "codes":
        return [_exact_coded(s["x"])]
    return _exact_layer(s) if case["kind"] == "layer" else _exact_loss(s)


# ---- what a pass cannot do without ----------------------------------------------------------------
def _code_bytes(n, dtype):
    return n + 2 * (8 if dtype == "f64" else 4) * -(-n // GROUP)


def work(case):
    if case["kind"] == "codes":
        n = math.prod(_shape(case))
        return dict(bytes=2 * n * _SIZES[case["dtype"]] + 2 * _code_bytes(n, case["dtype"]), flops=7 * n)
    if case["kind"] == "layer":
        x, y = case["inputs"] * case["batch"], case["neurons"] * case["batch"]
        # forward: x, y and the codes; backward: the codes, both gradients; the logits with their gradient and the wiring
        return dict(bytes=8 * x + 8 * y + 2 * _code_bytes(x, "f32") + case["neurons"] * (2 * 64 + 16), flops=7 * x + 20 * y)
    scores = case["rows"] * case["classes"]
    elements = scores * case["group"]
    return dict(bytes=elements * _SIZES[case["dtype"]] * (2 if case["grad"] else 1) + case["rows"] * 8, flops=elements + (10 if case["grad"] else 6) * scores)
