"""The head-to-loss operators on sizes that stand for their use.

Three operators of ``atomo_amd.ops``:

* ``linear_ops.linear_act``     y = act(x W^T + b) + residual, and its backward pass
* ``logit_ops.label_logprobs``  log probability of a given class, entropy, top alternatives
* ``logit_ops.distill_loss``    distillation from a teacher's top logits, and its gradient

``run`` computes them with elementary torch operations where ``own`` is
false, and through the framework where it is true.  ``exact`` is the
definition in 64 bits.
"""

import math

import torch

own = False

_DTYPE = {
    "float32": torch.float32,
    "bfloat16": torch.bfloat16,
    "float16": torch.float16,
}
_BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
_IGNORE = -100


# -- cases --------------------------------------------------------------------


def _answers(name, rows, classes, dtype, top, pad=0, masked=False):
    return {"name": name, "op": "answers", "rows": rows, "classes": classes,
            "dtype": dtype, "top": top, "pad": pad, "masked": masked}


def _distill(name, rows, classes, dtype, top, temperature, weight, train,
             pad=0):
    # 16-bit floats train with a scaled loss: their smallest steps would lose
    # most of the gradient otherwise
    return {"name": name, "op": "distill", "rows": rows, "classes": classes,
            "dtype": dtype, "top": top, "temperature": temperature,
            "weight": weight, "train": train, "pad": pad,
            "scale": 65536.0 if dtype == "float16" else 1.0}


def _linear(name, rows, inner, outer, dtype, activation, residual, train):
    return {"name": name, "op": "linear", "rows": rows, "inner": inner,
            "outer": outer, "dtype": dtype, "activation": activation,
            "residual": residual, "train": train}


def listed():
    return [
        # one batch of the evaluator (--test-batch-size 500, ten classes,
        # prec@5): launch latency is all that counts
        _answers("answers-test-batch", 500, 10, "float32", 5),
        # one new token over a wide vocabulary: a single row has to fill the card
        _answers("answers-one-row", 1, 131072, "bfloat16", 20),
        # scoring given tokens: an odd vocabulary in padded rows, a tenth of it
        # not allowed
        _answers("answers-odd-bf16", 2048, 50021, "bfloat16", 8, pad=27,
                 masked=True),
        # a teacher's answers for distillation
        _answers("answers-teacher-fp32", 4096, 32000, "float32", 64),
        # one training batch of the trainer (--batch-size 128, 100 classes)
        _distill("distill-train-batch", 128, 100, "float32", 10, 4.0, 0.9, True),
        # the largest: a wide vocabulary, both losses, some rows ignored
        _distill("distill-bf16", 4096, 65536, "bfloat16", 64, 2.0, 0.5, True),
        # odd rows and classes in padded rows, the teacher alone
        _distill("distill-fp16-odd", 1001, 50021, "float16", 17, 1.0, 1.0, True,
                 pad=11),
        # the same loss on a validation set: no gradient
        _distill("distill-loss-fp32", 4096, 32000, "float32", 32, 2.0, 0.9,
                 False),
        # the first layer of the FC network on one batch
        _linear("linear-fc", 128, 784, 800, "float32", "relu", False, True),
        # the first and widest layer of AlexNet's classifier on one batch
        _linear("linear-alexnet", 128, 9216, 4096, "float32", "relu", False,
                True),
        # the largest: a block's product over many tokens, in half precision
        _linear("linear-bf16", 8192, 4096, 4096, "bfloat16", "gelu", True,
                True),
        # one request: the weight is read for a single row
        _linear("linear-one-row", 1, 9216, 4096, "bfloat16", "relu", False,
                False),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["answers", "distill", "linear"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if op == "linear":
        rows = _log_int(rng, 1, 8192)
        inner = _log_int(rng, 64, 9216)
        outer = _log_int(rng, 10, 4096)
        train = rng.random() < 0.7
        activation = rng.choice(["none", "relu", "gelu", "silu"])
        residual = rng.random() < 0.4
        # no dearer than the largest listed product of the same type
        limit = 8192 * 4096 * 4096 if dtype != "float32" else 128 * 9216 * 4096
        rows = max(1, min(rows, limit // (inner * outer)))
        case = _linear(None, rows, inner, outer, dtype, activation, residual,
                       train)
    else:
        classes = _log_int(rng, 10, 131072)
        rows = _log_int(rng, 1, 8192)
        rows = max(1, min(rows, 4096 * 32000 // classes))
        top = min(_log_int(rng, 1, 64), classes)
        pad = rng.choice([0, 0, 5, 64])
        if op == "answers":
            case = _answers(None, rows, classes, dtype, top, pad,
                            rng.random() < 0.3 and classes >= 1000)
        else:
            case = _distill(None, rows, classes, dtype, top,
                            rng.choice([1.0, 2.0, 4.0]),
                            rng.choice([0.5, 0.9, 1.0]),
                            rng.random() < 0.7, pad)
    del case["name"]
    return case


def work(case):
    size = _BYTES[case["dtype"]]
    if case["op"] == "linear":
        m, k, n = case["rows"], case["inner"], case["outer"]
        elements = m * k + n * k + n + m * n * (2 if case["residual"] else 1)
        flops = 2.0 * m * n * k
        if case["train"]:
            # dy in; dx, dW, db out (the residual's gradient is dy itself)
            elements += m * n + m * k + n * k + n
            flops *= 3
        return {"bytes": float(elements * size), "flops": flops}
    n, v, k = case["rows"], case["classes"], case["top"]
    if case["op"] == "answers":
        # an index and a 32-bit value for each alternative; label, log
        # probability and entropy for each row
        return {"bytes": float(n * v * size + n * (k * 12 + 16)),
                "flops": 6.0 * n * v}
    moved = n * v * size * (2 if case["train"] else 1) + n * (k * 12 + 8)
    return {"bytes": float(moved),
            "flops": (10.0 if case["train"] else 6.0) * n * v}


# -- inputs -------------------------------------------------------------------


def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _logits(case, gen):
    """Logits as a trained head gives them: most classes within a few units,
    the right one raised by some; rows may lie in a wider buffer."""
    n, v = case["rows"], case["classes"]
    dtype = _DTYPE[case["dtype"]]
    labels = torch.randint(0, v, (n,), generator=gen, device="cuda")
    buffer = torch.empty(n, v + case["pad"], dtype=dtype, device="cuda")
    if case["pad"]:
        buffer[:, v:] = 0
    logits = buffer[:, :v]
    dark = None
    if case.get("masked"):
        dark = torch.rand(v, generator=gen, device="cuda") < 0.1
        dark[0] = False
        labels = torch.where(dark[labels], torch.zeros_like(labels), labels)
    step = max(1, (1 << 26) // v)
    for i in range(0, n, step):
        j = min(n, i + step)
        part = _randn(gen, j - i, v).mul_(2.5)
        raised = 6.0 + 2.0 * _randn(gen, j - i, 1)
        part.scatter_add_(1, labels[i:j, None], raised)
        if dark is not None:
            part.masked_fill_(dark, float("-inf"))
        logits[i:j] = part
    return logits, labels


def prepare(case, seed):
    gen = _generator(seed)
    state = {"case": dict(case)}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["inner"], case["outer"]
        dtype = _DTYPE[case["dtype"]]
        x = _randn(gen, m, k)
        weight = _randn(gen, n, k) / math.sqrt(k)
        bias = _randn(gen, n) * 0.1
        if case["activation"] == "relu":
            # on a grid on which 32-bit sums are exact, in any order: on which
            # side of relu's border a unit lies is then no matter of rounding
            x = (x * 16.0).round().clamp(-127.0, 127.0) / 16.0
            weight = (weight * 4096.0).round() / 4096.0
            bias = (bias * 4096.0).round() / 4096.0
        state["x"] = x.to(dtype)
        state["weight"] = weight.to(dtype)
        state["bias"] = bias.to(dtype)
        state["residual"] = (
            _randn(gen, m, n).to(dtype) if case["residual"] else None
        )
        if case["train"]:
            state["dy"] = (_randn(gen, m, n) * 0.1).to(dtype)
            for name in ("x", "weight", "bias", "residual"):
                if state[name] is not None:
                    state[name].requires_grad_()
        return state
    logits, labels = _logits(case, gen)
    state["logits"] = logits
    if case["op"] == "answers":
        state["labels"] = labels
        return state
    n, v, k = case["rows"], case["classes"], case["top"]
    values = torch.empty(n, k, device="cuda")
    index = torch.empty(n, k, dtype=torch.int64, device="cuda")
    step = max(1, (1 << 26) // v)
    for i in range(0, n, step):
        j = min(n, i + step)
        teacher = logits[i:j].float() * 0.8 + _randn(gen, j - i, v)
        values[i:j], index[i:j] = teacher.topk(k, dim=1)
    state["values"], state["index"] = values, index
    state["labels"] = None
    if case["weight"] < 1.0:
        # one row in eight is padding
        skip = torch.rand(n, generator=gen, device="cuda") < 0.125
        skip[0] = False
        state["labels"] = torch.where(
            skip, torch.full_like(labels, _IGNORE), labels)
    if case["train"]:
        state["logits"] = logits.detach().requires_grad_()
        state["scale"] = torch.tensor(case["scale"], device="cuda")
    return state


# -- one pass -----------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if op == "answers":
        return _run_answers(state)
    if op == "distill":
        return _run_distill(state)
    return _run_linear(state)


def _run_answers(state):
    case = state["case"]
    if own:
        from atomo_amd.ops import logit_ops

        out = logit_ops.label_logprobs(
            state["logits"], state["labels"], top=case["top"])
        return (out.logprob, out.entropy, out.top_logprob, out.top_index)
    z = state["logits"].float()
    peak = z.amax(1, keepdim=True)
    shifted = z - peak
    e = shifted.exp()
    total = e.sum(1, keepdim=True)
    log_total = total.log()
    # 0 * -inf of a class that is not allowed counts as nothing
    weighted = torch.where(e > 0, e * shifted, torch.zeros_like(e)).sum(1)
    entropy = log_total[:, 0] - weighted / total[:, 0]
    logprob = (shifted.gather(1, state["labels"][:, None]) - log_total)[:, 0]
    # the order of the floats as whole numbers, the lowest index first
    bits = (z + 0.0).view(torch.int32).to(torch.int64)
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF) - 1, bits)
    column = torch.arange(z.shape[1], device=z.device)
    key = (order << 32) + (0x7FFFFFFF - column)
    best = key.topk(case["top"], dim=1).values
    top_index = 0x7FFFFFFF - (best & 0xFFFFFFFF)
    top_logprob = shifted.gather(1, top_index) - log_total
    return (logprob, entropy, top_logprob, top_index)


def _run_distill(state):
    case = state["case"]
    tau, weight = case["temperature"], case["weight"]
    logits, labels = state["logits"], state["labels"]
    if own:
        from atomo_amd.ops import logit_ops

        loss = logit_ops.distill_loss(
            logits, state["values"], state["index"], labels,
            temperature=tau, weight=weight, ignore_index=_IGNORE)
        if not case["train"]:
            return (loss,)
        (grad,) = torch.autograd.grad(loss, logits, state["scale"])
        return (loss.detach(), grad)
    with torch.no_grad():
        z = logits.float()
        n = z.shape[0]
        t = state["values"] / tau
        t = t - t.amax(1, keepdim=True)
        log_q = t - t.exp().sum(1, keepdim=True).log()
        q = log_q.exp()
        soft = z / tau
        soft = soft - soft.amax(1, keepdim=True)
        e = soft.exp()
        total = e.sum(1, keepdim=True)
        log_p = soft.gather(1, state["index"]) - total.log()
        row = weight * tau * tau * (q * (log_q - log_p)).sum(1)
        grad = e / total if case["train"] else None
        if grad is not None:
            grad = grad.scatter_add(1, state["index"], -q) * (weight * tau)
        if labels is None:
            loss = row.sum() / n
            scale = torch.full((n, 1), 1.0 / n, device=z.device)
        else:
            counted = labels != _IGNORE
            label = labels.clamp_min(0)[:, None]
            hard = z - z.amax(1, keepdim=True)
            e = hard.exp()
            total = e.sum(1, keepdim=True)
            row = row + (1.0 - weight) * (
                total.log() - hard.gather(1, label))[:, 0]
            many = counted.sum()
            loss = torch.where(counted, row, torch.zeros_like(row)).sum() / many
            if grad is not None:
                rest = (e / total).scatter_add(
                    1, label, torch.full((n, 1), -1.0, device=z.device))
                grad = grad + (1.0 - weight) * rest
                scale = (counted.float() / many)[:, None]
        if grad is None:
            return (loss,)
        grad = grad * (scale * state["scale"])
        return (loss, grad.to(logits.dtype))


def _slope(name, h):
    if name == "none":
        return torch.ones_like(h)
    if name == "relu":
        return (h > 0).to(h.dtype)
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-h))
        return s * (1.0 + h * (1.0 - s))
    half = 0.5 * (1.0 + torch.erf(h * math.sqrt(0.5)))
    return half + h * torch.exp(-0.5 * h * h) * (1.0 / math.sqrt(2.0 * math.pi))


def _activate(name, h):
    if name == "none":
        return h
    if name == "relu":
        return h * (h > 0).to(h.dtype)
    if name == "silu":
        return h / (1.0 + torch.exp(-h))
    return h * (0.5 * (1.0 + torch.erf(h * math.sqrt(0.5))))


def _run_linear(state):
    case = state["case"]
    x, weight, bias = state["x"], state["weight"], state["bias"]
    residual = state["residual"]
    if own:
        from atomo_amd.ops import linear_ops

        y = linear_ops.linear_act(
            x, weight, bias, activation=case["activation"], residual=residual)
        if not case["train"]:
            return (y,)
        leaves = [x, weight, bias] + ([] if residual is None else [residual])
        return (y.detach(), *torch.autograd.grad(y, leaves, state["dy"]))
    with torch.no_grad():
        dtype = x.dtype
        wide_x, wide_w = x.float(), weight.float()
        h = wide_x @ wide_w.t() + bias.float()
        y = _activate(case["activation"], h)
        if residual is not None:
            y = y + residual.float()
        y = y.to(dtype)
        if not case["train"]:
            return (y,)
        dp = state["dy"].float() * _slope(case["activation"], h)
        out = [y, (dp @ wide_w).to(dtype), (dp.t() @ wide_x).to(dtype),
               dp.sum(0).to(dtype)]
        if residual is not None:
            out.append(state["dy"])
        return tuple(out)


# -- the definition in 64 bits ------------------------------------------------


def _row_parts(rows, classes):
    step = max(1, (1 << 25) // classes)
    return [(i, min(rows, i + step)) for i in range(0, rows, step)]


def exact(case, seed):
    with torch.no_grad():
        state = prepare(case, seed)
        if case["op"] == "answers":
            return _exact_answers(case, state)
        if case["op"] == "distill":
            return _exact_distill(case, state)
        return _exact_linear(case, state)


def _exact_answers(case, state):
    outs = []
    for i, j in _row_parts(case["rows"], case["classes"]):
        z = state["logits"][i:j].double()
        logp = z - torch.logsumexp(z, 1, keepdim=True)
        entropy = torch.special.entr(logp.exp()).sum(1)
        # a stable sort leaves equal values in the order of their index
        index = torch.sort(z, dim=1, descending=True, stable=True).indices
        index = index[:, : case["top"]].clone()
        label = state["labels"][i:j]
        outs.append((logp[torch.arange(j - i, device=z.device), label],
                     entropy, torch.take_along_dim(logp, index, 1), index))
    return tuple(torch.cat(part) for part in zip(*outs))


def _exact_distill(case, state):
    tau, weight = case["temperature"], case["weight"]
    labels = state["labels"]
    rows, classes = case["rows"], case["classes"]
    counted = rows if labels is None else int((labels != _IGNORE).sum())
    loss = torch.zeros((), dtype=torch.float64, device="cuda")
    grads = []
    for i, j in _row_parts(rows, classes):
        z = state["logits"][i:j].double()
        q = torch.zeros_like(z)
        q.scatter_add_(1, state["index"][i:j],
                       torch.softmax(state["values"][i:j].double() / tau, 1))
        log_p = torch.log_softmax(z / tau, 1)
        part = (torch.special.xlogy(q, q) - q * log_p).sum(1) * tau ** 2 * weight
        grad = weight * tau * (log_p.exp() - q)
        if labels is not None:
            y = labels[i:j]
            keep = (y != _IGNORE).double()
            hot = torch.zeros_like(z).scatter_(1, y.clamp_min(0)[:, None], 1.0)
            log_1 = torch.log_softmax(z, 1)
            part = (part - (1.0 - weight) * (hot * log_1).sum(1)) * keep
            grad = (grad + (1.0 - weight) * (log_1.exp() - hot)) * keep[:, None]
        loss = loss + part.sum() / counted
        if case["train"]:
            # 64 bits of the whole gradient stay within the card's memory
            grads.append(grad * (case["scale"] / counted))
    if not case["train"]:
        return (loss,)
    return (loss, torch.cat(grads))


def _exact_linear(case, state):
    name = case["activation"]
    x = state["x"].double()
    w = state["weight"].double()
    h = torch.addmm(state["bias"].double(), x, w.t())
    gauss = torch.special.ndtr(h)
    sig = torch.sigmoid(h)
    y = {"none": h, "relu": h.clamp_min(0), "gelu": h * gauss,
         "silu": h * sig}[name]
    if state["residual"] is not None:
        y = y + state["residual"].double()
    if not case["train"]:
        return (y,)
    density = torch.exp(-h.square() / 2) / math.sqrt(2 * math.pi)
    slope = {"none": torch.ones_like(h), "relu": torch.heaviside(
        h, torch.zeros_like(h)), "gelu": gauss + h * density,
        "silu": sig + y.new_tensor(1.0) * h * sig * (1 - sig)}[name]
    dy = state["dy"].double()
    dp = dy * slope
    out = [y, dp @ w, dp.t().contiguous() @ x, dp.sum(0)]
    if state["residual"] is not None:
        out.append(dy)
    return tuple(out)
