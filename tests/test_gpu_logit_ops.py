"""label_logprobs and distill_loss on the GPU against the 64-bit oracle on the
CPU, at the sizes and masks where the kernels can go wrong."""

import math

import pytest
import torch

from atomo_amd.ops import logit_ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of fp32, relative
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16

SIZES = [(1, 1), (4, 3), (500, 10), (37, 100), (3, 511), (2, 1025), (5, 4099),
         (2, 16385), (3, 50021), (1, 131072), (2, 70001)]


def _steps(classes, spread):
    """Roundings, in half steps, of a sum over the classes: a thread adds at
    most classes / 64 terms one after the other, some 64 more join the
    threads; exp(d) is off by its argument's rounding, 2 |d| half steps, and
    exp itself by 4."""
    return classes / 64 + 64 + 2 * spread + 4


def _spread(z):
    """The largest |d| that still counts: exp(-104) is 0 in fp32."""
    wide = z.double()
    finite = wide[torch.isfinite(wide)]
    return float(min(104.0, (finite.max() - finite.min()))) if finite.numel() else 0.0


def _logits(rows, classes, dtype, seed=0, mask=None, pad=0, offset=0):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(rows, classes, generator=g) * 3
    if mask == "some":
        z[torch.rand(rows, classes, generator=g) < 0.3] = -math.inf
    elif mask == "most":
        z[torch.rand(rows, classes, generator=g) < 0.995] = -math.inf
    elif mask == "lowest":
        low = torch.rand(rows, classes, generator=g) < 0.3
        z = z.to(dtype).masked_fill_(low, torch.finfo(dtype).min)
    elif mask == "odd":
        z[0] = -math.inf
        z[-1, classes // 2] = math.nan
        if rows > 2:
            z[1, -1] = math.inf
    elif mask == "ties":
        z = torch.randint(-2, 2, (rows, classes), generator=g) * -0.0 + \
            torch.randint(0, 2, (rows, classes), generator=g).float()
    elif mask == "flat":
        z[:] = 0.25
    elif mask == "rising":
        z = torch.linspace(-5, 5, classes).expand(rows, classes).contiguous()
    z = z.to(dtype)
    cuda = torch.zeros(rows, classes + pad + offset, dtype=dtype, device="cuda")
    cuda = cuda[:, offset:offset + classes]
    cuda.copy_(z)
    return z, cuda


def _same_odd(a, b):
    """Equal where infinite or NaN; masks those out."""
    assert torch.equal(a.isnan(), b.isnan())
    assert torch.equal(a.isinf(), b.isinf())
    assert torch.equal(a[a.isinf()], b[b.isinf()])
    return torch.isfinite(a)


def _check_logprobs(z, cuda, y, top):
    want = logit_ops.label_logprobs(z, y, top=top)
    got = logit_ops.label_logprobs(cuda, None if y is None else y.cuda(), top=top)
    classes = z.shape[1]
    u = U * _steps(classes, _spread(z))
    for a, b in ((got.logprob, want.logprob), (got.top_logprob, want.top_logprob)):
        if a is None:
            continue
        a, b = a.cpu().double(), b.double()
        ok = _same_odd(a, b)
        # log S: the sum's relative error; d: half a step of itself
        assert ((a - b).abs()[ok] <= u + 4 * U * b.abs()[ok] + 4 * U * math.log(classes + 1)).all()
    a, b = got.entropy.cpu().double(), want.entropy.double()
    ok = _same_odd(a, b)
    # T / S: two sums' errors on a quotient below the entropy
    assert ((a - b).abs()[ok] <= 3 * u * (1 + b.abs()[ok]) + 4 * U * math.log(classes + 1)).all()
    if top:
        assert torch.equal(got.top_index.cpu(), want.top_index)


def _labels(rows, classes, seed=3):
    g = torch.Generator().manual_seed(seed)
    y = torch.randint(0, classes, (rows,), generator=g)
    y[::3] = -100
    return y


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,classes", SIZES)
def test_logprobs_sizes(rows, classes, dtype):
    z, cuda = _logits(rows, classes, dtype, seed=classes)
    for top in sorted({0, 1, min(5, classes), min(128, classes)}):
        _check_logprobs(z, cuda, _labels(rows, classes), top)


@pytest.mark.parametrize("mask", ["some", "most", "lowest", "odd", "ties", "flat", "rising"])
@pytest.mark.parametrize("rows,classes,dtype", [
    (5, 10, F32), (4, 700, F16), (4, 5000, BF16), (3, 33333, F32), (600, 3000, BF16)])
def test_logprobs_masks(rows, classes, dtype, mask):
    z, cuda = _logits(rows, classes, dtype, seed=7, mask=mask)
    _check_logprobs(z, cuda, _labels(rows, classes), min(20, classes))


@pytest.mark.parametrize("pad,offset", [(1, 0), (0, 1), (5, 3), (64, 8)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_logprobs_strides(dtype, pad, offset):
    for rows, classes in ((9, 10), (6, 4097)):
        z, cuda = _logits(rows, classes, dtype, pad=pad, offset=offset)
        _check_logprobs(z, cuda, _labels(rows, classes), 7)
    z, cuda = _logits(1, 300, dtype)
    _check_logprobs(z.expand(5, 300), cuda.expand(5, 300), _labels(5, 300), 7)


def test_logprobs_labels_outside_and_other_stream():
    z, cuda = _logits(4, 50, F32)
    y = torch.tensor([-100, 50, -1, 2 ** 40])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = logit_ops.label_logprobs(cuda, y.cuda(), top=3)
    torch.cuda.current_stream().wait_stream(side)
    assert out.logprob[0] == 0 and out.logprob[1:].isnan().all()
    none = logit_ops.label_logprobs(cuda[:0], y[:0].cuda(), top=3)
    assert none.top_index.shape == (0, 3)


@pytest.mark.parametrize("classes,dtype", [(4300001, F32), (8500003, BF16)])
@pytest.mark.parametrize("mask", [None, "ties"])
def test_logprobs_of_parts_with_several_selections(classes, dtype, mask):
    z, cuda = _logits(2, classes, dtype, seed=9, mask=mask)
    _check_logprobs(z, cuda, torch.tensor([classes - 1, -100]), 33)


def test_more_rows_than_one_dimension_of_a_grid():
    rows, classes = 300001, 3
    z, cuda = _logits(rows, classes, F32)
    y = _labels(rows, classes)
    _check_logprobs(z, cuda, y, 2)
    value, index = _teacher(1, classes, 2)
    _check_distill(z, cuda, value.expand(rows, 2), index.expand(rows, 2).contiguous(), y, 2.0, 0.5)


@pytest.mark.parametrize("rows,classes", [(1, 100000), (300, 10), (70, 5000)])
def test_logprobs_in_a_graph(rows, classes):
    _, first = _logits(rows, classes, BF16, seed=1)
    y = _labels(rows, classes).cuda()
    static = first.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        logit_ops.label_logprobs(static, y, top=4)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = logit_ops.label_logprobs(static, y, top=4)
    for seed in range(4):
        _, now = _logits(rows, classes, BF16, seed=seed)
        static.copy_(now)
        graph.replay()
        want = logit_ops.label_logprobs(now, y, top=4)
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


# ---------------------------------------------------------------------------
def _teacher(rows, classes, k, seed=5, repeat=False):
    g = torch.Generator().manual_seed(seed)
    if repeat:
        index = torch.randint(0, classes, (rows, k), generator=g)
    else:
        index = torch.stack([torch.randperm(classes, generator=g)[:k] for _ in range(rows)])
    return torch.randn(rows, k, generator=g) * 2, index


def _terms(z, value, index, y, tau, weight):
    """Sizes of the parts that the loss and the gradient are made of, in 64
    bits: what roundings are relative to."""
    d = z.double()
    d = (d - d.amax(1, keepdim=True).clamp_min(-1e300)).nan_to_num(0, 0, -1e300)
    p1 = torch.softmax(d, 1)
    pt = torch.softmax(d / tau, 1)
    there = value != -math.inf
    t = value.double().masked_fill(~there, -1e300) / tau
    share = torch.softmax(t, 1) * there
    at = torch.where(there & (index >= 0) & (index < z.shape[1]), index, 0)
    q = torch.zeros_like(p1).scatter_add_(1, at, share)
    grad = weight * tau * (pt + q)
    low = math.log(z.shape[1] + 1)
    # roundings are relative to the distance itself, 3.4e38 for a class at the
    # type's lowest value (half a step of that is 2e31); -inf stands at 1e300
    # and only reaches losses that are infinite
    dist = -(d / tau)
    loss = weight * tau ** 2 * ((q * (dist + low)).sum(1) +
                                (share * (t - t.amax(1, keepdim=True)).abs().clamp_max(1e30)).sum(1) + low)
    if y is not None and weight < 1:
        hot = torch.zeros_like(p1).scatter_(1, y.clamp(0, z.shape[1] - 1)[:, None], 1.0)
        grad = grad + (1 - weight) * (p1 + hot)
        loss = loss + (1 - weight) * ((hot * -d).sum(1) + low)
    return loss, grad


def _check_distill(z, cuda, value, index, y, tau, weight, reduction="mean", up=1.0):
    rows, classes = z.shape
    leaf = z.clone().requires_grad_()
    kw = dict(temperature=tau, weight=weight, reduction=reduction)
    want = logit_ops.distill_loss(leaf, value, index, y, **kw)
    g = torch.Generator().manual_seed(11)
    up = torch.rand(want.shape, generator=g) + 0.5 if reduction == "none" else torch.tensor(up)
    # the oracle's gradient in 64 bits: of an fp32 leaf it rounds once more
    (ref,) = torch.autograd.grad(want, leaf, up)
    cl = cuda.detach().requires_grad_()
    yc = None if y is None else y.cuda()
    got = logit_ops.distill_loss(cl, value.cuda(), index.cuda(), yc, **kw)
    (grad,) = torch.autograd.grad(got, cl, up.cuda(), retain_graph=True)
    (again,) = torch.autograd.grad(got, cl, up.cuda())
    # the second pass gives what the first gave
    assert torch.equal(grad.isnan(), again.isnan())
    assert torch.equal(grad.nan_to_num(), again.nan_to_num())
    with torch.no_grad():
        plain = logit_ops.distill_loss(cuda, value.cuda(), index.cuda(), yc, **kw)
    assert torch.equal(plain.isnan(), got.isnan()) and torch.equal(plain.nan_to_num(), got.nan_to_num())
    k = value.shape[1]
    u = U * (_steps(classes, _spread(z) * max(1.0, 1 / tau)) + 2 * k + _spread(value))
    loss_size, grad_size = _terms(z, value, index, y, tau, weight)
    count = 1.0
    counted = torch.ones(rows, dtype=torch.bool) if y is None else y != -100
    if reduction == "mean":
        count = max(1, int(counted.sum()))
    a, b = got.cpu().double(), want.detach().double()
    ok = _same_odd(a, b)
    if reduction == "none":
        tol = 2 * u * loss_size
    else:
        # the rows' errors, and those of adding them up
        tol = (2 * u + U * (rows / 64 + 64)) * (loss_size * counted).sum() / count
    assert ((a - b).abs() <= tol)[ok].all()
    a, b = grad.cpu().double(), ref.double()
    ok = _same_odd(a, b)
    ups = up.double().abs()
    ups = ups[:, None] if ups.dim() else ups
    eps = torch.finfo(z.dtype).eps / 2
    tiny = torch.finfo(z.dtype).smallest_normal * torch.finfo(z.dtype).eps
    # the fp32 arithmetic, then one rounding on either side, then half a step
    # next to zero on either side
    tol = 2 * u * grad_size * ups / count + 2 * eps * b.abs() + 2 * tiny
    assert ((a - b).abs() <= tol)[ok].all()
    if y is not None:
        assert (grad[(y == -100).cuda()] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,classes", SIZES)
def test_distill_sizes(rows, classes, dtype):
    z, cuda = _logits(rows, classes, dtype, seed=classes)
    y = _labels(rows, classes)
    if rows == 1:
        y[0] = 0
    for k in sorted({1, min(10, classes), min(128, classes)}):
        value, index = _teacher(rows, classes, k)
        _check_distill(z, cuda, value, index, y, 2.0, 0.7)
        _check_distill(z, cuda, value, index, None, 1.0, 1.0, "sum")


@pytest.mark.parametrize("classes,dtype", [
    (4097, F32), (9000, BF16), (16385, F32), (40001, BF16), (32770, F32),
    (70001, BF16), (131072, BF16), (65537, F32), (131073, BF16), (9001, F16)])
def test_distill_long_rows_in_registers(classes, dtype):
    """Enough rows that each has a workgroup; lengths around what 64, 256, 512
    and 1024 threads hold, and beyond."""
    rows = 129
    z, cuda = _logits(rows, classes, dtype, seed=classes)
    z[3] = -math.inf
    z[4, 1:] = -math.inf
    cuda.copy_(z)
    value, index = _teacher(rows, classes, 5)
    y = _labels(rows, classes)
    leaf = cuda.detach().requires_grad_()
    args = (value.cuda(), index.cuda(), y.cuda())
    loss = logit_ops.distill_loss(leaf, *args, temperature=2.0, weight=0.7)
    (grad,) = torch.autograd.grad(loss, leaf)
    # against the same in 64 bits, on the device for speed
    wide = z[5:].cuda().double()
    count = int((y != -100).sum())
    q = torch.zeros_like(wide).scatter_(1, args[1][5:], torch.softmax(args[0][5:].double() / 2, 1))
    at = args[2][5:].clamp_min(0)[:, None]
    hot = torch.zeros_like(wide).scatter_(1, at, 1.0)
    pt, p1 = torch.softmax(wide / 2, 1), torch.softmax(wide, 1)
    keep = (args[2][5:] != -100).double()[:, None] / count
    want = (1.4 * (pt - q) + 0.3 * (p1 - hot)) * keep
    size = (1.4 * (pt + q) + 0.3 * (p1 + hot)) * keep
    u = U * (_steps(classes, _spread(z)) + 10 + _spread(value))
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    tol = 2 * u * size + half * want.abs() + tiny
    assert ((grad[5:].double() - want).abs() <= tol).all()
    assert (grad[3] == 0).all() and (grad[args[2] == -100] == 0).all()
    few = z[:5].clone()
    cpu = logit_ops.distill_loss(few, value[:5], index[:5], y[:5], temperature=2.0,
                                 weight=0.7, reduction="none")
    gpu = logit_ops.distill_loss(cuda[:5], *(t[:5] for t in args), temperature=2.0,
                                 weight=0.7, reduction="none").cpu()
    # a handful of rows goes another way
    loss_size, _ = _terms(few, value[:5], index[:5], y[:5], 2.0, 0.7)
    ok = _same_odd(gpu, cpu)
    assert ((gpu - cpu).abs() <= 2 * u * loss_size)[ok].all()
    rest = torch.cat([cpu.double(), (
        2.8 * (torch.special.xlogy(q, q) - q * torch.log_softmax(wide / 2, 1)).sum(1)
        - 0.3 * torch.log_softmax(wide, 1).gather(1, at)[:, 0]).cpu() * (y[5:] != -100)])
    if torch.isfinite(rest).all():
        total, _ = _terms(z, value, index, y, 2.0, 0.7)
        bound = (2 * u + U * (rows / 64 + 64)) * (total * (y != -100)).sum() / count
        assert abs(float(loss) - float(rest.sum() / count)) <= bound


@pytest.mark.parametrize("tau,weight,reduction,up", [
    (1.0, 0.5, "mean", 1.0), (4.0, 0.9, "none", 1.0), (0.25, 0.3, "sum", 3.0),
    (2.0, 0.0, "mean", 0.0), (3.0, 1.0, "mean", -1.5), (2.0, 0.5, "mean", 1024.0)])
@pytest.mark.parametrize("rows,classes,dtype", [(6, 100, F32), (5, 5003, BF16), (300, 1000, F16)])
def test_distill_forms(rows, classes, dtype, tau, weight, reduction, up):
    z, cuda = _logits(rows, classes, dtype)
    value, index = _teacher(rows, classes, 17, repeat=True)
    value[0, 3:] = -math.inf
    index[0, 5] = classes + 4  # absent: never looked at
    value[2] = -math.inf
    y = _labels(rows, classes)
    index[1, 0] = y[1]  # the label among the teacher's classes, twice
    index[1, 9] = y[1]
    _check_distill(z, cuda, value, index, y, tau, weight, reduction, up)


@pytest.mark.parametrize("mask", ["some", "lowest", "odd", "flat"])
@pytest.mark.parametrize("rows,classes,dtype", [(5, 10, F32), (4, 700, F16), (3, 33333, BF16)])
def test_distill_masks(rows, classes, dtype, mask):
    z, cuda = _logits(rows, classes, dtype, mask=mask)
    value, index = _teacher(rows, classes, 6)
    y = _labels(rows, classes)
    y[1] = 1
    for reduction in ("none", "mean"):
        _check_distill(z, cuda, value, index, y, 2.0, 0.6, reduction)


@pytest.mark.parametrize("classes", [50, 20000])
def test_distill_wrong_entries(classes):
    z, cuda = _logits(6, classes, F32)
    value, index = _teacher(6, classes, 3)
    index[0, 1], index[1, 2] = classes, -1
    value[2, 0] = math.nan
    y = torch.tensor([0, 0, 0, classes, -1, 2])
    _check_distill(z, cuda, value, index, y, 2.0, 0.6, "none")


@pytest.mark.parametrize("classes", [50, 20000])
def test_distill_infinite_teacher(classes):
    z, cuda = _logits(3, classes, F32)
    value, index = _teacher(3, classes, 4)
    value[1, 2] = math.inf
    y = torch.tensor([0, 1, -100])
    _check_distill(z, cuda, value, index, y, 2.0, 0.6, "none")


@pytest.mark.parametrize("pad,offset", [(1, 0), (5, 3), (64, 8)])
def test_distill_strides(pad, offset):
    for dtype in (F32, F16):
        z, cuda = _logits(6, 4097, dtype, pad=pad, offset=offset)
        value, index = _teacher(6, 4097, 9)
        _check_distill(z, cuda, value, index, None, 2.0, 1.0)


def test_distill_all_rows_ignored():
    _, cuda = _logits(3, 40, F32)
    value, index = _teacher(3, 40, 4)
    y = torch.full((3,), -100).cuda()
    leaf = cuda.requires_grad_()
    loss = logit_ops.distill_loss(leaf, value.cuda(), index.cuda(), y, weight=0.5)
    loss.backward()
    assert loss == 0 and (leaf.grad == 0).all()
    none = logit_ops.distill_loss(cuda[:0], value[:0].cuda(), index[:0].cuda())
    assert none == 0


def test_distill_refuses_a_second_derivative_and_a_changed_input():
    _, cuda = _logits(3, 40, F32)
    value, index = (t.cuda() for t in _teacher(3, 40, 4))
    leaf = cuda.requires_grad_()
    loss = logit_ops.distill_loss(leaf, value, index)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, leaf, create_graph=True)
    with pytest.raises(ValueError):
        logit_ops.distill_loss(leaf, value.cpu(), index)
    moved = leaf * 1.0
    loss = logit_ops.distill_loss(moved, value, index)
    with torch.no_grad():
        moved.mul_(2.0)
    with pytest.raises(RuntimeError):
        (2.0 * loss).backward()


@pytest.mark.parametrize("rows,classes,dtype", [(128, 100, F32), (3, 60000, BF16), (40, 5000, F16)])
def test_distill_in_a_graph(rows, classes, dtype):
    """Forward and backward captured, replayed between eager passes."""
    _, first = _logits(rows, classes, dtype)
    value, index = (t.cuda() for t in _teacher(rows, classes, 8))
    y = _labels(rows, classes).cuda()
    kw = dict(temperature=2.0, weight=0.5)
    static = first.clone().requires_grad_()

    def step(leaf):
        loss = logit_ops.distill_loss(leaf, value, index, y, **kw)
        (grad,) = torch.autograd.grad(loss, leaf)
        return loss.detach(), grad

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grad = step(static)
    for seed in range(4):
        _, now = _logits(rows, classes, dtype, seed=seed)
        with torch.no_grad():
            static.copy_(now)
        graph.replay()
        want_loss, want = step(now.clone().requires_grad_())
        torch.cuda.synchronize()
        assert torch.equal(loss, want_loss) and torch.equal(grad, want)


@pytest.mark.parametrize("rows,classes,dtype", [(128, 100, F32), (130, 20000, BF16)])
def test_distill_backward_in_a_graph_of_its_own(rows, classes, dtype):
    """The backward pass's graph makes the gradient on each replay, also where
    its last result was changed and no forward pass came between."""
    _, first = _logits(rows, classes, dtype)
    value, index = (t.cuda() for t in _teacher(rows, classes, 8))
    y = _labels(rows, classes).cuda()
    kw = dict(temperature=2.0, weight=0.5)
    static = first.clone().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(logit_ops.distill_loss(static, value, index, y, **kw), static)
    torch.cuda.current_stream().wait_stream(side)
    one = torch.ones((), device="cuda")
    ahead, back = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ahead, stream=side):
        loss = logit_ops.distill_loss(static, value, index, y, **kw)
    with torch.cuda.graph(back, pool=ahead.pool(), stream=side):
        (grad,) = torch.autograd.grad(loss, static, one)
    for seed in range(3):
        _, now = _logits(rows, classes, dtype, seed=seed)
        with torch.no_grad():
            static.copy_(now)
        leaf = now.clone().requires_grad_()
        want = logit_ops.distill_loss(leaf, value, index, y, **kw)
        (want_grad,) = torch.autograd.grad(want, leaf)
        ahead.replay()
        for _ in range(2):
            back.replay()
            torch.cuda.synchronize()
            assert torch.equal(loss.detach(), want.detach())
            assert torch.equal(grad, want_grad)
            grad.zero_()


def test_teacher_answers_feed_the_loss():
    """The two together, as they are used: a teacher's alternatives, the
    student's loss and gradient."""
    rows, classes = 33, 12345
    zt, teacher = _logits(rows, classes, BF16, seed=1)
    zs, student = _logits(rows, classes, BF16, seed=2)
    out = logit_ops.label_logprobs(teacher, top=64)
    cpu = logit_ops.label_logprobs(zt, top=64)
    assert torch.equal(out.top_index.cpu(), cpu.top_index)
    _check_distill(zs, student, out.top_logprob.cpu(), out.top_index.cpu(),
                   _labels(rows, classes), 2.0, 0.8)


@pytest.mark.parametrize("rows,classes,dtype", [
    (4, 50, F32), (4, 20000, F32), (130, 20000, BF16), (4, 3000, F16), (4, 9001, F16)])
@pytest.mark.parametrize("labelled", [False, True])
@pytest.mark.parametrize("reduction", ["none", "sum"])
def test_distill_absent_teacher_of_an_odd_student(rows, classes, dtype, labelled, reduction):
    """A teacher's row of absent entries adds nothing, to the gradient either,
    whatever the student's row holds."""
    z, _ = _logits(rows, classes, dtype)
    z[0, 3], z[1, classes - 1], z[2] = math.nan, math.inf, math.nan
    value, index = _teacher(rows, classes, 3)
    value[:3] = -math.inf
    y = torch.zeros(rows, dtype=torch.long) if labelled else None
    _check_distill(z, z.cuda(), value, index, y, 2.0, 1.0, reduction)
    leaf = z.cuda().requires_grad_()
    loss = logit_ops.distill_loss(leaf, value.cuda(), index.cuda(), None if y is None else y.cuda(),
                                  temperature=2.0, reduction="none")
    (grad,) = torch.autograd.grad(loss, leaf, torch.full((rows,), 0.5, device="cuda"))
    assert (loss[:3] == 0).all() and (grad[:3] == 0).all() and (grad[3] != 0).any()


@pytest.mark.parametrize("rows,classes,dtype", [(130, 100, F32), (3, 20000, F32)])
@pytest.mark.parametrize("weight", [1 - 1e-5, 1 - 1e-7, 1 - 1e-9])
def test_distill_labels_of_little_weight_have_their_share(rows, classes, dtype, weight):
    """The labels' share is 1 - weight as given, not as fp32 holds the weight:
    the teacher is absent, so nothing else is there."""
    z, cuda = _logits(rows, classes, dtype)
    value, index = _teacher(rows, classes, 2)
    value[:] = -math.inf
    y = torch.arange(rows) % classes
    leaf = cuda.detach().requires_grad_()
    kw = dict(temperature=2.0, weight=weight, reduction="sum")
    loss = logit_ops.distill_loss(leaf, value.cuda(), index.cuda(), y.cuda(), **kw)
    (grad,) = torch.autograd.grad(loss, leaf)
    log_p = torch.log_softmax(z.double(), 1)
    hot = torch.zeros_like(log_p).scatter_(1, y[:, None], 1.0)
    share = 1.0 - weight
    # fp32 arithmetic relative to its terms, as in _check_distill
    u = U * (_steps(classes, _spread(z)) + rows / 64 + 64)
    size = share * ((-log_p * hot).sum(1) + math.log(classes + 1)).sum()
    assert abs(float(loss.detach()) + float((log_p * hot).sum() * share)) <= 2 * u * size
    want = share * (log_p.exp() - hot)
    assert ((grad.cpu().double() - want).abs() <= 2 * u * share * (log_p.exp() + hot)).all()
    # a wrong label makes the row NaN at any share
    y[0] = classes
    loss = logit_ops.distill_loss(leaf, value.cuda(), index.cuda(), y.cuda(), **kw)
    assert loss.isnan()


@pytest.mark.parametrize("classes", [50, 20000])
def test_distill_teacher_of_next_to_no_weight_is_looked_at(classes):
    """A weight that fp32 rounds to 0 is not 0: a wrong class makes NaN."""
    z, cuda = _logits(3, classes, F32)
    value, index = _teacher(3, classes, 2)
    index[1, 0] = classes
    _check_distill(z, cuda, value, index, torch.tensor([1, 2, 3]), 2.0, 1e-50, "none")
