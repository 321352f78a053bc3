"""label_logprobs and distill_loss on the CPU: the oracle against plain
64-bit formulas and differences, refusals, the empty and the odd."""

import math

import pytest
import torch
import torch.nn.functional as F

from atomo_amd.ops import logit_ops


def _logits(rows, classes, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, classes, generator=g) * 3).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,classes,top", [(1, 1, 1), (3, 10, 5), (7, 129, 128)])
def test_logprobs_match_plain_64_bit(rows, classes, top, dtype):
    z = _logits(rows, classes, dtype=dtype)
    y = torch.arange(rows) % classes
    out = logit_ops.label_logprobs(z, y, top=top)
    logp = F.log_softmax(z.double(), 1)
    # the oracle rounds 64-bit results once: half a step of fp32
    tol = dict(rtol=2.0 ** -24, atol=1e-14)
    torch.testing.assert_close(out.logprob.double(), -F.nll_loss(logp, y, reduction="none"), **tol)
    torch.testing.assert_close(out.entropy.double(), -(logp.exp() * logp).sum(1), **tol)
    order = sorted(range(classes), key=lambda c: (-float(z[0, c]), c))[:top]
    assert out.top_index[0].tolist() == order
    torch.testing.assert_close(out.top_logprob.double(), logp.gather(1, out.top_index), **tol)
    assert out.top_index.dtype == torch.int64 and out.logprob.dtype == torch.float32


def test_logprobs_ties_go_to_the_lowest_class():
    z = torch.tensor([[1.0, 2.0, 2.0, -0.0, 0.0, 2.0]])
    out = logit_ops.label_logprobs(z, top=6)
    assert out.top_index.tolist() == [[1, 2, 5, 0, 3, 4]]
    assert out.logprob is None


def test_logprobs_odd_rows():
    inf, nan = math.inf, math.nan
    z = torch.tensor([
        [-inf, -inf, -inf],
        [-inf, 2.0, -inf],
        [nan, 1.0, 2.0],
        [inf, 1.0, 2.0],
        [torch.finfo(torch.float32).min] * 3,
    ])
    out = logit_ops.label_logprobs(z, torch.tensor([0, 1, 1, 1, 2]), top=3)
    assert out.logprob[:2].tolist() == [-inf, 0.0]
    assert out.logprob[2:4].isnan().all()
    assert out.logprob[4].item() == pytest.approx(-math.log(3), rel=2.0 ** -24)
    assert out.entropy[:2].tolist() == [0.0, 0.0]
    assert out.entropy[2:4].isnan().all()
    assert out.top_index[:4].tolist() == [[0, 1, 2], [1, 0, 2], [0, 2, 1], [0, 2, 1]]
    assert out.top_logprob[0].tolist() == [-inf] * 3
    assert out.top_logprob[1].tolist() == [0.0, -inf, -inf]


def test_logprobs_labels_outside():
    z = _logits(4, 5)
    out = logit_ops.label_logprobs(z, torch.tensor([-100, 5, -1, 4]))
    assert out.logprob[0] == 0.0
    assert out.logprob[1:3].isnan().all()
    assert out.top_index is None and out.top_logprob is None
    out = logit_ops.label_logprobs(z, torch.tensor([7, 0, 0, 0]), ignore_index=7)
    assert out.logprob[0] == 0.0


def test_logprobs_shapes_and_strides():
    z = _logits(24, 16)
    base = logit_ops.label_logprobs(z, torch.arange(24) % 11, top=4)
    lead = logit_ops.label_logprobs(
        z.view(2, 3, 4, 16), (torch.arange(24) % 11).view(2, 3, 4).int(), top=4)
    assert lead.top_index.shape == (2, 3, 4, 4)
    assert torch.equal(lead.top_index.view(24, 4), base.top_index)
    assert torch.equal(lead.logprob.view(-1), base.logprob)
    wide = torch.zeros(24, 32)
    wide[:, 3:19] = z
    assert torch.equal(logit_ops.label_logprobs(wide[:, 3:19]).entropy, base.entropy)
    assert torch.equal(logit_ops.label_logprobs(z.t().contiguous().t()).entropy, base.entropy)
    one = logit_ops.label_logprobs(z[0], torch.tensor(2), top=1)
    assert one.logprob.shape == () and one.top_index.shape == (1,)
    none = logit_ops.label_logprobs(z[:0], torch.empty(0, dtype=torch.long), top=2)
    assert none.logprob.shape == (0,) and none.top_index.shape == (0, 2)


@pytest.mark.parametrize("call,error", [
    (lambda z, y: logit_ops.label_logprobs(z.double(), y), TypeError),
    (lambda z, y: logit_ops.label_logprobs(z, y.float()), TypeError),
    (lambda z, y: logit_ops.label_logprobs(z, y[:2]), ValueError),
    (lambda z, y: logit_ops.label_logprobs(z, y, top=-1), ValueError),
    (lambda z, y: logit_ops.label_logprobs(z, y, top=6), ValueError),
    (lambda z, y: logit_ops.label_logprobs(_logits(3, 200), None, top=129), ValueError),
    (lambda z, y: logit_ops.label_logprobs(z[:, :0], y), ValueError),
    (lambda z, y: logit_ops.label_logprobs(torch.tensor(1.0), y), ValueError),
])
def test_logprobs_refusals(call, error):
    with pytest.raises(error):
        call(_logits(3, 5), torch.tensor([0, 1, 2]))


def _plain_loss(z, value, index, y, tau, weight, ignore=-100):
    """Differentiable, 64 bits, dense."""
    q = torch.zeros_like(z).scatter_add_(
        1, index, torch.softmax(value.double() / tau, 1))
    log_p = F.log_softmax(z / tau, 1)
    row = weight * tau ** 2 * (torch.special.xlogy(q, q) - q * log_p).sum(1)
    if y is None:
        return row
    ce = F.cross_entropy(z, y, reduction="none", ignore_index=ignore)
    return (row + (1 - weight) * ce) * (y != ignore)


def _teacher(rows, classes, k, seed=1):
    g = torch.Generator().manual_seed(seed)
    index = torch.stack([torch.randperm(classes, generator=g)[:k] for _ in range(rows)])
    return torch.randn(rows, k, generator=g) * 2, index


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("tau,weight,labelled", [
    (1.0, 1.0, False), (2.0, 0.5, True), (4.0, 0.9, True), (0.5, 0.0, True), (3.0, 1.0, True)])
def test_distill_matches_autograd(tau, weight, labelled, reduction):
    z = _logits(6, 11)
    value, index = _teacher(6, 11, 4)
    y = torch.tensor([0, 10, -100, 3, 3, -100]) if labelled else None
    leaf = z.clone().requires_grad_()
    loss = logit_ops.distill_loss(leaf, value, index, y, temperature=tau,
                                  weight=weight, reduction=reduction)
    wide = z.double().requires_grad_()
    row = _plain_loss(wide, value, index, y, tau, weight)
    count = 6 if y is None else 4
    want = {"none": row, "sum": row.sum(), "mean": row.sum() / count}[reduction]
    up = torch.rand_like(want) + 0.5
    (grad,) = torch.autograd.grad(loss, leaf, up.float())
    (ref,) = torch.autograd.grad(want, wide, up.float().double())
    # one rounding each of 64-bit results
    torch.testing.assert_close(loss.double(), want.detach(), rtol=2.0 ** -24, atol=1e-13)
    torch.testing.assert_close(grad.double(), ref, rtol=2.0 ** -24, atol=1e-13)


def test_distill_gradient_matches_differences():
    z = _logits(2, 5)
    value, index = _teacher(2, 5, 3)
    y = torch.tensor([4, 1])
    leaf = z.clone().requires_grad_()
    loss = logit_ops.distill_loss(leaf, value, index, y, temperature=2.0, weight=0.7)
    loss.backward()
    # central differences of step h = 2^-5 on an fp32 loss of about 2: the
    # truncation is h^2/6 times a third derivative (below 2), the rounding
    # 2 * 2^-24 / h
    h = 2.0 ** -5
    for r in range(2):
        for c in range(5):
            a, b = z.clone(), z.clone()
            a[r, c] += h
            b[r, c] -= h
            two = [logit_ops.distill_loss(t, value, index, y, temperature=2.0, weight=0.7)
                   for t in (a, b)]
            step = float(a[r, c] - b[r, c])
            got = float(two[0] - two[1]) / step
            assert abs(got - float(leaf.grad[r, c])) < 2 * h * h / 6 + 4 * 2.0 ** -24 / h


def test_distill_repeated_classes_add_up():
    z = _logits(2, 6)
    value, index = torch.tensor([[1.0, 1.0, 0.5]] * 2), torch.tensor([[2, 2, 4]] * 2)
    merged = torch.tensor([[1.0 + math.log(2.0), 0.5]] * 2)
    a = logit_ops.distill_loss(z, value, index)
    b = logit_ops.distill_loss(z, merged, index[:, 1:])
    # log 2 is rounded to fp32 in the merged values: a relative 2^-24 of 1.7
    assert float(a) == pytest.approx(float(b), abs=2.0 ** -22)


def test_distill_absent_and_wrong_entries():
    inf = math.inf
    z = _logits(5, 6).requires_grad_()
    value = torch.tensor([[1.0, -inf], [-inf, -inf], [1.0, 0.0], [1.0, 0.0], [0.0, math.nan]])
    index = torch.tensor([[2, 99], [-7, 99], [6, 1], [-1, 0], [0, 1]])
    loss = logit_ops.distill_loss(z, value, index, reduction="none")
    loss[:2].sum().backward()
    one = logit_ops.distill_loss(z.detach()[:1], value[:1, :1], index[:1, :1])
    assert loss[0].item() == pytest.approx(one.item(), rel=2.0 ** -23)
    assert loss[1] == 0.0 and (z.grad[1] == 0).all()
    assert loss[2:].isnan().all()
    bad = logit_ops.distill_loss(z, value[:, :1].nan_to_num(0, 0, 0), index[:, :1] * 0,
                                 torch.tensor([0, 6, -1, -100, 5]), weight=0.5,
                                 reduction="none")
    assert bad.isnan().tolist() == [False, True, True, False, False]


def test_distill_infinite_teacher():
    """A teacher's +inf leaves no distribution: loss and gradient of the row
    are NaN throughout."""
    z = _logits(2, 6).requires_grad_()
    value = torch.tensor([[1.0, math.inf], [1.0, 0.0]])
    loss = logit_ops.distill_loss(z, value, torch.tensor([[0, 1], [0, 1]]), reduction="none")
    loss.sum().backward()
    assert loss.isnan().tolist() == [True, False]
    assert z.grad[0].isnan().all() and torch.isfinite(z.grad[1]).all()


def test_distill_masked_student():
    inf = math.inf
    z = torch.tensor([[-inf] * 3, [0.0, -inf, 1.0], [0.0, -inf, 1.0]], requires_grad=True)
    value, index = torch.zeros(3, 1), torch.tensor([[0], [0], [1]])
    loss = logit_ops.distill_loss(z, value, index, reduction="none")
    loss[:2].sum().backward(retain_graph=True)
    assert loss[0] == 0 and torch.isfinite(loss[1]) and loss[2] == inf
    assert (z.grad[0] == 0).all() and torch.isfinite(z.grad).all() and z.grad[1, 1] == 0


def test_distill_nothing_counted():
    z = _logits(2, 4).requires_grad_()
    value, index = _teacher(2, 4, 2)
    loss = logit_ops.distill_loss(z, value, index, torch.tensor([-100, -100]), weight=0.5)
    loss.backward()
    assert loss == 0 and (z.grad == 0).all()
    none = logit_ops.distill_loss(z[:0], value[:0], index[:0])
    assert none == 0


def test_distill_second_derivative_is_refused():
    z = _logits(2, 4).requires_grad_()
    value, index = _teacher(2, 4, 2)
    loss = logit_ops.distill_loss(z, value, index)
    (grad,) = torch.autograd.grad(loss, z, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


@pytest.mark.parametrize("change,error", [
    (dict(temperature=1e-3), ValueError), (dict(temperature=1e3), ValueError),
    (dict(temperature=0.0), ValueError), (dict(temperature=math.inf), ValueError),
    (dict(temperature=math.nan), ValueError), (dict(weight=1.5), ValueError),
    (dict(weight=math.nan), ValueError), (dict(weight=0.5, labels=None), ValueError),
    (dict(reduction="max"), ValueError), (dict(labels=torch.zeros(3).long()), ValueError),
    (dict(labels=torch.zeros(2)), TypeError),
    (dict(teacher_index=torch.zeros(2, 3).long()), ValueError),
    (dict(teacher_index=torch.zeros(2, 2)), TypeError),
    (dict(teacher_value=torch.zeros(2, 2).double()), TypeError),
    (dict(teacher_value=torch.zeros(3, 2)), ValueError),
    (dict(teacher_value=torch.zeros(2, 0), teacher_index=torch.zeros(2, 0).long()), ValueError),
    (dict(teacher_value=torch.zeros(2, 129), teacher_index=torch.zeros(2, 129).long()), ValueError),
    (dict(logits=torch.zeros(2, 4).long()), TypeError),
])
def test_distill_refusals(change, error):
    call = dict(logits=_logits(2, 4), teacher_value=torch.zeros(2, 2),
                teacher_index=torch.zeros(2, 2).long(), labels=torch.zeros(2).long())
    call.update(change)
    with pytest.raises(error):
        logit_ops.distill_loss(**call)


def test_teacher_answers_feed_the_loss():
    """A student equal to its teacher, who gave all classes, has loss 0."""
    z = _logits(5, 9)
    out = logit_ops.label_logprobs(z, top=9)
    loss = logit_ops.distill_loss(z, out.top_logprob, out.top_index, temperature=2.0)
    # log probabilities rounded to fp32 (below 16): 2^-21 each, second order
    assert abs(float(loss)) < 4 * 2.0 ** -40 * 9 + 1e-10
