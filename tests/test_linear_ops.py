"""linear_act on the CPU: the oracle against plain formulas and differences,
refusals, the layer and the models that carry it."""

import math

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from atomo_amd.ops import linear_ops
from atomo_amd.ops.linear_ops import FusedLinear, linear_act

PLAIN = {"none": lambda h: h, "relu": F.relu, "gelu": F.gelu, "silu": F.silu}


def _inputs(m, k, n, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(m, k, generator=g).to(dtype),
            (torch.randn(n, k, generator=g) / math.sqrt(k)).to(dtype),
            torch.randn(n, generator=g).to(dtype), torch.randn(m, n, generator=g).to(dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("activation", sorted(PLAIN))
@pytest.mark.parametrize("with_bias,with_residual", [(True, True), (False, False)])
def test_matches_plain_64_bit(activation, with_bias, with_residual, dtype):
    x, w, b, r = _inputs(5, 7, 3, dtype)
    leaves = [x, w] + ([b] if with_bias else []) + ([r] if with_residual else [])
    for t in leaves:
        t.requires_grad_()
    y = linear_act(x, w, b if with_bias else None, activation, r if with_residual else None)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    h = F.linear(wide[0], wide[1], wide[2] if with_bias else None)
    want = PLAIN[activation](h)
    if with_residual:
        want = want + wide[-1]
    dy = torch.randn_like(y)
    got = torch.autograd.grad(y, leaves, dy)
    ref = torch.autograd.grad(want, wide, dy.double())
    # one rounding of 64-bit results; fp16 has no normal numbers below 6e-5
    half = torch.finfo(dtype).eps / 2
    floor = torch.finfo(dtype).smallest_normal * half + 1e-14
    for a, b in zip((y, *got), (want, *ref)):
        assert a.dtype == dtype
        torch.testing.assert_close(a.double(), b, rtol=half, atol=floor)


def test_gradient_matches_differences():
    x, w, b, r = _inputs(2, 3, 2)
    x.requires_grad_()
    linear_act(x, w, b, "gelu", r).sum().backward()
    # central differences of 2^-6: h^2/6 of a third derivative below 2 (the
    # weights are below 1.5, cubed), and the fp32 output's rounding over 2h
    h = 2.0 ** -6
    for i in range(2):
        for j in range(3):
            step = torch.zeros(2, 3)
            step[i, j] = h
            a = linear_act(x.detach() + step, w, b, "gelu", r).double().sum()
            c = linear_act(x.detach() - step, w, b, "gelu", r).double().sum()
            assert abs(float(a - c) / (2 * h) - float(x.grad[i, j])) < \
                2 * 2 * 1.5 ** 3 * h * h / 6 + 8 * 2.0 ** -22 / h


def test_shapes():
    x, w, b, _ = _inputs(24, 5, 3)
    want = linear_act(x, w, b)
    assert torch.equal(linear_act(x.view(2, 3, 4, 5), w, b).view(24, 3), want)
    assert torch.equal(linear_act(x[0], w, b), want[0])
    assert linear_act(x[:0], w, b).shape == (0, 3)


def test_infinite_inputs():
    w = torch.tensor([[1.0], [-1.0]])
    x = torch.tensor([[math.inf], [math.nan]])
    for activation in ("relu", "gelu", "silu"):
        y = linear_act(x, w, None, activation)
        assert y[0, 0] == math.inf and y[0, 1] == 0
        assert y[1].isnan().all()


@pytest.mark.parametrize("change,error", [
    (dict(activation="tanh"), ValueError),
    (dict(x=torch.zeros(2, 3).double()), TypeError),
    (dict(x=torch.zeros(2, 4)), ValueError),
    (dict(x=torch.tensor(1.0)), ValueError),
    (dict(weight=torch.zeros(4, 3).half()), TypeError),
    (dict(weight=torch.zeros(3)), ValueError),
    (dict(weight=torch.zeros(0, 3)), ValueError),
    (dict(x=torch.zeros(2, 0), weight=torch.zeros(4, 0)), ValueError),
    (dict(bias=torch.zeros(3)), ValueError),
    (dict(bias=torch.zeros(4, 1)), ValueError),
    (dict(bias=torch.zeros(4).half()), TypeError),
    (dict(residual=torch.zeros(4)), ValueError),
    (dict(residual=torch.zeros(2, 4).half()), TypeError),
])
def test_refusals(change, error):
    call = dict(x=torch.zeros(2, 3), weight=torch.zeros(4, 3), bias=torch.zeros(4))
    call.update(change)
    with pytest.raises(error):
        linear_act(**call)


def test_layer_takes_over_a_linear():
    linear = nn.Linear(6, 4)
    fused = FusedLinear.of(linear, "relu")
    assert fused.weight is linear.weight and fused.bias is linear.bias
    assert list(fused.state_dict()) == list(linear.state_dict())
    x = torch.randn(3, 6)
    # both sides round: the plain one each of at most 7 sums, of terms below
    torch.testing.assert_close(fused(x), linear(x).relu(), rtol=0,
                               atol=8 * 2.0 ** -24 * 6 * float(x.abs().max()))
    assert "activation=relu" in repr(fused)
    with pytest.raises(ValueError):
        FusedLinear(3, 4, activation="tanh")
    assert linear_ops.FusedLinear(3, 4, bias=False)(torch.zeros(2, 3)).shape == (2, 4)


def test_layer_under_autocast():
    fused = FusedLinear(6, 4, activation="relu")
    x = torch.randn(3, 6)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        y = fused(x)
        assert y.dtype == torch.bfloat16
        y.float().sum().backward()
    assert fused.weight.grad.dtype == torch.float32


@pytest.mark.parametrize("activation,slopes", [
    ("none", [1.0, 1.0, 1.0, 1.0, 1.0]), ("relu", [1.0, 0.0, 1.0, 0.0, 1.0]),
    ("gelu", [1.0, 0.0, 1.0, 0.0, math.nan]), ("silu", [1.0, 0.0, 1.0, 0.0, math.nan])])
def test_slopes_at_the_ends(activation, slopes):
    """Infinities have the slope that the activation tends to; NaN passes."""
    x = torch.tensor([[math.inf], [-math.inf], [3e4], [-3e4], [math.nan]], requires_grad=True)
    y = linear_act(x, torch.ones(1, 1), None, activation)
    (grad,) = torch.autograd.grad(y.sum(), x)
    torch.testing.assert_close(grad[:, 0], torch.tensor(slopes), rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("activation", sorted(PLAIN))
def test_layer_takes_what_a_linear_takes(activation):
    """fp64, which gradcheck asks for."""
    torch.manual_seed(0)
    linear = nn.Linear(6, 4).double()
    fused = FusedLinear.of(linear, activation)
    x = torch.randn(3, 6, dtype=torch.float64, requires_grad=True)
    r = torch.randn(3, 4, dtype=torch.float64)
    assert torch.equal(fused(x), PLAIN[activation](linear(x)))
    assert torch.equal(fused(x, r), PLAIN[activation](linear(x)) + r)
    assert torch.autograd.gradcheck(fused, (x,))
    with pytest.raises(TypeError):
        fused(x.float())


def test_double_precision_stays_under_autocast():
    linear = nn.Linear(6, 4).double()
    x = torch.randn(3, 6, dtype=torch.float64)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        y = FusedLinear.of(linear)(x)
        assert y.dtype == torch.float64 and torch.equal(y, linear(x))
