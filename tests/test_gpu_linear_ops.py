"""linear_act on the GPU: exactly, on grids where 32-bit sums are exact, and
against 64 bits within the roundings of fp32 sums elsewhere."""

import math

import pytest
import torch

from atomo_amd.ops import linear_ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16

# rows, in, out: single rows and columns, below and around a tile, ragged in
# each index, long sums, many rows
SIZES = [(1, 1, 1), (1, 784, 800), (2, 9216, 130), (5, 33, 7), (17, 100, 10),
         (33, 9, 257), (64, 512, 512), (100, 777, 129), (128, 784, 800),
         (129, 130, 131), (300, 64, 513), (1000, 257, 300), (2, 65, 4096),
         (4100, 40, 20), (520, 1100, 530), (1030, 1000, 1026)]


def _grid(shape, seed, dtype, high=6):
    """Whole numbers: sums of a few thousand products stay below 2^24."""
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-high, high + 1, shape, generator=g).to(dtype)


def _check_exact(m, k, n, dtype, activation="relu", residual=False, bias=True,
                 x=None, w=None):
    x = _grid((m, k), 1, dtype) if x is None else x
    w = _grid((n, k), 2, dtype) if w is None else w
    b = _grid((n,), 3, dtype) if bias else None
    r = _grid((m, n), 4, dtype) if residual else None
    dy = _grid((m, n), 5, dtype)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b, r) if t is not None]
    it = iter(leaves)
    cx, cw = next(it), next(it)
    cb = next(it) if bias else None
    cr = next(it) if residual else None
    y = linear_ops.linear_act(cx, cw, cb, activation, cr)
    grads = torch.autograd.grad(y, leaves, dy.cuda())
    h = x.double() @ w.double().t()
    if bias:
        h = h + b.double()
    slope = torch.ones_like(h)
    if activation == "relu":
        slope = (h > 0).double()
    want = h * slope + (r.double() if residual else 0)
    dp = dy.double() * slope
    assert torch.equal(y.cpu(), want.to(dtype))
    assert torch.equal(grads[0].cpu(), (dp @ w.double()).to(dtype))
    assert torch.equal(grads[1].cpu(), (dp.t() @ x.double()).to(dtype))
    if bias:
        assert torch.equal(grads[2].cpu(), dp.sum(0).to(dtype))
    if residual:
        assert torch.equal(grads[-1].cpu(), dy)
    with torch.no_grad():
        again = linear_ops.linear_act(cx, cw, cb, activation, cr)
    assert torch.equal(again, y)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_exact_sizes(m, k, n, dtype):
    _check_exact(m, k, n, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,k,n", [
    (64, 64, 64), (192, 128, 8), (8, 64, 320), (448, 192, 72), (72, 64, 128),
    (320, 1088, 576), (2048, 64, 2048), (1000, 448, 1992), (384, 2112, 328),
    (8, 4096, 64), (64, 4096, 8)])
def test_exact_sizes_of_whole_steps(m, k, n, dtype):
    """Multiples of eight, and of 64 where sums run over them: operands that
    go straight to LDS, in one step or an odd or even number, in tiles that
    pass the last row, and, each by one element, just not."""
    _check_exact(m, k, n, dtype)
    _check_exact(m, k, n, dtype, "none", True, False)
    x, w = (torch.zeros(rows, k + 16, dtype=dtype) for rows in (m, n))
    for left in (8, 3):
        vx, vw = x[:, left:left + k], w[:, left:left + k]
        vx.copy_(_grid((m, k), 6, dtype))
        vw.copy_(_grid((n, k), 7, dtype))
        cx, cw = x.cuda()[:, left:left + k], w.cuda()[:, left:left + k]
        dy = _grid((m, n + 8), 8, dtype).cuda()[:, :n]
        cx, cw = cx.detach().requires_grad_(), cw.detach().requires_grad_()
        y = linear_ops.linear_act(cx, cw)
        gx, gw = torch.autograd.grad(y, (cx, cw), dy)
        dd = dy.cpu().double()
        assert torch.equal(y.cpu(), (vx.double() @ vw.double().t()).to(dtype))
        assert torch.equal(gx.cpu(), (dd @ vw.double()).to(dtype))
        assert torch.equal(gw.cpu(), (dd.t() @ vx.double()).to(dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("activation,residual,bias", [
    ("none", False, False), ("none", True, True), ("relu", True, False)])
@pytest.mark.parametrize("m,k,n", [(1, 40, 9), (70, 513, 140), (600, 300, 260)])
def test_exact_forms(m, k, n, activation, residual, bias, dtype):
    _check_exact(m, k, n, dtype, activation, residual, bias)


def _check_near(m, k, n, dtype, activation, residual):
    g = torch.Generator().manual_seed(m + k + n)
    x = torch.randn(m, k, generator=g).to(dtype)
    w = (torch.randn(n, k, generator=g) / math.sqrt(k)).to(dtype)
    b = torch.randn(n, generator=g).to(dtype)
    r = torch.randn(m, n, generator=g).to(dtype) if residual else None
    dy = torch.randn(m, n, generator=g).to(dtype)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b, r) if t is not None]
    y = linear_ops.linear_act(*leaves[:3], activation, leaves[3] if residual else None)
    grads = torch.autograd.grad(y, leaves, dy.cuda())
    xd, wd, dyd = x.double(), w.double(), dy.double()
    h = xd @ wd.t() + b.double()
    # an fp32 sum of k products: k half steps of the sum of their sizes
    dh = (k + 2) * U * (xd.abs() @ wd.abs().t() + b.double().abs())
    if activation == "gelu":
        cdf = 0.5 * torch.erfc(-h / math.sqrt(2))
        pdf = torch.exp(-h * h / 2) / math.sqrt(2 * math.pi)
        want, slope = h * cdf, cdf + h * pdf
    elif activation == "silu":
        s = torch.sigmoid(h)
        want, slope = h * s, s * (1 + h * (1 - s))
    else:
        want, slope = h, torch.ones_like(h)
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * half * 2
    # slopes lie within 1.2, their own within 0.9; 32 half steps for the
    # functions themselves, whose parts are up to 1 + |h|
    err = 1.2 * dh + 32 * U * (1 + h.abs())
    if residual:
        want = want + r.double()
        err = err + U * want.abs()
    assert ((y.cpu().double() - want).abs() <= err + half * want.abs() + tiny).all()
    dp = dyd * slope
    # dy times the slope is rounded; the slope is, too, to fp32, or next to
    # 16-bit operands to 2^-15 steps; without an activation neither is
    part = 0.0 if activation == "none" else 2 * half + half * half
    dslope = 0.0 if activation == "none" else 0.9 * dh + 32 * U * (1 + h.abs())
    if activation != "none" and dtype != F32:
        part, dslope = half, dslope + 2.0 ** -16
    edp = dyd.abs() * (part * slope.abs() + dslope * (1 + part)) + tiny

    def near(got, value, error, terms, size):
        got = got.cpu().double()
        error = error + (terms + 2) * U * size
        assert ((got - value).abs() <= error + half * (value.abs() + error) + tiny).all()

    size = dp.abs() + edp
    near(grads[0], dp @ wd, edp @ wd.abs(), n, size @ wd.abs())
    near(grads[1], dp.t() @ xd, edp.t() @ xd.abs(), m, size.t() @ xd.abs())
    near(grads[2], dp.sum(0), edp.sum(0), m, size.sum(0))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("activation", ["none", "gelu", "silu"])
@pytest.mark.parametrize("m,k,n,residual", [(1, 300, 70, True), (9, 65, 33, False),
                                            (260, 200, 150, True), (128, 1030, 300, False)])
def test_near_64_bit(m, k, n, residual, activation, dtype):
    _check_near(m, k, n, dtype, activation, residual)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("m,k,n", [(1, 70, 33), (37, 100, 40), (150, 140, 260)])
def test_layouts(m, k, n, dtype):
    """Padded, shifted, transposed and repeated operands."""
    def padded(t, left, right):
        wide = torch.zeros(t.shape[0], left + t.shape[1] + right, dtype=t.dtype, device="cuda")
        view = wide[:, left:left + t.shape[1]]
        view.copy_(t)
        return view

    x, w, r, dy = _grid((m, k), 1, dtype), _grid((n, k), 2, dtype), \
        _grid((m, n), 3, dtype), _grid((m, n), 4, dtype)
    h = x.double() @ w.double().t() + r.double()
    for cx, cw, cr, cdy in [
        (padded(x, 1, 2), padded(w, 3, 0), padded(r, 1, 1), padded(dy, 5, 2)),
        (x.cuda().t().contiguous().t(), w.cuda().t().contiguous().t(),
         r.cuda().t().contiguous().t(), dy.cuda().t().contiguous().t()),
    ]:
        cx, cw, cr = (t.detach().requires_grad_() for t in (cx, cw, cr))
        y = linear_ops.linear_act(cx, cw, None, "none", cr)
        gx, gw, gr = torch.autograd.grad(y, (cx, cw, cr), cdy)
        assert torch.equal(y.cpu(), h.to(dtype))
        assert torch.equal(gx.cpu(), (dy.double() @ w.double()).to(dtype))
        assert torch.equal(gw.cpu(), (dy.double().t() @ x.double()).to(dtype))
        assert torch.equal(gr.cpu(), dy)
    # rows that share their elements, and end where their memory ends
    def sliding(rows, columns, seed):
        flat = _grid((rows + columns - 1,), seed, dtype)
        return (flat.as_strided((rows, columns), (1, 1)),
                flat.cuda().as_strided((rows, columns), (1, 1)))

    (hx, sx), (hd, sdy) = sliding(m, k, 8), sliding(m, n, 9)
    cx, cw = sx.detach().requires_grad_(), w.cuda().requires_grad_()
    y = linear_ops.linear_act(cx, cw)
    gx, gw = torch.autograd.grad(y, (cx, cw), sdy)
    assert torch.equal(y.cpu(), (hx.double() @ w.double().t()).to(dtype))
    assert torch.equal(gx.cpu(), (hd.double() @ w.double()).to(dtype))
    assert torch.equal(gw.cpu(), (hd.double().t() @ hx.double()).to(dtype))
    # one row for all, and a gradient that is one number
    cx = x[:1].cuda().requires_grad_()
    cw = w.cuda().requires_grad_()
    y = linear_ops.linear_act(cx.expand(m, k), cw)
    y.sum().backward()
    assert torch.equal(cx.grad.cpu(), (w.double().sum(0) * m).to(dtype)[None])
    assert torch.equal(cw.grad.cpu(), (x[:1].double() * m).to(dtype).expand(n, k))


def test_parts_of_the_gradient():
    x, w, b, r = (_grid(s, i, F32).cuda() for i, s in enumerate(
        ((40, 30), (20, 30), (20,), (40, 20))))
    for wanted in range(1, 16):
        args = [t.clone().requires_grad_(bool(wanted >> i & 1))
                for i, t in enumerate((x, w, b, r))]
        linear_ops.linear_act(*args[:3], "gelu", args[3]).sum().backward()
        for i, t in enumerate(args):
            assert (t.grad is not None) == bool(wanted >> i & 1)


def test_empty_batch_and_refusals():
    w = torch.ones(4, 3, device="cuda", requires_grad=True)
    b = torch.ones(4, device="cuda", requires_grad=True)
    x = torch.zeros(0, 3, device="cuda", requires_grad=True)
    y = linear_ops.linear_act(x, w, b, "relu")
    y.sum().backward()
    assert y.shape == (0, 4) and x.grad.shape == (0, 3)
    assert (w.grad == 0).all() and (b.grad == 0).all()
    with pytest.raises(ValueError):
        linear_ops.linear_act(x, w.cpu(), b)
    y = linear_ops.linear_act(torch.ones(2, 3, device="cuda"), w, b)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.sum(), w, create_graph=True)


def test_infinite_inputs():
    w = torch.tensor([[1.0], [-1.0]], device="cuda")
    x = torch.tensor([[math.inf], [math.nan]], device="cuda")
    for dtype in (F32, BF16, F16):
        for activation in ("relu", "gelu", "silu"):
            y = linear_ops.linear_act(x.to(dtype), w.to(dtype), None, activation)
            assert y[0, 0] == math.inf and y[0, 1] == 0
            assert y[1].isnan().all()


@pytest.mark.parametrize("m,k,n", [(3, 20, 5), (130, 200, 140), (40, 3000, 70)])
def test_single_infinities_and_extremes(m, k, n):
    """An infinity times finite numbers, one by one: what fp32 gives, and
    nothing next to it; operands at both ends of fp32."""
    x, w = _grid((m, k), 1, F32) + 20, _grid((n, k), 2, F32) + 10.5  # no zeros
    x[m // 2, k // 3], x[m - 1, k - 1] = math.inf, 3.4e38
    x[0], w[0, 0] = x[0] * 2.0 ** -120, math.nan
    cx, cw = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = linear_ops.linear_act(cx, cw)
    want = (x.double() @ w.double().t()).float()
    got = y.detach().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isinf(), want.isinf())
    ok = torch.isfinite(want)
    # products of 2^-120 parts: their third parts lie below fp32's normal
    # numbers, 2^-126, and may be taken for 0; else k half steps of the sums
    tiny = k * 2.0 ** -126 * 32
    size = x.abs().double() @ w.abs().double().t()
    assert ((got.double() - want.double()).abs() <= (k + 2) * U * size + tiny)[ok].all()
    gx, gw = torch.autograd.grad(y, (cx, cw), torch.ones_like(y))
    want = (torch.ones(m, n).double() @ w.double()).float()
    assert torch.equal(gx.cpu().isnan(), want.isnan())
    want = (torch.ones(n, m).double() @ x.double()).float()
    assert torch.equal(gw.cpu().isinf(), want.isinf())
    assert not gw.isnan().any()


@pytest.mark.parametrize("m,k,n,dtype", [(1, 500, 300, BF16), (128, 784, 800, F32), (300, 300, 600, F16)])
def test_in_a_graph(m, k, n, dtype):
    """Forward and backward captured together, replayed between eager passes
    on another stream than the first."""
    w, b = _grid((n, k), 2, dtype).cuda().requires_grad_(), _grid((n,), 3, dtype).cuda().requires_grad_()
    dy = _grid((m, n), 5, dtype).cuda()
    static = _grid((m, k), 1, dtype).cuda().requires_grad_()

    def step(x):
        y = linear_ops.linear_act(x, w, b, "relu")
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for seed in range(4):
        now = _grid((m, k), 10 + seed, dtype).cuda().requires_grad_()
        with torch.no_grad():
            static.copy_(now)
        graph.replay()
        want = step(now)
        torch.cuda.synchronize()
        for a, c in zip(out, want):
            assert torch.equal(a, c)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("k", [2, 64, 100])
@pytest.mark.parametrize("rows", [1, 1793])
def test_gelu_of_16_bits_is_rounded_once(rows, k, dtype):
    """h = -8..-1 in steps of 2^-8, as the sum of two numbers that the type
    holds: each result is the rounding of a number 2^-16 next to gelu(h)."""
    steps = torch.arange(-2048, -255) if rows > 1 else torch.tensor([-1027])
    h = steps.double() / 256
    x = torch.zeros(rows, k, dtype=dtype)
    x[:, 0] = torch.div(steps, 16, rounding_mode="trunc") / 16
    x[:, 1] = torch.fmod(steps, 16) / 256
    w = torch.zeros(24, k, dtype=dtype)
    w[:, :2] = 1
    y = linear_ops.linear_act(x.cuda(), w.cuda(), None, "gelu").cpu()
    want = h * 0.5 * torch.erfc(-h / math.sqrt(2))
    # exponents of at most 47, rounded twice: 47 * 2^-23; a dozen roundings
    low = (want * (1 + 2.0 ** -16)).to(dtype)[:, None]
    high = (want * (1 - 2.0 ** -16)).to(dtype)[:, None]
    assert ((low <= y) & (y <= high)).all()


def _tail(m, k, n, dtype, centre):
    """x, w, b >= 0 or whole steps of 2^-5: h = centre + 0..1 or so, exactly."""
    g = torch.Generator().manual_seed(m + k + n)
    x = (torch.rand(m, k, generator=g) < min(1.0, 4.0 / k)).to(dtype)
    w = (torch.randint(1, 5, (n, k), generator=g) / 32.0).to(dtype)
    return x, w, torch.full((n,), centre).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("activation,centre", [
    ("gelu", -4.0), ("gelu", -5.0), ("gelu", -6.0), ("silu", -10.0),
    ("silu", -13.0), ("silu", -15.0)])
@pytest.mark.parametrize("m,k,n", [(1, 100, 40), (7, 5, 9), (130, 64, 72), (64, 2048, 64), (33, 70, 41)])
def test_small_slopes_keep_their_digits(m, k, n, activation, centre, dtype):
    """Units that are saturated throughout: their gradients have the relative
    error of the type's own roundings."""
    x, w, b = _tail(m, k, n, dtype, centre)
    g = torch.Generator().manual_seed(0)
    # dp within fp16's normal numbers: slopes are above 4e-8 here
    dy = (torch.randint(1, 4, (m, n), generator=g) * 8192.0).to(dtype)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = linear_ops.linear_act(*leaves, activation)
    gx, gw, gb = torch.autograd.grad(y, leaves, dy.cuda())
    h = x.double() @ w.double().t() + b.double()
    if activation == "gelu":
        slope = 0.5 * torch.erfc(-h / math.sqrt(2)) + h * torch.exp(-h * h / 2) / math.sqrt(2 * math.pi)
    else:
        s = torch.sigmoid(h)
        slope = s * (1 + h * (1 - s))
    dp = dy.double() * slope
    assert (slope < 0).all() and dp.abs().min() > 2.0 ** -14
    half = torch.finfo(dtype).eps / 2
    # nothing cancels: all terms have one sign.  The functions: exponents of at
    # most 27 are rounded twice, 27 * 2^-23; a dozen roundings of 2^-24, and
    # cdf against h * density, which are one sign apart, at most 1.1 times
    own = 2.0 ** -17
    for got, want, rounded, terms in ((gx, dp @ w.double(), half, n), (gw, dp.t() @ x.double(), half, m),
                                      (gb, dp.sum(0), 0.0, m)):
        off = rounded + own + (terms + 4) * U
        tiny = torch.finfo(dtype).smallest_normal * half
        assert ((got.cpu().double() - want).abs() <= (off + half * (1 + off)) * want.abs() + tiny).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("activation", ["none", "relu", "gelu", "silu"])
def test_slopes_at_the_ends_are_the_oracles(activation, dtype):
    x = torch.tensor([[math.inf], [-math.inf], [3e4], [-3e4], [math.nan]], dtype=dtype)
    w = torch.ones(1, 1, dtype=dtype)
    for residual in (None, torch.zeros(5, 1, dtype=dtype)):
        cpu, gpu = x.clone().requires_grad_(), x.cuda().requires_grad_()
        y = linear_ops.linear_act(cpu, w, None, activation, residual)
        z = linear_ops.linear_act(gpu, w.cuda(), None, activation,
                                  None if residual is None else residual.cuda())
        torch.testing.assert_close(z.cpu(), y, rtol=0, atol=0, equal_nan=True)
        (a,), (b,) = torch.autograd.grad(y.sum(), cpu), torch.autograd.grad(z.sum(), gpu)
        torch.testing.assert_close(b.cpu(), a, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("m,k,n", [(1, 40, 9), (3, 5, 7), (70, 100, 40), (130, 64, 72), (64, 2048, 64)])
def test_relu_of_what_rounds_to_zero_has_its_slope(m, k, n, residual, dtype):
    """Sums of 2^-26, 0 and -2^-26: below fp16's smallest number, but of a
    sign."""
    x = torch.zeros(m, k, dtype=dtype)
    x[:, 0] = 2.0 ** -13 * (torch.arange(m) % 3 - 1 if m > 1 else 1)
    w = torch.zeros(n, k, dtype=dtype)
    w[:, 0] = 2.0 ** -13
    dy = _grid((m, n), 5, dtype)
    leaves = [t.cuda().requires_grad_() for t in (x, w)]
    r = torch.zeros(m, n, dtype=dtype, device="cuda") if residual else None
    y = linear_ops.linear_act(*leaves, None, "relu", r)
    gx, gw = torch.autograd.grad(y, leaves, dy.cuda())
    h = x.double() @ w.double().t()
    dp = dy.double() * (h > 0)
    assert torch.equal(y.cpu(), h.relu().to(dtype))
    assert torch.equal(gx.cpu(), (dp @ w.double()).to(dtype))
    assert torch.equal(gw.cpu(), (dp.t() @ x.double()).to(dtype))


@pytest.mark.parametrize("size", [-101, -112, -120])
@pytest.mark.parametrize("m,k,n", [(3, 50, 20), (130, 200, 140), (40, 3000, 70)])
def test_tiny_fp32_operands_are_held_to_2_126(m, k, n, size):
    """Times numbers of 2^100, so that what is lost shows in normal results."""
    g = torch.Generator().manual_seed(k)
    x = torch.randn(m, k, generator=g) * 2.0 ** size
    w = torch.randn(n, k, generator=g) * 2.0 ** 100
    y = linear_ops.linear_act(x.cuda(), w.cuda()).cpu().double()
    want = x.double() @ w.double().t()
    mass = x.abs().double() @ w.abs().double().t()
    # an operand's parts, each below 2^-126 (the second and third together
    # 1 + 2^-8 of it), dropped products and fp32's k sums
    lost = 2.0 ** -126 * (1 + 2.0 ** -8) * w.abs().double().sum(1)
    assert ((y - want).abs() <= lost + (k + 4) * U * mass).all()
