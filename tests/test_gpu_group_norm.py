"""Group norm with an activation and a gate against its formula in 64 bits, under autograd."""
import math

import pytest
import torch

from visionhope_b200.utils.group_norm import GroupNorm, group_norm, group_norm_rows

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def normal(seed, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device="cuda") * scale + shift).to(dtype)


def formula(x, groups, weight, bias, eps, activation, gate):
    """x [samples, channels, ...] in fp64."""
    n, c = x.shape[:2]
    per = (1, c) + (1,) * (x.dim() - 2)
    g = x.reshape(n, groups, -1)
    var, mean = torch.var_mean(g, 2, unbiased=False, keepdim=True)
    y = ((g - mean) / (var + eps).sqrt()).reshape(x.shape)
    if weight is not None:
        y = y * weight.view(per)
    if bias is not None:
        y = y + bias.view(per)
    if activation == "silu":
        y = y * torch.sigmoid(y)
    elif activation == "gelu":
        y = 0.5 * y * torch.erfc(-y / math.sqrt(2.0))
    return y if gate is None else y * gate * torch.sigmoid(gate)


def close(got, want, size, terms=1):
    """Half a step of the result's type, and 2^-20 of ``size`` (the largest of the terms that are summed to a
    value: a dozen roundings of 2^-24, and approximations of 2^-22) for each of sqrt(``terms``) of them."""
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() + 2 ** -20 * size * math.sqrt(terms) + (2 ** -25 if got.dtype == torch.float16 else 0)
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), f"worst {float((off / tol).max()):.3g} of the tolerance"


def check(x, groups, weight, bias, activation, gate, rows, eps=1e-5, spread=1.0):
    """Forward and backward; ``spread``: how many times its deviation a value may lie from zero, which a mean's
    rounding of 2^-24 of the values is multiplied by."""
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, gate, weight, bias)]
    norm = group_norm_rows if rows else group_norm
    y = norm(leaves[0], groups, leaves[2], leaves[3], eps, activation=activation, gate=leaves[1])
    assert y.shape == x.shape and y.dtype == x.dtype
    wide = [None if t is None else t.detach().double().requires_grad_() for t in (x, gate, weight, bias)]
    lay = (lambda t: t if t is None else t.reshape(-1, t.shape[-1])) if rows else (lambda t: t)
    want = formula(lay(wide[0]), groups, wide[2], wide[3], eps, activation, lay(wide[1])).view(x.shape)
    dy = torch.empty_like(x).copy_(normal(99, *x.shape))
    live = [t for t in leaves if t is not None]
    got = torch.autograd.grad(y, live, dy)
    exact = torch.autograd.grad(want, [t for t in wide if t is not None], dy.double())
    close(y, want.detach(), spread * (want.detach().abs().amax() + 1))
    with torch.no_grad():
        assert torch.equal(norm(x, groups, weight, bias, eps, activation=activation, gate=gate), y)
    for t, g, w in zip(live, got, exact):
        assert g.shape == t.shape and g.dtype == t.dtype
        terms = x.numel() // x.shape[-1 if rows else 1] if t is leaves[2] or t is leaves[3] else 1
        size = w.abs().amax() + 1e-3 if terms == 1 else dy.double().abs().amax() * 8
        close(g, w, 8 * spread * size, terms)


IMAGES = [(1, 32, 7, 7, 8), (2, 64, 14, 14, 32), (3, 96, 5, 9, 32), (1, 13 * 7, 6, 5, 7), (2, 48, 56, 56, 3), (1, 128, 128, 130, 32), (2, 768, 7, 7, 32),
          (4, 33, 1, 8, 1), (1, 6, 300, 301, 6), (5, 64, 1, 1, 2), (1, 2048, 3, 3, 1), (2, 40, 200, 33, 5)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", IMAGES)
@pytest.mark.parametrize("activation,gated", [(None, False), ("silu", True), ("gelu", False), ("silu", False)])
def test_images(dtype, shape, activation, gated):
    b, c, h, w, groups = shape
    x = normal(1, b, c, h, w, dtype=dtype, scale=2.0, shift=0.5).contiguous(memory_format=torch.channels_last)
    gate = normal(2, b, c, h, w, dtype=dtype).contiguous(memory_format=torch.channels_last) if gated else None
    check(x, groups, normal(3, c, scale=0.2, shift=1.0), normal(4, c, scale=0.2), activation, gate, False)


ROWS = [(1, 64, 1), (7, 256, 4), (300, 2048, 16), (5, 96, 1), (33, 350, 7), (1000, 300, 5), (9, 2048, 2), (6, 2048, 1), (3, 4100, 1), (4, 32, 8),
        (2, 5, 5 // 5), (50, 1024, 1), (3, 1200, 8)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", ROWS)
@pytest.mark.parametrize("activation,gated", [(None, True), ("silu", False), ("gelu", True)])
def test_rows(dtype, shape, activation, gated):
    """Rows by themselves, taken out of wider ones."""
    n, c, groups = shape
    wide = normal(1, n, 3 * c, dtype=dtype, scale=2.0, shift=0.5)
    check(wide[:, c:2 * c], groups, normal(3, c, scale=0.2, shift=1.0), normal(4, c, scale=0.2), activation, wide[:, 2 * c:] if gated else None, True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
def test_without_parameters(dtype, weight, bias):
    x = normal(1, 2, 64, 12, 11, dtype=dtype).contiguous(memory_format=torch.channels_last)
    w, b = normal(3, 64) if weight else None, normal(4, 64) if bias else None
    check(x, 8, w, b, "silu", None, False)
    check(normal(5, 20, 64, dtype=dtype), 8, w, b, "silu", None, True)


@pytest.mark.parametrize("shape", [(2, 64, 14, 14), (1, 128, 128, 130), (3, 64, 1, 1)])
def test_large_mean(shape):
    """A mean a thousand times the deviation: the variance is not a difference of squares."""
    b, c, h, w = shape
    x = normal(1, b, c, h, w, scale=1.0, shift=1000.0).contiguous(memory_format=torch.channels_last)
    check(x, 4, normal(3, c), normal(4, c), None, None, False, spread=1000.0)


def test_constant_groups():
    """No deviation at all: the bias, and gradients that are finite."""
    for c, h, w, groups in ((64, 9, 9, 4), (64, 300, 300, 4), (64, 1, 1, 64), (64, 1, 1, 4)):
        x = torch.full((2, c, h, w), 3.0, device="cuda").contiguous(memory_format=torch.channels_last).requires_grad_()
        b = normal(4, c)
        y = group_norm(x, groups, normal(3, c), b)
        assert torch.allclose(y, b.view(1, c, 1, 1).expand_as(y), atol=1e-3)
        assert torch.isfinite(torch.autograd.grad(y.sum(), x)[0]).all()


@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_values_that_are_not_finite_stay_in_their_group(bad):
    for shape in ((3, 64, 9, 9), (3, 64, 300, 301), (3, 64, 1, 1)):
        x = normal(1, *shape).contiguous(memory_format=torch.channels_last)
        clean = group_norm(x, 4, activation="silu")
        x[1, 20, 0, 0] = bad
        y = group_norm(x, 4, activation="silu")
        hit = torch.zeros(3, 64, dtype=torch.bool, device="cuda")
        hit[1, 16:32] = True
        assert torch.equal(y[~hit], clean[~hit]) and y[hit].isnan().all()


def test_extreme_gates_and_activations():
    """Arguments of the sigmoids far on either side."""
    x = normal(1, 40, 64)
    w = torch.full((64,), 60.0, device="cuda")
    gate = torch.linspace(-200, 200, 40 * 64, device="cuda").view(40, 64)
    for act in ("silu", "gelu"):
        y = group_norm_rows(x, 4, w, None, activation=act, gate=gate)
        want = formula(x.double(), 4, w.double(), None, 1e-5, act, gate.double())
        # the pre-activation is off by 2^-21 of up to 240, and an exponential by that much relatively
        assert bool(((y.double() - want).abs() <= 2e-4 * want.abs() + 1e-6 * 240 * gate.double().abs().clamp(min=1)).all())


def test_other_layouts_and_module():
    x = normal(1, 2, 64, 10, 12)
    m = GroupNorm(8, 64, activation="gelu").cuda()
    y = m(x)
    assert y.is_contiguous(memory_format=torch.channels_last)
    assert torch.equal(y, m(x.contiguous(memory_format=torch.channels_last)))
    assert torch.allclose(y, torch.nn.functional.gelu(torch.nn.functional.group_norm(x, 8)), atol=2e-5)
    x3 = normal(2, 3, 5, 64)
    assert torch.equal(group_norm_rows(x3, 4), group_norm_rows(x3.view(15, 64), 4).view(3, 5, 64))
    half = GroupNorm(8, 64).cuda().to(torch.bfloat16)
    out = half(x.bfloat16())
    g = torch.autograd.grad(out.float().sum(), [half.weight, half.bias])
    assert [t.dtype for t in g] == [torch.bfloat16] * 2
    # one channel, or one pixel: any strides count as channels-last
    one = normal(3, 4, 1, 6, 6)
    assert torch.allclose(group_norm(one, 1), torch.nn.functional.group_norm(one, 1), atol=1e-5)
    thin = normal(3, 4, 16, 1, 1).expand(4, 16, 1, 1)
    assert torch.allclose(group_norm(thin, 2), torch.nn.functional.group_norm(thin, 2), atol=1e-5)


def test_gradients_against_differences():
    x, gate = normal(1, 2, 32, 6, 7).contiguous(memory_format=torch.channels_last), normal(2, 2, 32, 6, 7).contiguous(memory_format=torch.channels_last)
    leaves = [t.clone(memory_format=torch.preserve_format).requires_grad_() for t in (x, gate, normal(3, 32), normal(4, 32))]

    def f(*t):
        return group_norm(t[0], 4, t[2], t[3], activation="silu", gate=t[1])

    wt = normal(5, 2, 32, 6, 7)
    grads = torch.autograd.grad(f(*leaves), leaves, wt.contiguous(memory_format=torch.channels_last))
    for i in range(4):
        d, h = normal(10 + i, *leaves[i].shape), 2 ** -7
        plus, minus = [t.detach() for t in leaves], [t.detach() for t in leaves]
        plus[i], minus[i] = plus[i] + h * d, minus[i] - h * d
        want = ((f(*plus).double() - f(*minus).double()) * wt.double()).sum() / (2 * h)
        got = (grads[i].double() * d.double()).sum()
        # third derivatives times h^2, and rounding of 2^-22 over h
        assert abs(float(got - want)) <= 0.05 + 2e-3 * abs(float(want))


def test_same_bits_streams_and_graphs():
    x = normal(1, 4, 64, 30, 31, dtype=torch.bfloat16).contiguous(memory_format=torch.channels_last).requires_grad_()
    w = normal(3, 64).requires_grad_()
    dy = torch.ones_like(x)
    runs = []
    for _ in range(2):
        y = group_norm(x, 8, w, activation="silu")
        runs.append((y, *torch.autograd.grad(y, (x, w), dy)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = group_norm(x, 8, w, activation="silu")
        torch.autograd.grad(y, (x, w), dy)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, runs[0][0])
    graph = torch.cuda.CUDAGraph()
    a, b = x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(group_norm(a, 8, b, activation="silu"), (a, b), dy)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        out = group_norm(a, 8, b, activation="silu")
        grads = torch.autograd.grad(out, (a, b), dy)
    with torch.no_grad():
        a.mul_(2)
    graph.replay()
    c = a.detach().clone().requires_grad_()
    want = group_norm(c, 8, b, activation="silu")
    assert torch.equal(out, want) and all(torch.equal(p, q) for p, q in zip(grads, torch.autograd.grad(want, (c, b), dy)))


def test_nothing_to_do():
    w = torch.ones(64, device="cuda", requires_grad=True)
    for x in (torch.zeros(0, 64, 3, 3, device="cuda", requires_grad=True), torch.zeros(2, 64, 0, 3, device="cuda", requires_grad=True)):
        y = group_norm(x, 4, w)
        assert y.shape == x.shape
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert dx.shape == x.shape and not dw.any()
    assert group_norm_rows(torch.zeros(0, 64, device="cuda"), 4).shape == (0, 64)


def test_refusals():
    x = torch.zeros(2, 64, 3, 3, device="cuda")
    w = torch.ones(64, device="cuda")
    with pytest.raises(ValueError, match="divisor"):
        group_norm(x, 7)
    with pytest.raises(ValueError, match="divisor"):
        group_norm(x, 0)
    with pytest.raises(ValueError, match="weight must have shape"):
        group_norm(x, 4, w[:32])
    with pytest.raises(TypeError, match="bias"):
        group_norm(x, 4, w, w.int())
    with pytest.raises(ValueError, match="activation"):
        group_norm(x, 4, activation="relu")
    with pytest.raises(ValueError, match="gate must have shape"):
        group_norm(x, 4, gate=x[:1])
    with pytest.raises(TypeError, match="gate must be"):
        group_norm(x, 4, gate=x.half())
    with pytest.raises(ValueError, match="x must be"):
        group_norm(x[0], 4)
    with pytest.raises(TypeError, match="unsupported dtype"):
        group_norm(x.double(), 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        group_norm(x.cpu(), 4)
    with pytest.raises(RuntimeError, match="weight must be on"):
        group_norm(x, 4, w.cpu())
    with pytest.raises(ValueError, match="divisor"):
        GroupNorm(3, 64)
    a = x.clone().requires_grad_()
    d, = torch.autograd.grad(group_norm(a, 4, w).sum(), a, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), a)
