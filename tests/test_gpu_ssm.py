"""Selective state space operators (visionhope_b200.ssm_core) on the GPU against the float64 oracle
(oracle/ssm.py) on the same, already rounded inputs.

Bars, on max|a - e| / max|e| per tensor, from the arithmetic:
- 16-bit outputs are fp32 results rounded once: half a unit in the last place is 2^-9 (bf16) and
  2^-12 (fp16) of a value; doubled for the fp32 part: 2^-8 and 2^-11.
- fp32 outputs of the convolution: sums of at most 9 products and a fast sigmoid (2 ulp division):
  about 12 roundings, 12 * 2^-24 < 1e-6; sums over tokens (weight gradients) add in blocks: 5e-6.
- fp32 outputs of the scan: a decay is off by at most 2^-22 (the exponential) + 2^-23 (its argument,
  for |s A| < 4) = 3.6e-7, the state by that times the tokens that it remembers, 1 / (1 - decay);
  steps here are about 0.7 and |A| >= 0.3, so at most 6 tokens: 2.2e-6; the gradients go through
  it twice and through sums of up to 600 terms in blocks: 2e-5.
"""
import pytest
import torch

from oracle import ssm as oracle

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
BAR16 = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _bar(t, fp32):
    return BAR16.get(t.dtype, fp32)


def _rel(a, e):
    a, e = a.detach().double().cpu(), e.detach().double().cpu()
    assert a.shape == e.shape
    if e.numel() == 0:
        return 0.0
    return float((a - e).abs().max() / e.abs().max().clamp_min(1e-30))


def _close(a, e, fp32, what=""):
    assert torch.isfinite(a).all(), what
    assert _rel(a, e) <= _bar(a, fp32), (what, _rel(a, e), _bar(a, fp32))


def _rand(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(dtype)


def _leaves(ts, wide):
    return {k: None if t is None else
            (t.double() if wide else t.to(DEV)).detach().requires_grad_(t.is_floating_point()) for k, t in ts.items()}


# ---- short convolution ------------------------------------------------------------------------
def _conv_case(gen, lead, count, d, k, dtype, bias=True, initial=True):
    return dict(x=_rand(gen, *lead, d, dtype=dtype), weight=_rand(gen, d, k, scale=k ** -0.5),
                bias=_rand(gen, d) if bias else None,
                initial_state=_rand(gen, count, k - 1, d, dtype=dtype) if initial else None)


def _conv_check(ts, dtype, gen, *, activation="silu", offsets=None, reverse=False):
    from visionhope_b200.ssm_core import short_conv

    dev, ref = _leaves(ts, False), _leaves(ts, True)
    seq = None if offsets is None else torch.tensor(offsets, device=DEV)
    y, final = short_conv(dev["x"], dev["weight"], dev["bias"], activation=activation,
                          initial_state=dev["initial_state"], return_final_state=True, seq_offsets=seq, reverse=reverse)
    ey, efinal = oracle.short_conv(ref["x"], ref["weight"], ref["bias"], activation=activation,
                                   initial_state=ref["initial_state"], offsets=offsets, reverse=reverse)
    assert y.dtype == dtype and final.dtype == dtype
    _close(y, ey, 1e-6, "y")
    assert torch.equal(final.double().cpu(), efinal.detach())
    gy, gf = _rand(gen, *y.shape, dtype=dtype), _rand(gen, *final.shape, dtype=dtype)
    names = [k for k in dev if dev[k] is not None]
    got = torch.autograd.grad([y, final], [dev[k] for k in names], [gy.to(DEV), gf.to(DEV)])
    exp = torch.autograd.grad([ey, efinal], [ref[k] for k in names], [gy.double(), gf.double()], allow_unused=True)
    exp = [torch.zeros_like(ref[k]) if e is None else e for k, e in zip(names, exp)]  # no token uses it
    for n, g, e in zip(names, got, exp):
        assert g.dtype == dev[n].dtype
        _close(g, e, 5e-6, "d_" + n)
    with torch.no_grad():  # without autograd, and without states
        y2 = short_conv(dev["x"], dev["weight"], dev["bias"], activation=activation,
                        initial_state=dev["initial_state"], seq_offsets=seq, reverse=reverse)
    assert torch.equal(y2, y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L", [1, 2, 3, 15, 16, 17, 31, 33, 70])
@pytest.mark.parametrize("d", [5, 8, 130])
def test_conv_lengths(dtype, L, d):
    gen = torch.Generator().manual_seed(L * 1000 + d)
    _conv_check(_conv_case(gen, (2, L), 2, d, 4, dtype), dtype, gen, reverse=bool(L % 2))


@pytest.mark.parametrize("k", [2, 3, 5, 6, 7, 8])
@pytest.mark.parametrize("bias,initial,activation", [(False, True, "silu"), (True, False, None)])
def test_conv_taps(k, bias, initial, activation):
    gen = torch.Generator().manual_seed(k)
    for lead, dtype in (((3, 5), torch.float32), ((1, 40), torch.bfloat16)):
        _conv_check(_conv_case(gen, lead, lead[0], 12, k, dtype, bias, initial), dtype, gen, activation=activation)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("offsets", [[0, 0, 1, 3, 50, 50, 115], [0, 70], [0, 0, 0], [0, 16, 32, 33, 64]])
def test_conv_packed(dtype, reverse, offsets):
    gen = torch.Generator().manual_seed(len(offsets))
    count = len(offsets) - 1
    _conv_check(_conv_case(gen, (offsets[-1],), count, 24, 4, dtype), dtype, gen, offsets=offsets, reverse=reverse)


def test_conv_views_and_expanded_gradient():
    """Strided halves of a projection, offset by an odd channel, and a broadcast dy."""
    from visionhope_b200.ssm_core import short_conv

    gen = torch.Generator().manual_seed(3)
    big = _rand(gen, 2, 37, 50, dtype=torch.bfloat16)
    w, b = _rand(gen, 16, 4), _rand(gen, 16)
    for view in (lambda t: t[..., 16:32], lambda t: t[..., 3:19], lambda t: t[:, ::2, 5:21],
                 lambda t: t.transpose(1, 2)[:, :, :16]):
        dev = view(big.to(DEV)).detach().requires_grad_()
        ref = view(big).double().detach().requires_grad_()
        y, ey = short_conv(dev, w.to(DEV), b.to(DEV), activation="silu"), oracle.short_conv(ref, w.double(), b.double(), activation="silu")[0]
        _close(y, ey, 1e-6)
        y.sum().backward()
        ey.sum().backward()
        _close(dev.grad, ref.grad, 5e-6)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,d,k", [(1, 7, 4), (5, 64, 4), (3, 130, 2), (2, 12, 8)])
def test_conv_steps_follow_the_sequence(dtype, b, d, k):
    """Token by token through the cache gives the sequence's y and final state; rows of slots in any
    order; a slot outside the cache is skipped and its y is 0."""
    from visionhope_b200.ssm_core import short_conv, short_conv_step

    gen = torch.Generator().manual_seed(b * 100 + d)
    ts = _conv_case(gen, (b, 6), b, d, k, dtype)
    dev = {n: t.to(DEV) for n, t in ts.items()}
    y, final = short_conv(dev["x"], dev["weight"], dev["bias"], activation="silu", initial_state=dev["initial_state"],
                          return_final_state=True)
    slots = torch.tensor([b + 1 - i for i in range(b)], device=DEV)
    cache = torch.zeros(b + 2, k - 1, d, dtype=dtype, device=DEV)
    cache[slots] = dev["initial_state"]
    before = cache[0].clone()
    for t in range(6):
        yt = short_conv_step(dev["x"][:, t], cache, dev["weight"], dev["bias"], activation="silu", slots=slots)
        assert torch.equal(yt, y[:, t])
    assert torch.equal(cache[slots], final)
    assert torch.equal(cache[0], before)
    kept = cache.clone()
    bad = slots.clone()
    bad[0] = b + 2 if b % 2 else -1
    out = torch.full_like(cache, 7.0)
    yt = short_conv_step(dev["x"][:, 0], cache, dev["weight"], dev["bias"], slots=bad, state_out=out)
    assert torch.equal(cache, kept) and (yt[0] == 0).all() and (out[slots[0]] == 7).all()


# ---- selective scan ----------------------------------------------------------------------------
def _scan_case(gen, lead, count, d, n, dtype, groups=1, z=True, skip=True, bias=True, initial=True):
    bc = (*lead, groups, n) if groups > 1 else (*lead, n)
    return dict(u=_rand(gen, *lead, d, dtype=dtype), delta=_rand(gen, *lead, d, dtype=dtype, scale=0.5),
                A=-(0.3 + torch.rand(d, n, generator=gen) * 3), B=_rand(gen, *bc, dtype=dtype),
                C=_rand(gen, *bc, dtype=dtype), D=_rand(gen, d) if skip else None,
                z=_rand(gen, *lead, d, dtype=dtype) if z else None, delta_bias=_rand(gen, d, scale=0.3) if bias else None,
                initial_state=_rand(gen, count, d, n) if initial else None)


def _scan_run(module_or_oracle, ts, *, softplus=True, offsets=None, reverse=False):
    a = dict(z=ts["z"], delta_bias=ts["delta_bias"], delta_softplus=softplus, initial_state=ts["initial_state"],
             reverse=reverse)
    args = [ts[k] for k in ("u", "delta", "A", "B", "C", "D")]
    if module_or_oracle is oracle:
        return oracle.ssm_scan(*args, offsets=offsets, **a)
    seq = None if offsets is None else torch.tensor(offsets, device=DEV, dtype=torch.int32)
    return module_or_oracle.ssm_scan(*args, return_final_state=True, seq_offsets=seq, **a)


def _scan_check(ts, dtype, gen, **kw):
    from visionhope_b200 import ssm_core

    dev, ref = _leaves(ts, False), _leaves(ts, True)
    y, final = _scan_run(ssm_core, dev, **kw)
    ey, efinal = _scan_run(oracle, ref, **kw)
    assert y.dtype == dtype and final.dtype == torch.float32
    _close(y, ey, 5e-6, "y")
    _close(final, efinal, 5e-6, "final")
    with torch.no_grad():
        y2, final2 = _scan_run(ssm_core, dev, **kw)
    assert torch.equal(y2, y) and torch.equal(final2, final)
    gy, gf = _rand(gen, *y.shape, dtype=dtype), _rand(gen, *final.shape)
    names = [k for k in dev if dev[k] is not None]
    got = torch.autograd.grad([y, final], [dev[k] for k in names], [gy.to(DEV), gf.to(DEV)])
    exp = torch.autograd.grad([ey, efinal], [ref[k] for k in names], [gy.double(), gf.double()], allow_unused=True)
    exp = [torch.zeros_like(ref[k]) if e is None else e for k, e in zip(names, exp)]  # no token uses it
    for n, g, e in zip(names, got, exp):
        assert g.dtype == dev[n].dtype
        _close(g, e, 2e-5, "d_" + n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L", [1, 3, 4, 5, 31, 32, 33, 67, 130])
def test_scan_lengths(dtype, L):
    gen = torch.Generator().manual_seed(L)
    _scan_check(_scan_case(gen, (2, L), 2, 40, 16, dtype), dtype, gen, reverse=bool(L % 2))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [4, 8, 16, 32, 64])
@pytest.mark.parametrize("d,groups", [(1, 1), (7, 1), (36, 1), (132, 1), (66, 2), (96, 3)])
def test_scan_states_channels_groups(dtype, n, d, groups):
    gen = torch.Generator().manual_seed(n * 1000 + d)
    _scan_check(_scan_case(gen, (2, 37), 2, d, n, dtype, groups), dtype, gen, reverse=d % 2 == 1)


@pytest.mark.parametrize("off", ["z", "skip", "bias", "initial", "all"])
@pytest.mark.parametrize("softplus", [False, True])
def test_scan_optional_inputs(off, softplus):
    gen = torch.Generator().manual_seed(11)
    kw = {k: not (off in (k, "all")) for k in ("z", "skip", "bias", "initial")}
    ts = _scan_case(gen, (3, 35), 3, 20, 16, torch.float32, **kw)
    if not softplus:  # steps as they are: positive, as softplus would make them
        ts["delta"], ts["delta_bias"] = 0.2 + ts["delta"].abs(), None if ts["delta_bias"] is None else ts["delta_bias"].abs()
    _scan_check(ts, torch.float32, gen, softplus=softplus)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("offsets", [[0, 0, 1, 4, 69, 69, 133], [0, 70], [0, 0, 0], [0, 32, 64, 65, 96]])
def test_scan_packed(dtype, reverse, offsets):
    gen = torch.Generator().manual_seed(len(offsets))
    ts = _scan_case(gen, (offsets[-1],), len(offsets) - 1, 48, 16, dtype, groups=2)
    _scan_check(ts, dtype, gen, offsets=offsets, reverse=reverse)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,offsets,reverse", [(16, None, False), (16, [0, 5, 700, 700, 2100], True), (8, None, True),
                                               (64, [0, 1100, 1101], False), (4, None, False)])
def test_scan_long_chains(dtype, n, offsets, reverse):
    """Few chains of up to 2100 tokens: many warps share a chain."""
    gen = torch.Generator().manual_seed(n)
    lead = (1, 2100) if offsets is None else (offsets[-1],)
    count = 1 if offsets is None else len(offsets) - 1
    _scan_check(_scan_case(gen, lead, count, 40, n, dtype), dtype, gen, offsets=offsets, reverse=reverse)


def test_scan_many_chains():
    """More than eight chains a multiprocessor: one warp walks each."""
    gen = torch.Generator().manual_seed(1)
    _scan_check(_scan_case(gen, (320, 37), 320, 132, 16, torch.float32), torch.float32, gen)


@pytest.mark.parametrize("chains", [480, 640, 800])
def test_scan_chains_around_the_choices(chains):
    """Forward and backward in segments, the forward alone, neither."""
    gen = torch.Generator().manual_seed(chains)
    _scan_check(_scan_case(gen, (chains, 67), chains, 9, 16, torch.float32), torch.float32, gen)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scan_views_and_expanded_gradient(dtype):
    """Slices of two projections at odd offsets, a broadcast z and a broadcast dy."""
    from visionhope_b200 import ssm_core

    gen = torch.Generator().manual_seed(5)
    wide, rows = _rand(gen, 2, 41, 101, dtype=dtype), _rand(gen, 2, 41, 40, dtype=dtype)
    base = _scan_case(gen, (2, 41), 2, 48, 16, dtype)
    grads = []
    for src, w, r in ((False, wide.to(DEV), rows.to(DEV)), (True, wide.double(), rows.double())):
        ts = _leaves(base, src)
        ts["u"] = w[..., 2:50].detach().requires_grad_()
        ts["delta"] = w[..., 52:100].detach().requires_grad_()
        ts["B"], ts["C"] = (r[..., i:i + 16].detach().requires_grad_() for i in (3, 20))
        ts["z"] = w[:, :1, 1:49].expand(2, 41, 48).detach().requires_grad_()
        y, _ = _scan_run(oracle if src else ssm_core, ts)
        grads.append((y, *torch.autograd.grad(y.sum(), [ts[k] for k in ("u", "delta", "B", "C", "z", "A")])))
    for a, e in zip(*grads):
        _close(a, e, 2e-5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,d,n,groups", [(1, 7, 16, 1), (5, 64, 16, 2), (3, 130, 8, 1), (2, 12, 64, 3), (2, 9, 4, 1)])
def test_scan_steps_follow_the_sequence(dtype, b, d, n, groups):
    from visionhope_b200.ssm_core import ssm_scan_step

    gen = torch.Generator().manual_seed(b * 100 + d)
    ts = _scan_case(gen, (b, 6), b, d, n, dtype, groups)
    ey, efinal = _scan_run(oracle, {k: t.double() for k, t in ts.items()})
    dev = {k: t.to(DEV) for k, t in ts.items()}
    slots = torch.tensor([b + 1 - i for i in range(b)], device=DEV, dtype=torch.int32)
    cache = torch.zeros(b + 2, d, n, device=DEV)
    cache[slots.long()] = dev["initial_state"]

    def step(t, **kw):
        return ssm_scan_step(dev["u"][:, t], dev["delta"][:, t], dev["A"], dev["B"][:, t], dev["C"][:, t], cache,
                             dev["D"], z=dev["z"][:, t], delta_bias=dev["delta_bias"], delta_softplus=True, **kw)

    for t in range(6):
        _close(step(t, slots=slots), ey[:, t], 5e-6)
    _close(cache[slots.long()], efinal, 5e-6)
    assert (cache[0] == 0).all()
    kept, out = cache.clone(), torch.full_like(cache, 7.0)
    bad = slots.clone()
    bad[0] = b + 2 if b % 2 else -1
    y = step(0, slots=bad, state_out=out)
    assert torch.equal(cache, kept) and (y[0] == 0).all() and (out[slots[0].long()] == 7).all()


def test_scan_gradient_against_differences():
    """Central differences of the kernels' own loss along a random direction of all inputs.  The
    loss sums 3000 outputs of size 1 weighted by normals, so its rounding noise is below 1e-6 * 60
    = 6e-5, over 2 eps = 0.02: 3e-3; the gradient along a direction of norm 50 is about 50; the
    third-order term is eps^2 of it: together well under 1e-3 of the gradient's norm."""
    from visionhope_b200 import ssm_core

    gen = torch.Generator().manual_seed(21)
    ts = _leaves(_scan_case(gen, (2, 37), 2, 40, 16, torch.float32), False)
    names = list(ts)
    gy = _rand(gen, 2, 37, 40).to(DEV)
    dirs = {k: _rand(gen, *ts[k].shape).to(DEV) * (0.1 if k == "A" else 1.0) for k in names}

    def loss(eps):
        with torch.no_grad():
            y, _ = _scan_run(ssm_core, {k: ts[k] + eps * dirs[k] for k in names})
            return float((y.double() * gy.double()).sum())

    y, _ = _scan_run(ssm_core, ts)
    grads = torch.autograd.grad(y, [ts[k] for k in names], gy)
    want = sum(float((g.double() * dirs[k].double()).sum()) for g, k in zip(grads, names))
    norm = sum(float(g.double().norm() * dirs[k].double().norm()) for g, k in zip(grads, names))
    eps = 0.01
    assert abs((loss(eps) - loss(-eps)) / (2 * eps) - want) <= 1e-3 * norm


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_backward_is_deterministic(dtype):
    from visionhope_b200 import ssm_core

    gen = torch.Generator().manual_seed(8)
    ts = _leaves(_scan_case(gen, (3, 300), 3, 200, 16, dtype, groups=2), False)
    cs = _leaves(_conv_case(gen, (3, 300), 3, 200, 4, dtype), False)
    gy = _rand(gen, 3, 300, 200, dtype=dtype).to(DEV)
    runs = []
    for _ in range(2):
        y, _ = _scan_run(ssm_core, ts)
        c = ssm_core.short_conv(cs["x"], cs["weight"], cs["bias"], activation="silu")
        runs.append([*torch.autograd.grad(y, list(ts.values()), gy),
                     *torch.autograd.grad(c, [cs[k] for k in ("x", "weight", "bias")], gy)])
    for a, b in zip(*runs):
        assert torch.equal(a, b)


def test_steps_of_zero_keep_the_state_and_large_ones_forget_it():
    """softplus(-inf) = 0 leaves the state untouched whatever A is; a large step times A = -1e30 or
    -inf forgets it; neither makes a NaN."""
    from visionhope_b200.ssm_core import ssm_scan

    gen = torch.Generator().manual_seed(4)
    ts = {k: t.to(DEV) for k, t in _scan_case(gen, (1, 9), 1, 32, 16, torch.float32, z=False, skip=False, bias=False).items()
          if t is not None}
    ts["A"][:, 0], ts["A"][:, 1] = -1e30, -float("inf")
    h0 = ts["initial_state"]
    ts["delta"].fill_(-float("inf"))
    y, h = ssm_scan(ts["u"], ts["delta"], ts["A"], ts["B"], ts["C"], delta_softplus=True, initial_state=h0,
                    return_final_state=True)
    assert torch.equal(h, h0) and torch.isfinite(y).all()
    ts["delta"].fill_(50.0)
    y, h = ssm_scan(ts["u"], ts["delta"], ts["A"], ts["B"], ts["C"], delta_softplus=True, initial_state=h0,
                    return_final_state=True)
    last = 50.0 * ts["u"][0, -1, :, None] * ts["B"][0, -1]
    assert torch.allclose(h[0, :, :2], last[:, :2], rtol=1e-6) and torch.isfinite(y).all()


@pytest.mark.parametrize("d", [40, 37])
def test_nan_and_inf_stay_in_their_channel_and_sequence(d):
    from visionhope_b200 import ssm_core

    gen = torch.Generator().manual_seed(6)
    offsets = [0, 30, 30, 70]
    ts = {k: t.to(DEV) for k, t in _scan_case(gen, (70,), 3, d, 16, torch.float32).items()}
    clean_y, clean_h = _scan_run(ssm_core, ts, offsets=offsets)
    ts["u"][35, 3], ts["z"][40, 5], ts["delta"][50, d - 1] = float("nan"), float("inf"), float("nan")
    y, h = _scan_run(ssm_core, ts, offsets=offsets)
    hit = torch.zeros(70, d, dtype=torch.bool, device=DEV)
    hit[35:, 3] = hit[40, 5] = hit[50:, d - 1] = True
    assert torch.equal(y[~hit], clean_y[~hit])
    assert y[35:, 3].isnan().all() and y[50:, d - 1].isnan().all() and not y[40, 5].isfinite()
    assert torch.equal(h[:2], clean_h[:2]) and h[2, 3].isnan().all() and h[2, d - 1].isnan().all()
    x = ts["z"]
    w, b = _rand(gen, d, 4).to(DEV), _rand(gen, d).to(DEV)
    seq = torch.tensor(offsets, device=DEV)
    x[40, 5] = 0.0
    clean = ssm_core.short_conv(x, w, b, seq_offsets=seq)
    x[28, 2] = x[69, d - 1] = float("nan")
    y = ssm_core.short_conv(x, w, b, seq_offsets=seq)
    hit.zero_()
    hit[28:30, 2] = hit[69, d - 1] = True
    assert torch.equal(y[~hit], clean[~hit]) and y[hit].isnan().all()


def test_offsets_out_of_range_are_clamped():
    """Offsets that the host cannot see: values outside the tokens, or tokens before the first
    sequence, touch nothing outside the tokens."""
    from visionhope_b200 import ssm_core

    gen = torch.Generator().manual_seed(9)
    ts = {k: t.to(DEV) for k, t in _scan_case(gen, (50,), 3, 32, 16, torch.float32).items()}
    want, h = _scan_run(ssm_core, ts, offsets=[0, 20, 20, 50])
    got, h2 = _scan_run(ssm_core, ts, offsets=[-5, 20, 20, 900])
    assert torch.equal(h, h2) and torch.equal(got, want)
    x, w = ts["u"], _rand(gen, 32, 4).to(DEV)
    a = ssm_core.short_conv(x, w, seq_offsets=torch.tensor([0, 20, 20, 50], device=DEV))
    b = ssm_core.short_conv(x, w, seq_offsets=torch.tensor([-5, 20, 20, 900], device=DEV))
    assert torch.equal(a, b)
    late = ssm_core.short_conv(x, w, seq_offsets=torch.tensor([40, 50], device=DEV))
    assert torch.equal(late[43:], a[43:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [5, 24])
@pytest.mark.parametrize("op", ["conv", "scan"])
def test_rows_of_no_sequence_are_zero(op, d, dtype):
    """A packed buffer longer than its sequences: NaN before and behind them reaches nothing."""
    from visionhope_b200 import ssm_core

    gen = torch.Generator().manual_seed(d)
    if op == "conv":
        base, rows = _conv_case(gen, (54,), 3, d, 4, dtype), ("x",)
        bars = dict(y=1e-6, final=1e-6, grad=5e-6)
    else:
        base, rows = _scan_case(gen, (54,), 3, d, 16, dtype), ("u", "delta", "B", "C", "z")
        bars = dict(y=5e-6, final=5e-6, grad=2e-5)
    gy, inside = _rand(gen, 54, d, dtype=dtype), slice(3, 57)

    def padded(t):
        out = torch.full((70, *t.shape[1:]), float("nan"), dtype=t.dtype)
        out[inside] = t
        return out

    ref = _leaves(base, True)
    dev = _leaves({k: padded(t) if k in rows else t for k, t in base.items()}, False)
    if op == "conv":
        y, final = ssm_core.short_conv(dev["x"], dev["weight"], dev["bias"], activation="silu",
                                       initial_state=dev["initial_state"], return_final_state=True,
                                       seq_offsets=torch.tensor([3, 10, 10, 57], device=DEV))
        ey, efinal = oracle.short_conv(ref["x"], ref["weight"], ref["bias"], activation="silu",
                                       initial_state=ref["initial_state"], offsets=[0, 7, 7, 54])
    else:
        y, final = _scan_run(ssm_core, dev, offsets=[3, 10, 10, 57])
        ey, efinal = _scan_run(oracle, ref, offsets=[0, 7, 7, 54])
    gf = _rand(gen, *final.shape, dtype=final.dtype)
    got = torch.autograd.grad([y, final], list(dev.values()), [padded(gy).to(DEV), gf.to(DEV)])
    exp = torch.autograd.grad([ey, efinal], list(ref.values()), [gy.double(), gf.double()])
    results = {"y": (y, ey, bars["y"]), "final": (final, efinal, bars["final"])}
    results.update({"d_" + n: (g, e, bars["grad"]) for n, g, e in zip(dev, got, exp)})
    for n, (a, e, bar) in results.items():
        if a.shape[0] == 70:
            assert (a[:3] == 0).all() and (a[57:] == 0).all(), n
            a = a[inside]
        _close(a, e, bar, n)


def test_side_stream_and_empty_inputs():
    from visionhope_b200 import ssm_core

    gen = torch.Generator().manual_seed(2)
    ts = {k: t.to(DEV) for k, t in _scan_case(gen, (2, 64), 2, 64, 16, torch.bfloat16).items()}
    want, hw = _scan_run(ssm_core, ts)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, hg = _scan_run(ssm_core, ts)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(hg, hw)
    empty = {k: t[:, :0].contiguous() if k in ("u", "delta", "B", "C", "z") else t for k, t in ts.items()}
    empty = _leaves(empty, False)
    y, h = _scan_run(ssm_core, empty)
    assert y.shape == (2, 0, 64) and torch.equal(h, ts["initial_state"])
    gh = torch.autograd.grad(h.sum(), empty["initial_state"])[0]
    assert (gh == 1).all()
    x = torch.zeros(2, 0, 8, device=DEV)
    y, s = ssm_core.short_conv(x, torch.ones(8, 4, device=DEV), return_final_state=True)
    assert y.shape == x.shape and s.shape == (2, 3, 8) and (s == 0).all()


def test_long_strides_pass_32_bits():
    """Token rows whose offsets exceed 2^31 elements: a view with a large token stride over one
    allocation of about 4.4 GB, a row every 2^28 elements."""
    from visionhope_b200 import ssm_core

    gen = torch.Generator().manual_seed(7)
    d, stride, L = 32, 1 << 28, 9
    big = torch.zeros(stride * (L - 1) + d, dtype=torch.bfloat16, device=DEV)
    rows = big.as_strided((1, L, d), (0, stride, 1))
    x = _rand(gen, 1, L, d, dtype=torch.bfloat16).to(DEV)
    rows.copy_(x)
    w = _rand(gen, d, 4).to(DEV)
    assert torch.equal(ssm_core.short_conv(rows, w), ssm_core.short_conv(x, w))
    ts = {k: t.to(DEV) for k, t in _scan_case(gen, (1, L), 1, d, 16, torch.bfloat16).items()}
    want, _ = _scan_run(ssm_core, {**ts, "u": x})
    got, _ = _scan_run(ssm_core, {**ts, "u": rows})
    assert torch.equal(got, want)


def test_second_derivatives_are_refused():
    """The backward's kernels are not differentiable themselves: asking for it raises instead of
    giving the wrong second derivative."""
    from visionhope_b200.ssm_core import short_conv

    x = torch.randn(1, 5, 8, device=DEV, requires_grad=True)
    w = torch.randn(8, 4, device=DEV, requires_grad=True)
    g = torch.autograd.grad(short_conv(x, w, activation="silu").sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_python_refusals():
    from visionhope_b200 import ssm_core

    x, w = torch.zeros(2, 5, 8, device=DEV), torch.zeros(8, 4, device=DEV)
    A, B = torch.zeros(8, 16, device=DEV), torch.zeros(2, 5, 16, device=DEV)
    conv, scan = ssm_core.short_conv, ssm_core.ssm_scan
    off = torch.tensor([0, 5], device=DEV)
    for exc, call in [
        (ValueError, lambda: conv(x[0], w)), (ValueError, lambda: conv(x, w[:4])), (ValueError, lambda: conv(x, w[:, :1])),
        (ValueError, lambda: conv(x, torch.zeros(8, 9, device=DEV))), (TypeError, lambda: conv(x.double(), w)),
        (ValueError, lambda: conv(x, w, seq_offsets=off)), (TypeError, lambda: conv(x[0], w, seq_offsets=off.float())),
        (ValueError, lambda: conv(x[0], w, seq_offsets=off[:1])), (RuntimeError, lambda: conv(x[0], w, seq_offsets=off.cpu())),
        (RuntimeError, lambda: conv(x, w.cpu())), (ValueError, lambda: conv(x, w, torch.zeros(7, device=DEV))),
        (ValueError, lambda: conv(x, w, initial_state=torch.zeros(2, 4, 8, device=DEV))),
        (TypeError, lambda: conv(x, w, initial_state=torch.zeros(2, 3, 8, device=DEV, dtype=torch.bfloat16))),
        (ValueError, lambda: conv(x, w, activation="gelu")),
        (ValueError, lambda: scan(x, x[:, :4], A, B, B)), (TypeError, lambda: scan(x, x.half(), A, B, B)),
        (ValueError, lambda: scan(x, x, A[:, :12], B[..., :12], B[..., :12])), (ValueError, lambda: scan(x, x, A, B[..., :8], B)),
        (ValueError, lambda: scan(x, x, A, B.view(2, 5, 1, 16).expand(2, 5, 3, 16), B)),
        (ValueError, lambda: scan(x, x, A[:4], B, B)), (RuntimeError, lambda: scan(x, x, A.cpu(), B, B)),
        (TypeError, lambda: scan(x, x, A, B, B, initial_state=torch.zeros(2, 8, 16, device=DEV, dtype=torch.bfloat16))),
        (ValueError, lambda: scan(x, x, A, B, B, torch.zeros(9, device=DEV))),
        (ValueError, lambda: ssm_core.ssm_scan_step(x, x, A, B, B, torch.zeros(2, 8, 16, device=DEV))),
        (ValueError, lambda: ssm_core.ssm_scan_step(x[:, 0], x[:, 0], A, B[:, 0], B[:, 0], torch.zeros(1, 8, 16, device=DEV))),
        (TypeError, lambda: ssm_core.ssm_scan_step(x[:, 0], x[:, 0], A, B[:, 0], B[:, 0], torch.zeros(2, 8, 16, device=DEV).half())),
        (ValueError, lambda: ssm_core.short_conv_step(x[:, 0], torch.zeros(2, 8, 3, device=DEV).transpose(1, 2), w)),
        (ValueError, lambda: ssm_core.short_conv_step(x[:, 0], torch.zeros(1, 3, 8, device=DEV), w)),
        (ValueError, lambda: ssm_core.short_conv_step(x[:, 0], torch.zeros(2, 3, 8, device=DEV), w, slots=off[:1])),
    ]:
        with pytest.raises(exc):
            call()
