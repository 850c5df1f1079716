"""The selective state space operators over the whole range of their inputs: the functions inside
them where they saturate, the lowest and infinite values that masks are made of.

Bars, from the arithmetic.  A sigmoid is 1 / (1 + 2^(-x log2 e)) by ex2.approx (2^-22) and rcp.approx
(2^-23); its argument carries the rounding of the product and of the constant, |x| (2^-24 + 2^-25).
Relative to the value that is REL(x) = |x| 1e-7 + 1e-6 with the products behind it.  Below x = -87 the
sigmoid is less than fp32's smallest normal number, 1.2e-38, and may be zero: TINY = |x| 1.2e-38 for
|x| up to 104, past which the true value is smaller still: 2e-36.  A 16-bit
result has to lie between the two ends of that interval rounded to 16 bits.  silu' = sg (1 + x (1 - sg)) is
held to REL(x) of the sum of its terms' sizes, sg (1 + |x| (1 - sg)), and for x > 0 to the rounding of
1 - sg, 2^-23, times x where it is not exactly zero (x < 18).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
TINY = 2e-36


def _values(dtype):
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    v = [low, -1e30, -1e20, -1e18, -60000.0, -1000.0, -200.0, -104.0, -90.0, -60.0, -42.0, -41.0, -20.0, -5.0, -1.0,
         -1e-3, 0.0, 1e-3, 1.0, 5.0, 17.0, 20.0, 60.0, 100.0, 1000.0, 60000.0, 1e18, 1e30, high, -float("inf")]
    return [x for x in v if x == -float("inf") or low <= x <= high]


def _table(dtype, d=24):
    """[sequences, 1, d]: every value beside many others, since neighbouring channels share instructions."""
    v = _values(dtype)
    rows = [[v[(b + c * (c + 1) // 2) % len(v)] for c in range(d)] for b in range(len(v))]
    return torch.tensor(rows, dtype=torch.float64).to(dtype)[:, None]


def _rel(x):
    return x.abs().clamp_max(1e4) * 1e-7 + 1e-6


def _check(got, want, bar, dtype):
    got, want, bar = got.detach().double().cpu(), want.double(), bar.double()
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan)
    got, want, bar = got[~nan], want[~nan], bar[~nan]
    low, high = want - bar - TINY, want + bar + TINY
    if dtype != torch.float32:
        low, high = low.to(dtype).double(), high.to(dtype).double()
    off = torch.maximum(low - got, got - high)
    worst = int(off.argmax())
    assert float(off[worst]) <= 0, (float(got[worst]), float(want[worst]), float(bar[worst]))


def _silu(x):
    x = x.double()
    y = x * torch.sigmoid(x)
    return y, _rel(x) * y.abs()


def _silu_slope(x):
    x = x.double()
    sg = torch.sigmoid(x)
    rest = torch.sigmoid(-x)
    slope = sg + x * sg * rest
    slope[x == float("-inf")] = float("nan")
    bar = _rel(x) * sg * (1 + x.abs() * rest) + torch.where((x > 0) & (x < 18), x * 2.0 ** -23, torch.zeros_like(x))
    bar = bar + torch.where(x >= 17, x.clamp(0, 1e3) * rest, torch.zeros_like(x))  # 1 - sg rounded away
    return slope, bar


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [24, 7])
def test_convolution_silu_saturates(dtype, d):
    """One token through a convolution that passes it on: silu(x), its gradient and its step."""
    from visionhope_b200.ssm_core import short_conv, short_conv_step

    x = _table(dtype, d)
    dev = x.to(DEV).requires_grad_()
    w = torch.tensor([[0.0, 1.0]], device=DEV).expand(d, 2).contiguous()
    y = short_conv(dev, w, activation="silu")
    _check(y, *_silu(x), dtype)
    g = torch.autograd.grad(y, dev, torch.ones_like(y))[0]
    _check(g, *_silu_slope(x), dtype)
    state = torch.zeros(x.shape[0], 1, d, dtype=dtype, device=DEV)
    step = short_conv_step(dev.detach()[:, 0], state, w, activation="silu")
    _check(step[:, None], *_silu(x), dtype)


def _scan_args(x, dtype):
    """A scan whose state stays zero and whose inner output is u = 1."""
    b, _, d = x.shape
    one, none = torch.ones(b, 1, d, dtype=dtype, device=DEV), torch.zeros(b, 1, 16, dtype=dtype, device=DEV)
    return one, one, -torch.ones(d, 16, device=DEV), none, none, torch.ones(d, device=DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [24, 7])
def test_scan_gate_saturates(dtype, d):
    """An inner output of one behind the gate: silu(z), its gradient and the step's."""
    from visionhope_b200.ssm_core import ssm_scan, ssm_scan_step

    z = _table(dtype, d)
    dev = z.to(DEV).requires_grad_()
    u, delta, A, B, C, D = _scan_args(z, dtype)
    u = u.requires_grad_()
    y = ssm_scan(u, delta, A, B, C, D, z=dev)
    _check(y, *_silu(z), dtype)
    gz, gu = torch.autograd.grad(y, [dev, u], torch.ones_like(y))
    _check(gz, *_silu_slope(z), dtype)
    _check(gu, *_silu(z), dtype)
    state = torch.zeros(z.shape[0], d, 16, device=DEV)
    step = ssm_scan_step(u.detach()[:, 0], delta[:, 0], A, B[:, 0], C[:, 0], state, D, z=dev.detach()[:, 0])
    _check(step[:, None], *_silu(z), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [24, 7])
def test_masked_steps_get_no_gradient(dtype, d):
    """softplus' derivative at the lowest value and at -inf is zero; at large values it is one."""
    from visionhope_b200.ssm_core import ssm_scan

    delta = torch.tensor([torch.finfo(dtype).min, -float("inf"), -200.0, -0.5, 0.5, 300.0], dtype=torch.float64).to(dtype)
    delta = delta[(torch.arange(6)[:, None] + torch.arange(d) * (torch.arange(d) + 1) // 2) % 6][:, None]
    dev = delta.to(DEV).requires_grad_()
    u = torch.ones(6, 1, d, dtype=dtype, device=DEV)
    bc = torch.ones(6, 1, 16, dtype=dtype, device=DEV)
    y = ssm_scan(u, dev, torch.zeros(d, 16, device=DEV), bc, bc, delta_softplus=True)
    g = torch.autograd.grad(y, dev, torch.ones_like(y))[0]
    want = 16 * torch.sigmoid(delta.double())  # y = 16 softplus(delta)
    _check(g, want, _rel(delta.double().clamp(-104, 104)) * want, dtype)
    assert (g[delta.to(DEV) < -150] == 0).all()


@pytest.mark.parametrize("packed", [False, True])
def test_entry_points_pass_states_on_without_tokens(packed):
    """The C entry points with a length of 0: states and their gradients pass through, parameters get
    zeros.  (The Python functions answer such calls themselves.)"""
    import ctypes

    from visionhope_b200 import _lib

    lib = _lib.load()
    b, d, n, k = 3, 40, 16, 4
    gen = torch.Generator(device=DEV).manual_seed(1)
    row = torch.zeros(64, device=DEV)  # stands for rows that are never read
    off = torch.zeros(b + 1, dtype=torch.int32, device=DEV) if packed else None
    h0, gf = (torch.randn(b, d, n, generator=gen, device=DEV) for _ in range(2))
    s0, gs = (torch.randn(b, k - 1, d, generator=gen, device=DEV) for _ in range(2))
    A, w = -torch.rand(d, n, generator=gen, device=DEV), torch.randn(d, k, generator=gen, device=DEV)
    stream = _lib.stream_handle(DEV)
    _lib.ensure_device(row)

    def ptr(t):
        return None if t is None else t.data_ptr()

    r = row.data_ptr()
    final, ck = torch.full_like(h0, 7.0), torch.zeros(b * 2 * 512, device=DEV)
    a = _lib.VhSsmScanArgs(u=r, delta=r, z=None, b=r, c=r, u_token_stride=d, delta_token_stride=d, b_token_stride=n,
                           c_token_stride=n, a=ptr(A), initial_state=ptr(h0), y=r, final_state=ptr(final),
                           checkpoints=ptr(ck), seq_offsets=ptr(off), length=0, dtype=0, batch=b, channels=d, states=n,
                           groups=1)
    assert lib.vh_ssm_scan_checkpoint_bytes(ctypes.byref(a)) <= ck.numel() * 4
    need = lib.vh_ssm_scan_fwd_workspace_bytes(ctypes.byref(a))
    ws = torch.empty(need + 16, dtype=torch.uint8, device=DEV)
    _lib.check(lib.vh_ssm_scan_fwd(ctypes.byref(a), ptr(ws), need, stream), "vh_ssm_scan_fwd")
    assert torch.equal(final, h0)
    gi, ga, gd, gb = torch.full_like(h0, 7.0), torch.full_like(A, 7.0), torch.full((d,), 7.0, device=DEV), torch.full((d,), 7.0, device=DEV)
    g = _lib.VhSsmScanBwdArgs(fwd=a, grad_y=r, grad_final=ptr(gf), grad_u=r, grad_delta=r, grad_z=None, grad_b=r, grad_c=r,
                              grad_a=ptr(ga), grad_d_skip=ptr(gd), grad_delta_bias=ptr(gb), grad_initial=ptr(gi))
    need = lib.vh_ssm_scan_bwd_workspace_bytes(ctypes.byref(g))
    ws = torch.empty(need + 16, dtype=torch.uint8, device=DEV)
    _lib.check(lib.vh_ssm_scan_bwd(ctypes.byref(g), ptr(ws), need, stream), "vh_ssm_scan_bwd")
    assert torch.equal(gi, gf) and not ga.any() and not gd.any() and not gb.any()
    kept, gw, gi = torch.full_like(s0, 7.0), torch.full_like(w, 7.0), torch.full_like(s0, 7.0)
    c = _lib.VhShortConvArgs(x=r, x_token_stride=d, weight=ptr(w), initial_state=ptr(s0), y=r, final_state=ptr(kept),
                             seq_offsets=ptr(off), length=0, dtype=0, activation=1, taps=k, batch=b, channels=d)
    _lib.check(lib.vh_short_conv_fwd(ctypes.byref(c), stream), "vh_short_conv_fwd")
    assert torch.equal(kept, s0)
    need = lib.vh_short_conv_bwd_workspace_bytes(ctypes.byref(c))
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    _lib.check(lib.vh_short_conv_bwd(ctypes.byref(c), r, ptr(gs), r, ptr(gw), None, ptr(gi), ptr(ws), need, stream),
               "vh_short_conv_bwd")
    assert torch.equal(gi, gs) and not gw.any()
    assert not row.any()


def test_far_offsets_are_clamped():
    """Offsets of 2^32 + 5 mean the end of the tokens, not token 5."""
    from visionhope_b200.ssm_core import short_conv, ssm_scan

    gen = torch.Generator(device=DEV).manual_seed(2)
    x, bc = torch.randn(50, 32, generator=gen, device=DEV), torch.randn(50, 16, generator=gen, device=DEV)
    w, A = torch.randn(32, 4, generator=gen, device=DEV), -torch.rand(32, 16, generator=gen, device=DEV)
    near = torch.tensor([0, 20, 20, 50], device=DEV)
    far = torch.tensor([-(1 << 32), 20, 20, (1 << 32) + 5], device=DEV)
    assert torch.equal(short_conv(x, w, seq_offsets=near), short_conv(x, w, seq_offsets=far))
    args = x, x, A, bc, bc
    near, far = (ssm_scan(*args, delta_softplus=True, seq_offsets=o, return_final_state=True) for o in (near, far))
    assert torch.equal(near[0], far[0]) and torch.equal(near[1], far[1])


def _shifted(t):
    """The same values one element past an aligned address."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    view = flat[1:].view(t.shape)
    view.copy_(t)
    assert view.data_ptr() % 16
    return view


@pytest.mark.parametrize("dtype", DTYPES)
def test_views_into_larger_buffers(dtype):
    """Parameters, states, rows and incoming gradients at odd addresses give the same bits.  Only the
    convolution's sums over tokens (weight, bias) are added in another order where its loads are
    narrower: 5e-6 of the largest, as against the oracle."""
    from visionhope_b200.ssm_core import short_conv, short_conv_step, ssm_scan, ssm_scan_step

    gen = torch.Generator(device=DEV).manual_seed(3)
    b, L, d, n, k = 2, 70, 32, 16, 4

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device=DEV).to(dtype)

    scan = [normal(b, L, d, dtype=dtype) for _ in range(2)] + [-normal(d, n).abs()] + [normal(b, L, n, dtype=dtype) for _ in range(2)]
    scan += [normal(d), normal(b, d, n), normal(d), normal(b, L, d, dtype=dtype)]
    conv = [normal(b, L, d, dtype=dtype), normal(d, k), normal(d), normal(b, k - 1, d, dtype=dtype)]
    dy, dh, ds = normal(b, L, d, dtype=dtype), normal(b, d, n), normal(b, k - 1, d, dtype=dtype)
    results = []
    for put in (lambda t: t.clone(), _shifted):
        u, delta, A, B, C, D, h0, bias, z = ts = [put(t).requires_grad_() for t in scan]
        x, w, wb, s0 = cs = [put(t).requires_grad_() for t in conv]
        y, h = ssm_scan(u, delta, A, B, C, D, z=z, delta_bias=bias, delta_softplus=True, initial_state=h0, return_final_state=True)
        c, s = short_conv(x, w, wb, activation="silu", initial_state=s0, return_final_state=True)
        out = [y, h, c, s, *torch.autograd.grad([y, h], ts, [put(dy), put(dh)]), *torch.autograd.grad([c, s], cs, [put(dy), put(ds)])]
        with torch.no_grad():
            out.append(ssm_scan_step(put(u[:, 0]), put(delta[:, 0]), A, put(B[:, 0]), put(C[:, 0]), h0.clone(), D, z=put(z[:, 0]),
                                     delta_bias=bias, delta_softplus=True))
            cache = put(s0)
            out += [short_conv_step(put(x[:, 0]), cache, w, wb, activation="silu"), cache]
        results.append(out)
    sums = (4 + len(scan) + 1, 4 + len(scan) + 2)
    for i, (a, e) in enumerate(zip(*results)):
        assert float((a - e).abs().max()) <= 5e-6 * float(e.abs().max()) if i in sums else torch.equal(a, e), i


@pytest.mark.parametrize("name", ["B", "C"])
@pytest.mark.parametrize("n,d", [(16, 32), (8, 64)])
@pytest.mark.parametrize("L", [1, 2, 3, 4, 5, 7, 33, 130, 131])
def test_an_infinite_last_token(L, n, d, name):
    """B or C infinite in one state of the last token: the others' results and whatever does not meet
    that value stay finite, whether the tokens fill their last group of four or not.  All inputs are
    positive, so that no sum has infinities of both signs but the steps' gradient.  Finite values to
    the scan's fp32 bar for gradients, 2e-5 of the largest."""
    from oracle import ssm as oracle
    from visionhope_b200 import ssm_core

    gen = torch.Generator().manual_seed(L)
    ts = dict(u=torch.rand(2, L, d, generator=gen) + 0.1, delta=torch.rand(2, L, d, generator=gen) + 0.1,
              A=-0.3 - torch.rand(d, n, generator=gen), B=torch.rand(2, L, n, generator=gen) + 0.1,
              C=torch.rand(2, L, n, generator=gen) + 0.1, D=torch.rand(d, generator=gen) + 0.1,
              initial_state=torch.rand(2, d, n, generator=gen) + 0.1)
    ts[name][:, -1, 1] = float("inf")
    out = []
    for module, put in ((ssm_core, lambda t: t.to(DEV)), (oracle, lambda t: t.double())):
        v = {k: put(t).requires_grad_() for k, t in ts.items()}
        kw = dict(return_final_state=True) if module is ssm_core else {}
        y, h = module.ssm_scan(v["u"], v["delta"], v["A"], v["B"], v["C"], v["D"], initial_state=v["initial_state"], **kw)
        out.append({"y": y, "final": h, **dict(zip(v, torch.autograd.grad([y, h], list(v.values()),
                                                                        [torch.ones_like(y), torch.ones_like(h)])))})
    for k, e in out[1].items():
        g, e = out[0][k].detach().double().cpu(), e.detach()
        assert torch.equal(g.isnan(), e.isnan()) and torch.equal(g.isinf(), e.isinf()), k
        keep = e.isfinite()
        if keep.any():
            assert float((g - e)[keep].abs().max()) <= 2e-5 * float(e[keep].abs().max()), k
        assert (g[e.isinf()] == e[e.isinf()]).all(), k


@pytest.mark.parametrize("L", [64, 300, 1100, 2100])
def test_growing_states_that_are_zero_stay_zero(L):
    """Rates above zero let a state grow by e^3 a token.  Rows of zeros before the first input (padding),
    and tokens behind the last one with a gradient, keep states and gradients at zero however many
    there are.  Finite values to the scan's fp32 bars: 5e-6, gradients 2e-5 of the largest."""
    from oracle import ssm as oracle
    from visionhope_b200 import ssm_core

    gen = torch.Generator().manual_seed(L)
    d, n = 40, 16
    ts = dict(u=torch.zeros(1, L, d), delta=torch.rand(1, L, d, generator=gen) + 1.5, A=1.0 + torch.rand(d, n, generator=gen),
              B=torch.randn(1, L, n, generator=gen), C=torch.randn(1, L, n, generator=gen))
    ts["u"][:, -3:] = torch.randn(1, 3, d, generator=gen)
    head = torch.zeros(1, L, d)
    head[:, :3] = torch.randn(1, 3, d, generator=gen)
    out = []
    for module, put in ((ssm_core, lambda t: t.to(DEV)), (oracle, lambda t: t.double())):
        v = {k: put(t).requires_grad_() for k, t in ts.items()}
        kw = dict(return_final_state=True) if module is ssm_core else {}
        y, h = module.ssm_scan(*v.values(), **kw)
        out.append([y, h, *torch.autograd.grad(y, list(v.values()), put(head))])
    for i, (g, e) in enumerate(zip(*out)):
        g, e = g.detach().double().cpu(), e.detach()
        assert float((g - e).abs().max()) <= (5e-6 if i < 2 else 2e-5) * float(e.abs().max()), i
    assert out[0][0][:, :-3].eq(0).all() and out[0][2][:, 3:].eq(0).all()


def _segments(L, d, n, dtype, offsets=None):
    """Segments of the forward, over all chains of one channel tile, as its workspace tells."""
    import ctypes

    from visionhope_b200 import _lib

    p = 256  # not read by the query
    a = _lib.VhSsmScanArgs(u=p, delta=p, b=p, c=p, a=p, y=p, seq_offsets=p if offsets else None, length=L,
                           dtype=_lib.DTYPES[dtype], batch=len(offsets) - 1 if offsets else 2, channels=d, states=n, groups=1)
    width = 512 // n
    tiles = -(-d // width)
    return _lib.load().vh_ssm_scan_fwd_workspace_bytes(ctypes.byref(a)) // (4 * (512 + width)) // tiles


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype,n", [(torch.float32, 16), (torch.bfloat16, 16), (torch.float32, 8), (torch.float32, 64),
                                     (torch.bfloat16, 4)])
@pytest.mark.parametrize("L", [300, 700, 1024])
def test_chains_of_nine_to_thirty_two_segments(L, dtype, n, reverse):
    """States and gradients carried over four runs of segments.  Bars: as every other length's."""
    from tests.test_gpu_ssm import _scan_case, _scan_check

    assert 9 <= _segments(L, 40, n, dtype) // 2 <= 32
    gen = torch.Generator().manual_seed(L + n)
    _scan_check(_scan_case(gen, (2, L), 2, 40, n, dtype), dtype, gen, reverse=reverse)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("offsets,d", [([0, 3, 690, 700], 40), ([0, 400, 401, 401, 1100, 1300, 2500, 3900, 4000], 1280)])
def test_packed_chains_over_four_runs(offsets, d, reverse):
    """Packed sequences of which one has most segments; few chains with up to 32, and more than twice as
    many chains as multiprocessors.  (The oracle runs on the GPU too: on the CPU it takes a minute.)"""
    from oracle import ssm as oracle
    from tests.test_gpu_ssm import _close, _scan_case
    from visionhope_b200 import ssm_core

    assert _segments(offsets[-1], d, 16, torch.float32, offsets) > 8
    gen = torch.Generator().manual_seed(d)
    ts = _scan_case(gen, (offsets[-1],), len(offsets) - 1, d, 16, torch.float32)
    ts["delta"], ts["delta_bias"] = 0.2 + ts["delta"].abs(), ts["delta_bias"].abs()  # steps as softplus would make them
    gy, gf = torch.randn(offsets[-1], d, generator=gen).to(DEV), torch.randn(len(offsets) - 1, d, 16, generator=gen).to(DEV)
    out = []
    for module, dtype, kw in ((ssm_core, torch.float32, dict(seq_offsets=torch.tensor(offsets, device=DEV), return_final_state=True)),
                              (oracle, torch.float64, dict(offsets=offsets))):
        v = {k: t.to(DEV, dtype).requires_grad_() for k, t in ts.items()}
        y, h = module.ssm_scan(*(v[k] for k in ("u", "delta", "A", "B", "C", "D")), z=v["z"], delta_bias=v["delta_bias"],
                               initial_state=v["initial_state"], reverse=reverse, **kw)
        out.append({"y": y, "final": h, **dict(zip(v, torch.autograd.grad([y, h], list(v.values()), [gy.to(dtype), gf.to(dtype)])))})
    for k, e in out[1].items():
        _close(out[0][k], e, 5e-6 if k in ("y", "final") else 2e-5, k)


def _sweep(low, high, count, seed):
    gen = torch.Generator().manual_seed(seed)
    even = torch.linspace(low, high, count)
    near = torch.randn(count, generator=gen) * torch.logspace(-6, 1, count)
    return torch.cat([even, near.clamp(low, high), torch.rand(count, generator=gen) * (high - low) + low])


def _within(got, want, rel):
    """Relative to each value; below fp32's normal numbers (1.2e-38) a result may be zero."""
    got, want = got.detach().double().cpu(), want.double()
    assert torch.isfinite(got).all()
    off = (got - want).abs() - rel * want.abs() - TINY / 100
    worst = int(off.argmax())
    assert float(off.flatten()[worst]) <= 0, (float(got.flatten()[worst]), float(want.flatten()[worst]))


def test_softplus_over_its_range():
    """One token with A = 0, B = u = 1 leaves softplus(delta) in a state that was zero.  e = exp(-|x|) is
    within 2^-22 (ex2.approx) and, by the constant's rounding of 1.34e-8, |x| 1.34e-8; log1p(e) / e adds
    3e-8 (the fit) and about four roundings, the sum one: 6e-7 + |x| 1.34e-8."""
    from visionhope_b200.ssm_core import ssm_scan, ssm_scan_step

    x = torch.cat([_sweep(-120, 120, 4096, 1), torch.tensor([-3e38, -1e4, -104.0, -87.0, 0.0, 88.0, 1e4, 3e38])])
    d = x.numel()
    want = torch.logaddexp(x.double(), torch.zeros((), dtype=torch.float64))
    rel = 6e-7 + x.double().abs().clamp_max(104) * 1.34e-8
    one, A, bc, state = torch.ones(1, d, device=DEV), torch.zeros(d, 4, device=DEV), torch.ones(1, 4, device=DEV), torch.zeros(1, d, 4, device=DEV)
    ssm_scan_step(one, x[None].to(DEV), A, bc, bc, state, delta_softplus=True)
    _, final = ssm_scan(one[None], x[None, None].to(DEV), A, bc[None], bc[None], delta_softplus=True, return_final_state=True)
    for got in (state, final):
        for n in range(4):
            _within(got[0, :, n], want, rel)


def test_decays_over_their_range():
    """One token with u = 0 leaves exp(delta A) in states that were one.  log2(e) A carries its rounding
    and the constant's, 7.3e-8 of the exponent.  The polynomial (the step; the scan's lowest quarter of
    the states) adds 2e-7, past an exponent of 126 the hardware's 2^-22 and the argument's rounding; the
    hardware function (the other states) adds that everywhere: 4e-7 and 1.4e-7 of the exponent."""
    from visionhope_b200.ssm_core import ssm_scan, ssm_scan_step

    s = _sweep(0.0, 12.0, 2048, 2).abs()
    d, n = s.numel(), 16
    gen = torch.Generator().manual_seed(3)
    A = -torch.rand(d, n, generator=gen) * torch.tensor([0.01, 0.1, 1.0, 11.0]).repeat(d, n // 4)
    A[::7] *= -0.5  # growing states too
    x = s.double()[:, None] * A.double()
    want = torch.exp(x)
    zero, bc = torch.zeros(1, d, device=DEV), torch.ones(1, n, device=DEV)
    state = torch.ones(1, d, n, device=DEV)
    _, final = ssm_scan(zero[None], s[None, None].to(DEV), A.to(DEV), bc[None], bc[None], initial_state=state, return_final_state=True)
    ssm_scan_step(zero, s[None].to(DEV), A.to(DEV), bc, bc, state)
    hardware = 4e-7 + x.abs() * 1.4e-7
    poly = torch.where(x.abs() * 1.4427 < 125, 2e-7 + x.abs() * 7.3e-8, hardware)
    _within(state[0], want, poly)
    _within(final[0, :, :n // 4], want[:, :n // 4], poly[:, :n // 4])
    _within(final[0, :, n // 4:], want[:, n // 4:], hardware[:, n // 4:])


@pytest.mark.parametrize("dtype", DTYPES)
def test_silu_over_its_range(dtype):
    """Dense values between the saturated ends, through the convolution and its gradient."""
    from visionhope_b200.ssm_core import short_conv

    x = _sweep(-110, 110, 4096, 4).to(dtype)[:, None, None].expand(-1, 1, 2).contiguous()
    dev = x.to(DEV).requires_grad_()
    w = torch.tensor([[0.0, 1.0]], device=DEV).expand(2, 2).contiguous()
    y = short_conv(dev, w, activation="silu")
    _check(y, *_silu(x), dtype)
    _check(torch.autograd.grad(y, dev, torch.ones_like(y))[0], *_silu_slope(x), dtype)
