"""What autograd is told about the selective state space operators: caches that change in place, and
derivatives that there are none of."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda")


def _conv(gen, b=2, L=5, d=8, k=4):
    x, cache = torch.randn(b, L, d, generator=gen, device=DEV), torch.randn(b, k - 1, d, generator=gen, device=DEV)
    return x, cache, torch.randn(d, k, generator=gen, device=DEV)


def _scan(gen, b=2, L=5, d=8, n=16):
    u, delta = (torch.randn(b, L, d, generator=gen, device=DEV) for _ in range(2))
    B, C = (torch.randn(b, L, n, generator=gen, device=DEV) for _ in range(2))
    return [u, delta, -torch.rand(d, n, generator=gen, device=DEV), B, C], torch.randn(b, d, n, generator=gen, device=DEV)


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("op", ["conv", "scan"])
def test_a_step_on_a_saved_cache_is_noticed(op, apart):
    """Sequences that started from a cache, then a step that changes it, then the backward: it needs
    the cache as it was, and raises.  A step into another tensor leaves the cache alone."""
    from visionhope_b200.ssm_core import short_conv, short_conv_step, ssm_scan, ssm_scan_step

    gen = torch.Generator(device=DEV).manual_seed(1)
    if op == "conv":
        x, cache, w = _conv(gen)
        w.requires_grad_()
        y = short_conv(x, w, initial_state=cache, activation="silu")
        out = torch.empty_like(cache) if apart else None
        with torch.no_grad():
            short_conv_step(x[:, 0], cache, w, state_out=out)
    else:
        (u, delta, A, B, C), cache = _scan(gen)
        w = A.requires_grad_()
        y = ssm_scan(u, delta, A, B, C, initial_state=cache, delta_softplus=True)
        out = torch.empty_like(cache) if apart else None
        with torch.no_grad():
            ssm_scan_step(u[:, 0], delta[:, 0], A, B[:, 0], C[:, 0], cache, state_out=out)
    if apart:
        y.sum().backward()
        assert torch.isfinite(w.grad).all()
        assert out._version > 0 and cache._version == 0
    else:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


@pytest.mark.parametrize("inside", [False, True])
def test_steps_on_a_cache_of_inference_mode(inside):
    """Inference tensors have no version to move; steps on them run, in and out of that mode."""
    from visionhope_b200.ssm_core import short_conv_step, ssm_scan_step

    gen = torch.Generator(device=DEV).manual_seed(2)
    with torch.inference_mode():
        x, cache, w = _conv(gen)
        (u, delta, A, B, C), state = _scan(gen)
    before = cache.clone(), state.clone()
    with torch.inference_mode(inside):
        short_conv_step(x[:, 0], cache, w)
        ssm_scan_step(u[:, 0], delta[:, 0].abs(), A, B[:, 0], C[:, 0], state)
    assert torch.equal(cache[:, :-1], before[0][:, 1:]) and torch.equal(cache[:, -1], x[:, 0])
    assert not torch.equal(state, before[1])


def test_steps_have_no_backward():
    """Inputs or parameters that require gradients: the step runs, and a backward through its y raises
    in place of leaving them out.  A cache that requires gradients is refused and stays as it is."""
    from visionhope_b200.ssm_core import short_conv_step, ssm_scan_step

    gen = torch.Generator(device=DEV).manual_seed(3)
    x, cache, w = _conv(gen)
    (u, delta, A, B, C), state = _scan(gen)
    bias = torch.zeros(8, device=DEV)
    conv = dict(x=x[:, 0], state=cache, weight=w, bias=bias)
    scan = dict(u=u[:, 0], delta=delta[:, 0].abs(), A=A, B=B[:, 0], C=C[:, 0], state=state, D=bias, z=x[:, 0], delta_bias=bias)
    for step, args in ((short_conv_step, conv), (ssm_scan_step, scan)):
        plain = {k: t.clone() for k, t in args.items()}
        want = step(**plain)
        assert not want.requires_grad
        for name in args:
            given = {k: t.clone() for k, t in args.items()}
            given[name].requires_grad_()
            if name == "state":
                with pytest.raises(RuntimeError, match="cache requires gradients"):
                    step(**given)
                assert torch.equal(given["state"], args["state"])
                out = torch.zeros_like(args["state"])  # read only: as any other input
                y = step(**given, state_out=out)
                assert torch.equal(out, plain["state"])
            else:
                y = step(**given)
                assert torch.equal(given["state"], plain["state"])
            assert torch.equal(y, want)
            with pytest.raises(RuntimeError, match="not differentiable"):
                y.sum().backward()
            given["state"] = args["state"].clone().requires_grad_()
            with torch.no_grad():
                y = step(**given)
            assert not y.requires_grad and torch.equal(given["state"], plain["state"])


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(grad):
    """There is no forward-mode rule: a tangent raises instead of vanishing, under no_grad too (which
    does not switch forward mode off).  Inputs without one run inside a level as outside."""
    import torch.autograd.forward_ad as fwd

    from visionhope_b200.ssm_core import short_conv, short_conv_step, ssm_scan, ssm_scan_step

    gen = torch.Generator(device=DEV).manual_seed(4)
    x, cache, w = _conv(gen)
    (u, delta, A, B, C), state = _scan(gen)
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        for run, args in ((short_conv, [x, w, torch.zeros(8, device=DEV)]), (ssm_scan, [u, delta, A, B, C]),
                              (short_conv_step, [x[:, 0], cache, w]),
                              (ssm_scan_step, [u[:, 0], delta[:, 0], A, B[:, 0], C[:, 0], state])):
            run(*args)
            for i in range(len(args)):
                dual = list(args)
                dual[i] = fwd.make_dual(args[i].clone(), torch.ones_like(args[i]))
                with pytest.raises((NotImplementedError, RuntimeError), match="forward mode|not differentiable"):
                    run(*dual)


def test_function_transforms_are_refused():
    """torch.func's tangents and batch dimensions do not reach the kernels as plain memory either."""
    from visionhope_b200.ssm_core import short_conv

    gen = torch.Generator(device=DEV).manual_seed(5)
    x, _, w = _conv(gen)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(lambda t: short_conv(t, w), (x,), (torch.ones_like(x),))
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.vmap(lambda t: short_conv(t, w))(torch.stack([x, x]))


@pytest.mark.parametrize("shape", [(2, 5, 0), (2, 0, 8), (0, 5, 8)])
def test_empty_inputs_get_zero_gradients(shape):
    """Without channels, tokens or sequences every gradient that has elements is zero (an initial
    state's is the final one's).  Blocks full of NaN are freed first: gradients left unwritten would
    show them."""
    from visionhope_b200.ssm_core import short_conv, ssm_scan

    b, L, d = shape
    n, k = 16, 4
    u, delta = (torch.ones(shape, device=DEV, requires_grad=True) for _ in range(2))
    B, C = (torch.ones(b, L, n, device=DEV, requires_grad=True) for _ in range(2))
    A, D = torch.ones(d, n, device=DEV, requires_grad=True), torch.ones(d, device=DEV, requires_grad=True)
    w, h0 = torch.ones(d, k, device=DEV, requires_grad=True), torch.ones(b, d, n, device=DEV, requires_grad=True)
    x, s0 = torch.ones(shape, device=DEV, requires_grad=True), torch.ones(b, k - 1, d, device=DEV, requires_grad=True)
    y, h = ssm_scan(u, delta, A, B, C, D, initial_state=h0, return_final_state=True)
    c, s = short_conv(x, w, initial_state=s0, return_final_state=True)
    for t in [torch.full((m,), float("nan"), device=DEV) for m in (b * L * n, d * n, d, d * k, b * d * n) for _ in range(8)]:
        del t
    scan_in, conv_in = (u, delta, A, B, C, D), (x, w)
    grads = torch.autograd.grad([y, h], [*scan_in, h0], [torch.ones_like(y), torch.full_like(h, 2.0)])
    grads = [*grads, *torch.autograd.grad([c, s], [*conv_in, s0], [torch.ones_like(c), torch.full_like(s, 2.0)])]
    for g, t in zip(grads, [*scan_in, h0, *conv_in, s0]):
        assert g.shape == t.shape and (g == (2.0 if t is h0 or t is s0 else 0.0)).all()
