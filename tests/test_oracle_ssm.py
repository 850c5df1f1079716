"""The selective state space oracle (oracle/ssm.py) on the CPU: its gradients against finite
differences, its convolution and scan against closed forms, and the operators' argument checks
that need no GPU."""
import ctypes

import pytest
import torch
import torch.nn.functional as F

from oracle import ssm


def _leaf(*shape, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * scale).requires_grad_()


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("offsets", [None, [0, 0, 1, 5]])
def test_scan_gradients_against_differences(reverse, offsets):
    lead = (2, 5) if offsets is None else (5,)
    count, d, n, groups = (2 if offsets is None else 3), 4, 3, 2
    u, delta, z = (_leaf(*lead, d, seed=i) for i in range(3))
    B, C = (_leaf(*lead, groups, n, seed=3 + i) for i in range(2))
    A = (-_leaf(d, n, seed=6).detach().abs() - 0.1).requires_grad_()
    D, bias, h0 = _leaf(d, seed=7), _leaf(d, seed=8), _leaf(count, d, n, seed=9)

    def f(u, delta, A, B, C, D, z, bias, h0):
        return ssm.ssm_scan(u, delta, A, B, C, D, z=z, delta_bias=bias, delta_softplus=True, initial_state=h0,
                            offsets=offsets, reverse=reverse)

    assert torch.autograd.gradcheck(f, (u, delta, A, B, C, D, z, bias, h0))


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("offsets", [None, [0, 0, 1, 5]])
def test_conv_gradients_against_differences(reverse, offsets):
    lead = (2, 5) if offsets is None else (5,)
    count, d, k = (2 if offsets is None else 3), 3, 4
    x, w, b, s0 = _leaf(*lead, d, seed=1), _leaf(d, k, seed=2), _leaf(d, seed=3), _leaf(count, k - 1, d, seed=4)

    def f(x, w, b, s0):
        return ssm.short_conv(x, w, b, activation="silu", initial_state=s0, offsets=offsets, reverse=reverse)

    assert torch.autograd.gradcheck(f, (x, w, b, s0))


def test_conv_is_a_padded_grouped_convolution():
    x, w, b = _leaf(2, 11, 6, seed=1).detach(), _leaf(6, 4, seed=2).detach(), _leaf(6, seed=3).detach()
    want = F.conv1d(F.pad(x.transpose(1, 2), (3, 0)), w[:, None], b, groups=6).transpose(1, 2)
    y, state = ssm.short_conv(x, w, b)
    assert torch.allclose(y, want, atol=1e-12)
    assert torch.equal(state, x[:, -3:])


def test_scan_with_constant_steps_is_a_geometric_sum():
    """Constant step s, input 1, B = C = 1: h_t = s (1 - q^t) / (1 - q), q = exp(s A)."""
    L, s, a = 9, 0.3, -0.7
    one = torch.ones(1, L, 1, dtype=torch.float64)
    y, h = ssm.ssm_scan(one, s * one, torch.full((1, 1), a, dtype=torch.float64), one, one)
    q = torch.exp(torch.tensor(s * a, dtype=torch.float64))
    t = torch.arange(1, L + 1, dtype=torch.float64)
    assert torch.allclose(y[0, :, 0], s * (1 - q ** t) / (1 - q), atol=1e-12)
    assert torch.allclose(h[0, 0, 0], y[0, -1, 0], atol=1e-12)


def _fake():
    buf = ctypes.create_string_buffer(1 << 16)
    return (ctypes.addressof(buf) + 255) & ~255, buf


def _err(lib):
    return lib.vh_last_error().decode()


def _conv_args(L, p, **kw):
    a = dict(x=p, x_batch_stride=64, x_token_stride=8, weight=p, bias=p, initial_state=None, y=p, final_state=None,
             seq_offsets=None, length=8, dtype=1, activation=1, taps=4, batch=2, channels=8, reverse=0)
    a.update(kw)
    return L.VhShortConvArgs(**a)


def _scan_args(L, p, **kw):
    a = dict(u=p, delta=p, z=p, b=p, c=p, u_batch_stride=64, u_token_stride=8, delta_batch_stride=64,
             delta_token_stride=8, z_batch_stride=64, z_token_stride=8, b_batch_stride=128, b_token_stride=16,
             b_group_stride=0, c_batch_stride=128, c_token_stride=16, c_group_stride=0, a=p, d_skip=p, delta_bias=p,
             initial_state=None, y=p, final_state=None, checkpoints=None, seq_offsets=None, length=8, dtype=1, batch=2,
             channels=8, states=16, groups=1, delta_softplus=1, reverse=0)
    a.update(kw)
    return L.VhSsmScanArgs(**a)


def test_struct_layouts_match_the_header():
    from tests.test_abi import _c_layout
    from visionhope_b200 import _lib

    for cls, name in ((_lib.VhShortConvArgs, "vh_short_conv_args"), (_lib.VhSsmScanArgs, "vh_ssm_scan_args"),
                      (_lib.VhSsmScanBwdArgs, "vh_ssm_scan_bwd_args")):
        fields = [f[0] for f in cls._fields_]
        size, offsets = _c_layout(name, fields)
        assert size == ctypes.sizeof(cls)
        assert offsets == [getattr(cls, f).offset for f in fields]


def test_packed_structs_match_their_mirrors():
    from visionhope_b200 import _lib
    from visionhope_b200.ssm_core import conv, scan

    def packed(cls):
        """(offset, size) of every value that ``struct`` packs, from the mirror's fields."""
        return [(getattr(cls, f[0]).offset, ctypes.sizeof(f[1])) for f in cls._fields_]

    def values(fmt, count, size):
        ones = [fmt.unpack(bytes(i) + b"\xff" + bytes(size - i - 1)) for i in range(size)]
        return [(min(i for i in range(size) if ones[i][k]), sum(1 for i in range(size) if ones[i][k])) for k in range(count)]

    for cls, fmt in ((_lib.VhShortConvArgs, conv._ARGS), (_lib.VhSsmScanArgs, scan._ARGS)):
        assert fmt.size == ctypes.sizeof(cls)
        assert values(fmt, len(cls._fields_), fmt.size) == packed(cls)
    assert scan._ARGS.size + scan._GRADS.size == ctypes.sizeof(_lib.VhSsmScanBwdArgs)


@pytest.mark.parametrize("change,code,text", [
    (dict(x=None), -1, "null"), (dict(dtype=7), -3, "dtype"), (dict(taps=1), -2, "taps"), (dict(taps=9), -2, "taps"),
    (dict(activation=2), -1, "activation"), (dict(batch=0), -2, "positive"), (dict(channels=-4), -2, "positive"),
    (dict(length=-1), -2, "length"), (dict(length=1 << 31), -6, "tokens")])
def test_conv_entry_points_refuse(change, code, text):
    from visionhope_b200 import _lib

    lib, (p, keep) = _lib.load(), _fake()
    a = _conv_args(_lib, p, **change)
    assert lib.vh_short_conv_fwd(ctypes.byref(a), None) == code
    assert text in _err(lib)
    assert lib.vh_short_conv_bwd(ctypes.byref(a), p, None, p, p, p, None, p, 1 << 30, None) == code


def test_conv_refuses_misaligned_and_short_workspace():
    from visionhope_b200 import _lib

    lib, (p, keep) = _lib.load(), _fake()
    assert lib.vh_short_conv_fwd(ctypes.byref(_conv_args(_lib, p, x=p + 1)), None) == -5
    a = _conv_args(_lib, p)
    need = lib.vh_short_conv_bwd_workspace_bytes(ctypes.byref(a))
    assert need > 0
    assert lib.vh_short_conv_bwd(ctypes.byref(a), p, None, p, p, p, None, p, need - 4, None) == -1
    assert "workspace" in _err(lib)
    assert lib.vh_short_conv_fwd(None, None) == -1
    assert lib.vh_short_conv_step(p, 8, 1, p, p, 1, None, p, None, 2, p, 2, 8, 4, None) == -1
    assert lib.vh_short_conv_step(p, 8, 1, p, p, 1, p, p, None, 1, p, 2, 8, 4, None) == -2
    assert "slots" in _err(lib)


@pytest.mark.parametrize("change,code,text", [
    (dict(u=None), -1, "null"), (dict(a=None), -1, "null"), (dict(dtype=3), -3, "dtype"),
    (dict(states=12), -2, "states"), (dict(groups=3), -2, "multiple"), (dict(groups=0), -2, "positive"),
    (dict(batch=-1), -2, "positive"), (dict(length=-1), -2, "length"), (dict(length=1 << 31), -6, "tokens")])
def test_scan_entry_points_refuse(change, code, text):
    from visionhope_b200 import _lib

    lib, (p, keep) = _lib.load(), _fake()
    a = _scan_args(_lib, p, **change)
    assert lib.vh_ssm_scan_fwd(ctypes.byref(a), p, 1 << 40, None) == code
    assert text in _err(lib)
    if "length" not in change:
        assert lib.vh_ssm_scan_step(ctypes.byref(a), p, p, None, 4, None) == code


def test_scan_backward_refuses():
    from visionhope_b200 import _lib

    lib, (p, keep) = _lib.load(), _fake()

    def bwd(**kw):
        a = dict(fwd=_scan_args(_lib, p, checkpoints=p), grad_y=p, grad_final=None, grad_u=p, grad_delta=p, grad_z=p,
                 grad_b=p, grad_c=p, grad_a=p, grad_d_skip=p, grad_delta_bias=p, grad_initial=None)
        a.update(kw)
        return _lib.VhSsmScanBwdArgs(**a)

    need = lib.vh_ssm_scan_bwd_workspace_bytes(ctypes.byref(bwd()))
    assert need > 0
    assert lib.vh_ssm_scan_bwd(ctypes.byref(bwd()), p, need - 4, None) == -1
    assert "workspace" in _err(lib)
    assert lib.vh_ssm_scan_bwd(ctypes.byref(bwd(fwd=_scan_args(_lib, p))), p, need, None) == -1
    assert "checkpoints" in _err(lib)
    assert lib.vh_ssm_scan_bwd(ctypes.byref(bwd(grad_z=None)), p, need, None) == -1
    assert lib.vh_ssm_scan_bwd(ctypes.byref(bwd(grad_u=p + 1)), p, need, None) == -5
    assert lib.vh_ssm_scan_step(ctypes.byref(_scan_args(_lib, p)), p, p, None, 1, None) == -2
    assert "slots" in _err(lib)


def test_operators_refuse_cpu_tensors():
    from visionhope_b200.ssm_core import short_conv, short_conv_step, ssm_scan, ssm_scan_step

    x, w = torch.zeros(1, 4, 8), torch.zeros(8, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        short_conv(x, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        short_conv_step(x[:, 0], torch.zeros(1, 3, 8), w)
    A, B = torch.zeros(8, 16), torch.zeros(1, 4, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ssm_scan(x, x, A, B, B)
    with pytest.raises(RuntimeError, match="CUDA"):
        ssm_scan_step(x[:, 0], x[:, 0], A, B[:, 0], B[:, 0], torch.zeros(1, 8, 16))
    with pytest.raises(ValueError, match="activation"):
        short_conv(x, w, activation="relu")
