"""Selective scan over token rows (``vh_ssm_scan_fwd``, ``_bwd``, ``_step``)."""
import ctypes

import torch

from .. import _lib
from . import _args

STATES = (4, 8, 16, 32, 64)


def _grouped(t, lead, n, name, like):
    """B or C as [..., groups, states] rows; a tensor without a group dim has one group."""
    if t.dim() == len(lead) + 1:
        t = t.unsqueeze(-2)
    if t.dim() != len(lead) + 2 or tuple(t.shape[:-2]) != lead or t.shape[-1] != n:
        raise ValueError(f"{name} must be [{', '.join(map(str, lead))}, (groups,) {n}], got {tuple(t.shape)}")
    return _args.rows(t, tuple(t.shape), name, like)


class _Call:
    """One call's checked arguments: the C struct, and the tensors that it points to."""

    def __init__(self, u, delta, A, B, C, D, z, delta_bias, softplus, initial, offsets, reverse, one_token=False):
        if one_token:
            _lib.ensure_device(u)
            _lib.dtype_code(u.dtype)
            if u.dim() != 2:
                raise ValueError(f"u must be [batch, channels], got {tuple(u.shape)}")
            count, length = u.shape[0], 1
        else:
            count, length, offsets = _args.sequences(u, offsets, "u")
        shape, d = tuple(u.shape), u.shape[-1]
        if A.dim() != 2 or A.shape[0] != d:
            raise ValueError(f"A must be [{d}, states], got {tuple(A.shape)}")
        n = A.shape[1]
        if n not in STATES:
            raise ValueError(f"ssm_scan takes {', '.join(map(str, STATES))} states, got {n}")
        dev = u.device
        u = _args.rows(u, shape, "u", u)
        delta = _args.rows(delta, shape, "delta", u)
        z = _args.rows(z, shape, "z", u)
        B, C = _grouped(B, shape[:-1], n, "B", u), _grouped(C, shape[:-1], n, "C", u)
        groups = B.shape[-2]
        if C.shape[-2] != groups or groups == 0 or d % groups:
            raise ValueError(f"B and C must have the same number of groups, a divisor of {d}; got {groups} and "
                             f"{C.shape[-2]}")
        A = _args.fp32(A, (d, n), "A", dev)
        D = _args.fp32(D, (d,), "D", dev)
        delta_bias = _args.fp32(delta_bias, (d,), "delta_bias", dev)
        initial = _args.state(initial, (count, d, n), "initial_state", torch.float32, dev)
        if initial is not None and initial.requires_grad:
            initial = initial.detach()
        self.kept = u, delta, A, B, C, D, z, delta_bias, initial, offsets
        self.state_shape = count, d, n
        ut = u.stride(-2)
        self.args = _lib.VhSsmScanArgs(
            u.data_ptr(), delta.data_ptr(), _lib.ptr(z), B.data_ptr(), C.data_ptr(),
            u.stride(0), ut, delta.stride(0), delta.stride(-2),
            0 if z is None else z.stride(0), 0 if z is None else z.stride(-2),
            B.stride(0), 0 if one_token else B.stride(-3), B.stride(-2) if groups > 1 else 0,
            C.stride(0), 0 if one_token else C.stride(-3), C.stride(-2) if groups > 1 else 0,
            A.data_ptr(), _lib.ptr(D), _lib.ptr(delta_bias), _lib.ptr(initial), None, None, None, _lib.ptr(offsets),
            length, _lib.DTYPES[u.dtype], count, d, n, groups, int(bool(softplus)), int(bool(reverse)))

    def forward(self, want_final, want_checkpoints=False):
        u, initial = self.kept[0], self.kept[8]
        dev = u.device
        y = torch.empty(u.shape, dtype=u.dtype, device=dev)
        final = torch.empty(self.state_shape, dtype=torch.float32, device=dev) if want_final else None
        if y.numel() == 0:  # no tokens: every state leaves as it entered
            if final is not None:
                final.copy_(initial) if initial is not None else final.zero_()
            return y, final, None
        lib, a = _lib.load(), self.args
        ck = None
        if want_checkpoints:
            ck = _args.workspace(lib.vh_ssm_scan_checkpoint_bytes(ctypes.byref(a)), dev)
        a.y, a.final_state, a.checkpoints = y.data_ptr(), _lib.ptr(final), _lib.ptr(ck)
        nbytes = lib.vh_ssm_scan_fwd_workspace_bytes(ctypes.byref(a))
        ws = _args.workspace(nbytes, dev) if nbytes else None
        _lib.check(lib.vh_ssm_scan_fwd(ctypes.byref(a), _lib.ptr(ws), nbytes, _lib.stream_handle(dev)), "vh_ssm_scan_fwd")
        return y, final, ck

    def backward(self, dy, dfinal, ck, want_initial):
        u, delta, A, B, C, D, z, delta_bias, _, _ = self.kept
        dev = u.device
        like = lambda t: None if t is None else torch.empty(t.shape, dtype=t.dtype, device=dev)  # noqa: E731
        du, dd, dz, dB, dC, dA, dD, dbias = (like(t) for t in (u, delta, z, B, C, A, D, delta_bias))
        di = torch.empty(self.state_shape, dtype=torch.float32, device=dev) if want_initial else None
        if u.numel() == 0:
            for t in (dA, dD, dbias):
                if t is not None:
                    t.zero_()
            if di is not None:
                di.copy_(dfinal) if dfinal is not None else di.zero_()
            return du, dd, dA, dB, dC, dD, dz, dbias, di
        lib = _lib.load()
        self.args.checkpoints = ck.data_ptr()
        args = _lib.VhSsmScanBwdArgs(self.args, dy.data_ptr(), _lib.ptr(dfinal), du.data_ptr(), dd.data_ptr(),
                                     _lib.ptr(dz), dB.data_ptr(), dC.data_ptr(), dA.data_ptr(), _lib.ptr(dD),
                                     _lib.ptr(dbias), _lib.ptr(di))
        ws = _args.workspace(lib.vh_ssm_scan_bwd_workspace_bytes(ctypes.byref(args)), dev)
        _lib.check(lib.vh_ssm_scan_bwd(ctypes.byref(args), ws.data_ptr(), ws.numel(), _lib.stream_handle(dev)),
                   "vh_ssm_scan_bwd")
        return du, dd, dA, dB, dC, dD, dz, dbias, di


class _SsmScanFunction(torch.autograd.Function):
    """Saves the inputs and the state before every 32nd token (2 bytes per element at 16 states)."""

    @staticmethod
    def forward(ctx, u, delta, A, B, C, D, z, delta_bias, initial, softplus, want_final, offsets, reverse):
        call = _Call(u, delta, A, B, C, D, z, delta_bias, softplus, initial, offsets, reverse)
        y, final, ck = call.forward(want_final, want_checkpoints=True)
        ctx.save_for_backward(u, delta, A, B, C, D, z, delta_bias, initial, call.kept[9], ck)
        ctx.options = softplus, reverse
        ctx.set_materialize_grads(False)
        return (y, final) if want_final else y

    @staticmethod
    @_lib.on_input_device
    def backward(ctx, dy, dfinal=None):
        *inputs, offsets, ck = ctx.saved_tensors
        u, delta, A, B, C, D, z, delta_bias, initial = inputs
        softplus, reverse = ctx.options
        if dy is None and dfinal is None:
            return (None,) * 13
        call = _Call(u, delta, A, B, C, D, z, delta_bias, softplus, initial, offsets, reverse)
        dy = torch.zeros(u.shape, dtype=u.dtype, device=u.device) if dy is None else _args.grad_rows(dy)
        dfinal = None if dfinal is None else _args.grad_rows(dfinal)
        grads = call.backward(dy, dfinal, ck, initial is not None and ctx.needs_input_grad[8])
        grads = [None if g is None else g.view(t.shape).to(t.dtype) for g, t in zip(grads, inputs)]
        return (*grads, None, None, None, None)


@_lib.on_input_device
def ssm_scan(u, delta, A, B, C, D=None, *, z=None, delta_bias=None, delta_softplus=False, initial_state=None,
             return_final_state=False, seq_offsets=None, reverse=False):
    """The selective scan: with ``s_t = softplus(delta_t + delta_bias)`` (the sum itself without
    ``delta_softplus``), per channel d and state n

        h_t = exp(s_t A[d, n]) h_{t-1} + s_t u_t B_t[n]
        y_t = (sum_n C_t[n] h_t + D[d] u_t) * silu(z_t)

    u, delta, z: [B, L, C] of one dtype (fp32, bf16 or fp16; any batch and token strides), or
    packed [T, C] with ``seq_offsets`` (as :func:`short_conv`).  B, C: [B, L, states] or [B, L,
    groups, states] of that dtype (packed: without the batch); channel d uses group d // (C /
    groups).  A: [C, states], 4, 8, 16, 32 or 64 states; D, delta_bias: [C].  initial_state: fp32
    [B, C, states] (zeros when None).  reverse reads every sequence from its last token to its
    first.  The state is fp32 throughout; y, of u's dtype, is rounded once.  Returns y, or (y,
    final_state) with ``return_final_state``.  Differentiable in every tensor, through y and the
    final state; the sums of the backward run in a fixed order."""
    tensors = (u, delta, A, B, C, D, z, delta_bias, initial_state)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return _SsmScanFunction.apply(*tensors, bool(delta_softplus), bool(return_final_state), seq_offsets,
                                      bool(reverse))
    call = _Call(*tensors[:8], delta_softplus, initial_state, seq_offsets, reverse)
    y, final, _ = call.forward(return_final_state)
    return (y, final) if return_final_state else y


@torch.no_grad()
@_lib.on_input_device
def ssm_scan_step(u, delta, A, B, C, state, D=None, *, z=None, delta_bias=None, delta_softplus=False, slots=None,
                  state_out=None):
    """One token of ``B`` cached streams: u, delta, z [B, C]; B, C [B, (groups,) states]; state fp32
    [slots, C, states], advanced in place (or into ``state_out``).  slots: as
    :func:`short_conv_step`.  Returns y [B, C]."""
    call = _Call(u, delta, A, B, C, D, z, delta_bias, delta_softplus, None, None, False, one_token=True)
    u = call.kept[0]
    b, d, n = call.state_shape
    slots = _args.slot_index(slots, b, u.device)
    state, state_out = _args.cache(state, state_out, (d, n), b, slots, torch.float32, u.device)
    y = torch.empty((b, d), dtype=u.dtype, device=u.device)
    if y.numel() == 0:
        return y
    call.args.y = y.data_ptr()
    _lib.check(_lib.load().vh_ssm_scan_step(ctypes.byref(call.args), state.data_ptr(), state_out.data_ptr(),
                                            _lib.ptr(slots), state.shape[0], _lib.stream_handle(u.device)),
               "vh_ssm_scan_step")
    return y
