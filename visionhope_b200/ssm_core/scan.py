"""Selective scan over token rows (``vh_ssm_scan_fwd``, ``_bwd``, ``_step``)."""
import struct

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from . import _args
from ._args import ptr

STATES = (4, 8, 16, 32, 64)
_ARGS = struct.Struct("5Q12q8Qq7i4x")  # vh_ssm_scan_args
_GRADS = struct.Struct("11Q")          # the rest of vh_ssm_scan_bwd_args
_NONE = (0, 0, 0)


def _grouped(t, lead, n, name, dtype, device):
    """B or C as [..., groups, states] rows, and (groups, batch, token and group strides); a tensor
    without a group dim has one group."""
    shape, ranks = t.shape, len(lead) + 1
    if len(shape) not in (ranks, ranks + 1) or shape[:ranks - 1] != lead or shape[-1] != n:
        raise ValueError(f"{name} must be [{', '.join(map(str, lead))}, (groups,) {n}], got {tuple(shape)}")
    t = _args.rows(t, shape, name, dtype, device)
    stride = t.stride()
    if len(shape) == ranks:
        return t, 1, (stride[0], stride[-2], 0)
    return t, shape[-2], (stride[0], stride[-3], stride[-2])


class _Call:
    """One call's checked arguments; ``args`` packs them with the output pointers."""

    __slots__ = ("u", "delta", "A", "B", "C", "D", "z", "bias", "initial", "offsets", "state_shape", "head", "tail")

    def __init__(self, u, delta, A, B, C, D, z, delta_bias, softplus, initial, offsets, reverse, one_token=False):
        if one_token:
            _lib.ensure_device(u)
            if u.dim() != 2:
                raise ValueError(f"u must be [batch, channels], got {tuple(u.shape)}")
            count, length = u.shape[0], 1
        else:
            count, length, offsets = _args.sequences(u, offsets, "u")
        shape, device, dtype = u.shape, u.device, u.dtype
        code = _lib.dtype_code(dtype)
        d, lead = shape[-1], shape[:-1]
        if A.dim() != 2 or A.shape[0] != d:
            raise ValueError(f"A must be [{d}, states], got {tuple(A.shape)}")
        n = A.shape[1]
        if n not in STATES:
            raise ValueError(f"ssm_scan takes {', '.join(map(str, STATES))} states, got {n}")
        self.u = u = _args.rows(u, shape, "u", dtype, device)
        self.delta = delta = _args.rows(delta, shape, "delta", dtype, device)
        self.z = z = _args.rows(z, shape, "z", dtype, device)
        self.B, groups, bs = _grouped(B, lead, n, "B", dtype, device)
        self.C, cgroups, cs = _grouped(C, lead, n, "C", dtype, device)
        if cgroups != groups or groups == 0 or d % groups:
            raise ValueError(f"B and C must have the same number of groups, a divisor of {d}; got {groups} and {cgroups}")
        self.A = A = _args.fp32(A, (d, n), "A", device)
        self.D = D = _args.fp32(D, (d,), "D", device)
        self.bias = bias = _args.fp32(delta_bias, (d,), "delta_bias", device)
        self.state_shape = count, d, n
        self.initial = _args.state(initial, self.state_shape, "initial_state", torch.float32, device)
        self.offsets = offsets
        us, ds = u.stride(), delta.stride()
        zs = _NONE if z is None else z.stride()
        self.head = (u.data_ptr(), delta.data_ptr(), ptr(z), self.B.data_ptr(), self.C.data_ptr(),
                     us[0], us[-2], ds[0], ds[-2], zs[0], zs[-2], *bs, *cs,
                     A.data_ptr(), ptr(D), ptr(bias), ptr(self.initial))
        self.tail = (ptr(offsets), length, code, count, d, n, groups, 1 if softplus else 0, 1 if reverse else 0)

    def args(self, y=0, final=0, checkpoints=0):
        return _ARGS.pack(*self.head, y, final, checkpoints, *self.tail)

    def forward(self, want_final, want_checkpoints=False):
        u, initial = self.u, self.initial
        dev = u.device
        y = torch.empty(u.shape, dtype=u.dtype, device=dev)
        final = torch.empty(self.state_shape, dtype=torch.float32, device=dev) if want_final else None
        if y.numel() == 0:  # no tokens: every state leaves as it entered
            if final is not None:
                final.copy_(initial.detach()) if initial is not None else final.zero_()
            return y, final, None
        lib = _lib.load()
        args = self.args(y.data_ptr(), ptr(final))
        nbytes = lib.vh_ssm_scan_fwd_workspace_bytes(args)
        ws = _args.workspace(nbytes, dev) if nbytes else None
        ck = None
        if want_checkpoints:
            ck = _args.workspace(lib.vh_ssm_scan_checkpoint_bytes(args), dev)
            args = self.args(y.data_ptr(), ptr(final), ck.data_ptr())
        _lib.check(lib.vh_ssm_scan_fwd(args, ptr(ws), nbytes, _lib.stream_handle(dev)), "vh_ssm_scan_fwd")
        return y, final, ck

    def backward(self, dy, dfinal, ck, want_initial):
        u, dev, dtype = self.u, self.u.device, self.u.dtype

        def like(t, kind):
            return None if t is None else torch.empty(t.shape, dtype=kind, device=dev)

        du, dd, dz, dB, dC = (like(t, dtype) for t in (u, self.delta, self.z, self.B, self.C))
        dA, dD, dbias = (like(t, torch.float32) for t in (self.A, self.D, self.bias))
        di = torch.empty(self.state_shape, dtype=torch.float32, device=dev) if want_initial else None
        if u.numel() == 0:  # without channels B and C still have elements
            for t in (dA, dB, dC, dD, dbias):
                if t is not None:
                    t.zero_()
            if di is not None:
                di.copy_(dfinal) if dfinal is not None else di.zero_()
            return du, dd, dA, dB, dC, dD, dz, dbias, di
        lib = _lib.load()
        args = self.args(checkpoints=ck.data_ptr()) + _GRADS.pack(
            dy.data_ptr(), ptr(dfinal), du.data_ptr(), dd.data_ptr(), ptr(dz), dB.data_ptr(), dC.data_ptr(),
            dA.data_ptr(), ptr(dD), ptr(dbias), ptr(di))
        ws = _args.workspace(lib.vh_ssm_scan_bwd_workspace_bytes(args), dev)
        _lib.check(lib.vh_ssm_scan_bwd(args, ws.data_ptr(), ws.numel(), _lib.stream_handle(dev)), "vh_ssm_scan_bwd")
        return du, dd, dA, dB, dC, dD, dz, dbias, di


class _SsmScanFunction(torch.autograd.Function):
    """Saves the inputs and the state before every 32nd token (states / 8 bytes per element of u); the
    backward's workspace takes states^2 / 64 bytes per element."""

    @staticmethod
    def forward(ctx, u, delta, A, B, C, D, z, delta_bias, initial, softplus, want_final, offsets, reverse):
        call = _Call(u, delta, A, B, C, D, z, delta_bias, softplus, initial, offsets, reverse)
        y, final, ck = call.forward(want_final, want_checkpoints=True)
        ctx.save_for_backward(u, delta, A, B, C, D, z, delta_bias, initial, call.offsets, ck)
        ctx.options = softplus, reverse
        ctx.set_materialize_grads(False)
        return (y, final) if want_final else y

    @staticmethod
    @once_differentiable
    @_lib.on_input_device
    def backward(ctx, dy, dfinal=None):
        if dy is None and dfinal is None:
            return (None,) * 13
        *inputs, offsets, ck = ctx.saved_tensors
        u, delta, A, B, C, D, z, delta_bias, initial = inputs
        softplus, reverse = ctx.options
        call = _Call(u, delta, A, B, C, D, z, delta_bias, softplus, initial, offsets, reverse)
        dy = torch.zeros(u.shape, dtype=u.dtype, device=u.device) if dy is None else _args.grad_rows(dy)
        dfinal = None if dfinal is None else _args.grad_rows(dfinal)
        grads = call.backward(dy, dfinal, ck, initial is not None and ctx.needs_input_grad[8])
        return (*map(_args.grad_like, grads, inputs), None, None, None, None)


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
    final state; the sums of the backward run in a fixed order.  Steps times A are meant to be at most 0,
    so that states decay: where they grow, a state other than zero may overflow sooner than token by
    token, because long chains are computed in segments."""
    tensors = (u, delta, A, B, C, D, z, delta_bias, initial_state)
    if _args.tracked(tensors):
        return _SsmScanFunction.apply(*tensors, bool(delta_softplus), bool(return_final_state), seq_offsets,
                                      bool(reverse))
    call = _Call(*tensors[:8], delta_softplus, initial_state, seq_offsets, reverse)
    y, final, _ = call.forward(return_final_state)
    return (y, final) if return_final_state else y


@_lib.on_input_device
def ssm_scan_step(u, delta, A, B, C, state, D=None, *, z=None, delta_bias=None, delta_softplus=False, slots=None,
                  state_out=None):
    """One token of ``B`` cached streams: u, delta, z [B, C]; B, C [B, (groups,) states]; state fp32
    [slots, C, states] and 16-byte aligned, advanced in place (or into ``state_out``).  slots: as
    :func:`short_conv_step`.  Returns y [B, C].  Not differentiable, as :func:`short_conv_step`."""
    tensors = u, delta, A, B, C, state, D, z, delta_bias, state_out
    if A.data_ptr() % 16:  # a view into a larger buffer: the kernel reads four rates at a time
        A = A.detach().clone()
    marked = _args.step_derivatives("ssm_scan_step", tensors, state, state_out)
    call = _Call(u, delta, A, B, C, D, z, delta_bias, delta_softplus, None, None, False, one_token=True)
    device = u.device
    b, d, n = call.state_shape
    slots = _args.slot_index(slots, b, device)
    state, state_out = _args.cache(state, state_out, (d, n), b, slots, torch.float32, device)
    y = torch.empty_like(u, memory_format=torch.contiguous_format)
    if b * d == 0:
        return y
    _lib.check(_lib.load().vh_ssm_scan_step(call.args(y.data_ptr()), state.data_ptr(), state_out.data_ptr(),
                                            ptr(slots), state.shape[0], _lib.stream_handle(device)), "vh_ssm_scan_step")
    _args.wrote(state_out)
    return _args.no_backward(y, "ssm_scan_step", tensors) if marked else y
