"""Short causal convolution over token rows (``vh_short_conv_fwd``, ``_bwd``, ``_step``)."""
import ctypes

import torch

from .. import _lib
from . import _args

_ACTIVATIONS = {None: 0, "silu": 1}


def _activation(activation):
    try:
        return _ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"activation must be None or 'silu', got {activation!r}") from None


def _taps(weight, channels):
    if weight.dim() != 2 or weight.shape[0] != channels:
        raise ValueError(f"weight must be [{channels}, taps], got {tuple(weight.shape)}")
    if not 2 <= weight.shape[1] <= 8:
        raise ValueError(f"short_conv takes 2 to 8 taps, got {weight.shape[1]}")
    return weight.shape[1]


class _Call:
    """One call's checked arguments: the C struct, and the tensors that it points to."""

    def __init__(self, x, weight, bias, activation, initial, offsets, reverse):
        count, length, offsets = _args.sequences(x, offsets, "x")
        d = x.shape[-1]
        k = _taps(weight, d)
        x = _args.rows(x, tuple(x.shape), "x", x)
        weight = _args.fp32(weight, (d, k), "weight", x.device)
        bias = _args.fp32(bias, (d,), "bias", x.device)
        initial = _args.state(initial, (count, k - 1, d), "initial_state", x.dtype, x.device)
        if initial is not None and initial.requires_grad:
            initial = initial.detach()
        self.kept = x, weight, bias, initial, offsets
        self.state_shape = count, k - 1, d
        self.args = _lib.VhShortConvArgs(
            x.data_ptr(), x.stride(0), x.stride(-2), weight.data_ptr(), _lib.ptr(bias), _lib.ptr(initial), None, None,
            _lib.ptr(offsets), length, _lib.DTYPES[x.dtype], activation, k, count, d, int(bool(reverse)))

    def forward(self, want_final):
        x, initial = self.kept[0], self.kept[3]
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        final = torch.empty(self.state_shape, dtype=x.dtype, device=x.device) if want_final else None
        if y.numel() == 0:  # no tokens: every state leaves as it entered
            if final is not None:
                final.copy_(initial) if initial is not None else final.zero_()
            return y, final
        self.args.y, self.args.final_state = y.data_ptr(), _lib.ptr(final)
        _lib.check(_lib.load().vh_short_conv_fwd(ctypes.byref(self.args), _lib.stream_handle(x.device)),
                   "vh_short_conv_fwd")
        return y, final

    def backward(self, dy, dfinal, want_bias, want_initial):
        x, weight = self.kept[:2]
        dev, d, k = x.device, weight.shape[0], weight.shape[1]
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
        dw = torch.empty((d, k), dtype=torch.float32, device=dev)
        db = torch.empty((d,), dtype=torch.float32, device=dev) if want_bias else None
        di = torch.empty(self.state_shape, dtype=x.dtype, device=dev) if want_initial else None
        if x.numel() == 0:
            dw.zero_()
            if db is not None:
                db.zero_()
            if di is not None:
                di.copy_(dfinal) if dfinal is not None else di.zero_()
            return dx, dw, db, di
        lib = _lib.load()
        ws = _args.workspace(lib.vh_short_conv_bwd_workspace_bytes(ctypes.byref(self.args)), dev)
        _lib.check(lib.vh_short_conv_bwd(
            ctypes.byref(self.args), dy.data_ptr(), _lib.ptr(dfinal), dx.data_ptr(), dw.data_ptr(), _lib.ptr(db),
            _lib.ptr(di), ws.data_ptr(), ws.numel(), _lib.stream_handle(dev)), "vh_short_conv_bwd")
        return dx, dw, db, di


class _ShortConvFunction(torch.autograd.Function):
    """Saves the inputs; the backward computes the pre-activation again."""

    @staticmethod
    def forward(ctx, x, weight, bias, initial, activation, want_final, offsets, reverse):
        call = _Call(x, weight, bias, activation, initial, offsets, reverse)
        y, final = call.forward(want_final)
        ctx.save_for_backward(x, weight, bias, initial, call.kept[4])
        ctx.options = activation, reverse
        ctx.set_materialize_grads(False)
        return (y, final) if want_final else y

    @staticmethod
    @_lib.on_input_device
    def backward(ctx, dy, dfinal=None):
        x, weight, bias, initial, offsets = ctx.saved_tensors
        activation, reverse = ctx.options
        if dy is None and dfinal is None:
            return (None,) * 8
        call = _Call(x, weight, bias, activation, initial, offsets, reverse)
        dy = torch.zeros(x.shape, dtype=x.dtype, device=x.device) if dy is None else _args.grad_rows(dy)
        dfinal = None if dfinal is None else _args.grad_rows(dfinal)
        dx, dw, db, di = call.backward(dy, dfinal, bias is not None,
                                       initial is not None and ctx.needs_input_grad[3])
        return (dx, dw.to(weight.dtype), None if db is None else db.to(bias.dtype), di, None, None, None, None)


@_lib.on_input_device
def short_conv(x, weight, bias=None, *, activation=None, initial_state=None, return_final_state=False,
               seq_offsets=None, reverse=False):
    """``y_t = act(bias + sum_k weight[:, k] x_{t - taps + 1 + k})`` per channel and sequence.

    x: [B, L, C] (fp32, bf16 or fp16; any batch and token strides), or packed [T, C] with
    ``seq_offsets`` [B + 1] (int32 or int64 on x's device: 0 first, never decreasing, T last;
    sequences may be empty; the offsets are not read on the host).  weight: [C, taps], 2 to 8
    taps.  activation: None or "silu".  initial_state: [B, taps - 1, C] of x's dtype, the inputs
    before each sequence, oldest first (zeros when None).  reverse reads every sequence from its
    last token to its first.  Sums run in fp32 and y, of x's dtype, is rounded once.  Returns y,
    or (y, final_state) with ``return_final_state``, the last taps - 1 inputs.  Differentiable in
    x, weight, bias and initial_state, through y and the final state."""
    act = _activation(activation)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, initial_state)):
        return _ShortConvFunction.apply(x, weight, bias, initial_state, act, bool(return_final_state), seq_offsets,
                                        bool(reverse))
    y, final = _Call(x, weight, bias, act, initial_state, seq_offsets, reverse).forward(return_final_state)
    return (y, final) if return_final_state else y


@torch.no_grad()
@_lib.on_input_device
def short_conv_step(x, state, weight, bias=None, *, activation=None, slots=None, state_out=None):
    """One token of ``B`` cached streams: x [B, C], state [slots, taps - 1, C] of x's dtype, whose
    rows move up by one with x as the newest (in place, or into ``state_out``).  slots: int32 or
    int64 [B], each stream's row of the state (row b without it); a stream whose slot lies outside
    the state is skipped and its y is 0; no two streams may name one slot.  Returns y [B, C]."""
    act = _activation(activation)
    _lib.ensure_device(x)
    code = _lib.dtype_code(x.dtype)
    if x.dim() != 2:
        raise ValueError(f"x must be [batch, channels], got {tuple(x.shape)}")
    b, d = x.shape
    k = _taps(weight, d)
    x = _args.rows(x, (b, d), "x", x)
    weight = _args.fp32(weight, (d, k), "weight", x.device)
    bias = _args.fp32(bias, (d,), "bias", x.device)
    slots = _args.slot_index(slots, b, x.device)
    state, state_out = _args.cache(state, state_out, (k - 1, d), b, slots, x.dtype, x.device)
    y = torch.empty((b, d), dtype=x.dtype, device=x.device)
    if y.numel() == 0:
        return y
    _lib.check(_lib.load().vh_short_conv_step(
        x.data_ptr(), x.stride(0), code, weight.data_ptr(), _lib.ptr(bias), act, state.data_ptr(), state_out.data_ptr(),
        _lib.ptr(slots), state.shape[0], y.data_ptr(), b, d, k, _lib.stream_handle(x.device)), "vh_short_conv_step")
    return y
