"""Short causal convolution over token rows (``vh_short_conv_fwd``, ``_bwd``, ``_step``)."""
import struct

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from . import _args
from ._args import ptr

_ACTIVATIONS = {None: 0, "silu": 1}
_ARGS = struct.Struct("QqqQQQQQQqiiiiii")  # vh_short_conv_args


def _activation(activation):
    try:
        return _ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"activation must be None or 'silu', got {activation!r}") from None


def _taps(weight, channels):
    if weight.dim() != 2 or weight.shape[0] != channels:
        raise ValueError(f"weight must be [{channels}, taps], got {tuple(weight.shape)}")
    k = weight.shape[1]
    if not 2 <= k <= 8:
        raise ValueError(f"short_conv takes 2 to 8 taps, got {k}")
    return k


class _Call:
    """One call's checked arguments; ``args`` packs them with the output pointers."""

    __slots__ = ("x", "weight", "bias", "initial", "offsets", "state_shape", "head", "tail")

    def __init__(self, x, weight, bias, activation, initial, offsets, reverse):
        count, length, offsets = _args.sequences(x, offsets, "x")
        shape, device, dtype = x.shape, x.device, x.dtype
        d = shape[-1]
        k = _taps(weight, d)
        self.x = x = _args.rows(x, shape, "x", dtype, device)
        self.weight = weight = _args.fp32(weight, (d, k), "weight", device)
        self.bias = bias = _args.fp32(bias, (d,), "bias", device)
        self.state_shape = count, k - 1, d
        self.initial = initial = _args.state(initial, self.state_shape, "initial_state", dtype, device)
        self.offsets = offsets
        stride = x.stride()
        self.head = (x.data_ptr(), stride[0], stride[-2], weight.data_ptr(), ptr(bias), ptr(initial))
        self.tail = (ptr(offsets), length, _lib.DTYPES[dtype], activation, k, count, d, 1 if reverse else 0)

    def args(self, y=0, final=0):
        return _ARGS.pack(*self.head, y, final, *self.tail)

    def forward(self, want_final):
        x = self.x
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        final = torch.empty(self.state_shape, dtype=x.dtype, device=x.device) if want_final else None
        if y.numel() == 0:  # no tokens: every state leaves as it entered
            if final is not None:
                final.copy_(self.initial.detach()) if self.initial is not None else final.zero_()
            return y, final
        _lib.check(_lib.load().vh_short_conv_fwd(self.args(y.data_ptr(), ptr(final)), _lib.stream_handle(x.device)),
                   "vh_short_conv_fwd")
        return y, final

    def backward(self, dy, dfinal, want_initial):
        x, weight = self.x, self.weight
        dev, dtype = x.device, x.dtype
        dx = torch.empty(x.shape, dtype=dtype, device=dev)
        dw = torch.empty(weight.shape, dtype=torch.float32, device=dev)
        db = None if self.bias is None else torch.empty(self.bias.shape, dtype=torch.float32, device=dev)
        di = torch.empty(self.state_shape, dtype=dtype, device=dev) if want_initial else None
        if x.numel() == 0:
            dw.zero_()
            if db is not None:
                db.zero_()
            if di is not None:
                di.copy_(dfinal) if dfinal is not None else di.zero_()
            return dx, dw, db, di
        lib, args = _lib.load(), self.args()
        ws = _args.workspace(lib.vh_short_conv_bwd_workspace_bytes(args), dev)
        _lib.check(lib.vh_short_conv_bwd(args, dy.data_ptr(), ptr(dfinal), dx.data_ptr(), dw.data_ptr(), ptr(db), ptr(di),
                                         ws.data_ptr(), ws.numel(), _lib.stream_handle(dev)), "vh_short_conv_bwd")
        return dx, dw, db, di


class _ShortConvFunction(torch.autograd.Function):
    """Saves the inputs; the backward computes the pre-activation again."""

    @staticmethod
    def forward(ctx, x, weight, bias, initial, activation, want_final, offsets, reverse):
        call = _Call(x, weight, bias, activation, initial, offsets, reverse)
        y, final = call.forward(want_final)
        ctx.save_for_backward(x, weight, bias, initial, call.offsets)
        ctx.options = activation, reverse
        ctx.set_materialize_grads(False)
        return (y, final) if want_final else y

    @staticmethod
    @once_differentiable
    @_lib.on_input_device
    def backward(ctx, dy, dfinal=None):
        if dy is None and dfinal is None:
            return (None,) * 8
        x, weight, bias, initial, offsets = ctx.saved_tensors
        activation, reverse = ctx.options
        call = _Call(x, weight, bias, activation, initial, offsets, reverse)
        dy = torch.zeros(x.shape, dtype=x.dtype, device=x.device) if dy is None else _args.grad_rows(dy)
        dfinal = None if dfinal is None else _args.grad_rows(dfinal)
        dx, dw, db, di = call.backward(dy, dfinal, initial is not None and ctx.needs_input_grad[3])
        return dx, _args.grad_like(dw, weight), _args.grad_like(db, bias), di, None, None, None, None


@_lib.on_input_device
def short_conv(x, weight, bias=None, *, activation=None, initial_state=None, return_final_state=False,
               seq_offsets=None, reverse=False):
    """``y_t = act(bias + sum_k weight[:, k] x_{t - taps + 1 + k})`` per channel and sequence.

    x: [B, L, C] (fp32, bf16 or fp16; any batch and token strides), or packed [T, C] with
    ``seq_offsets`` [B + 1] (int32 or int64 on x's device, never decreasing, from 0 to T; sequences
    may be empty; rows before the first offset and from the last one on belong to none and give
    zeros, y's and the gradients'; the offsets are not read on the host).  weight: [C, taps], 2 to 8
    taps.  activation: None or "silu".  initial_state: [B, taps - 1, C] of x's dtype, the inputs
    before each sequence, oldest first (zeros when None).  reverse reads every sequence from its
    last token to its first.  Sums run in fp32 and y, of x's dtype, is rounded once.  Returns y,
    or (y, final_state) with ``return_final_state``, the last taps - 1 inputs.  Differentiable in
    x, weight, bias and initial_state, through y and the final state."""
    act = _activation(activation)
    if _args.tracked((x, weight, bias, initial_state)):
        return _ShortConvFunction.apply(x, weight, bias, initial_state, act, bool(return_final_state), seq_offsets,
                                        bool(reverse))
    y, final = _Call(x, weight, bias, act, initial_state, seq_offsets, reverse).forward(return_final_state)
    return (y, final) if return_final_state else y


@_lib.on_input_device
def short_conv_step(x, state, weight, bias=None, *, activation=None, slots=None, state_out=None):
    """One token of ``B`` cached streams: x [B, C], state [slots, taps - 1, C] of x's dtype, whose
    rows move up by one with x as the newest (in place, or into ``state_out``).  slots: int32 or
    int64 [B], each stream's row of the state (row b without it); a stream whose slot lies outside
    the state is skipped and its y is 0; no two streams may name one slot.  Returns y [B, C].  Not
    differentiable: a backward through y raises, and so does a cache that requires gradients, unless
    the call is under ``torch.no_grad()``."""
    act = _activation(activation)
    tensors = x, state, weight, bias, state_out
    marked = _args.step_derivatives("short_conv_step", tensors, state, state_out)
    _lib.ensure_device(x)
    device, dtype = x.device, x.dtype
    code = _lib.dtype_code(dtype)
    if x.dim() != 2:
        raise ValueError(f"x must be [batch, channels], got {tuple(x.shape)}")
    b, d = shape = x.shape
    k = _taps(weight, d)
    x = _args.rows(x, shape, "x", dtype, device)
    weight = _args.fp32(weight, (d, k), "weight", device)
    bias = _args.fp32(bias, (d,), "bias", device)
    slots = _args.slot_index(slots, b, device)
    state, state_out = _args.cache(state, state_out, (k - 1, d), b, slots, dtype, device)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    if b * d == 0:
        return y
    _lib.check(_lib.load().vh_short_conv_step(
        x.data_ptr(), x.stride(0), code, weight.data_ptr(), ptr(bias), act, state.data_ptr(), state_out.data_ptr(),
        ptr(slots), state.shape[0], y.data_ptr(), b, d, k, _lib.stream_handle(device)), "vh_short_conv_step")
    _args.wrote(state_out)
    return _args.no_backward(y, "short_conv_step", tensors) if marked else y
