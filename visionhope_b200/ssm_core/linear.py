"""Linear attention with a decay for each head (``vh_linear_attention_fwd``, ``_bwd``, ``_step``)."""
import struct

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from . import _args
from ._args import ptr

MAX_DIM = 128
_ARGS = struct.Struct("3Q9q5Qqf6i4x")  # vh_linear_attention_args


class _Call:
    """One call's checked arguments; ``args`` packs them with the output pointers."""

    __slots__ = ("q", "k", "v", "log_decay", "initial", "offsets", "state_shape", "head", "tail")

    def __init__(self, q, k, v, log_decay, scale, initial, offsets, reverse, one_token=False):
        _lib.ensure_device(q)
        device, dtype, shape = q.device, q.dtype, q.shape
        code = _lib.dtype_code(dtype)
        if one_token:
            if len(shape) != 3:
                raise ValueError(f"q must be [batch, heads, key dim], got {tuple(shape)}")
            count, length = shape[0], 1
        elif offsets is None:
            if len(shape) != 4:
                raise ValueError("q must be [batch, length, heads, key dim], or [tokens, heads, key dim] with seq_offsets; "
                                 f"got {tuple(shape)}")
            count, length = shape[0], shape[1]
        else:
            if len(shape) != 3:
                raise ValueError(f"q must be [tokens, heads, key dim] with seq_offsets, got {tuple(shape)}")
            offsets = _args.offsets_like(offsets, device)
            count, length = offsets.numel() - 1, shape[0]
        lead, heads, dk = shape[:-2], shape[-2], shape[-1]
        if v.dim() != len(shape):
            raise ValueError(f"v must be [{', '.join(map(str, (*lead, heads)))}, value dim], got {tuple(v.shape)}")
        dv = v.shape[-1]
        if not (1 <= dk <= MAX_DIM and 1 <= dv <= MAX_DIM):
            raise ValueError(f"linear_attention takes key and value dims of 1 to {MAX_DIM}, got {dk} and {dv}")
        self.q = q = _args.rows(q, shape, "q", dtype, device)
        self.k = k = _args.rows(k, shape, "k", dtype, device)
        self.v = v = _args.rows(v, (*lead, heads, dv), "v", dtype, device)
        self.log_decay = log_decay = _args.fp32(log_decay, (heads,), "log_decay", device)
        self.state_shape = count, heads, dk, dv
        self.initial = _args.state(initial, self.state_shape, "initial_state", torch.float32, device)
        self.offsets = offsets
        qs, ks, vs = q.stride(), k.stride(), v.stride()
        self.head = (q.data_ptr(), k.data_ptr(), v.data_ptr(), qs[0], qs[-3], qs[-2], ks[0], ks[-3], ks[-2],
                     vs[0], vs[-3], vs[-2], log_decay.data_ptr(), ptr(self.initial))
        self.tail = (ptr(offsets), length, dk ** -0.5 if scale is None else float(scale), code, count, heads, dk, dv,
                     1 if reverse else 0)

    def args(self, o=0, final=0):
        return _ARGS.pack(*self.head, o, final, *self.tail)

    def forward(self, want_final):
        v, initial, dev = self.v, self.initial, self.v.device
        o = torch.empty(v.shape, dtype=v.dtype, device=dev)
        final = torch.empty(self.state_shape, dtype=torch.float32, device=dev) if want_final else None
        if o.numel() == 0:  # no tokens: every state leaves as it entered
            if final is not None:
                final.copy_(initial.detach()) if initial is not None else final.zero_()
            return o, final
        lib = _lib.load()
        args = self.args(o.data_ptr(), ptr(final))
        nbytes = lib.vh_linear_attention_fwd_workspace_bytes(args)
        ws = _args.workspace(nbytes, dev) if nbytes else None
        _lib.check(lib.vh_linear_attention_fwd(args, ptr(ws), nbytes, _lib.stream_handle(dev)), "vh_linear_attention_fwd")
        return o, final

    def backward(self, do, dfinal, want_initial):
        dev = self.q.device
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (self.q, self.k, self.v))
        di = torch.empty(self.state_shape, dtype=torch.float32, device=dev) if want_initial else None
        if dq.numel() == 0:
            if di is not None:
                di.copy_(dfinal) if dfinal is not None else di.zero_()
            return dq, dk, dv, di
        lib = _lib.load()
        args = self.args()
        nbytes = lib.vh_linear_attention_bwd_workspace_bytes(args)
        ws = _args.workspace(nbytes, dev) if nbytes else None
        _lib.check(lib.vh_linear_attention_bwd(args, do.data_ptr(), ptr(dfinal), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                               ptr(di), ptr(ws), nbytes, _lib.stream_handle(dev)), "vh_linear_attention_bwd")
        return dq, dk, dv, di


class _LinearAttentionFunction(torch.autograd.Function):
    """Saves its inputs alone: the backward runs the recurrences again."""

    @staticmethod
    def forward(ctx, q, k, v, initial, log_decay, scale, want_final, offsets, reverse):
        call = _Call(q, k, v, log_decay, scale, initial, offsets, reverse)
        o, final = call.forward(want_final)
        ctx.save_for_backward(q, k, v, initial, call.log_decay, call.offsets)
        ctx.options = scale, reverse
        ctx.set_materialize_grads(False)
        return (o, final) if want_final else o

    @staticmethod
    @once_differentiable
    @_lib.on_input_device
    def backward(ctx, do, dfinal=None):
        if do is None and dfinal is None:
            return (None,) * 9
        q, k, v, initial, log_decay, offsets = ctx.saved_tensors
        scale, reverse = ctx.options
        call = _Call(q, k, v, log_decay, scale, initial, offsets, reverse)
        do = torch.zeros(v.shape, dtype=v.dtype, device=v.device) if do is None else _args.grad_rows(do)
        dfinal = None if dfinal is None else _args.grad_rows(dfinal)
        return (*call.backward(do, dfinal, initial is not None and ctx.needs_input_grad[3]), None, None, None, None, None)


def _constant(log_decay):
    if _args.tracked((log_decay,)):
        raise ValueError("log_decay is a constant of the layer and has no gradient: detach it")


@_lib.on_input_device
def linear_attention(q, k, v, log_decay, *, scale=None, initial_state=None, return_final_state=False, seq_offsets=None,
                     reverse=False):
    """Linear attention whose state decays by ``exp(log_decay[h])`` a token: per sequence and head h

        S_t = exp(log_decay[h]) S_{t-1} + k_t v_t^T          (S: [key dim, value dim])
        o_t = scale q_t^T S_t

    q, k: [B, L, H, key dim] and v: [B, L, H, value dim] of one dtype (fp32, bf16 or fp16; any batch,
    token and head strides), or packed [T, H, dim] with ``seq_offsets`` (as :func:`short_conv`).  Dims
    of 1 to 128.  log_decay: [H], at most 0 (minus infinity forgets everything), a constant: it gets no
    gradient.  scale: key dim ** -0.5 when None.  initial_state: fp32 [B, H, key dim, value dim] (zeros
    when None).  reverse reads every sequence from its last token to its first.  The state is fp32
    throughout; o, of v's dtype, is rounded once, and its terms' scores and states, as operands of a
    matrix product, to bf16 (bf16 inputs), 16 bits (fp16) or 24 bits (fp32).  A value that is not finite
    reaches its own and later tokens only.  Returns o, or (o, final_state) with
    ``return_final_state``.  Differentiable in q, k, v and the initial state, through o and the final
    state; the sums of the backward run in a fixed order."""
    _constant(log_decay)
    tensors = (q, k, v, initial_state)
    if _args.tracked(tensors):
        return _LinearAttentionFunction.apply(*tensors, log_decay, scale, bool(return_final_state), seq_offsets, bool(reverse))
    o, final = _Call(q, k, v, log_decay, scale, initial_state, seq_offsets, reverse).forward(return_final_state)
    return (o, final) if return_final_state else o


@_lib.on_input_device
def linear_attention_step(q, k, v, log_decay, state, *, scale=None, slots=None, state_out=None):
    """One token of ``B`` cached streams: q, k [B, H, key dim]; v [B, H, value dim]; state fp32 [slots, H,
    key dim, value dim], advanced in place (or into ``state_out``).  slots: as :func:`short_conv_step`.
    Returns o [B, H, value dim].  Not differentiable, as :func:`short_conv_step`."""
    tensors = q, k, v, log_decay, state, state_out
    marked = _args.step_derivatives("linear_attention_step", tensors, state, state_out)
    call = _Call(q, k, v, log_decay, scale, None, None, False, one_token=True)
    device = q.device
    b, h, dk, dv = call.state_shape
    slots = _args.slot_index(slots, b, device)
    state, state_out = _args.cache(state, state_out, (h, dk, dv), b, slots, torch.float32, device)
    o = torch.empty((b, h, dv), dtype=q.dtype, device=device)
    if o.numel() == 0:
        return o
    _lib.check(_lib.load().vh_linear_attention_step(call.args(o.data_ptr()), state.data_ptr(), state_out.data_ptr(),
                                                    ptr(slots), state.shape[0], _lib.stream_handle(device)),
               "vh_linear_attention_step")
    _args.wrote(state_out)
    return _args.no_backward(o, "linear_attention_step", tensors) if marked else o
