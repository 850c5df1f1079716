"""Group norm over channels-last data with an activation and a gate (``vh_group_norm_fwd``, ``_bwd``).

    pre = (x - mean) / sqrt(var + eps) * weight + bias,      y = act(pre) * silu(gate)

``group_norm`` takes images, with statistics over a group's channels at all pixels; ``group_norm_rows``
token rows, each by itself, as behind the heads of ``ssm_core.linear_attention``.  Statistics, sums and
parameters are fp32; y has x's dtype and is rounded once.  There is no CPU path: CPU tensors raise.
"""
import struct

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from .. import _lib
from ..ssm_core import _args
from ..ssm_core._args import ptr

__all__ = ["GroupNorm", "group_norm", "group_norm_rows"]

_ARGS = struct.Struct("2Q4q5Q2qf4i4x")  # vh_group_norm_args
_ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2}


class _Call:
    """One call's checked arguments; ``args`` packs them with the output pointers.  x and gate: [samples,
    channels] (unit stride last) or contiguous [samples, pixels, channels]."""

    __slots__ = ("x", "gate", "weight", "bias", "samples", "groups", "head", "tail")

    def __init__(self, x, gate, weight, bias, groups, eps, activation):
        shape, device, xs = x.shape, x.device, x.stride()
        n, c = shape[0], shape[-1]
        self.x, self.gate, self.samples, self.groups = x, gate, n, groups
        self.weight = weight = _args.fp32(weight, (c,), "weight", device)
        self.bias = bias = _args.fp32(bias, (c,), "bias", device)
        gs = (0, 0) if gate is None else gate.stride()
        self.head = (x.data_ptr(), ptr(gate), xs[0], xs[-2], gs[0], gs[-2], ptr(weight), ptr(bias))
        self.tail = n, shape[1] if len(shape) == 3 else 1, eps, _lib.DTYPES[x.dtype], c, groups, activation

    def args(self, y=0, mean=None, rstd=None):
        return _ARGS.pack(*self.head, y, ptr(mean), ptr(rstd), *self.tail)

    def forward(self, want_stats):
        x = self.x
        dev = x.device
        y = torch.empty(x.shape, dtype=x.dtype, device=dev)
        mean = rstd = None
        if want_stats:
            mean, rstd = torch.empty((2, self.samples, self.groups), dtype=torch.float32, device=dev)
        if y.numel() == 0:
            return y, mean, rstd
        lib = _lib.load()
        args = self.args(y.data_ptr(), mean, rstd)
        nbytes = lib.vh_group_norm_fwd_workspace_bytes(args)
        ws = _args.workspace(nbytes, dev) if nbytes else None
        _lib.check(lib.vh_group_norm_fwd(args, ptr(ws), nbytes, _lib.stream_handle(dev)), "vh_group_norm_fwd")
        return y, mean, rstd

    def backward(self, dy, mean, rstd, want_gate):
        x, dev = self.x, self.x.device
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
        dgate = torch.empty(x.shape, dtype=x.dtype, device=dev) if want_gate else None
        both = torch.empty((2, x.shape[-1]), dtype=torch.float32, device=dev)
        dw, db = None if self.weight is None else both[0], None if self.bias is None else both[1]
        if dx.numel() == 0:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
            return dx, dgate, dw, db
        lib = _lib.load()
        args = self.args(0, mean, rstd)
        nbytes = lib.vh_group_norm_bwd_workspace_bytes(args)
        ws = _args.workspace(nbytes, dev)
        _lib.check(lib.vh_group_norm_bwd(args, dy.data_ptr(), dx.data_ptr(), ptr(dgate), ptr(dw), ptr(db), ws.data_ptr(), nbytes,
                                         _lib.stream_handle(dev)), "vh_group_norm_bwd")
        return dx, dgate, dw, db


def _check(x, channels, groups, activation, gate):
    _lib.ensure_device(x)
    if x.dtype not in _lib.DTYPES:
        _lib.dtype_code(x.dtype)
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be None, 'silu' or 'gelu', got {activation!r}")
    if groups < 1 or channels % groups:
        raise ValueError(f"groups must be a divisor of {channels}, got {groups}")
    if gate is not None:
        if gate.shape != x.shape:
            _args.refuse_shape("gate", x.shape, gate.shape)
        if gate.dtype is not x.dtype:
            raise TypeError(f"gate must be {x.dtype} as x, got {gate.dtype}")
        if gate.device != x.device:
            _args.refuse_device("gate", x.device, gate.device)


def _flat(t):
    """[..., C] as [rows, C] with unit stride last: a view where the strides allow it."""
    c = t.shape[-1]
    if t.dim() != 2:
        t = t.reshape(t.numel() // c if c else 0, c)
    return t if t.stride(-1) == 1 or c == 1 else t.contiguous()


def _pixels(t):
    """[B, C, H, W] as contiguous [B, H * W, C]: a view of a channels-last tensor."""
    t = t.contiguous(memory_format=torch.channels_last).permute(0, 2, 3, 1)
    # a single row of pixels or channel lets a tensor count as channels-last with any strides
    return (t if t.is_contiguous() else t.contiguous()).flatten(1, 2)


def _shaped(t, like):
    """[rows, C] or [B, H * W, C] in the shape of the call's x, an image channels-last."""
    if t is None or t.shape == like.shape:
        return t
    if t.dim() == 2:
        return t.view(like.shape)
    b, c, h, w = like.shape
    return t.view(b, h, w, c).permute(0, 3, 1, 2)


class _GroupNormFunction(torch.autograd.Function):
    """Saves its inputs and each group's mean and 1 / standard deviation.  Takes x as the caller has it: views
    outside would be nodes of the graph, some 10 us of host time each."""

    @staticmethod
    def forward(ctx, x, gate, weight, bias, layout, groups, eps, activation):
        y, mean, rstd = _Call(layout(x), None if gate is None else layout(gate), weight, bias, groups, eps, activation).forward(True)
        ctx.save_for_backward(x, gate, weight, bias, mean, rstd)
        ctx.options = groups, eps, activation
        ctx.layout = layout
        return _shaped(y, x)

    @staticmethod
    @once_differentiable
    @_lib.on_input_device
    def backward(ctx, dy):
        x, gate, weight, bias, mean, rstd = ctx.saved_tensors
        layout = ctx.layout
        call = _Call(layout(x), None if gate is None else layout(gate), weight, bias, *ctx.options)
        dx, dgate, dw, db = call.backward(_args.grad_rows(layout(dy)), mean, rstd, gate is not None and ctx.needs_input_grad[1])
        return (_shaped(dx, x), None if dgate is None else _shaped(dgate, gate), _args.grad_like(dw, weight),
                _args.grad_like(db, bias), None, None, None, None)


def _run(x, gate, weight, bias, layout, groups, eps, activation):
    options = int(groups), float(eps), _ACTIVATIONS[activation]
    if _args.tracked((x, gate, weight, bias)):
        return _GroupNormFunction.apply(x, gate, weight, bias, layout, *options)
    call = _Call(layout(x), None if gate is None else layout(gate), weight, bias, *options)
    return _shaped(call.forward(False)[0], x)


@_lib.on_input_device
def group_norm(x, groups, weight=None, bias=None, eps=1e-5, *, activation=None, gate=None):
    """Group norm of images x [B, C, H, W] stored channels-last (other layouts are converted), fp32, bf16
    or fp16: statistics over the C / groups channels of a group at all pixels of an image.  weight, bias:
    [C] (1 and 0 when None).  activation: None, "silu" or "gelu" (by the error function).  gate: as x, or
    None; multiplies the result by silu(gate).  Returns y, channels-last, of x's dtype.  Differentiable in
    every tensor; the sums of the backward run in a fixed order."""
    if x.dim() != 4:
        raise ValueError(f"x must be [batch, channels, height, width], got {tuple(x.shape)}")
    _check(x, x.shape[1], groups, activation, gate)
    return _run(x, gate, weight, bias, _pixels, groups, eps, activation)


@_lib.on_input_device
def group_norm_rows(x, groups, weight=None, bias=None, eps=1e-5, *, activation=None, gate=None):
    """As :func:`group_norm` for rows x [..., C], each normalised by itself: statistics over the C /
    groups channels of a group.  x and gate may be parts of wider rows (unit stride last)."""
    if x.dim() < 1:
        raise ValueError("x must be [..., channels]")
    _check(x, x.shape[-1], groups, activation, gate)
    return _run(x, gate, weight, bias, _flat, groups, eps, activation)


class GroupNorm(nn.Module):
    """Group norm of channels-last images with an activation (``group_norm``); one weight and bias a channel."""

    def __init__(self, groups, dim, eps=1e-5, activation=None):
        super().__init__()
        if groups < 1 or dim % groups:
            raise ValueError(f"groups must be a divisor of {dim}, got {groups}")
        if activation not in _ACTIVATIONS:
            raise ValueError(f"activation must be None, 'silu' or 'gelu', got {activation!r}")
        self.weight = nn.Parameter(torch.ones(dim, dtype=torch.float32))
        self.bias = nn.Parameter(torch.zeros(dim, dtype=torch.float32))
        self.groups, self.eps, self.activation = int(groups), float(eps), activation

    def forward(self, x, gate=None):
        return group_norm(x, self.groups, self.weight, self.bias, self.eps, activation=self.activation, gate=gate)

    def extra_repr(self):
        return f"groups={self.groups}, dim={self.weight.numel()}, eps={self.eps}, activation={self.activation}"
