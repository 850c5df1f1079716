"""Argument checks and layouts shared by the selective state space operators.

A step of a small batch takes the GPU a few microseconds, so the host's part counts: the C structs are
packed in one go (``struct.Struct``) and every check runs on values that are already at hand."""
import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from .. import _lib

_F32 = torch.float32


def refuse_shape(name, want, got):
    raise ValueError(f"{name} must have shape {tuple(want)}, got {tuple(got)}")


def refuse_device(name, want, got):
    raise RuntimeError(f"{name} must be on {want}, got {got}")


def refuse_dtype(name, want, got):
    raise TypeError(f"{name} must be {want}, got {got}")


def fp32(t, shape, name, device):
    """A parameter as contiguous fp32 of ``shape`` on ``device`` (None stays None)."""
    if t is None:
        return None
    if t.shape != shape:
        refuse_shape(name, shape, t.shape)
    if t.device != device:
        refuse_device(name, device, t.device)
    if t.dtype is not _F32:
        if not t.is_floating_point():
            raise TypeError(f"{name} must be a floating-point tensor, got {t.dtype}")
        t = t.detach().float()
    return t if t.is_contiguous() else t.detach().contiguous()


def rows(t, shape, name, dtype, device):
    """Token rows of ``shape`` with the dtype and device of the others, unit stride last."""
    if t is None:
        return None
    if t.shape != shape:
        refuse_shape(name, shape, t.shape)
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype} as the other sequences, got {t.dtype}")
    if t.device != device:
        refuse_device(name, device, t.device)
    return t if t.stride(-1) == 1 or shape[-1] == 1 else t.detach().contiguous()


def state(t, shape, name, dtype, device):
    """An initial state: contiguous, of ``shape`` and ``dtype`` on ``device`` (None stays None)."""
    if t is None:
        return None
    if t.shape != shape:
        refuse_shape(name, shape, t.shape)
    if t.dtype is not dtype:
        refuse_dtype(name, dtype, t.dtype)
    if t.device != device:
        refuse_device(name, device, t.device)
    return t if t.is_contiguous() else t.detach().contiguous()


def offsets_like(seq_offsets, device):
    """Sequence offsets as contiguous int32 on ``device``; the kernels clamp them to the tokens."""
    if seq_offsets.dim() != 1 or seq_offsets.numel() < 2:
        raise ValueError("seq_offsets must hold at least two offsets, one more than there are sequences")
    if seq_offsets.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"seq_offsets must be int32 or int64, got {seq_offsets.dtype}")
    if seq_offsets.device != device:
        refuse_device("seq_offsets", device, seq_offsets.device)
    if seq_offsets.dtype is torch.int32 and seq_offsets.is_contiguous():
        return seq_offsets
    if seq_offsets.dtype is torch.int64:
        # past int32 an offset is outside any tokens, and must not wrap into them
        seq_offsets = seq_offsets.clamp(-1, 0x7fffffff).to(torch.int32)
    return seq_offsets.contiguous()


def sequences(x, seq_offsets, name):
    """(sequences, tokens per sequence or in all, offsets) of ``x``: [B, L, C], or [T, C] with
    ``seq_offsets`` (int32 or int64, [sequences + 1], on x's device)."""
    _lib.ensure_device(x)
    if x.dtype not in _lib.DTYPES:
        _lib.dtype_code(x.dtype)
    if seq_offsets is None:
        if x.dim() != 3:
            raise ValueError(f"{name} must be [batch, length, channels], or [tokens, channels] with seq_offsets; "
                             f"got {tuple(x.shape)}")
        return x.shape[0], x.shape[1], None
    if x.dim() != 2:
        raise ValueError(f"{name} must be [tokens, channels] with seq_offsets, got {tuple(x.shape)}")
    seq_offsets = offsets_like(seq_offsets, x.device)
    return seq_offsets.numel() - 1, x.shape[0], seq_offsets


def slot_index(slots, batch, device):
    """The step's stream slots as contiguous int32 [batch] (None: stream b is slot b)."""
    if slots is None:
        return None
    if slots.shape != (batch,):
        refuse_shape("slots", (batch,), slots.shape)
    if slots.device != device:
        refuse_device("slots", device, slots.device)
    if slots.dtype is not torch.int32:
        if slots.dtype is not torch.int64:
            raise TypeError(f"slots must be int32 or int64, got {slots.dtype}")
        # past int32 a slot is outside any cache, and must not wrap into one
        slots = slots.clamp(-1, 0x7fffffff).to(torch.int32)
    return slots if slots.is_contiguous() else slots.contiguous()


def cache(t, out, tail, batch, slots, dtype, device):
    """The step's state and where its successor goes (in place when ``out`` is None): both
    contiguous [slots, *tail] of ``dtype``, large enough for ``batch`` when there is no index."""
    for name, s in (("state", t),) if out is None else (("state", t), ("state_out", out)):
        if s.dim() != len(tail) + 1 or s.shape[1:] != tail:
            raise ValueError(f"{name} must have shape [slots, {', '.join(map(str, tail))}], got {tuple(s.shape)}")
        if s.dtype is not dtype:
            refuse_dtype(name, dtype, s.dtype)
        if s.device != device:
            refuse_device(name, device, s.device)
        if not s.is_contiguous():
            raise ValueError(f"{name} must be contiguous: the kernel updates it in place")
    if out is None:
        out = t
    elif out.shape[0] != t.shape[0]:
        raise ValueError(f"state_out must have {t.shape[0]} slots, got {out.shape[0]}")
    if slots is None and t.shape[0] < batch:
        raise ValueError(f"the state has {t.shape[0]} slots for {batch} streams")
    return t, out


def wrote(t):
    """Tells autograd that a kernel changed ``t`` in place, as an in-place operation would: a backward
    that saved it then raises instead of reading the new values."""
    if not t.is_inference():
        increment_version((t,))


def tracked(tensors):
    """Whether a derivative by one of the tensors (None among them) is wanted: they require gradients,
    or carry a forward-mode tangent (which an autograd function without a rule for it refuses)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return forward_ad._current_level >= 0 and _tangent(tensors)


def _tangent(tensors):
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


class _NoBackward(torch.autograd.Function):
    """The identity for a step's y; its backward raises."""

    @staticmethod
    def forward(ctx, y, name, *tensors):
        ctx.name = name
        return y.view_as(y)

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError(f"{ctx.name} is not differentiable: run the tokens as a sequence instead")


def step_derivatives(name, tensors, state, state_out):
    """A step keeps nothing for a backward.  Refuses what could only end in a wrong derivative: tangents,
    and a cache that is written and takes part in a graph (under ``torch.no_grad()`` it may).  Returns
    whether others of ``tensors`` (all of them, the states too) require gradients, which
    :func:`no_backward` then marks y with."""
    if not tracked(tensors):
        return False
    if forward_ad._current_level >= 0 and _tangent(tensors):
        raise RuntimeError(f"{name} is not differentiable in forward mode")
    if (state if state_out is None else state_out).requires_grad:
        raise RuntimeError(f"{name} is not differentiable and its cache requires gradients: call it under torch.no_grad() "
                           "or detach the cache")
    return True


def no_backward(y, name, tensors):
    """y of a step some of whose tensors require gradients: a backward through it raises."""
    return _NoBackward.apply(y, name, *tensors)


def ptr(t):
    return 0 if t is None else t.data_ptr()


def workspace(nbytes, device):
    return torch.empty(nbytes if nbytes > 16 else 16, dtype=torch.uint8, device=device)


def grad_rows(dy):
    """An incoming gradient as contiguous rows (expanded or permuted ones are copied)."""
    return dy if dy.is_contiguous() else dy.contiguous()


def grad_like(g, t):
    """A gradient in the shape and dtype of its input."""
    if g is None:
        return None
    if g.shape != t.shape:
        g = g.view(t.shape)
    return g if g.dtype is t.dtype else g.to(t.dtype)
