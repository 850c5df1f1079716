"""Argument checks and layouts shared by the selective state space operators."""
import torch

from .. import _lib


def fp32(t, shape, name, device):
    """A parameter as contiguous fp32 of ``shape`` on ``device`` (None stays None)."""
    if t is None:
        return None
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    if t.device != device:
        raise RuntimeError(f"{name} must be on {device}, got {t.device}")
    if not t.is_floating_point():
        raise TypeError(f"{name} must be a floating-point tensor, got {t.dtype}")
    if t.requires_grad:
        t = t.detach()
    if t.dtype != torch.float32:
        t = t.float()
    return t if t.is_contiguous() else t.contiguous()


def rows(t, shape, name, like):
    """Token rows of ``shape`` with the dtype and device of ``like``, unit stride last."""
    if t is None:
        return None
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    if t.dtype != like.dtype:
        raise TypeError(f"{name} must be {like.dtype} as the other sequences, got {t.dtype}")
    if t.device != like.device:
        raise RuntimeError(f"{name} must be on {like.device}, got {t.device}")
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def state(t, shape, name, dtype, device):
    """A cached state: contiguous, of ``shape`` and ``dtype`` on ``device``."""
    if t is None:
        return None
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise RuntimeError(f"{name} must be on {device}, got {t.device}")
    return t if t.is_contiguous() else t.contiguous()


def sequences(x, seq_offsets, name):
    """(sequences, tokens per sequence or in all, offsets) of ``x``: [B, L, C], or [T, C] with
    ``seq_offsets`` (int32 or int64, [sequences + 1], on x's device)."""
    _lib.ensure_device(x)
    _lib.dtype_code(x.dtype)
    if seq_offsets is None:
        if x.dim() != 3:
            raise ValueError(f"{name} must be [batch, length, channels], or [tokens, channels] with seq_offsets; "
                             f"got {tuple(x.shape)}")
        return x.shape[0], x.shape[1], None
    if x.dim() != 2:
        raise ValueError(f"{name} must be [tokens, channels] with seq_offsets, got {tuple(x.shape)}")
    if seq_offsets.dim() != 1 or seq_offsets.numel() < 2:
        raise ValueError("seq_offsets must hold at least two offsets, one more than there are sequences")
    if seq_offsets.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"seq_offsets must be int32 or int64, got {seq_offsets.dtype}")
    if seq_offsets.device != x.device:
        raise RuntimeError(f"seq_offsets must be on {x.device}, got {seq_offsets.device}")
    return seq_offsets.numel() - 1, x.shape[0], seq_offsets.to(torch.int32).contiguous()


def slot_index(slots, batch, device):
    """The step's stream slots as contiguous int32 [batch] (None: stream b is slot b)."""
    if slots is None:
        return None
    if tuple(slots.shape) != (batch,):
        raise ValueError(f"slots must have shape {(batch,)}, got {tuple(slots.shape)}")
    if slots.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"slots must be int32 or int64, got {slots.dtype}")
    if slots.device != device:
        raise RuntimeError(f"slots must be on {device}, got {slots.device}")
    return slots.to(torch.int32).contiguous()


def cache(t, out, tail, batch, slots, dtype, device):
    """The step's state and where its successor goes (in place when ``out`` is None): both
    contiguous [slots, *tail] of ``dtype``, large enough for ``batch`` when there is no index."""
    out = t if out is None else out
    for name, s in (("state", t), ("state_out", out)):
        if s.dim() != len(tail) + 1 or tuple(s.shape[1:]) != tail:
            raise ValueError(f"{name} must have shape [slots, {', '.join(map(str, tail))}], got {tuple(s.shape)}")
        if s.dtype != dtype:
            raise TypeError(f"{name} must be {dtype}, got {s.dtype}")
        if s.device != device:
            raise RuntimeError(f"{name} must be on {device}, got {s.device}")
        if not s.is_contiguous():
            raise ValueError(f"{name} must be contiguous: the kernel updates it in place")
    if out.shape[0] != t.shape[0]:
        raise ValueError(f"state_out must have {t.shape[0]} slots, got {out.shape[0]}")
    if slots is None and t.shape[0] < batch:
        raise ValueError(f"the state has {t.shape[0]} slots for {batch} streams")
    return t, out


def workspace(nbytes, device):
    return torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=device)


def grad_rows(dy):
    """An incoming gradient as contiguous rows (expanded or permuted ones are copied)."""
    return dy if dy.is_contiguous() else dy.contiguous()
