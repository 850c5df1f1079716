"""A token-row mixer on linear attention with a decay for each head.

``RetentionMixer``: one input projection into queries, keys, values and a gate, linear attention whose
states decay head by head, a group norm of each head's outputs times silu(gate), and an output
projection.  The projections are plain GEMMs; the attention and the norm run on ``libvhope.so``.

Rows are ``[batch, length, dim]``, or packed ``[tokens, dim]`` with ``seq_offsets``, such as the tokens of
a channels-last image (``ssm_mixer.image_rows``), read forward or, with ``reverse=True``, backward.  For
streams, ``prefill`` runs prompts and leaves one state per stream and head, and ``step`` advances any of
its slots by one token.

    mixer = RetentionMixer(128, heads=4).cuda()
    y = mixer(image_rows(x))                                  # training and whole sequences
    y, cache = mixer.prefill(rows, seq_offsets=offsets)       # ragged prompts
    y = mixer.step(token, cache, slots=slots)                 # one token of some of them
"""
from __future__ import annotations

import torch
from torch import nn

from .ssm_core import linear_attention, linear_attention_step
from .utils.group_norm import group_norm_rows


class RetentionMixer(nn.Module):
    """``out_proj(norm(attention(q, k, v)) * silu(gate))`` over token rows.

    dim: row width; heads * key_dim is dim by default and the values are expand * dim wide in all, both
    at most 128 a head.  windows: how many tokens the first and the last head remember; head h
    forgets by 1 - 1 / window, with windows spread evenly over their logarithm."""

    def __init__(self, dim: int, *, heads: int = 4, key_dim: int | None = None, expand: int = 2,
                 windows: tuple[float, float] = (4.0, 512.0), eps: float = 1e-5):
        super().__init__()
        if dim <= 0 or heads <= 0 or expand <= 0 or (expand * dim) % heads or (key_dim is None and dim % heads):
            raise ValueError("dim, heads and expand must be positive and heads divide dim and expand * dim")
        self.dim, self.heads, self.eps = int(dim), int(heads), float(eps)
        self.key_dim = dim // heads if key_dim is None else int(key_dim)
        self.value_dim = expand * dim // heads
        if not (1 <= self.key_dim <= 128 and self.value_dim <= 128):
            raise ValueError(f"keys and values of at most 128 a head, got {self.key_dim} and {self.value_dim}")
        if not 1.0 <= windows[0] <= windows[1]:
            raise ValueError("windows must be at least 1 and ascend")
        inner = heads * self.value_dim
        self.in_proj = nn.Linear(dim, 2 * heads * self.key_dim + 2 * inner, bias=False)
        self.norm_weight = nn.Parameter(torch.ones(inner))
        self.norm_bias = nn.Parameter(torch.zeros(inner))
        self.out_proj = nn.Linear(inner, dim, bias=False)
        low, high = (torch.tensor(w, dtype=torch.float64).log() for w in windows)
        window = torch.exp(low + (high - low) * torch.arange(heads, dtype=torch.float64) / max(1, heads - 1))
        self.register_buffer("log_decay", torch.log1p(-1.0 / window).float())

    def _split(self, x):
        """(q, k, v, gate) of rows x; views of one projection."""
        h, dk, dv = self.heads, self.key_dim, self.value_dim
        q, k, v, gate = self.in_proj(x).split((h * dk, h * dk, h * dv, h * dv), dim=-1)
        return q.unflatten(-1, (h, dk)), k.unflatten(-1, (h, dk)), v.unflatten(-1, (h, dv)), gate

    def _finish(self, o, gate):
        return self.out_proj(group_norm_rows(o.flatten(-2), self.heads, self.norm_weight, self.norm_bias, self.eps, gate=gate))

    def forward(self, x, *, seq_offsets=None, reverse=False):
        """Rows [B, L, dim] (or packed [T, dim] with ``seq_offsets``) -> rows of the same shape."""
        q, k, v, gate = self._split(x)
        return self._finish(linear_attention(q, k, v, self.log_decay, seq_offsets=seq_offsets, reverse=reverse), gate)

    def prefill(self, x, *, cache: torch.Tensor | None = None, seq_offsets=None):
        """As ``forward``, from ``cache`` (one slot per sequence) if given; also returns the cache after
        the last token of every sequence, fp32 [sequences, heads, key dim, value dim]."""
        q, k, v, gate = self._split(x)
        o, state = linear_attention(q, k, v, self.log_decay, initial_state=cache, return_final_state=True, seq_offsets=seq_offsets)
        return self._finish(o, gate), state

    def empty_cache(self, slots: int) -> torch.Tensor:
        """Zero states for ``slots`` streams."""
        return torch.zeros(slots, self.heads, self.key_dim, self.value_dim, dtype=torch.float32, device=self.log_decay.device)

    @torch.no_grad()
    def step(self, x, cache: torch.Tensor, *, slots=None):
        """One token [B, dim] of the streams in ``slots`` (int32 or int64 [B]; all slots in order without
        it) -> [B, dim]; the cache advances in place."""
        q, k, v, gate = self._split(x)
        return self._finish(linear_attention_step(q, k, v, self.log_decay, cache, slots=slots), gate)
