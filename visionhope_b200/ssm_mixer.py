"""A token-row mixer on the selective state space operators.

``SelectiveMixer`` is the layer that the operators of ``visionhope_b200.ssm_core`` are for: an input
projection into a value and a gate, the short causal convolution with SiLU, projections of the
convolved rows into step, B and C, the selective scan with its gate, and an output projection.  The
projections are plain GEMMs; the convolution and the scan run on ``libvhope.so``.

Rows are ``[batch, length, dim]``, or packed ``[tokens, dim]`` with ``seq_offsets``.  The tokens of a
channels-last image are such rows without a copy (``image_rows``), read forward or, with
``reverse=True``, backward.  For streams, ``prefill`` runs prompts and leaves a ``MixerCache`` of two
small states per stream, and ``step`` advances any of its slots by one token.

    mixer = SelectiveMixer(128).cuda()
    y = mixer(image_rows(x))                                  # training and whole sequences
    y, cache = mixer.prefill(rows, seq_offsets=offsets)       # ragged prompts
    y = mixer.step(token, cache, slots=slots)                 # one token of some of them
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch
from torch import nn

from .ssm_core import short_conv, short_conv_step, ssm_scan, ssm_scan_step


class MixerCache(NamedTuple):
    """The states of a batch of streams: the last taps - 1 inputs of the convolution
    [slots, taps - 1, inner], and the scan's state, fp32 [slots, inner, states]."""

    conv: torch.Tensor
    scan: torch.Tensor


def image_rows(x: torch.Tensor) -> torch.Tensor:
    """The tokens of an image [B, C, H, W] in row-major order, [B, H * W, C]: a view of a
    channels-last tensor, a copy of another."""
    b, c, h, w = x.shape
    return x.permute(0, 2, 3, 1).reshape(b, h * w, c)


class SelectiveMixer(nn.Module):
    """``out_proj(scan(conv(value)) * silu(gate))`` over token rows.

    dim: row width; the inner width is expand * dim.  states: 4, 8, 16, 32 or 64 per inner channel.
    groups: groups of B and C.  step_range: the steps' softplus(bias) is initialised log-uniformly
    in it; the decay rates as -1, -2, ... -states."""

    def __init__(self, dim: int, *, expand: int = 2, states: int = 16, taps: int = 4, groups: int = 1,
                 step_rank: int | None = None, step_range: tuple[float, float] = (1e-3, 1e-1)):
        super().__init__()
        if dim <= 0 or expand <= 0 or groups <= 0 or (expand * dim) % groups:
            raise ValueError("dim, expand and groups must be positive and groups divide expand * dim")
        self.dim, self.inner = int(dim), int(expand * dim)
        self.states, self.taps, self.groups = int(states), int(taps), int(groups)
        self.step_rank = max(1, math.ceil(dim / 16)) if step_rank is None else int(step_rank)
        d, n = self.inner, self.states
        self.in_proj = nn.Linear(dim, 2 * d, bias=False)
        self.conv_weight = nn.Parameter(torch.empty(d, taps))
        self.conv_bias = nn.Parameter(torch.zeros(d))
        self.x_proj = nn.Linear(d, self.step_rank + 2 * groups * n, bias=False)
        self.step_proj = nn.Linear(self.step_rank, d, bias=False)
        self.step_bias = nn.Parameter(torch.empty(d))
        self.rate_log = nn.Parameter(torch.empty(d, n))  # A = -exp(rate_log)
        self.skip = nn.Parameter(torch.ones(d))
        self.out_proj = nn.Linear(d, dim, bias=False)
        self.step_range = step_range
        self.reset_parameters()

    @torch.no_grad()
    def reset_parameters(self):
        nn.init.uniform_(self.conv_weight, -self.taps ** -0.5, self.taps ** -0.5)
        self.conv_bias.zero_()
        nn.init.uniform_(self.step_proj.weight, -self.step_rank ** -0.5, self.step_rank ** -0.5)
        low, high = (math.log(v) for v in self.step_range)
        step = torch.exp(torch.rand_like(self.step_bias) * (high - low) + low)
        self.step_bias.copy_(step + torch.log(-torch.expm1(-step)))  # softplus of it is `step`
        rates = torch.arange(1, self.states + 1, dtype=torch.float32, device=self.rate_log.device)
        self.rate_log.copy_(rates.log().expand_as(self.rate_log))
        self.skip.fill_(1.0)

    def _scan_inputs(self, rows):
        """(step, B, C) of convolved rows [..., inner]."""
        r, n = self.step_rank, self.groups * self.states
        step, b, c = self.x_proj(rows).split((r, n, n), dim=-1)
        if self.groups > 1:
            b, c = (t.unflatten(-1, (self.groups, self.states)) for t in (b, c))
        return self.step_proj(step), b, c

    def _run(self, x, seq_offsets, reverse, cache, want_cache):
        value, gate = self.in_proj(x).chunk(2, dim=-1)
        value, conv = short_conv(value, self.conv_weight, self.conv_bias, activation="silu",
                                 initial_state=None if cache is None else cache.conv, return_final_state=True,
                                 seq_offsets=seq_offsets, reverse=reverse)
        step, b, c = self._scan_inputs(value)
        y, scan = ssm_scan(value, step, -torch.exp(self.rate_log.float()), b, c, self.skip, z=gate,
                           delta_bias=self.step_bias, delta_softplus=True,
                           initial_state=None if cache is None else cache.scan, return_final_state=True,
                           seq_offsets=seq_offsets, reverse=reverse)
        return self.out_proj(y), MixerCache(conv, scan) if want_cache else None

    def forward(self, x, *, seq_offsets=None, reverse=False):
        """Rows [B, L, dim] (or packed [T, dim] with ``seq_offsets``) -> rows of the same shape."""
        return self._run(x, seq_offsets, reverse, None, False)[0]

    def prefill(self, x, *, cache: MixerCache | None = None, seq_offsets=None):
        """As ``forward``, from ``cache`` (one slot per sequence) if given; also returns the cache
        after the last token of every sequence."""
        return self._run(x, seq_offsets, False, cache, True)

    def empty_cache(self, slots: int, dtype=None) -> MixerCache:
        """Zero states for ``slots`` streams; dtype: that of the projected rows (the parameters'
        by default; the autocast dtype under autocast)."""
        device = self.conv_weight.device
        if dtype is None:
            dtype = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else self.in_proj.weight.dtype
        return MixerCache(torch.zeros(slots, self.taps - 1, self.inner, dtype=dtype, device=device),
                          torch.zeros(slots, self.inner, self.states, dtype=torch.float32, device=device))

    @torch.no_grad()
    def step(self, x, cache: MixerCache, *, slots=None):
        """One token [B, dim] of the streams in ``slots`` (int32 or int64 [B]; all slots in order
        without it) -> [B, dim]; the cache advances in place."""
        value, gate = self.in_proj(x).chunk(2, dim=-1)
        value = short_conv_step(value, cache.conv, self.conv_weight, self.conv_bias, activation="silu", slots=slots)
        step, b, c = self._scan_inputs(value)
        y = ssm_scan_step(value, step, -torch.exp(self.rate_log.float()), b, c, cache.scan, self.skip, z=gate,
                          delta_bias=self.step_bias, delta_softplus=True, slots=slots)
        return self.out_proj(y)
