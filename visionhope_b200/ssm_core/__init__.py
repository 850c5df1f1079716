"""Recurrent operators over token rows: a short causal convolution, a selective scan and linear
attention with a decay for each head.

    short_conv              causal convolution of 2 to 8 taps over token rows, forward and backward
    short_conv_step         the same for one token of a batch of cached streams
    ssm_scan                diagonal selective scan over token rows, forward and backward
    ssm_scan_step           the same for one token of a batch of cached streams
    linear_attention        matrix states with a decay for each head, forward and backward
    linear_attention_step   the same for one token of a batch of cached streams

Token rows are channels-last, ``[batch, length, channels]``, or packed ``[tokens, channels]`` with
``seq_offsets``; those of linear attention have heads, ``[..., heads, dim]``.  The kernels are in
``csrc/short_conv.cu``, ``csrc/ssm_scan.cu``, ``csrc/ssm_scan_bwd.cu`` and
``csrc/linear_attention.cu``; ``visionhope_b200.ssm_mixer`` and ``visionhope_b200.retention_mixer`` are
layers that run them.
"""
from .conv import short_conv, short_conv_step  # noqa: F401
from .linear import linear_attention, linear_attention_step  # noqa: F401
from .scan import ssm_scan, ssm_scan_step  # noqa: F401

__all__ = ["short_conv", "short_conv_step", "ssm_scan", "ssm_scan_step", "linear_attention",
           "linear_attention_step"]
