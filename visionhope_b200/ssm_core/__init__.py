"""Selective state space operators: a short causal convolution and a selective scan.

    short_conv        causal convolution of 2 to 8 taps over token rows, forward and backward
    short_conv_step   the same for one token of a batch of cached streams
    ssm_scan          diagonal selective scan over token rows, forward and backward
    ssm_scan_step     the same for one token of a batch of cached streams

Token rows are channels-last, ``[batch, length, channels]``, or packed ``[tokens, channels]`` with
``seq_offsets``.  The kernels are in ``csrc/short_conv.cu``, ``csrc/ssm_scan.cu`` and
``csrc/ssm_scan_bwd.cu``; ``visionhope_b200.ssm_mixer`` is a layer that runs all four.
"""
from .conv import short_conv, short_conv_step  # noqa: F401
from .scan import ssm_scan, ssm_scan_step  # noqa: F401

__all__ = ["short_conv", "short_conv_step", "ssm_scan", "ssm_scan_step"]
