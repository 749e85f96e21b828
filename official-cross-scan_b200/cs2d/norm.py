"""Layer normalisation over the channels, with the SiLU gate that scan blocks put behind it.

    y = ((x - mean) / sqrt(var + eps) * weight + bias) * silu(gate)

in one pass each way, statistics and sums in float32.  Besides rows of tokens ``(..., dim)`` with contiguous channels it takes
channel-major images as the scans write them, seen through ``permute``: ``x = image.permute(0, 2, 3, 1)`` is read and its
gradient written in the image's own layout, without a transposed copy.
"""
from __future__ import annotations

from . import _lib


def layer_norm(x, weight=None, bias=None, gate=None, eps=1e-5):
    """Differentiable layer norm over the last dimension; ``y`` is contiguous, of the dtype of ``x``.

    ``x``: ``(..., dim)``, float32, float16 or bfloat16.  ``weight``, ``bias``: ``(dim,)``, float32 or the dtype of ``x``, or None.  ``gate``:
    the shape and dtype of ``x``, or None for no gate.  Other strides than those of token rows and channel-major images cost a copy.
    The gradients of ``weight`` and ``bias`` are sums over the rows in float32 and a fixed order: every result comes out
    with the same bits on every run.  No forward-mode derivative: an input with a tangent is refused.
    """
    return _lib.native().layer_norm(x, weight, bias, gate, float(eps))
