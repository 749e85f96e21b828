"""Gated linear recurrence over tokens: the scan of a sequence, where ``selective_scan_2d`` scans an image.

    h[t] = a[t] * h[t-1] + b[t],    y[t] = h[t]

per channel, with the factor ``a`` from the gate and the input term ``b`` from ``u``:

===========  ==========================  =====================
``form``     ``a``                       ``b`` if ``weighted``
===========  ==========================  =====================
"sigmoid"    ``1 / (1 + exp(-gate))``    ``(1 - a) * u``
"log"        ``exp(gate)``               ``(1 - a) * u``
"direct"     ``gate``                    ``(1 - a) * u``
===========  ==========================  =====================

and ``b = u`` otherwise.  The state is float32 throughout, whatever the type of ``u`` and ``gate``; ``y`` is rounded once
per element.  Factors above one are allowed as long as the product of 512 consecutive ones stays inside float32.
Results and gradients come out with the same bits on every run.  As everywhere in this package there is no CPU or
PyTorch fallback.
"""
from __future__ import annotations

from . import _lib

_FORMS = {"sigmoid": 0, "log": 1, "direct": 2}


def _form(form):
    try:
        return _FORMS[form]
    except (KeyError, TypeError):
        raise RuntimeError(f"form must be one of {', '.join(_FORMS)}; got {form!r}") from None


def gated_scan_1d(u, gate, h0=None, offsets=None, form="sigmoid", weighted=True):
    """Differentiable scan; returns ``(y, h_last)``.

    ``u, gate``: ``(batch, length, dim)``, float32, float16 or bfloat16, any strides (a channel stride other than 1 costs a
    copy).  ``h0``: float32 ``(batch, dim)`` or None (zeros).  ``h_last``: float32 ``(batch, dim)``, the state behind the last token,
    which is the ``h0`` of a call that goes on from there and the ``h`` of ``gated_scan_step``.

    With ``offsets`` (int32 or int64 on the GPU, ``(sequences + 1,)``, ascending) ``u, gate`` are ``(total, dim)`` and sequence ``s``
    is rows ``offsets[s]:offsets[s+1]``; ``h0`` and ``h_last`` are ``(sequences, dim)``.  Sequences may be empty: their state passes
    through.  What rows of no sequence hold (padding before the first or behind the last) does not matter, NaN included; ``y`` and the
    gradients are zero there.
    Offsets that do not ascend or leave the tensor are found on the GPU and reported by ``cs2d.device_status()``.

    Gradients go to ``u``, ``gate`` and ``h0``, from ``y`` and ``h_last``.  When nothing can ask for one, no state is kept.
    No forward-mode derivative: an input with a tangent is refused, here and in ``gated_scan_step``.
    """
    return _lib.native().gated_scan(u, gate, h0, offsets, _form(form), bool(weighted))


def gated_scan_step(u, gate, h, form="sigmoid", weighted=True):
    """One token of ``gated_scan_1d``: ``u, gate`` ``(batch, dim)``; ``h``, float32 ``(batch, dim)``, is updated in place.  Returns ``y``.

    Not differentiable.  The rows of ``h`` may be rows of a larger pool of states, but must not overlap.
    """
    return _lib.native().gated_step(u, gate, h, _form(form), bool(weighted))
