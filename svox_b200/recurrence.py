"""The gated linear recurrence along samples: scanned states, and samples composited to colours.

A ray that passes a sample of thickness ``g`` (density times length) keeps ``exp(-g)`` of what it
carried and takes ``1 - exp(-g)`` of the sample's value,

    h[t] = exp(-g[t]) h[t-1] + (1 - exp(-g[t])) x[t]

which is what the renderer accumulates inside its march (svox/csrc/rt_kernel.cu:261-316), here for
samples that the caller has chosen and evaluated, and for any sequence that is gated in this way.
No counterpart in the reference, whose users composite with tensor operations.
"""
from torch.autograd import forward_ad as _fwd

from . import csrc as _C

__all__ = ["gated_scan", "composite"]


def gated_scan(values, thickness, initial=None, offsets=None, reverse=False, premultiplied=False):
    """All states of the recurrence and the last one: ``(states, last)``.

    ``values`` is ``(B, T, C)``, or ``(N, C)`` with ``offsets`` ``(B + 1,)`` int64 for rows of any
    length (row b has the steps ``offsets[b]`` up to ``offsets[b + 1]``; none is fine), float32,
    bfloat16 or float16, with any strides.  ``thickness`` is ``(B, T)`` for all channels or
    ``(B, T, H)`` for H groups of ``C / H`` neighbouring ones (packed: ``(N,)``, ``(N, H)``), not
    negative, float32 or of the type of ``values``.  ``initial``, the state before the first step,
    broadcasts to ``(B, C)`` (zeros by default).  ``reverse`` runs from the last step of a row to the
    first.  ``premultiplied``: ``values`` are added as they are, without the factor
    ``1 - exp(-thickness)``.

    ``states`` is shaped and typed like ``values``; ``last``, ``(B, C)``, is float32, as is the state
    that is carried: pass it as ``initial`` to go on, one step at a time if need be.  Steps that no
    row covers have states and gradients of zero.  A step of no thickness adds nothing whatever its
    value (NaN included), and nothing from before a step of infinite thickness (of more than about 87,
    whose ``exp(-thickness)`` is 0 in 32 bits) gets past it; a state that is not a number gets past any
    other.

    Differentiable, once, with respect to ``values``, ``thickness`` and ``initial``.  Offsets are
    read on the device: one out of order or range is noticed by ``csrc.check_device_status()``, and
    the outputs are undefined then (all accesses stay within the arrays).
    """
    if _fwd._current_level >= 0:
        _C.refuse_tangents(values, thickness, initial)
    return _C.host().gated_scan(values, thickness, initial, offsets, reverse, premultiplied, True,
                                "initial")


def composite(values, thickness, background=None, offsets=None, premultiplied=False):
    """Samples of rays, front to back, to what is seen: ``(B, C)`` float32.

    The last state alone of :func:`gated_scan` run from the far end of each ray, where it starts as
    ``background`` (``(B, C)`` or what broadcasts to it; nothing by default).  Arguments and
    gradients as there; a ray without samples shows its background.  Behind samples that together
    leave nothing of the light in 32 bits (thicknesses of 87 and more), a value that is not finite may
    count or not, none of them being opaque by itself.
    """
    if _fwd._current_level >= 0:
        _C.refuse_tangents(values, thickness, background)
    return _C.host().gated_scan(values, thickness, background, offsets, True, premultiplied, False,
                                "background")
