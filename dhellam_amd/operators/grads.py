"""The norm of a step's gradients and their clipping.

The reference leaves both to Megatron's optimiser; these operators follow its wrapper convention (``stream=None`` means the current
stream, trailing elapsed-ms return).  The norm stays on the device: nothing here synchronises.  The two halves are apart so that ranks
that hold parts of one model add up their ``sum_sq`` in between.
"""
from __future__ import annotations

from .. import _host, _lib
from ._util import issue


def grad_norm(grads, stream=None, profiling=False):
    """grads: tensors of any number, sizes and types (fp32, bf16, fp16), each filling its memory -> (sum_sq fp64 [1], ms), the sum
    of the squares of all elements, added in 64 bits and the same bits on every call.  Zero for an empty list."""
    return issue(_host.grad_norm, stream, profiling, list(grads))


def clip_grads(grads, sum_sq, max_norm, scale=1.0, out=None, stream=None, profiling=False):
    """out = factor * grads with norm = |scale| sqrt(sum_sq), factor = scale min(1, max_norm / (norm + 1e-6)); in place without ``out``.
    ``scale`` undoes a loss scale on the way; ``max_norm=inf`` clips nothing.  ``out``: a tensor for each gradient, of its layout and its
    type or fp32 (the optimiser's copies), memory of its own or the gradient itself.  Where the norm is not finite, or past fp32's
    largest number, the factor is 0 and zeros are written, whatever the gradients hold: such a step moves no weight.  Returns (found fp32 [2] on the device: norm, factor; ms)."""
    grads = list(grads)
    out = None if out is None else list(out)
    _lib.mark_written(*(grads if out is None else out))
    return issue(_host.grad_clip, stream, profiling, grads, sum_sq, float(max_norm), float(scale), out)
