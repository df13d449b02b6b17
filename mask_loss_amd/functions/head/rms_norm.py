"""Root-mean-square norm over the last dimension with the residual's addition in front
of it, with the gradients of input, residual and weight, and with an output in
microscaled values for the products behind it.  No counterpart in the reference, whose
operators start at the logits.

Outputs have the input's dtype (float32, bfloat16 or float16), the weight that dtype or
float32, and its gradient its own.  The statistics are float32.  Gradients are not
differentiated a second time, and forward-mode derivatives raise."""
from __future__ import annotations

import mask_loss_amd  # noqa: F401  (registers the `mask_loss` extension)
import mask_loss


class RMSNormFunction:
    """``apply(input, weight, eps, residual)``, a C++ autograd node; weight and residual
    may be None."""

    @staticmethod
    def apply(input, weight=None, eps=1e-6, residual=None):
        out = mask_loss.rms_norm_autograd(input, weight, residual, eps)
        return out[0] if residual is None else tuple(out)


def rms_norm(input, weight=None, eps=1e-6, residual=None):
    """``s / sqrt(mean(s ** 2) + eps) * weight`` over the last dimension of ``input``
    (..., D); ``weight``: (D,) or None.

    Without a residual s is the input and the result the norm.  With a ``residual`` of the
    input's shape and dtype s is their sum, rounded to that dtype, and the result is
    (norm, s): s is the residual of the next layer, and its gradient comes back
    through both."""
    out = mask_loss.rms_norm(input, weight, residual, eps)
    return out[0] if residual is None else (out[0], out[1])


def rms_norm_mx(input, weight=None, eps=1e-6, residual=None, format="e4m3"):
    """``rms_norm`` whose norm comes out quantised from float32, as ``mx_quantize``
    does it: (codes, scales), or (codes, scales, s) with a residual.  D is a multiple of 32.
    For inference: no gradient is provided."""
    codes, scales, s = mask_loss.rms_norm_mx_forward(input, weight, residual, eps, format)
    return (codes, scales) if residual is None else (codes, scales, s)
