"""Microscaled values (the OCP microscaling formats) for inference: 32 consecutive values
of a row share a power of two.  No counterpart in the reference.

Values are kept as ``e2m1`` (4 bits: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives, two to a
byte of a uint8 tensor, the first in the low bits) or ``e4m3`` (``torch.float8_e4m3fn``), scales
as ``torch.float8_e8m0fnu``, one for 32 values."""
from __future__ import annotations

import mask_loss_amd  # noqa: F401  (registers the `mask_loss` extension)
import mask_loss


def mx_quantize(input, format="e4m3"):
    """(codes, scales) of ``input`` (..., D), D a multiple of 32: codes (..., D), or (..., D / 2)
    for e2m1, scales (..., D / 32).

    A scale brings its block's largest magnitude into the format's last binade
    (2^(floor(log2 max) - 2) for e2m1, - 8 for e4m3); values are divided by it, rounded to
    nearest, ties to even, and held to the format's largest.  A block with a NaN or an infinity has the
    scale NaN and reads as NaN.  No gradient is provided."""
    return tuple(mask_loss.mx_quantize(input.contiguous(), format))
