"""Layer norm over the last dimension, with the gradients of input, weight and
bias: the norm of a decoder's queries (L,B,Q,C) in front of their mask and class
logits.  No counterpart in the reference, whose operators start at the logits.

The output has the input's dtype (float32, bfloat16 or float16); weight and bias
have that dtype or are float32, and their gradients come back in their own.  The
statistics are float32.  Gradients are not differentiable a second time, and
forward-mode derivatives raise."""
from __future__ import annotations

import torch

import mask_loss_amd  # noqa: F401  (registers the `mask_loss` extension)
import mask_loss


class LayerNormFunction:
    """``apply(input, weight, bias, eps)``, a C++ autograd node; weight and bias may
    be None (ones, zeros)."""

    @staticmethod
    def apply(input, weight, bias, eps):
        return mask_loss.layer_norm_autograd(input, weight, bias, float(eps))


def layer_norm(input, weight=None, bias=None, eps=1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension of
    ``input`` (..., D), var being the mean squared deviation.  ``weight`` and
    ``bias``: (D,) or None."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (input, weight, bias)):
        return LayerNormFunction.apply(input, weight, bias, eps)
    return mask_loss.layer_norm_forward(input.contiguous(), None if weight is None else weight.contiguous(),
                                        None if bias is None else bias.contiguous(), float(eps))[0]
