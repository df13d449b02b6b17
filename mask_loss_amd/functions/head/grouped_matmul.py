"""Products of ragged groups of rows with one matrix per group, with the gradients
of both: an image's queries times its feature map (``mask_logits``), or the rows
of an expert or a class times its weights.  No counterpart in the reference, whose
operators start at the mask logits.

Tensors are float32, bfloat16 or float16, input and weight alike; sums are float32
and rounded once.  Gradients are not differentiable a second time, and forward-mode
derivatives raise."""
from __future__ import annotations

import torch

import mask_loss_amd  # noqa: F401  (registers the `mask_loss` extension)
import mask_loss


class GroupedMatmulFunction:
    """``apply(input, weight, offsets, transposed)``, a C++ autograd node."""

    @staticmethod
    def apply(input, weight, offsets, transposed=False):
        return mask_loss.grouped_matmul_autograd(input, weight, offsets, bool(transposed))


def grouped_matmul(input, weight, offsets=None, transposed=False):
    """``input[r] @ weight[g % M]`` for every row r of group g.

    ``weight``: M matrices, (M, K, N), or (M, N, K) with ``transposed`` (as linear
    layers keep theirs).  With ``offsets`` (G + 1,), int64 on the input's device,
    ``input`` is (R, K) and group g its rows offsets[g] .. offsets[g + 1], possibly
    none; the result is (R, N).  Rows in no group, before the first or behind the
    last, give zeros and take no part in the gradients.  Without offsets ``input``
    is (G, n, K), n rows to a group, and the result (G, n, N).  G is a multiple of
    M: groups g, g + M, ... share a matrix, and its gradient is their sum.

    The offsets are read on the GPU only; they must not decrease (each is held to
    0 .. R and to at least the one before)."""
    if torch.is_grad_enabled() and (input.requires_grad or weight.requires_grad):
        return GroupedMatmulFunction.apply(input, weight, offsets, transposed)
    return mask_loss.grouped_matmul_forward(input.contiguous(), weight.contiguous(),
                                            None if offsets is None else offsets.contiguous(), bool(transposed))
