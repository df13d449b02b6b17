"""Mask logits of queries: what ``MaskMatchingFunction`` and the pairwise costs take,
made from the queries' mask embeddings and the images' feature maps.  No counterpart
in the reference, whose operators start at the mask logits."""
from __future__ import annotations

import torch

import mask_loss_amd  # noqa: F401  (registers the `mask_loss` extension)
import mask_loss


def mask_logits(queries, features, offsets=None):
    """Products of every image's queries with its feature map, differentiable in both
    (once, in reverse mode): the products of ``grouped_matmul`` with an image as a group.

    ``features``: (B, C, H, W).  ``queries``: (L, B, Q, C), every query of L layers,
    giving (L, B, Q, H, W); or (R, C) with ``offsets`` (B + 1,), int64, a set of its own
    size per image (matched queries, kept predictions): rows offsets[b] ..
    offsets[b + 1] are image b's, giving (R, H, W).  Rows in no image's set give
    zeros."""
    if torch.is_grad_enabled() and (queries.requires_grad or features.requires_grad):
        return mask_loss.mask_logits_autograd(queries, features, offsets)
    return mask_loss.mask_logits_forward(queries.contiguous(), features.contiguous(),
                                         None if offsets is None else offsets.contiguous())
