"""Mask logits of queries: what ``MaskMatchingFunction`` and the pairwise costs take,
made from the queries' mask embeddings and the images' feature maps.  No counterpart
in the reference, whose operators start at the mask logits."""
from __future__ import annotations

from ..head.grouped_matmul import grouped_matmul


def mask_logits(queries, features, offsets=None):
    """Products of every image's queries with its feature map, differentiable in both.

    ``features``: (B, C, H, W).  ``queries``: (L, B, Q, C), every query of L layers,
    giving (L, B, Q, H, W); or (R, C) with ``offsets`` (B + 1,), a set of its own
    size per image (matched queries, kept predictions): rows offsets[b] ..
    offsets[b + 1] are image b's, giving (R, H, W).  Rows in no image's set give
    zeros (``grouped_matmul``)."""
    if features.dim() != 4:
        raise ValueError(f"features must be (B, C, H, W), got {tuple(features.shape)}")
    B, C, H, W = features.shape
    if queries.dim() != (4 if offsets is None else 2) or queries.shape[-1] != C:
        want = "(L, B, Q, C)" if offsets is None else "(R, C) with offsets"
        raise ValueError(f"queries must be {want} for features (B, C, H, W) = {tuple(features.shape)}, "
                         f"got {tuple(queries.shape)}")
    maps = features.flatten(2)
    if offsets is not None:
        if offsets.dim() != 1 or offsets.shape[0] != B + 1:
            raise ValueError(f"offsets must have shape (B + 1,) = ({B + 1},), got {tuple(offsets.shape)}")
        return grouped_matmul(queries, maps, offsets).unflatten(1, (H, W))
    L, Bq, Q, _ = queries.shape
    if Bq != B:
        raise ValueError(f"queries and features must have the same batch size, got {Bq} and {B}")
    if L * B == 0:  # no image, or no layer
        return queries.new_zeros(L, B, Q, H, W) * (queries.sum() + features.sum())
    return grouped_matmul(queries.flatten(0, 1), maps).view(L, B, Q, H, W)
