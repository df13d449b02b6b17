"""Rows on their way to their experts and back, around ``grouped_matmul``: expert numbers
sorted by expert, the tokens' rows at their experts' places, the experts' rows summed
back with weights, with their gradients.  No counterpart in the reference.

    order = sort_by_expert(ids, experts)             # (T, k) int64
    rows = to_experts(x, order)                      # (T, D) -> (T * k, D)
    rows = grouped_matmul(rows, w, order.offsets)    # expert e: rows offsets[e] .. offsets[e + 1]
    out = from_experts(rows, order, weights)         # -> (T, N)

An expert number outside 0 .. experts - 1 drops its assignment (a token over an expert's
capacity): its place, behind all experts', holds zeros, and it counts for no sum and no
gradient.  Nothing is read back to the host.  Gradients are not differentiated a second
time, and forward-mode derivatives raise.

An order that does not come from ``sort_by_expert`` has to name each place below
``offsets[experts]`` once in ``slots``: rows of places that it leaves out are uninitialised,
in ``to_experts`` and in the row gradient of ``from_experts``."""
from __future__ import annotations

from typing import NamedTuple

import torch

import mask_loss_amd  # noqa: F401  (registers the `mask_loss` extension)
import mask_loss


class ExpertOrder(NamedTuple):
    """order (T * k,): the assignments t * k + j by expert, those of one expert in their
    order, the dropped ones last.  slots (T, k): each assignment's place in it.  offsets
    (experts + 1,): each expert's first place, and the end of the last one's.  All int64."""
    order: torch.Tensor
    slots: torch.Tensor
    offsets: torch.Tensor


class ToExpertsFunction:
    """``apply(input, slots, offsets)``, a C++ autograd node."""

    @staticmethod
    def apply(input, slots, offsets):
        return mask_loss.to_experts_autograd(input, slots, offsets)


class FromExpertsFunction:
    """``apply(input, slots, offsets, weights)``, a C++ autograd node; weights may be None
    (ones)."""

    @staticmethod
    def apply(input, slots, offsets, weights=None):
        return mask_loss.from_experts_autograd(input, slots, offsets, weights)


def sort_by_expert(ids, experts):
    """The order of (T, k) int64 expert numbers by expert (at most 4,000 experts)."""
    return ExpertOrder(*mask_loss.sort_by_expert(ids, experts))


def to_experts(input, order):
    """Row ``order.slots[t, j]`` of the result (T * k, D) is ``input[t]``, for input (T, D) of
    any dtype (gradients: float32, bfloat16 or float16); zeros in the dropped places."""
    return mask_loss.to_experts(input, order.slots, order.offsets)


def from_experts(input, order, weights=None):
    """``sum_j weights[t, j] * input[order.slots[t, j]]`` for every token t, in float32 and
    rounded once; input (T * k, D), weights (T, k) in its dtype or float32, or None for
    ones."""
    return mask_loss.from_experts(input, order.slots, order.offsets, weights)
