"""A learned bias by distance: ``distance_buckets`` and ``relative_bias``, with the gradient of its table.

A graph has no order in which one node follows another; what stands for the relative position of two nodes is their
edge vector.  Its length falls into one of the buckets between ascending boundaries, and every bucket has a learned row of a
table: a bias for each attention head (added to the logits by ``graph_softmax`` in one launch), or a weight for each
path and channel of a convolution.  Buckets of other quantities (bonds, hops) are int32 tensors of the caller's own.

The bias is constant within a bucket, so nothing flows back to the edge vectors.
"""

from __future__ import annotations

import torch

from . import _native
from .conv import is_compiling


@torch.library.custom_op("lunaeq::distance_buckets", mutates_args=())
def distance_buckets_op(vec: torch.Tensor, boundaries: torch.Tensor) -> torch.Tensor:
    return _native.binding().distance_buckets(vec, boundaries)


@distance_buckets_op.register_fake
def _(vec, boundaries):
    return vec.new_empty(vec.shape[:-1], dtype=torch.int32)


@torch.library.custom_op("lunaeq::relative_bias_forward", mutates_args=())
def relative_bias_forward_op(table: torch.Tensor, buckets: torch.Tensor) -> torch.Tensor:
    return _native.binding().relative_bias_forward(table, buckets)


@relative_bias_forward_op.register_fake
def _(table, buckets):
    return table.new_empty((*buckets.shape, table.shape[1]))


@torch.library.custom_op("lunaeq::relative_bias_backward", mutates_args=(),
                         schema="(Tensor g, Tensor buckets, SymInt num_buckets) -> Tensor")
def relative_bias_backward_op(g, buckets, num_buckets):
    return _native.binding().relative_bias_backward(g, buckets, num_buckets)


@relative_bias_backward_op.register_fake
def _(g, buckets, num_buckets):
    return g.new_empty((num_buckets, g.shape[-1]))


def _forward_setup(ctx, inputs, output):
    table, buckets = inputs
    ctx.num_buckets = table.shape[0]
    ctx.save_for_backward(buckets)


def _forward_backward(ctx, g):
    (buckets,) = ctx.saved_tensors
    return relative_bias_backward_op(g, buckets, ctx.num_buckets), None


def _backward_setup(ctx, inputs, output):
    ctx.save_for_backward(inputs[1])


def _backward_backward(ctx, r):
    (buckets,) = ctx.saved_tensors
    return relative_bias_forward_op(r, buckets), None, None


relative_bias_forward_op.register_autograd(_forward_backward, setup_context=_forward_setup)
relative_bias_backward_op.register_autograd(_backward_backward, setup_context=_backward_setup)


def distance_buckets(vec, boundaries):
    """The bucket of every vector ``vec[..., 3]``: how many of the ``boundaries`` are at most its length (int32).

    ``boundaries`` is an ascending tensor without negative numbers, of the type (float32 or float64) and on the device of
    ``vec``.  Lengths and boundaries are compared as squares in double precision.  A length that is no number is in
    bucket 0.
    """
    if is_compiling():
        return torch.ops.lunaeq.distance_buckets.default(vec.detach(), boundaries)
    return _native.binding().distance_buckets(vec, boundaries)


def relative_bias(table, buckets):
    """``table[buckets]`` for a table ``[buckets, heads]`` and int32 ``buckets`` of any shape.

    A bucket that is no row of the table (-1 marks an edge without a bias) gives zeros and adds nothing to the table's
    gradient, which is a sum without atomics: the same bits for the same sizes, alignment and device.  Sums are held in 32 bits, in 64 for
    float64.  Differentiable to any order.
    """
    if is_compiling():
        return torch.ops.lunaeq.relative_bias_forward.default(table, buckets)
    return _native.binding().relative_bias(table, buckets)


__all__ = ["distance_buckets", "relative_bias"]
