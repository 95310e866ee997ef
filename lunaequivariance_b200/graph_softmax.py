"""``graph_softmax``: softmax over the in-edges of every node, with a learned bias by buckets added on the way.

The logits of an edge are one number per attention head, in the edge order of a graph (sorted by destination).  The result
with one head is the ``env`` of a convolution: attention over a node's neighbours is a convolution whose messages are
scaled by it.  Forward, backward (logits and bias table) and second order, without atomics.
"""

from __future__ import annotations

import torch

from . import _native
from .conv import is_compiling
from .graph import LunaTPGraph


def _mask(needs) -> int:
    return sum(1 << bit for bit, need in enumerate(needs) if need)


# ----------------------------------------------------------------------------------------------- custom ops
# A traced program carries the row pointers alone: rows are not cut, however long.


def _rows(rowptr, edges):
    return _native.binding().Rows(rowptr, edges, None, None, None, None)


def _narrow(t):
    return t.dtype in (torch.bfloat16, torch.float16)


@torch.library.custom_op("lunaeq::graph_softmax_forward", mutates_args=(),
                         schema="(Tensor logits, Tensor? table, Tensor? buckets, Tensor? mask, Tensor rowptr, SymInt edges)"
                                " -> (Tensor, Tensor)")
def graph_softmax_forward_op(logits, table, buckets, mask, rowptr, edges):
    """The result, and for 16-bit types the result before it was rounded (else nothing).

    The second order's cotangent of a 16-bit result comes back through the latter: its rounding would count many times."""
    alpha, wide = _native.binding().graph_softmax_forward(_rows(rowptr, edges), logits, table, buckets, mask)
    return alpha, logits.new_empty(0, dtype=torch.float32) if wide is None else wide


@graph_softmax_forward_op.register_fake
def _(logits, table, buckets, mask, rowptr, edges):
    alpha = torch.empty_like(logits, memory_format=torch.contiguous_format)
    return alpha, alpha.new_empty(alpha.shape if _narrow(logits) else (0,), dtype=torch.float32)


@torch.library.custom_op("lunaeq::graph_softmax_backward", mutates_args=(),
                         schema="(Tensor alpha, Tensor wide, Tensor g, Tensor? buckets, SymInt num_buckets, Tensor rowptr,"
                                " bool[] needs) -> (Tensor?, Tensor?)")
def graph_softmax_backward_op(alpha, wide, g, buckets, num_buckets, rowptr, needs):
    return tuple(_native.binding().graph_softmax_backward(_rows(rowptr, alpha.shape[0]), alpha, wide, g, buckets,
                                                          num_buckets, _mask(needs)))


@graph_softmax_backward_op.register_fake
def _(alpha, wide, g, buckets, num_buckets, rowptr, needs):
    heads = alpha.shape[1] if alpha.ndim == 2 else 1
    return (torch.empty_like(alpha, memory_format=torch.contiguous_format) if needs[0] else None,
            alpha.new_empty((num_buckets, heads)) if needs[1] else None)


@torch.library.custom_op("lunaeq::graph_softmax_double_backward", mutates_args=(),
                         schema="(Tensor alpha, Tensor wide, Tensor g, Tensor? buckets, Tensor? r, Tensor? rtable, Tensor rowptr,"
                                " bool[] needs) -> (Tensor?, Tensor?)")
def graph_softmax_double_backward_op(alpha, wide, g, buckets, r, rtable, rowptr, needs):
    return tuple(_native.binding().graph_softmax_double(_rows(rowptr, alpha.shape[0]), alpha, wide, g, buckets, r, rtable,
                                                        _mask(needs)))


@graph_softmax_double_backward_op.register_fake
def _(alpha, wide, g, buckets, r, rtable, rowptr, needs):
    return (torch.empty_like(alpha, dtype=torch.float32 if _narrow(alpha) else None, memory_format=torch.contiguous_format) if needs[0] else None,
            torch.empty_like(g, memory_format=torch.contiguous_format) if needs[1] else None)


def _forward_setup(ctx, inputs, output):
    _, table, buckets, _, rowptr, _ = inputs
    ctx.num_buckets = 0 if table is None else table.shape[0]
    ctx.save_for_backward(*output, buckets, rowptr)
    if not _narrow(output[0]):
        ctx.mark_non_differentiable(output[1])
    ctx.set_materialize_grads(False)


def _forward_backward(ctx, g, wide_g):
    if wide_g is not None:
        g = wide_g if g is None else wide_g + g
    if g is None:
        return (None,) * 6
    alpha, wide, buckets, rowptr = ctx.saved_tensors
    needs = [ctx.needs_input_grad[0], bool(ctx.num_buckets) and ctx.needs_input_grad[1]]
    return (*graph_softmax_backward_op(alpha, wide, g, buckets, ctx.num_buckets, rowptr, needs), None, None, None, None)


def _backward_setup(ctx, inputs, output):
    alpha, wide, g, buckets, _, rowptr, _ = inputs
    ctx.save_for_backward(alpha, wide, g, buckets, rowptr)
    ctx.set_materialize_grads(False)


def _backward_backward(ctx, r, rtable):
    if r is None and rtable is None:
        return (None,) * 7
    alpha, wide, g, buckets, rowptr = ctx.saved_tensors
    widened = _narrow(alpha) and wide.numel() > 0  # what the launches read in the place of alpha
    needs = [ctx.needs_input_grad[1 if widened else 0], ctx.needs_input_grad[2]]
    halpha, hg = graph_softmax_double_backward_op(alpha, wide, g, buckets, r, rtable, rowptr, needs)
    if widened:
        return None, halpha, hg, None, None, None, None
    return None if halpha is None else halpha.to(alpha.dtype), None, hg, None, None, None, None


graph_softmax_forward_op.register_autograd(_forward_backward, setup_context=_forward_setup)
graph_softmax_backward_op.register_autograd(_backward_backward, setup_context=_backward_setup)


def graph_softmax(logits, graph, *, mask=None, table=None, buckets=None):
    """Softmax of ``logits[edges]`` or ``logits[edges, heads]`` over the in-edges of every node of ``graph``.

    ``table[buckets, heads]`` (of the type of the logits) and ``buckets[edges]`` (int32, as from ``distance_buckets``)
    add a learned bias to the logits; a bucket that is no row of the table adds nothing.  ``mask[edges]`` (bool) keeps the
    edges that are ``True``; what stands in the others' logits does not matter, and their result is zero.  A node whose
    edges are all masked, or have logits of minus infinity only, gets zeros.  Where the result is zero nothing flows back.

    Of a gradient's gradient, what is asked for with respect to the result itself leaves out a constant of a node's edges, which the
    softmax takes out behind it; in 16-bit types it reaches the logits from the result before it was rounded, past the result.

    The first call with a graph reads its largest degree, and makes tables if a node has very many in-edges.  It waits for the
    GPU; make it before a CUDA graph is captured (``graph.row_holder()`` does that and nothing else).  Traced programs carry the
    row pointers alone, and walk a node's edges in one warp or one block, however many: graphs with hubs are faster in eager calls.
    """
    if not isinstance(graph, LunaTPGraph):
        raise TypeError("graph must come from make_graph")
    if (table is None) != (buckets is None):
        raise TypeError("a bias table and the edges' buckets come together")
    if is_compiling():
        return torch.ops.lunaeq.graph_softmax_forward.default(logits, table, buckets, mask, graph.dst_rowptr,
                                                              graph.num_edges)[0]
    if not logits.is_cuda:
        raise RuntimeError("CUDA is required for the softmax over in-edges in this library")
    if graph.src.device != logits.device and graph.num_edges:
        raise ValueError("logits and graph must share one CUDA device")
    return _native.binding().graph_softmax(graph.row_holder(), logits, table, buckets, mask)


__all__ = ["graph_softmax"]
