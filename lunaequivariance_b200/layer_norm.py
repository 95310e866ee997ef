"""``layer_norm``: layer norm over irreps, its configuration object and its custom ops.

Every block ``mul x l`` of a row is normalised alone: scalars (``0e``) lose their mean, every block is divided by
``sqrt(share * sum of squares + eps)`` and multiplied by one weight per channel, and scalars get one bias per channel.
``share`` is one over the elements of the block (``normalization="component"``) or over its channels (``"norm"``).
With the irreps of scalars alone, or their number, this is the layer norm of a radial or a readout network.

Float32, float64, bfloat16 and float16 on CUDA, sums in 32 bits (64 for float64); forward, backward and second order (a force
step differentiates the norm of its radial network twice); the sums of the weights' gradients are the same bits
for the same sizes, alignment of the tensors and device.
"""

from __future__ import annotations

import json
from functools import lru_cache

import torch

from . import _native
from .conv import is_compiling
from .irreps import Irreps, as_irreps

_NORMALIZATIONS = {"component": 0, "norm": 1}


class LayerNormConfig:
    """Static description of one layer norm: blocks, normalization and ``eps``."""

    def __init__(self, irreps, eps=1e-5, normalization="component"):
        if isinstance(irreps, int):
            if irreps < 1:
                raise ValueError("layer norm needs a positive number of scalars")
            irreps = Irreps([(irreps, (0, 1))])
        self.irreps = as_irreps(irreps).remove_zero_multiplicities()
        if not len(self.irreps):
            raise ValueError("layer norm needs nonempty irreps")
        if normalization not in _NORMALIZATIONS:
            raise ValueError("normalization must be component or norm")
        eps = float(eps)
        if not 0.0 <= eps < float("inf"):
            raise ValueError("eps must be finite and not negative")
        self.eps, self.normalization = eps, normalization
        self.dim = self.irreps.dim
        self.weight_numel = sum(mul for mul, _ in self.irreps)
        self.bias_numel = sum(mul for mul, ir in self.irreps if ir.is_scalar())
        self._descriptor = json.dumps([str(self.irreps), eps, normalization])
        self._holder = None

    def descriptor(self) -> str:
        return self._descriptor

    def holder(self):
        """This norm for the C++ launch path."""
        if self._holder is None:
            blocks = [(mul, ir.dim, int(ir.is_scalar())) for mul, ir in self.irreps]
            self._holder = _native.binding().Norm(blocks, _NORMALIZATIONS[self.normalization], self.eps)
        return self._holder

    def __getstate__(self):
        return dict(self.__dict__, _holder=None)


@lru_cache(maxsize=256)
def _config(irreps, eps, normalization) -> LayerNormConfig:
    return LayerNormConfig(irreps, eps, normalization)


@lru_cache(maxsize=256)
def _config_from_descriptor(descriptor: str) -> LayerNormConfig:
    return LayerNormConfig(*json.loads(descriptor))


def _mask(needs) -> int:
    return sum(1 << bit for bit, need in enumerate(needs) if need)


# ----------------------------------------------------------------------------------------------- custom ops


def _stats_like(x, blocks):
    dim = x.shape[-1]
    return x.new_empty((blocks, x.numel() // dim if dim else 0, 2),
                       dtype=torch.float64 if x.dtype == torch.float64 else torch.float32)


@torch.library.custom_op("lunaeq::layer_norm_forward", mutates_args=())
def layer_norm_forward_op(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None,
                          config: str) -> tuple[torch.Tensor, torch.Tensor]:
    return tuple(_native.binding().layer_norm_forward(_config_from_descriptor(config).holder(), x, weight, bias))


@layer_norm_forward_op.register_fake
def _(x, weight, bias, config):
    return (torch.empty_like(x, memory_format=torch.contiguous_format),
            _stats_like(x, len(_config_from_descriptor(config).irreps)))


@torch.library.custom_op("lunaeq::layer_norm_backward", mutates_args=(),
                         schema="(Tensor x, Tensor? weight, Tensor stats, Tensor g, bool[] needs, str config)"
                                " -> (Tensor?, Tensor?, Tensor?)")
def layer_norm_backward_op(x, weight, stats, g, needs, config):
    return tuple(_native.binding().layer_norm_backward(_config_from_descriptor(config).holder(), x, weight, stats, g,
                                                       _mask(needs)))


@layer_norm_backward_op.register_fake
def _(x, weight, stats, g, needs, config):
    op = _config_from_descriptor(config)
    return (torch.empty_like(x, memory_format=torch.contiguous_format) if needs[0] else None,
            x.new_empty(op.weight_numel) if needs[1] else None, x.new_empty(op.bias_numel) if needs[2] else None)


@torch.library.custom_op("lunaeq::layer_norm_double_backward", mutates_args=(),
                         schema="(Tensor x, Tensor? weight, Tensor stats, Tensor g, Tensor? rx, Tensor? rw, Tensor? rb,"
                                " bool[] needs, str config) -> (Tensor?, Tensor?, Tensor?)")
def layer_norm_double_backward_op(x, weight, stats, g, rx, rw, rb, needs, config):
    return tuple(_native.binding().layer_norm_double(_config_from_descriptor(config).holder(), x, weight, stats, g, rx,
                                                     rw, rb, _mask(needs)))


@layer_norm_double_backward_op.register_fake
def _(x, weight, stats, g, rx, rw, rb, needs, config):
    return tuple(torch.empty_like(t, memory_format=torch.contiguous_format) if need else None
                 for t, need in zip((x, x.new_empty(_config_from_descriptor(config).weight_numel), x), needs))


def _norm_setup(ctx, inputs, output):
    x, weight, bias, ctx.config = inputs
    ctx.save_for_backward(x, weight, output[1])
    ctx.mark_non_differentiable(output[1])
    ctx.set_materialize_grads(False)


def _norm_forward_backward(ctx, g, _):
    if g is None:
        return None, None, None, None
    x, weight, stats = ctx.saved_tensors
    return (*layer_norm_backward_op(x, weight, stats, g, list(ctx.needs_input_grad[:3]), ctx.config), None)


def _norm_backward_setup(ctx, inputs, output):
    x, weight, stats, g, _, ctx.config = inputs
    ctx.save_for_backward(x, weight, stats, g)
    ctx.set_materialize_grads(False)


def _norm_backward_backward(ctx, rx, rw, rb):
    if rx is None and rw is None and rb is None:
        return (None,) * 6
    x, weight, stats, g = ctx.saved_tensors
    needs = [ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.needs_input_grad[3]]
    hx, hw, hg = layer_norm_double_backward_op(x, weight, stats, g, rx, rw, rb, needs, ctx.config)
    return hx, hw, None, hg, None, None


layer_norm_forward_op.register_autograd(_norm_forward_backward, setup_context=_norm_setup)
layer_norm_backward_op.register_autograd(_norm_backward_backward, setup_context=_norm_backward_setup)


def layer_norm(x, irreps=None, weight=None, bias=None, *, eps=1e-5, normalization="component", config=None):
    """Normalise ``x[..., irreps.dim]`` block by block.

    ``irreps`` are irreps, a string, or a number of scalars; ``weight`` has one entry per channel of every block, ``bias``
    one per channel of the ``0e`` blocks, both of the type of ``x``, and both may be left out.  Pass a prepared
    ``config`` (:class:`LayerNormConfig`) instead of ``irreps``, ``eps`` and ``normalization`` to save their lookup.
    """
    if config is None:
        if irreps is None:
            raise TypeError("Supply irreps or a prepared config")
        config = _config(irreps if isinstance(irreps, (int, str, Irreps)) else as_irreps(irreps), eps, normalization)
    if is_compiling():
        return torch.ops.lunaeq.layer_norm_forward.default(x, weight, bias, config.descriptor())[0]
    return _native.binding().layer_norm(config.holder(), x, weight, bias)


__all__ = ["layer_norm", "LayerNormConfig"]
