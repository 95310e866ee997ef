"""The operators of attention over a node's neighbours in 64 bits on the CPU, from their definitions; derivatives by autograd."""

from __future__ import annotations

import torch

from lunaequivariance_b200.irreps import as_irreps


def layer_norm(x, irreps, weight=None, bias=None, eps=1e-5, normalization="component"):
    """Block by block: mean out (0e only), divided by the root of the mean square, times a weight per channel, plus a bias."""
    rows, at, channel, scalar = x.reshape(-1, x.shape[-1]), 0, 0, 0
    done = []
    for mul, ir in as_irreps(irreps).remove_zero_multiplicities():
        v = rows[:, at:at + mul * ir.dim].reshape(-1, mul, ir.dim)
        if ir.is_scalar():
            v = v - v.mean((1, 2), keepdim=True)
        power = (v * v).sum((1, 2), keepdim=True) / (mul * ir.dim if normalization == "component" else mul)
        v = v / torch.sqrt(power + eps)
        if weight is not None:
            v = v * weight[channel:channel + mul].reshape(1, mul, 1)
        if bias is not None and ir.is_scalar():
            v = v + bias[scalar:scalar + mul].reshape(1, mul, 1)
        done.append(v.reshape(-1, mul * ir.dim))
        at, channel, scalar = at + mul * ir.dim, channel + mul, scalar + (mul if ir.is_scalar() else 0)
    return torch.cat(done, 1).reshape(x.shape)


def distance_buckets(vec, boundaries):
    v, b = vec.double(), boundaries.double()
    squared = (v[..., 0] * v[..., 0] + v[..., 1] * v[..., 1]) + v[..., 2] * v[..., 2]
    return (b * b <= squared.unsqueeze(-1)).sum(-1).to(torch.int32)


def relative_bias(table, buckets):
    inside = (buckets >= 0) & (buckets < table.shape[0])
    return torch.where(inside.unsqueeze(-1), table[torch.where(inside, buckets, 0).long()], 0.0)


def graph_softmax(logits, dst, nodes, mask=None, table=None, buckets=None):
    """Node by node.  Rows without anything left are zeros, and nothing flows through what is masked."""
    flat = logits.ndim == 1
    z = logits.unsqueeze(-1) if flat else logits
    if table is not None:
        z = z + relative_bias(table, buckets)
    gone = torch.zeros(z.shape, dtype=torch.bool) if mask is None else (~mask).unsqueeze(-1).expand_as(z)
    gone = gone | (z.detach() == -float("inf"))
    z = torch.where(gone, 0.0, z)
    out = torch.zeros_like(z)
    counts = torch.bincount(dst.long(), minlength=nodes).tolist()
    rows, begin = [], 0
    for count in counts:
        if count:
            row, dead = z[begin:begin + count], gone[begin:begin + count]
            top = torch.where(dead, -float("inf"), row).amax(0, keepdim=True).detach()
            top = torch.where(top == -float("inf"), 0.0, top)
            e = torch.where(dead, 0.0, torch.exp(row - top))
            total = e.sum(0, keepdim=True)
            rows.append(e / torch.where(total == 0.0, 1.0, total))
            begin += count
    out = torch.cat(rows) if rows else out
    return out.squeeze(-1) if flat else out
