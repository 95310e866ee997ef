"""The operators of attention over neighbours where their numbers meet: masks beside NaN, cotangents far from zero, sums of many runs."""

import pytest
import torch

import lunaequivariance_b200 as luna
from oracle import attention as oracle

pytestmark = pytest.mark.gpu
DEVICE = "cuda"
F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
INF, NAN = float("inf"), float("nan")


def step(dtype):
    return torch.finfo(dtype).eps / 2


def inner(dtype):
    return step(F64 if dtype == F64 else F32)


def graph_of(degrees, generator):
    dst = torch.repeat_interleave(torch.arange(len(degrees)), torch.tensor(degrees))
    src = torch.randint(len(degrees), (dst.numel(),), generator=generator)
    return luna.make_graph(src.to(DEVICE), dst.to(DEVICE), len(degrees)), dst


# Rows of a warp's part, of a warp that walks them, of a whole CTA, and cut ones.
ROWS = {"short": [6, 0, 9, 3] * 20, "warps": [60, 200, 33] * 4, "ctas": [700, 0, 1000, 999], "cut": [3, 2500, 0, 1024, 1025, 7]}


@pytest.mark.parametrize("dtype", [F32, F64, BF16, F16])
@pytest.mark.parametrize("heads", [1, 2, 3, 8, 40])
@pytest.mark.parametrize("rows", list(ROWS))
def test_what_is_masked_stays_zero_beside_what_is_no_number(rows, heads, dtype):
    """A NaN or an infinity in one head of a row makes that head of its other edges NaN, and nothing else."""
    generator = torch.Generator().manual_seed(heads)
    degrees = ROWS[rows]
    graph, dst = graph_of(degrees, generator)
    edges = dst.numel()
    mask = torch.rand(edges, generator=generator) < 0.6
    logits = torch.randn(edges, heads, generator=generator, dtype=F64).to(dtype)
    g = torch.randn(edges, heads, generator=generator, dtype=F64).to(dtype)
    bad = torch.zeros(len(degrees), heads, dtype=torch.bool)
    broken, begin = logits.clone(), 0
    for node, count in enumerate(degrees):
        there = mask[begin:begin + count].nonzero().flatten()
        if there.numel() and node % 3 != 2:
            head = node % heads
            broken[begin + there[-1], head] = NAN if node % 2 else INF
            bad[node, head] = True
        begin += count
    buckets = torch.where(mask, torch.randint(1, 4, (edges,), generator=generator), 0).to(torch.int32)  # bucket 0: masked edges only
    table = torch.randn(4, heads, generator=generator, dtype=F64).to(dtype)

    def run(z):
        z, t = z.to(DEVICE).requires_grad_(True), table.to(DEVICE).requires_grad_(True)
        alpha = luna.graph_softmax(z, graph, mask=mask.to(DEVICE), table=t, buckets=buckets.to(DEVICE))
        gz, gt = torch.autograd.grad(alpha, (z, t), g.to(DEVICE))
        return alpha.detach().cpu(), gz.cpu(), gt.cpu()

    clean, got = run(logits), run(broken)
    lost = bad[dst] & mask[:, None]
    for a, b in zip(got[:2], clean[:2]):
        assert a[lost].isnan().all()
        assert not a[~mask].any() and not a[~mask].isnan().any()
        fine = ~bad[dst] & mask[:, None]
        assert torch.equal(a[fine], b[fine])
    assert not got[2][0].any() and not got[2][0].isnan().any()
