"""Softmax over in-edges with a bias by buckets: forward, backward and second order against the definition in 64 bits."""

import pytest
import torch

import lunaequivariance_b200 as luna
from oracle import attention as oracle
from oracle import uvu_conv as oracle_conv

pytestmark = pytest.mark.gpu
DEVICE = "cuda"
F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
INF = float("inf")


def step(dtype):
    return torch.finfo(dtype).eps / 2


def degrees_of(kind, generator):
    if kind == "mixed":  # empty rows, single edges, rows about and beyond what a warp holds
        return [0, 1, 0, 2, 31, 32, 33, 0, 64, 65, 127, 300, 5, 0]
    if kind == "small":
        return torch.randint(0, 9, (150,), generator=generator).tolist()
    if kind == "long":  # rows that are cut into pieces, between others that are not
        return [3, 2500, 0, 1024, 1025, 7, 4097, 0]
    if kind == "one":
        return [1]
    if kind == "few":  # rows of several hundred edges: a CTA each
        return [700, 0, 1000, 999]
    return [40] * 25


def graph_of(degrees, generator):
    dst = torch.repeat_interleave(torch.arange(len(degrees)), torch.tensor(degrees))
    src = torch.randint(len(degrees), (dst.numel(),), generator=generator)
    return luna.make_graph(src.to(DEVICE), dst.to(DEVICE), len(degrees)), dst


def problem(kind, heads, buckets, masked, dtype, seed=0):
    generator = torch.Generator().manual_seed(seed)
    degrees = degrees_of(kind, generator)
    graph, dst = graph_of(degrees, generator)
    edges = dst.numel()
    rand = lambda *shape: torch.randn(*shape, generator=generator, dtype=F64).to(dtype)  # noqa: E731
    shape = (edges,) if heads is None else (edges, heads)
    p = dict(logits=2 * rand(*shape), g=rand(*shape), r=rand(*shape), table=None, buckets=None, mask=None, rt=None)
    if buckets:
        p["table"], p["rt"] = rand(buckets, heads or 1), rand(buckets, heads or 1)
        p["buckets"] = torch.randint(-1, buckets + 1, (edges,), generator=generator, dtype=torch.int32)
    if masked:
        p["mask"] = torch.rand(edges, generator=generator) >= masked
        p["mask"][:degrees[0] + degrees[1] if len(degrees) > 1 else 1] = False  # a row without anything
    return graph, dst, len(degrees), p


def derivatives(softmax, p):
    z, g = (p[k].clone().requires_grad_(True) for k in ("logits", "g"))
    t = None if p["table"] is None else p["table"].clone().requires_grad_(True)
    alpha = softmax(z, t)
    inputs = (z,) if t is None else (z, t)
    first = torch.autograd.grad(alpha, inputs, g, create_graph=True)
    second = torch.autograd.grad(first, (*inputs, g), (p["r"],) if t is None else (p["r"], p["rt"]))
    found = dict(alpha=alpha, gz=first[0], hz=second[0], hg=second[-1])
    if t is not None:
        found.update(gt=first[1], ht=second[1])
    # no graph is left behind: the autograd engine cannot capture a backward pass while an eager graph of the leaves lives
    return {k: v.detach() for k, v in found.items()}


def compare(got, want, p, dtype, degrees, what):
    """The rounding of each result, and of what it is made of.

    alpha is rounded to its type before the gradients are made of it: a relative error of a step, and of a step of the sums'
    type for the arithmetic: the logit's sum (its size times a step, in the exponent), the exponential (two), and the
    sums over a row (at most its edges, one after the other).  D = sum alpha g is as exact as the largest g, and every
    gradient multiplies alpha with differences of such sums; the second order has three of them.
    """
    inner = step(F64 if dtype == F64 else F32)
    span = float(p["logits"].double().abs().max()) + (0.0 if p["table"] is None else float(p["table"].double().abs().max())) if p["logits"].numel() else 0.0
    relative = inner * (4 * span + min(max(degrees, default=1), 64) + 30)
    coarse = relative + (step(dtype) if dtype in (BF16, F16) else 0.0)
    tiny = 2.0 ** -25 if dtype == F16 else 1e-40 if dtype != F64 else 1e-300
    g, r = p["g"].double().abs().max(), p["r"].double().abs().max() + (0 if p["rt"] is None else p["rt"].double().abs().max())
    alpha = want["alpha"].detach()
    bounds = {"alpha": relative * alpha, "gz": 4 * coarse * alpha * 2 * g, "hg": 4 * coarse * alpha * 2 * r,
              "hz": 24 * coarse * alpha * 2 * g * r}
    # the cotangents of the second order are themselves rounded results of the types: hz is made of d/dalpha
    for k, bound in bounds.items():
        extra = step(dtype) * (want[k].detach().abs() + (8 * alpha * g * r if k == "hz" else 0))
        over = (got[k].detach().cpu().double() - want[k].detach()).abs() / (bound + extra + tiny * (1 + (8 * g * r if k == "hz" else 2 * r + 2 * g)))
        assert got[k].dtype == dtype and got[k].shape == want[k].shape, (what, k)
        assert not over.numel() or over.max().item() <= 1.0, f"{what} {k}: {over.max().item():.3g} of what is allowed"
    for k, source in (("gt", "gz"), ("ht", "hz")):
        if k in want:  # sums of what the logits' gradient has, whose errors they may all have
            allowed = ((bounds[source] + step(dtype) * (want[source].detach().abs() + (8 * alpha * g * r if k == "ht" else 0)) + 4 * tiny * (1 + g * r)).sum()
                       + step(dtype) * want[k].detach().abs().max() + 200 * inner * want[source].detach().abs().sum())
            assert got[k].dtype == dtype and (got[k].detach().cpu().double() - want[k].detach()).abs().max() <= allowed, (what, k)


def check(kind, heads, buckets, masked, dtype, seed=0):
    graph, dst, nodes, p = problem(kind, heads, buckets, masked, dtype, seed)
    up = {k: None if v is None else v.to(DEVICE) for k, v in p.items()}
    wide = {k: v.double() if v is not None and v.is_floating_point() else v for k, v in p.items()}
    want = derivatives(lambda z, t: oracle.graph_softmax(z, dst, nodes, p["mask"], t, p["buckets"]), wide)
    got = derivatives(lambda z, t: luna.graph_softmax(z, graph, mask=up["mask"], table=t, buckets=up["buckets"]), up)
    compare(got, want, p, dtype, torch.bincount(dst, minlength=1).tolist(), f"{kind} {heads} heads")
    again = derivatives(lambda z, t: luna.graph_softmax(z, graph, mask=up["mask"], table=t, buckets=up["buckets"]), up)
    assert all(torch.equal(got[k], again[k]) for k in got)
    return graph, got


@pytest.mark.parametrize("dtype", [F32, F64, BF16, F16])
@pytest.mark.parametrize("heads,buckets,masked", [(None, 0, 0.0), (1, 16, 0.3), (2, 0, 0.1), (3, 5, 0.0), (4, 32, 0.5), (5, 0, 0.2), (8, 64, 0.125),
                                                  (12, 7, 0.0), (16, 300, 0.9), (33, 3, 0.0), (64, 0, 0.4), (200, 4, 0.1)])
@pytest.mark.parametrize("kind", ["mixed", "small", "even"])
def test_all_orders(kind, heads, buckets, masked, dtype):
    check(kind, heads, buckets, masked, dtype)


@pytest.mark.parametrize("dtype", [F32, F64, BF16])
@pytest.mark.parametrize("heads,buckets,masked", [(None, 4, 0.2), (3, 0, 0.0), (8, 32, 0.1), (40, 0, 0.0)])
@pytest.mark.parametrize("kind", ["long", "few", "one"])
def test_long_rows(kind, heads, buckets, masked, dtype):
    check(kind, heads, buckets, masked, dtype)


def test_rows_that_must_stay_whole():
    """A graph that refuses to be cut: one CTA or one warp walks the whole row."""
    for degrees in ([5000, 3, 0, 9], [5000] + [2] * 4000):
        generator = torch.Generator().manual_seed(1)
        dst = torch.repeat_interleave(torch.arange(len(degrees)), torch.tensor(degrees))
        whole = luna.make_graph(torch.zeros_like(dst).to(DEVICE), dst.to(DEVICE), len(degrees), split=False)
        logits = torch.randn(dst.numel(), 4, generator=generator, dtype=F64)
        want = oracle.graph_softmax(logits, dst, len(degrees))
        assert torch.allclose(luna.graph_softmax(logits.to(DEVICE), whole).cpu(), want, rtol=1e-12, atol=0)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_sums_by_bucket_are_not_made_of_rounded_parts(dtype):
    """Almost all edges of a row in one bucket: its gradient is what is left of sums that cancel, as exact as its own rounding."""
    generator = torch.Generator().manual_seed(3)
    graph, dst = graph_of([50] * 200, generator)
    buckets = (torch.rand(10_000, generator=generator) < 0.05).to(torch.int32)
    z, g = ((2 * torch.randn(10_000, 4, generator=generator, dtype=F64)).to(dtype) for _ in range(2))
    table = torch.randn(2, 4, generator=generator, dtype=F64).to(dtype)
    leaf = table.to(DEVICE).requires_grad_(True)
    got, = torch.autograd.grad(luna.graph_softmax(z.to(DEVICE), graph, table=leaf, buckets=buckets.to(DEVICE)), leaf, g.to(DEVICE))
    reference = table.double().requires_grad_(True)
    alpha = oracle.graph_softmax(z.double(), dst, 200, table=reference, buckets=buckets)
    want, = torch.autograd.grad(alpha, reference, g.double())
    # the rounding of the result, and 200 roundings in single precision of what is added up: alpha times twice the largest g
    allowed = step(dtype) * want.abs() + 200 * step(F32) * (alpha.detach() * 2 * g.double().abs().max()).sum(0)
    assert ((got.cpu().double() - want).abs() <= allowed).all()


def test_gradient_against_differences():
    for kind, buckets in (("mixed", 0), ("small", 6)):
        graph, _, _, p = problem(kind, 2, buckets, 0.2, F64)
        up = {k: None if v is None else v.to(DEVICE) for k, v in p.items()}
        inputs = [up["logits"].requires_grad_(True)] + ([up["table"].requires_grad_(True)] if buckets else [])
        call = lambda z, t=None: luna.graph_softmax(z, graph, mask=up["mask"], table=t, buckets=up["buckets"])  # noqa: E731, B023
        assert torch.autograd.gradcheck(call, inputs, fast_mode=True) and torch.autograd.gradgradcheck(call, inputs, fast_mode=True)


@pytest.mark.parametrize("dtype", [F32, BF16, F64])
def test_rows_without_anything(dtype):
    """Masked rows, rows of minus infinity, rows of the lowest number; NaN and infinities behind the mask."""
    degrees = [3, 2, 4, 0, 2, 3]
    graph, dst = graph_of(degrees, torch.Generator().manual_seed(0))
    low = torch.finfo(dtype).min
    logits = torch.tensor([1.0, float("nan"), 2.0, -INF, -INF, low, low, low, low, INF, -INF, 0.5, 0.5, float("nan")], dtype=F64).to(dtype)
    mask = torch.tensor([True, False, True, True, True, True, True, True, True, False, False, True, True, False])
    z = logits.to(DEVICE).requires_grad_(True)
    alpha = luna.graph_softmax(z, graph, mask=mask.to(DEVICE))
    got = alpha.detach().cpu().double()
    want = [1 / (1 + torch.e), 0.0, torch.e / (1 + torch.e), 0.0, 0.0, 0.25, 0.25, 0.25, 0.25, 0.0, 0.0, 0.5, 0.5, 0.0]
    assert torch.allclose(got, torch.tensor(want, dtype=F64), rtol=4 * step(dtype), atol=0)
    g = torch.tensor([1.0, float("nan"), -1.0, INF, float("nan"), 1.0, 2.0, 3.0, 4.0, float("nan"), INF, 1.0, 1.0, -INF], dtype=F64).to(dtype)
    gz, = torch.autograd.grad(alpha, z, g.to(DEVICE).requires_grad_(True), create_graph=True)
    assert gz.isfinite().all() and not gz.detach()[[1, 3, 4, 9, 10, 13]].any()
    hz, = torch.autograd.grad(gz, z, torch.ones_like(gz))
    assert hz.isfinite().all()


def test_infinities_that_are_not_masked():
    """What the definition makes of them: a row with an infinite logit or a NaN is NaN, other rows are as they were."""
    degrees = [2, 3, 2, 2000, 1500]
    graph, dst = graph_of(degrees, torch.Generator().manual_seed(0))
    logits = torch.randn(dst.numel(), device=DEVICE)
    clean = luna.graph_softmax(logits, graph)
    logits[1], logits[3], logits[1000] = INF, float("nan"), float("nan")
    got = luna.graph_softmax(logits, graph)
    rows = torch.tensor(degrees).cumsum(0).tolist()
    assert got[:5].isnan().all() and got[7:rows[3]].isnan().all()
    assert torch.equal(got[5:7], clean[5:7]) and torch.equal(got[rows[3]:], clean[rows[3]:])
    nan_only = torch.full((dst.numel(),), float("nan"), device=DEVICE)
    assert luna.graph_softmax(nan_only, graph).isnan().all()


def test_values_beyond_32_bits():
    """More than 2^31 logits: the last rows are what they are in a small graph."""
    nodes, degree, heads = 34_000, 1000, 64

    def run(nodes, logits, g):
        dst = torch.arange(nodes, device=DEVICE).repeat_interleave(degree)
        graph = luna.make_graph(torch.zeros_like(dst), dst, nodes)
        z = logits.requires_grad_(True)
        alpha = luna.graph_softmax(z, graph)
        return alpha.detach()[-2 * degree:], torch.autograd.grad(alpha, z, g)[0][-2 * degree:]

    generator = torch.Generator(device=DEVICE).manual_seed(0)
    tail, gtail = (torch.randn(5 * degree, heads, generator=generator, device=DEVICE).to(BF16) for _ in range(2))
    logits = torch.zeros(nodes * degree, heads, device=DEVICE, dtype=BF16)
    assert logits.numel() > 1 << 31
    g = torch.zeros_like(logits)
    logits[-5 * degree:], g[-5 * degree:] = tail, gtail
    for a, b in zip(run(nodes, logits, g), run(5, tail.clone(), gtail)):
        assert torch.equal(a, b)


def test_two_streams_at_once():
    """Calls that overlap share nothing."""
    graph, _, _, p = problem("even", 8, 16, 0.1, F32)
    long, _, _, q = problem("long", 8, 16, 0.1, F32)
    problems = [(graph, {k: None if v is None else v.to(DEVICE) for k, v in p.items()}),
                (long, {k: None if v is None else v.to(DEVICE) for k, v in q.items()})]

    def step(graph, p):
        return derivatives(lambda z, t: luna.graph_softmax(z, graph, mask=p["mask"], table=t, buckets=p["buckets"]), p)

    want = [step(*x) for x in problems]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in problems]
    found = []
    for _ in range(10):
        for stream, x in zip(streams, problems):
            with torch.cuda.stream(stream):
                found.append(step(*x))
    torch.cuda.synchronize()
    for i, f in enumerate(found):
        assert all(torch.equal(f[k], want[i % 2][k]) for k in f)


def test_memory_orders():
    generator = torch.Generator(device=DEVICE).manual_seed(0)
    graph, dst = graph_of([40] * 30, torch.Generator().manual_seed(0))
    flat = torch.randn(1 + 1200 * 8, generator=generator, device=DEVICE)
    want = luna.graph_softmax(flat[1:].reshape(1200, 8).clone(), graph)
    assert torch.allclose(luna.graph_softmax(flat[1:].reshape(1200, 8), graph), want, rtol=1e-6, atol=0)
    turned = flat[1:].reshape(8, 1200).t()
    assert torch.equal(luna.graph_softmax(turned, graph), luna.graph_softmax(turned.contiguous(), graph))
    z = flat[1:].reshape(1200, 8).clone().requires_grad_(True)
    mask = torch.ones(2400, dtype=torch.bool, device=DEVICE)[::2]
    alpha = luna.graph_softmax(z, graph, mask=mask)
    one, = torch.autograd.grad(alpha.sum(), z)  # an expanded cotangent: the sums of a row do not depend on the logits
    assert one.abs().max().item() <= 64 * step(F32)


@pytest.mark.parametrize("kind", ["even", "long"])
def test_streams_and_captured_graphs(kind):
    graph, dst, nodes, p = problem(kind, 4, 8, 0.1, F32)
    p = {k: None if v is None else v.to(DEVICE) for k, v in p.items()}
    call = lambda z, t: luna.graph_softmax(z, graph, mask=p["mask"], table=t, buckets=p["buckets"])  # noqa: E731
    eager = derivatives(call, p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        aside = derivatives(call, p)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(eager[k], aside[k]) for k in eager)
    graphs = []
    for _ in range(2):
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            found = derivatives(call, p)
        graphs.append((captured, found))
    _, _, _, new = problem(kind, 4, 8, 0.1, F32, 5)
    for k, v in new.items():
        if v is not None and p[k].shape == v.shape:
            p[k].copy_(v)
    want = derivatives(call, p)
    for captured, _ in graphs:
        captured.replay()
    for _, found in graphs:
        assert all(torch.equal(found[k], want[k]) for k in want)


@pytest.mark.parametrize("dtype", [F64, BF16])
def test_custom_ops(dtype):
    graph, _, _, p = problem("small", 3, 6, 0.2, dtype)
    p = {k: None if v is None else v.to(DEVICE) for k, v in p.items()}
    ops = lambda z, t: torch.ops.lunaeq.graph_softmax_forward(z, t, p["buckets"], p["mask"], graph.dst_rowptr, graph.num_edges)[0]  # noqa: E731
    own = lambda z, t: luna.graph_softmax(z, graph, mask=p["mask"], table=t, buckets=p["buckets"])  # noqa: E731
    want, got = derivatives(own, p), derivatives(ops, p)
    assert all(torch.equal(got[k], want[k]) for k in want)
    traced = torch.compile(own, fullgraph=True)
    z, t = p["logits"].clone().requires_grad_(True), p["table"].clone().requires_grad_(True)
    alpha = traced(z, t)
    assert torch.equal(alpha, want["alpha"])
    assert all(torch.equal(a, want[k]) for k, a in zip(("gz", "gt"), torch.autograd.grad(alpha, (z, t), p["g"])))
    torch.library.opcheck(torch.ops.lunaeq.graph_softmax_forward.default,
                          (z, t, p["buckets"], p["mask"], graph.dst_rowptr, graph.num_edges))


def test_parts_of_the_gradient():
    """The table's gradient alone, the logits' alone, the second order with the table's cotangent alone."""
    graph, dst, nodes, p = problem("mixed", 4, 6, 0.2, F64)
    up = {k: None if v is None else v.to(DEVICE) for k, v in p.items()}
    whole = derivatives(lambda z, t: luna.graph_softmax(z, graph, mask=up["mask"], table=t, buckets=up["buckets"]), up)
    for name, k in (("logits", "gz"), ("table", "gt")):
        t = {n: up[n].clone().requires_grad_(n == name) for n in ("logits", "table")}
        alpha = luna.graph_softmax(t["logits"], graph, mask=up["mask"], table=t["table"], buckets=up["buckets"])
        g, = torch.autograd.grad(alpha, t[name], up["g"])
        assert torch.equal(g, whole[k])
    for softmax, q in ((lambda z, t: luna.graph_softmax(z, graph, mask=up["mask"], table=t, buckets=up["buckets"]), up),
                       (lambda z, t: oracle.graph_softmax(z, dst, nodes, p["mask"], t, p["buckets"]), p)):
        z, t = q["logits"].clone().requires_grad_(True), q["table"].clone().requires_grad_(True)
        gt, = torch.autograd.grad(softmax(z, t), t, q["g"], create_graph=True)
        found = torch.autograd.grad(gt, (z, t), q["rt"])
        if q is up:
            got = found
    for a, b in zip(got, found):
        # sums of up to a thousand terms of alpha g r: far within a thousand roundings of the largest
        assert (a.cpu() - b).abs().max().item() <= 1000 * step(F64) * 100


def test_attention_with_a_convolution():
    """Norm of the features, logits, bias by distance, softmax, and the messages' sum: energy, forces, and a force loss."""
    generator = torch.Generator().manual_seed(4)
    nodes, edges = 20, 160
    dst = torch.sort(torch.randint(nodes, (edges,), generator=generator))[0]
    src = torch.randint(nodes, (edges,), generator=generator)
    irreps = "8x0e+8x1o"
    instructions = [(0, 0, 0, "uvu", True), (1, 1, 0, "uvu", True), (0, 1, 1, "uvu", True), (1, 0, 1, "uvu", True)]
    rand = lambda *shape: torch.randn(*shape, generator=generator, dtype=F64)  # noqa: E731
    pos, x, mix, weight = 2 * rand(nodes, 3), rand(nodes, 32), rand(8, 1), rand(edges, 32)
    table, gain, shift = rand(5, 1), 1 + 0.1 * rand(16), rand(8)
    borders = torch.tensor([0.5, 1.5, 2.5, 4.0], dtype=F64)
    conv = luna.TensorProductConv(irreps, "1x0e+1x1o", irreps, instructions, internal_weights=False, shared_weights=False, dtype=F64)
    meta = oracle_conv.build_specs(irreps, "1x0e+1x1o", irreps, instructions)
    from oracle import spherical_harmonics as oracle_sh

    def loss(norm, harmonics, bucketed, softmax, convolve, tensors):
        pos, x, mix, weight, table, gain, shift, src, dst, borders = tensors
        vec = pos[src] - pos[dst]
        h = norm(x, gain, shift)
        logits = (h[src, :8] * h[dst, :8]) @ mix - vec.square().sum(1, keepdim=True) / 8
        alpha = softmax(logits, table, bucketed(vec.detach(), borders))
        out = convolve(h, harmonics(vec), weight * alpha)
        energy = (out ** 2).sum() / 100
        force, = torch.autograd.grad(energy, pos, create_graph=True)
        total = energy + (force ** 2).sum() / 100
        return (energy, force, *torch.autograd.grad(total, (x, mix, weight, table, gain, shift)))

    def leaves(device):
        return [t.to(device).clone().requires_grad_(True) for t in (pos, x, mix, weight, table, gain, shift)] + [
            t.to(device) for t in (src, dst, borders)]

    graph = conv.create_graph(src.to(DEVICE), dst.to(DEVICE), nodes)
    got = loss(lambda x, w, b: luna.layer_norm(x, irreps, w, b), lambda v: luna.spherical_harmonics([0, 1], v, True, "component"),
               luna.distance_buckets, lambda z, t, b: luna.graph_softmax(z, graph, table=t, buckets=b),
               lambda x, y, w: conv(x, y, w, graph=graph), leaves(DEVICE))
    want = loss(lambda x, w, b: oracle.layer_norm(x, irreps, w, b), lambda v: oracle_sh.spherical_harmonics((0, 1), v, True, "component"),
                oracle.distance_buckets, lambda z, t, b: oracle.graph_softmax(z, dst, nodes, None, t, b),
                lambda x, y, w: oracle_conv.conv_forward(meta, x, y, w, src, dst, nodes), leaves("cpu"))
    for k, a, b in zip(("energy", "force", "x", "mix", "weight", "table", "gain", "shift"), got, want):
        # the package's bound for chains in double precision
        assert (a.cpu() - b).abs().max().item() <= 1e-11 * max(b.abs().max().item(), 1.0), k
    # one head's softmax as the envelope of the messages
    env = luna.graph_softmax(torch.randn(edges, device=DEVICE, dtype=F64), graph)
    y = luna.spherical_harmonics([0, 1], torch.randn(edges, 3, device=DEVICE, dtype=F64), True, "component")
    w, feats = weight.to(DEVICE), x.to(DEVICE)
    assert torch.allclose(conv(feats, y, w, graph=graph, env=env), conv(feats, y, w * env[:, None], graph=graph), rtol=1e-11, atol=1e-11)


def test_refusals():
    graph, _ = graph_of([2, 3], torch.Generator().manual_seed(0))
    z = torch.zeros(5, 2, device=DEVICE)
    buckets = torch.zeros(5, dtype=torch.int32, device=DEVICE)
    for bad in (z[:4], z[:, :0], z.unsqueeze(0)):
        with pytest.raises(ValueError, match="shape"):
            luna.graph_softmax(bad, graph)
    with pytest.raises(TypeError, match="float32"):
        luna.graph_softmax(z.int(), graph)
    with pytest.raises(TypeError, match="mask"):
        luna.graph_softmax(z, graph, mask=buckets)
    with pytest.raises(ValueError, match="mask"):
        luna.graph_softmax(z, graph, mask=torch.ones(4, dtype=torch.bool, device=DEVICE))
    with pytest.raises(ValueError, match="table"):
        luna.graph_softmax(z, graph, table=torch.zeros(3, 1, device=DEVICE), buckets=buckets)
    with pytest.raises(TypeError, match="table"):
        luna.graph_softmax(z, graph, table=torch.zeros(3, 2, device=DEVICE, dtype=F64), buckets=buckets)
    with pytest.raises(TypeError, match="buckets"):
        luna.graph_softmax(z, graph, table=torch.zeros(3, 2, device=DEVICE), buckets=buckets.long())
    with pytest.raises(ValueError, match="buckets"):
        luna.graph_softmax(z, graph, table=torch.zeros(3, 2, device=DEVICE), buckets=buckets[:4])
    with pytest.raises(ValueError, match="share one CUDA device"):
        luna.graph_softmax(z, luna.make_graph(torch.zeros(5).int(), torch.zeros(5).int(), 1))
    leaf = z.clone().requires_grad_(True)
    g, = torch.autograd.grad(luna.graph_softmax(leaf, graph).square().sum(), leaf, create_graph=True)
    h, = torch.autograd.grad(g.square().sum(), leaf, create_graph=True)
    with pytest.raises(NotImplementedError, match="third-order"):
        torch.autograd.grad(h.sum(), leaf)


def test_no_edges():
    graph = luna.make_graph(torch.zeros(0, dtype=torch.int64, device=DEVICE), torch.zeros(0, dtype=torch.int64, device=DEVICE), 4)
    z = torch.zeros(0, 3, device=DEVICE, requires_grad=True)
    t = torch.zeros(5, 3, device=DEVICE, requires_grad=True)
    alpha = luna.graph_softmax(z, graph, table=t, buckets=torch.zeros(0, dtype=torch.int32, device=DEVICE))
    gz, gt = torch.autograd.grad(alpha, (z, t), torch.zeros(0, 3, device=DEVICE))
    assert alpha.shape == gz.shape == (0, 3) and not gt.any()
