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


def softmax_orders(softmax, z, t, g, r, rt):
    z, t, g = (v.clone().requires_grad_(True) for v in (z, t, g))
    alpha = softmax(z, t)
    gz, gt = torch.autograd.grad(alpha, (z, t), g, create_graph=True)
    hz, ht, hg = torch.autograd.grad((gz, gt), (z, t, g), (r, rt))
    return {k: v.detach() for k, v in dict(alpha=alpha, gz=gz, gt=gt, hz=hz, ht=ht, hg=hg).items()}


@pytest.mark.parametrize("dtype,shift,spread", [(BF16, 0, 1), (BF16, 3, 1), (BF16, 10, 1), (BF16, 0, 300), (F16, 0, 100), (F16, 100, 30), (F16, 10, 1),
                                                (F32, 0, 1), (F32, 1e5, 1), (F64, 1e6, 1)])
@pytest.mark.parametrize("rows,heads", [("short", 3), ("warps", 8), ("warps", 1), ("ctas", 4), ("cut", 2)])
def test_second_order_of_the_softmax_far_from_zero(rows, heads, dtype, shift, spread):
    """Cotangents that are far from zero, or large: the second order is made of their distances from the row's means.

    With D, R the means of g and r by alpha, sg, sr the largest distances from them and G, R the largest cotangents:
    hz = alpha ((g - D)(r - R) - their mean).  alpha, the means and their sums are off by `relative` of what goes into them: the exponent's
    size, 64 additions one after the other and thirty operations.  So a distance is off by relative G, and a product by relative (G sr + sg R +
    sg sr + relative G R); it is there twice, itself and in the mean, and alpha's own error weighs the same once more: eight of them are above all.
    """
    generator = torch.Generator().manual_seed(heads)
    degrees = ROWS[rows]
    graph, dst = graph_of(degrees, generator)
    nodes, edges, count = len(degrees), dst.numel(), 5
    rand = lambda *shape: torch.randn(*shape, generator=generator, dtype=F64)  # noqa: E731
    p = [t.to(dtype) for t in (2 * rand(edges, heads), rand(count, heads), shift + spread * rand(edges, heads), shift + spread * rand(edges, heads),
                               0 * rand(count, heads))]
    mask = torch.rand(edges, generator=generator) < 0.8
    buckets = torch.randint(-1, count, (edges,), generator=generator, dtype=torch.int32)
    # a constant in all of g or of r changes nothing, so the definition is asked without it
    want = softmax_orders(lambda z, t: oracle.graph_softmax(z, dst, nodes, mask, t, buckets),
                          *(t.double() - c for t, c in zip(p, (0, 0, shift, shift, 0))))
    got = softmax_orders(lambda z, t: luna.graph_softmax(z, graph, mask=mask.to(DEVICE), table=t, buckets=buckets.to(DEVICE)),
                         *(t.to(DEVICE) for t in p))
    z, t, g, r, _ = (v.double() for v in p)
    span = z.abs().max() + t.abs().max()
    relative = inner(dtype) * (4 * span + 64 + 30)
    alpha = want["alpha"]

    def mean(v):
        return torch.zeros(nodes, heads, dtype=F64).index_add_(0, dst, alpha * v)[dst]

    def largest(v):
        return torch.zeros(nodes, heads, dtype=F64).index_reduce_(0, dst, torch.where(mask[:, None], v.abs(), 0.0), "amax")[dst]

    G, R, sg, sr = largest(g), largest(r), largest(g - mean(g)), largest(r - mean(r))
    tiny = 2.0 ** -24 if dtype == F16 else 1e-30 if dtype != F64 else 1e-300
    error = {"gz": 4 * relative * alpha * G, "hg": 4 * relative * alpha * R, "hz": 8 * relative * alpha * (G * sr + sg * R + sg * sr + relative * G * R)}
    for k, allowed in error.items():
        over = (got[k].cpu().double() - want[k]).abs() / (step(dtype) * want[k].abs() + allowed + tiny)
        assert got[k].dtype == dtype and over.max().item() <= 1.0, f"{k}: {over.max().item():.3g} of what is allowed"
    for k, source in (("gt", "gz"), ("ht", "hz")):
        # by bucket: the parts' errors, and 200 additions of them one after the other
        inside = buckets >= 0
        parts = (error[source] + 200 * inner(dtype) * want[source].abs())[inside]
        allowed = torch.zeros(count, heads, dtype=F64).index_add_(0, buckets[inside].long(), parts) + step(dtype) * want[k].abs() + tiny
        over = (got[k].cpu().double() - want[k]).abs() / allowed
        assert got[k].dtype == dtype and over.max().item() <= 1.0, f"{k}: {over.max().item():.3g} of what is allowed"


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_both_orders_in_one_pass(dtype):
    """A loss of alpha and of its gradient: both cotangents of alpha meet before the logits' gradient is rounded."""
    generator = torch.Generator().manual_seed(1)
    graph, dst = graph_of([30] * 20, generator)
    z, g, r, q = ((torch.randn(600, 4, generator=generator, dtype=F64)).to(dtype) for _ in range(4))

    def run(softmax, z, g, r, q):
        z, g = z.clone().requires_grad_(True), g.clone().requires_grad_(True)
        alpha = softmax(z)
        gz, = torch.autograd.grad(alpha, z, g, create_graph=True)
        return torch.autograd.grad((alpha, gz), z, (q, r))[0].detach()

    want = run(lambda z: oracle.graph_softmax(z, dst, 20), *(t.double() for t in (z, g, r, q)))
    got = run(lambda z: luna.graph_softmax(z, graph), *(t.to(DEVICE) for t in (z, g, r, q)))
    alpha = oracle.graph_softmax(z.double(), dst, 20)
    G, R, Q = (t.double().abs().max() for t in (g, r, q))
    # one rounding of the result; the sums' type as in the test above
    allowed = step(dtype) * want.abs() + 8 * inner(dtype) * (4 * z.double().abs().max() + 94) * alpha * (8 * G * R + Q) + 2.0 ** -24
    assert ((got.cpu().double() - want).abs() <= allowed).all()


@pytest.mark.parametrize("dtype,shift", [(F32, 0.0), (F32, 1e4), (F64, 1e6), (BF16, 100.0), (F16, 100.0)])
@pytest.mark.parametrize("irreps,rows", [(3, 40), (64, 301), (50, 130), (1001, 37), (5000, 5), ("64x0e+16x1o", 100), ("32x0e+5x0o+17x0e", 33)])
def test_second_order_of_the_layer_norm_far_from_zero(irreps, rows, dtype, shift):
    """Cotangents with a common offset, which a block of scalars takes out: what is left depends on their distances from the mean.

    With r', c' the distances of r and c = g from their means (ones as weights), R and C the largest of r and c themselves, and H the
    largest normalised value: r' is off by a few roundings of R, so a product of r' and c' by those of R C' + C R' + R' C'.  hx is s^2
    times such a product by h and two by a projection, |P t| <= max|t| (2 + H q) with q the root of the components; hg is s P r with
    those of R.  A hundred roundings, as the row's sums are twenty additions and ten levels of a tree, and each output has three of them.
    """
    config = luna.LayerNormConfig(irreps)
    generator = torch.Generator().manual_seed(rows)
    rand = lambda *shape: torch.randn(*shape, generator=generator, dtype=F64)  # noqa: E731
    x, g, r = (t.to(dtype) for t in (1.5 * rand(rows, config.dim) + 0.3, rand(rows, config.dim) + shift, rand(rows, config.dim) + shift))

    def run(norm, x, g, r):
        w = torch.ones(config.weight_numel, dtype=x.dtype, device=x.device, requires_grad=True)
        x, g = x.clone().requires_grad_(True), g.clone().requires_grad_(True)
        gx, = torch.autograd.grad(norm(x, w), x, g, create_graph=True)
        return [t.detach() for t in (gx, *torch.autograd.grad(gx, (x, w, g), r))]

    # a constant in a scalar block's g or r changes nothing but the weights' sums, which g is a factor of: the definition is asked without it
    constant = torch.cat([torch.full((mul * ir.dim,), shift if ir.is_scalar() else 0.0, dtype=F64) for mul, ir in config.irreps])
    plain = lambda x, w: oracle.layer_norm(x, config.irreps, w)  # noqa: E731
    want = run(plain, x.double(), g.double() - constant, r.double() - constant)
    want[2] = run(plain, x.double(), g.double(), r.double() - constant)[2]
    got = run(lambda x, w: luna.layer_norm(x, config.irreps, w), *(t.to(DEVICE) for t in (x, g, r)))
    at = channel = 0
    top = lambda t: t.abs().amax(1, keepdim=True)  # noqa: E731
    for mul, ir in config.irreps:
        block = slice(at, at + mul * ir.dim)
        v, e, t = (a.double()[:, block] for a in (x, g, r))
        centred = (lambda a: a - a.mean(1, keepdim=True)) if ir.is_scalar() else (lambda a: a)
        s = (centred(v).square().mean(1, keepdim=True) + config.eps).rsqrt()
        H, R, C, near_r, near_c = top(centred(v) * s), top(t), top(e), top(centred(t)), top(centred(e))
        project = 2 + H * ir.dim ** 0.5
        weigh = 100 * inner(dtype) * (top(v) * s).clamp_min(1.0)
        error = {0: s * C * project * weigh, 1: s * s * ir.dim * (R * near_c + C * near_r + near_r * near_c) * (H + 2 * project) * weigh,
                 3: s * R * project * weigh}
        for k, allowed in error.items():
            over = (got[k].cpu().double()[:, block] - want[k][:, block]).abs() / (step(dtype) * want[k][:, block].abs() + allowed + 2.0 ** -24 * (dtype == F16))
            assert got[k].dtype == dtype and over.max().item() <= 1.0, f"{('gx', 'hx', 'hw', 'hg')[k]} of {mul}x{ir}: {over.max().item():.3g} of what is allowed"
        # the weights': sums of s (P r) g over rows and components
        allowed = (s * R * C * project * weigh).sum() * ir.dim
        a, b = got[2].cpu()[channel:channel + mul], want[2][channel:channel + mul]
        beyond = b.to(dtype).isinf()  # of the range of 16 bits
        assert torch.equal(a[beyond], b.to(dtype)[beyond])
        over = ((a.double() - b).abs() / (step(dtype) * b.abs() + allowed))[~beyond]
        assert not over.numel() or over.max().item() <= 1.0, f"hw of {mul}x{ir}: {over.max().item():.3g} of what is allowed"
        at, channel = at + mul * ir.dim, channel + mul


def test_first_calls_of_two_streams():
    """The tables of cut rows are made in the first call; one on another stream right behind it finds them finished."""
    generator = torch.Generator().manual_seed(0)
    dst = torch.repeat_interleave(torch.arange(300), torch.tensor(([3] * 99 + [3000]) * 3)).to(DEVICE)
    z = torch.randn(dst.numel(), 2, generator=generator).to(DEVICE)
    want = luna.graph_softmax(z, luna.make_graph(torch.zeros_like(dst), dst, 300))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        graph = luna.make_graph(torch.zeros_like(dst), dst, 300)
        torch.cuda.synchronize()
        found = []
        for stream in streams:
            with torch.cuda.stream(stream):
                found.append(luna.graph_softmax(z, graph))
        torch.cuda.synchronize()
        assert all(torch.equal(f, want) for f in found)


def test_tables_outlive_the_work_of_other_streams():
    """Memory of tables that no caller sees is not handed out again while a stream that they were used on is busy."""
    dst = torch.repeat_interleave(torch.arange(300), torch.tensor(([3] * 99 + [3000]) * 3)).to(DEVICE)
    z = torch.randn(dst.numel(), 2, device=DEVICE)
    graph = luna.make_graph(torch.zeros_like(dst), dst, 300)
    want = luna.graph_softmax(z, graph)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)  # a fifth of a second
        got = luna.graph_softmax(z, graph)
    tables = graph._tables["rows"].tensors
    places, sizes = {t.data_ptr() for t in tables}, [t.numel() for t in tables]
    del graph, tables
    again = [torch.empty(n, dtype=torch.int32, device=DEVICE) for n in sizes for _ in range(4)]
    assert not side.query()  # still asleep
    assert not places & {t.data_ptr() for t in again}
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [F32, F64, BF16])
@pytest.mark.parametrize("irreps,rows", [(4, 300_001), (64, 60_000), ("16x0e+16x1o", 40_000), (1024, 5000)])
def test_packets_are_read_before_they_are_refilled(irreps, rows, dtype):
    """The gradient of the weights alone asks for the next rows right behind its reads: the same bits as beside the rows' gradient."""
    config = luna.LayerNormConfig(irreps)
    generator = torch.Generator(device=DEVICE).manual_seed(0)
    x, g = (torch.randn(rows, config.dim, generator=generator, device=DEVICE).to(dtype).requires_grad_(True) for _ in range(2))
    w = torch.rand(config.weight_numel, generator=generator, device=DEVICE).to(dtype).requires_grad_(True)
    _, both = torch.autograd.grad(luna.layer_norm(x, config.irreps, w), (x, w), g)
    for _ in range(20):
        alone, = torch.autograd.grad(luna.layer_norm(x.detach(), config.irreps, w), w, g)
        assert torch.equal(alone, both)


def test_statistics_of_another_call_are_refused():
    """The operators behind the layer norm take the forward's statistics as an argument, and follow them by the sizes of the rows."""
    ops, config = torch.ops.lunaeq, luna.LayerNormConfig("8x0e+4x1o").descriptor()
    x, g = torch.randn(6, 20, device=DEVICE), torch.randn(6, 20, device=DEVICE)
    stats = ops.layer_norm_forward(x, None, None, config)[1]
    assert stats.shape == (2, 6, 2)
    needs = [True, False, False]
    want = ops.layer_norm_backward(x, None, stats, g, needs, config)[0]
    # in another order of memory they are what they were
    assert torch.equal(ops.layer_norm_backward(x, None, stats.permute(2, 1, 0).contiguous().permute(2, 1, 0), g, needs, config)[0], want)
    for bad, error in ((stats[:, :3], ValueError), (stats[:1], ValueError), (stats.flatten(), ValueError), (stats.double(), TypeError), (stats.cpu(), ValueError)):
        with pytest.raises(error, match="stats"):
            ops.layer_norm_backward(x, None, bad, g, needs, config)
        with pytest.raises(error, match="stats"):
            ops.layer_norm_double_backward(x, None, bad, g, x, None, None, needs, config)


def test_borders_are_there_before_the_first_call():
    """A module that is captured, or compiled, before it has ever been called."""
    module = luna.RelativeBias([0.5, 1.0, 2.0], 4, device=DEVICE)
    with torch.no_grad():
        module.weight.normal_()
    vec = torch.randn(50, 3, device=DEVICE)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        luna.distance_buckets(vec, torch.zeros(1, device=DEVICE))
    torch.cuda.current_stream().wait_stream(side)
    captured = torch.cuda.CUDAGraph()
    with torch.cuda.graph(captured):
        found = module.buckets(vec)
    captured.replay()
    want = oracle.distance_buckets(vec.cpu(), torch.tensor([0.5, 1.0, 2.0]))
    assert torch.equal(found.cpu(), want)
    fresh = luna.RelativeBias([0.5, 1.0, 2.0], 4, device=DEVICE)
    fresh._borders = {}
    assert torch.equal(torch.compile(lambda v: fresh.buckets(v), fullgraph=True)(vec).cpu(), want)
    assert not fresh._borders and torch.equal(fresh.buckets(vec).cpu(), want)


@pytest.mark.parametrize("dtype", [F32, F64, BF16, F16])
@pytest.mark.parametrize("edges,buckets,heads", [(600_007, 128, 16), (900_001, 64, 8), (400_003, 32, 1), (700_009, 25, 3), (300_013, 16, 33),
                                                 (200_003, 5000, 12), (150_001, 7, 130), (1_000_003, 2, 4)])
def test_sums_by_bucket_of_many_runs(edges, buckets, heads, dtype):
    """Whole numbers that differ from edge to edge, in tens of runs of each copy of the table: their sums are exact, however they are made."""
    generator = torch.Generator(device=DEVICE).manual_seed(edges)
    g = torch.randint(-8, 9, (edges, heads), generator=generator, device=DEVICE).to(dtype)
    index = torch.randint(-1, buckets + 1, (edges + 1,), generator=generator, device=DEVICE, dtype=torch.int32)
    index[: edges // 3] = index[: edges // 3].sort()[0]  # long stretches of one bucket, then none
    table = torch.zeros(buckets, heads, device=DEVICE, dtype=dtype, requires_grad=True)
    for those in (index[:-1], index[1:]):  # aligned to whole packets and not
        got, = torch.autograd.grad(luna.relative_bias(table, those), table, g)
        inside = (those >= 0) & (those < buckets)
        sums = torch.zeros(buckets, heads, dtype=F64, device=DEVICE).index_add_(0, those[inside].long(), g[inside].double())
        assert sums.abs().max() < 2 ** 24 and torch.equal(got, sums.to(dtype))


@pytest.mark.parametrize("dtype", [F32, F64, BF16])
def test_sums_by_bucket_behind_a_softmax_of_many_edges(dtype):
    """The table's gradient, bucket by bucket: the parts' errors as in the tests above, and 300 additions one after the other."""
    nodes, degree, heads, buckets = 8000, 50, 8, 64
    generator = torch.Generator(device=DEVICE).manual_seed(0)
    rand = lambda *shape: torch.randn(*shape, generator=generator, device=DEVICE).to(dtype)  # noqa: E731
    dst = torch.arange(nodes, device=DEVICE).repeat_interleave(degree)
    z, t, g = rand(nodes * degree, heads), rand(buckets, heads), rand(nodes * degree, heads)
    index = torch.randint(buckets, (nodes * degree,), generator=generator, device=DEVICE, dtype=torch.int32)
    leaf = t.clone().requires_grad_(True)
    got, = torch.autograd.grad(luna.graph_softmax(z, luna.make_graph(dst, dst, nodes), table=leaf, buckets=index), leaf, g)
    alpha = (z.double() + t.double()[index.long()]).reshape(nodes, degree, heads).softmax(1)
    e = g.double().reshape(nodes, degree, heads)
    gz = (alpha * (e - (alpha * e).sum(1, keepdim=True))).reshape(-1, heads)
    want = torch.zeros(buckets, heads, dtype=F64, device=DEVICE).index_add_(0, index.long(), gz)
    relative = inner(dtype) * (4 * (z.double().abs().max() + t.double().abs().max()) + 64 + 30)
    parts = 4 * relative * alpha.reshape(-1, heads) * e.abs().max() + 300 * inner(dtype) * gz.abs()
    allowed = torch.zeros_like(want).index_add_(0, index.long(), parts) + step(dtype) * want.abs()
    assert ((got.double() - want).abs() <= allowed).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_operators_of_the_second_order(dtype):
    """The operators that a traced program names, with cotangents of either type; third orders are refused in every type."""
    generator = torch.Generator().manual_seed(2)
    graph, _ = graph_of([5, 0, 40, 9], generator)
    z, g, r = (torch.randn(54, 3, generator=generator, dtype=F64).to(dtype).to(DEVICE) for _ in range(3))
    table = torch.randn(4, 3, generator=generator, dtype=F64).to(dtype).to(DEVICE)
    buckets = torch.randint(4, (54,), generator=generator, dtype=torch.int32).to(DEVICE)
    ops = torch.ops.lunaeq
    alpha, wide = ops.graph_softmax_forward(z, table, buckets, None, graph.dst_rowptr, graph.num_edges)
    kind = ("test_schema", "test_faketensor")
    for cotangent in {g.dtype, torch.float32 if dtype in (BF16, F16) else dtype}:
        args = (alpha, wide, g.to(cotangent), buckets, 4, graph.dst_rowptr, [True, True])
        torch.library.opcheck(ops.graph_softmax_backward.default, args, test_utils=kind)
        assert all(t.dtype == dtype for t in ops.graph_softmax_backward(*args))
        args = (alpha, wide, g.to(cotangent), buckets, r, table, graph.dst_rowptr, [True, True])
        torch.library.opcheck(ops.graph_softmax_double_backward.default, args, test_utils=kind)
        halpha, hg = ops.graph_softmax_double_backward(*args)
        assert halpha.dtype == (F32 if dtype in (BF16, F16) else dtype) and hg.dtype == cotangent
    # an alpha that was rounded, without what it was before: its own type comes back
    if dtype in (BF16, F16):
        leaf = alpha.clone().requires_grad_(True)
        gz, _ = ops.graph_softmax_backward(leaf, wide[:0], g, buckets, 4, graph.dst_rowptr, [True, False])
        assert torch.autograd.grad(gz, leaf, r)[0].dtype == dtype
    for softmax in (lambda z: luna.graph_softmax(z, graph, table=table, buckets=buckets),
                    lambda z: ops.graph_softmax_forward(z, table, buckets, None, graph.dst_rowptr, graph.num_edges)[0]):
        leaf = z.clone().requires_grad_(True)
        first, = torch.autograd.grad(softmax(leaf).square().sum(), leaf, create_graph=True)
        second, = torch.autograd.grad(first.square().sum(), leaf, create_graph=True)
        with pytest.raises((NotImplementedError, RuntimeError), match="third-order|does not require grad|autograd"):
            torch.autograd.grad(second.sum(), leaf)
