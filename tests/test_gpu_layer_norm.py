"""Layer norm over irreps: forward, backward and second order against the definition in 64 bits."""

import pytest
import torch

import lunaequivariance_b200 as luna
from oracle import attention as oracle

pytestmark = pytest.mark.gpu
DEVICE = "cuda"
F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16


def step(dtype):
    """Half a unit in the last place of one."""
    return torch.finfo(dtype).eps / 2


def inner(dtype):
    """The step of the type that sums are held in."""
    return step(F64 if dtype == F64 else F32)


def close(got, want, dtype, size, what, roundings=100):
    """Every number is within the rounding of its type, and `roundings` of the sums' type on what went into it, `size`.

    A row's sum is at most 20 additions one after the other and ten levels of a tree; an output has four such sums in it
    (mean, power, and two projections) and about twenty operations more: a hundred and forty, which do not all fall to one
    side.
    """
    want = want.detach()
    allowed = step(dtype) * want.abs() + roundings * inner(dtype) * size + 1e-300
    if dtype == F16:
        allowed = allowed + 2.0 ** -25  # half the smallest number of the type
    over = ((got.detach().cpu().double() - want).abs() / allowed)
    assert got.dtype == dtype and got.shape == want.shape, what
    assert not want.numel() or over.max().item() <= 1.0, f"{what}: {over.max().item():.3g} of what is allowed"


def problem(irreps, rows, dtype, seed=0, shift=0.3):
    config = luna.LayerNormConfig(irreps)
    generator = torch.Generator().manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=generator, dtype=F64)  # noqa: E731
    p = dict(x=1.5 * rand(rows, config.dim) + shift, weight=1 + 0.3 * rand(config.weight_numel), bias=0.3 * rand(config.bias_numel),
             g=rand(rows, config.dim), rx=rand(rows, config.dim), rw=rand(config.weight_numel), rb=rand(config.bias_numel))
    return config, {k: v.to(dtype) for k, v in p.items()}


def derivatives(norm, p, second=True):
    x, w, b, g = (p[k].clone().requires_grad_(True) for k in ("x", "weight", "bias", "g"))
    y = norm(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), g, create_graph=second, allow_unused=True)
    if gb is None:  # the definition does not use an empty bias
        gb = torch.zeros_like(b)
    found = dict(y=y, gx=gx, gw=gw, gb=gb)
    if second:
        terms = [(gx, p["rx"]), (gw, p["rw"])] + ([(gb, p["rb"])] if b.numel() else [])
        found.update(zip(("hx", "hw", "hg"), torch.autograd.grad([t for t, _ in terms], (x, w, g), [r for _, r in terms])))
    # no graph is left behind: the autograd engine cannot capture a backward pass while an eager graph of the leaves lives
    return {k: v.detach() for k, v in found.items()}


def sizes(config, p):
    """Bounds on the magnitude of what is added up in every output, row by row; for the sums over rows, of all rows.

    With h the normalised values, H the largest, q the root of the components: share sum|h| <= q, so |P t| <= max|t| (2 + H q);
    the two dot products of the second order are at most max|r| max|c| d per unit of share, together 2 d.  A rounding of x
    itself weighs |x| s instead of one, which `relative` multiplies everything with.
    """
    at = channel = scalar = 0
    x, w, b, g, rx, rw, rb = (p[k].double() for k in ("x", "weight", "bias", "g", "rx", "rw", "rb"))
    blocks = []
    for mul, ir in config.irreps:
        n, d = mul * ir.dim, ir.dim
        v, e, r = (t[:, at:at + n] for t in (x, g, rx))
        mean = v.mean(1, keepdim=True) if ir.is_scalar() else 0.0
        s = ((v - mean).square().sum(1, keepdim=True) / (n if config.normalization == "component" else mul) + config.eps).rsqrt()
        top = lambda t: t.abs().amax(1, keepdim=True)  # noqa: E731
        wide = lambda t: t.repeat_interleave(d)  # noqa: E731
        W, Q = w[channel:channel + mul].abs().max(), top(e * wide(rw[channel:channel + mul]))
        H, q, R, C, G = top((v - mean) * s), d ** 0.5, top(r), top(e * wide(w[channel:channel + mul])), top(e)
        B, RB = (b[scalar:scalar + mul].abs().max(), rb[scalar:scalar + mul].abs().max()) if ir.is_scalar() else (0.0, 0.0)
        project = 2 + H * q
        relative = (top(v) * s).clamp_min(1.0)
        blocks.append({"y": (W * H + B) * relative, "gx": s * C * project * relative,
                       "hx": (s * s * (2 * d * R * C * H + 2 * C * q * R * project) + s * Q * project) * relative,
                       "hg": (W * s * R * project + rw.abs().max() * H + RB) * relative,
                       "gw": (G * H * relative * d).sum(), "gb": G.sum(), "hw": (s * R * project * G * relative * d).sum()})
        at, channel, scalar = at + n, channel + mul, scalar + (mul if ir.is_scalar() else 0)
    return {k: torch.stack([block[k] for block in blocks]).amax(0) for k in blocks[0]}


@pytest.mark.parametrize("dtype", [F32, F64, BF16, F16])
@pytest.mark.parametrize("normalization", ["component", "norm"])
@pytest.mark.parametrize("irreps,rows", [
    (1, 5), (7, 1), (64, 1), (64, 301), (50, 130), (1001, 37), ("5x0e+5x1o", 33), ("64x0e+64x1o+64x2e", 100),
    ("3x0o+4x0e+2x3o+6x1e", 1000), ("1x0e+1x1o", 2500), ("128x0e+128x1o+128x2e+128x3o", 19), ("700x2e", 9), ("256x0e", 2000)])
def test_all_orders(irreps, rows, normalization, dtype):
    config, p = problem(irreps, rows, dtype)
    config = luna.LayerNormConfig(irreps, 1e-5, normalization)
    want = derivatives(lambda x, w, b: oracle.layer_norm(x, config.irreps, w, b, 1e-5, normalization), {k: v.double() for k, v in p.items()})
    got = derivatives(lambda x, w, b: luna.layer_norm(x, config.irreps, w, b, normalization=normalization),
                      {k: v.to(DEVICE) for k, v in p.items()})
    for k, size in sizes(config, p).items():
        close(got[k], want[k], dtype, size, k)


@pytest.mark.parametrize("dtype,width", [(F32, 4096), (F32, 4999), (F32, 16384), (F32, 5000), (F64, 2051), (F64, 16384), (F64, 9000), (BF16, 16384),
                                         (BF16, 4097), (F16, 8192), (F32, 16383)])
def test_wide_rows(dtype, width):
    config, p = problem(width, 7, dtype)
    want = derivatives(lambda x, w, b: oracle.layer_norm(x, config.irreps, w, b), {k: v.double() for k, v in p.items()})
    got = derivatives(lambda x, w, b: luna.layer_norm(x, width, w, b), {k: v.to(DEVICE) for k, v in p.items()})
    for k, size in sizes(config, p).items():
        close(got[k], want[k], dtype, size, k)


def test_blocks_beside_a_wide_one():
    """A row of one block that takes a whole CTA and of short ones, and as many blocks as there may be."""
    for irreps, rows in (("6000x0e+2x1o+24x0o+500x0e", 11), ("+".join("2x0e+1x1o" for _ in range(16)), 50)):
        config, p = problem(irreps, rows, F64)
        want = derivatives(lambda x, w, b: oracle.layer_norm(x, irreps, w, b), {k: v for k, v in p.items()})
        got = derivatives(lambda x, w, b: luna.layer_norm(x, irreps, w, b), {k: v.to(DEVICE) for k, v in p.items()})
        for k, size in sizes(config, p).items():
            close(got[k], want[k], F64, size, k)


@pytest.mark.parametrize("wants", [("x",), ("weight",), ("bias",), ("x", "bias"), ("weight", "bias")])
def test_some_gradients(wants):
    irreps = "33x0e+20x1o"
    config, p = problem(irreps, 77, F64)

    def run(norm, p):
        t = {k: p[k].clone().requires_grad_(k in wants) for k in ("x", "weight", "bias")}
        return torch.autograd.grad(norm(t["x"], t["weight"], t["bias"]), [t[k] for k in wants], p["g"])

    want = run(lambda x, w, b: oracle.layer_norm(x, irreps, w, b), p)
    got = run(lambda x, w, b: luna.layer_norm(x, irreps, w, b), {k: v.to(DEVICE) for k, v in p.items()})
    for k, a, b in zip(wants, got, want):
        close(a, b, F64, 77 * b.abs().max(), k)


@pytest.mark.parametrize("parts", [(True, False), (False, False)])
def test_without_parameters(parts):
    irreps = "12x0e+4x1o"
    config, p = problem(irreps, 40, F32)
    w, b = (p["weight"] if parts[0] else None), (p["bias"] if parts[1] else None)
    up = lambda t: None if t is None else t.to(DEVICE)  # noqa: E731
    double = lambda t: None if t is None else t.double()  # noqa: E731

    def run(norm, x, w, b, g, r):
        x, g = x.clone().requires_grad_(True), g.clone().requires_grad_(True)
        gx, = torch.autograd.grad(norm(x, w, b), x, g, create_graph=True)
        return (gx, *torch.autograd.grad(gx, (x, g), r))

    want = run(lambda *a: oracle.layer_norm(a[0], irreps, *a[1:]), p["x"].double(), double(w), double(b), p["g"].double(), p["rx"].double())
    got = run(lambda *a: luna.layer_norm(a[0], irreps, *a[1:]), up(p["x"]), up(w), up(b), up(p["g"]), up(p["rx"]))
    for k, a, c in zip(("gx", "hx", "hg"), got, want):
        close(a, c, F32, 10 * c.abs().max(), k)


@pytest.mark.parametrize("slot", [0, 1, 2])
@pytest.mark.parametrize("irreps,dtype", [("64x0e+16x1o", F64), ("51x0e", F64), ("33x0e", BF16)])
def test_second_order_of_one_gradient(irreps, dtype, slot):
    """The cotangent of gx, of gw or of gb alone."""
    config, p = problem(irreps, 70, dtype)

    def run(norm, p):
        x, w, b, g = (p[k].clone().requires_grad_(True) for k in ("x", "weight", "bias", "g"))
        first = torch.autograd.grad(norm(x, w, b), (x, w, b), g, create_graph=True)[slot]
        return [t for t in torch.autograd.grad(first, (x, w, g), p[("rx", "rw", "rb")[slot]], allow_unused=True)]

    want = run(lambda x, w, b: oracle.layer_norm(x, irreps, w, b), {k: v.double() for k, v in p.items()})
    got = run(lambda x, w, b: luna.layer_norm(x, irreps, w, b), {k: v.to(DEVICE) for k, v in p.items()})
    bounds = sizes(config, p)
    for k, a, b in zip(("hx", "hw", "hg"), got, want):
        if b is None:  # the definition has no path there: a derivative of zero
            assert a is None or not a.any(), k
        else:
            close(a, b, dtype, bounds[k], k)


def test_gradient_against_differences():
    irreps = "6x0e+3x1o+2x2e"
    config, p = problem(irreps, 4, F64)
    t = [p[k].to(DEVICE).requires_grad_(True) for k in ("x", "weight", "bias")]
    assert torch.autograd.gradcheck(lambda x, w, b: luna.layer_norm(x, irreps, w, b), t)
    assert torch.autograd.gradgradcheck(lambda x, w, b: luna.layer_norm(x, irreps, w, b), t)


def test_memory_orders():
    """Batched, transposed, strided and unaligned rows are what their copies are."""
    generator = torch.Generator(device=DEVICE).manual_seed(3)
    flat = torch.randn(1 + 4 * 6 * 20, generator=generator, device=DEVICE)
    w = torch.rand(20, generator=generator, device=DEVICE)
    plain = flat[1:].reshape(4, 6, 20)
    # rows that are not aligned are read number by number and summed in another order: each result is within a hundred roundings
    # of |h| <= sqrt(20) times what a rounding of x weighs, |x| s
    a, b = luna.layer_norm(plain, 20, w), luna.layer_norm(plain.clone(), 20, w)
    relative = (plain.abs().amax(-1) / plain.std(-1, correction=0)).max().item()
    assert (a - b).abs().max().item() <= 2 * 100 * step(F32) * 20 ** 0.5 * max(relative, 1.0)
    for view in (flat[:-1].reshape(6, 4, 20).transpose(0, 1), flat[:480].reshape(20, 24).t().reshape(24, 20)[::2], flat[:24].reshape(4, 6, 1).expand(4, 6, 20)):
        assert torch.equal(luna.layer_norm(view, 20, w), luna.layer_norm(view.clone(memory_format=torch.contiguous_format), 20, w))
    x = flat[:-1].reshape(4, 6, 20).transpose(0, 1).requires_grad_(True)
    g = torch.randn(6, 20, 4, generator=generator, device=DEVICE).transpose(1, 2)
    a, = torch.autograd.grad(luna.layer_norm(x, 20, w), x, g)
    y = x.detach().contiguous().requires_grad_(True)
    b, = torch.autograd.grad(luna.layer_norm(y, 20, w), y, g.contiguous())
    assert torch.equal(a, b)
    expanded = torch.ones((), device=DEVICE).expand(6, 4, 20)
    c, = torch.autograd.grad(luna.layer_norm(y, 20, w), y, expanded)
    d, = torch.autograd.grad(luna.layer_norm(y, 20, w), y, expanded.contiguous())
    assert torch.equal(c, d)


def test_no_rows():
    x = torch.zeros(0, 16, device=DEVICE, requires_grad=True)
    w, b = torch.ones(10, device=DEVICE, requires_grad=True), torch.ones(7, device=DEVICE, requires_grad=True)
    y = luna.layer_norm(x, "7x0e+3x1o", w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.zeros(0, 16, device=DEVICE), create_graph=True)
    assert y.shape == gx.shape == (0, 16) and not gw.any() and not gb.any()
    hw, = torch.autograd.grad(gx.sum() + gw.sum(), w, allow_unused=True)
    assert hw is None or not hw.any()


def test_rows_do_not_touch_each_other():
    """Rows of zeros, infinities and NaN beside others: those are what they are alone."""
    x = torch.randn(40, 24, device=DEVICE, generator=torch.Generator(device=DEVICE).manual_seed(1))
    want = luna.layer_norm(x, "12x0e+4x1o")
    x[3], x[11, 2], x[12, 20], x[39] = 0.0, float("nan"), float("inf"), -float("inf")
    got = luna.layer_norm(x, "12x0e+4x1o")
    fine = [i for i in range(40) if i not in (3, 11, 12, 39)]
    assert torch.equal(got[fine], want[fine]) and not got[3].any()
    assert got[11, :12].isnan().all() and torch.equal(got[11, 12:], want[11, 12:])
    assert torch.equal(got[12, :12], want[12, :12])
    zeros = torch.zeros(3, 16, device=DEVICE, requires_grad=True)
    g, = torch.autograd.grad(luna.layer_norm(zeros, "4x0e+4x1o").sum(), zeros)
    assert g.isfinite().all()


@pytest.mark.parametrize("shift", [1e3, 1e4])
def test_far_means(shift):
    """A mean much larger than the spread: the variance is made of differences, not of squares."""
    generator = torch.Generator().manual_seed(2)
    x = (torch.randn(50, 256, generator=generator, dtype=F64) + shift).float()
    want = oracle.layer_norm(x.double(), "256x0e")
    got = luna.layer_norm(x.to(DEVICE), 256).cpu().double()
    # the mean is off by at most 14 roundings (16 values in a thread's turn and tree of 32) of its own size: all outputs shift by it
    assert (got - want).abs().max().item() <= 20 * step(F32) * shift / x.double().std(1).min().item()


def test_same_bits_every_time():
    config, p = problem("64x0e+64x1o", 5000, F32)
    p = {k: v.to(DEVICE) for k, v in p.items()}
    norm = lambda x, w, b: luna.layer_norm(x, "64x0e+64x1o", w, b)  # noqa: E731
    first = derivatives(norm, p)
    for _ in range(3):
        again = derivatives(norm, p)
        assert all(torch.equal(first[k], again[k]) for k in first)


def test_rows_beyond_32_bits():
    """More than 2^31 elements."""
    rows, dim = (1 << 31) // 64 + 5, 64
    x = torch.zeros(rows, dim, device=DEVICE, dtype=BF16)
    x[-3:] = torch.randn(3, dim, device=DEVICE, generator=torch.Generator(device=DEVICE).manual_seed(0)).to(BF16)
    y = luna.layer_norm(x, dim)
    assert torch.equal(y[-3:], luna.layer_norm(x[-3:].clone(), dim)) and not y[:-3].any()


def test_stream_and_captured_graph():
    config, p = problem("16x0e+16x1o", 300, F32)
    p = {k: v.to(DEVICE) for k, v in p.items()}
    norm = lambda x, w, b: luna.layer_norm(x, "16x0e+16x1o", w, b)  # noqa: E731
    eager = derivatives(norm, p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        aside = derivatives(norm, p)
        derivatives(norm, p)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(eager[k], aside[k]) for k in eager)
    graphs = []
    for _ in range(2):  # two graphs, replayed in turn
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            found = derivatives(norm, p)
        graphs.append((captured, found))
    for seed in (5, 6):
        _, new = problem("16x0e+16x1o", 300, F32, seed)
        for k, v in new.items():
            p[k].copy_(v)
        want = derivatives(norm, p)
        for captured, found in graphs:
            captured.replay()
        for captured, found in graphs:
            assert all(torch.equal(found[k], want[k]) for k in want)


def test_module_and_compile():
    module = luna.LayerNorm("8x0e+8x1o", dtype=F64, device=DEVICE)
    with torch.no_grad():
        module.weight.uniform_(0.5, 1.5)
        module.bias.uniform_(-1, 1)
    assert [tuple(p.shape) for p in module.parameters()] == [(16,), (8,)]
    x = torch.randn(9, 32, device=DEVICE, dtype=F64, requires_grad=True)

    def energy_and_force(module, x):
        y = module(x)
        g, = torch.autograd.grad((y ** 3).sum(), x, create_graph=True)
        return y, g

    y, g = energy_and_force(module, x)
    want = torch.autograd.grad((g ** 2).sum(), (x, *module.parameters()), allow_unused=True)
    traced = torch.compile(lambda x: module(x), fullgraph=True)
    assert torch.equal(traced(x), y)
    ops = lambda x: torch.ops.lunaeq.layer_norm_forward(x, module.weight, module.bias, module._config.descriptor())[0]  # noqa: E731
    y2, g2 = energy_and_force(ops, x)
    got = torch.autograd.grad((g2 ** 2).sum(), (x, *module.parameters()), allow_unused=True)
    assert torch.equal(y, y2) and torch.equal(g, g2) and all(torch.equal(a, b) for a, b in zip(want, got))
    torch.library.opcheck(torch.ops.lunaeq.layer_norm_forward.default, (x, module.weight, module.bias, module._config.descriptor()))


def test_refusals():
    x = torch.randn(4, 8, device=DEVICE)
    with pytest.raises(ValueError, match="shape"):
        luna.layer_norm(x, 9)
    with pytest.raises(TypeError, match="float32"):
        luna.layer_norm(x.int(), 8)
    with pytest.raises(TypeError, match="weight"):
        luna.layer_norm(x, 8, torch.ones(8, device=DEVICE, dtype=F64))
    with pytest.raises(ValueError, match="weight"):
        luna.layer_norm(x, "2x0e+2x1o", torch.ones(8, device=DEVICE))
    with pytest.raises(ValueError, match="bias"):
        luna.layer_norm(x, "2x0e+2x1o", None, torch.ones(4, device=DEVICE))
    with pytest.raises(ValueError, match="must be on"):
        luna.layer_norm(x, 8, torch.ones(8))
    with pytest.raises(NotImplementedError, match="16384"):
        luna.layer_norm(torch.zeros(1, 16385, device=DEVICE), 16385)
    leaf = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(luna.layer_norm(leaf, 8).square().sum(), leaf, create_graph=True)
    h, = torch.autograd.grad(g.square().sum(), leaf, create_graph=True)
    with pytest.raises(NotImplementedError, match="third-order"):
        torch.autograd.grad(h.sum(), leaf)
