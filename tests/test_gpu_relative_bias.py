"""Buckets of edge vectors, the bias they get from a table, and the table's gradient, against their definitions."""

import pytest
import torch

import lunaequivariance_b200 as luna
from oracle import attention as oracle

pytestmark = pytest.mark.gpu
DEVICE = "cuda"
F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16


def step(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype", [F32, F64])
@pytest.mark.parametrize("count,edges", [(0, 5), (1, 1), (7, 100), (31, 1), (127, 5000), (2048, 300), (2049, 300)])
def test_buckets(count, edges, dtype):
    generator = torch.Generator().manual_seed(count)
    vec = (3 * torch.randn(edges, 3, generator=generator, dtype=F64)).to(dtype)
    boundaries = (6 * torch.rand(count, generator=generator, dtype=F64)).sort()[0].to(dtype)
    got = luna.distance_buckets(vec.to(DEVICE), boundaries.to(DEVICE))
    assert got.dtype == torch.int32 and torch.equal(got.cpu(), oracle.distance_buckets(vec, boundaries))


def test_lengths_on_a_border():
    """3-4-5 triangles, axis vectors and the neighbours of a border in its type; nothing, infinities and NaN."""
    boundaries = torch.tensor([0.0, 1.0, 5.0, 5.0, 7.5])
    up, down = torch.nextafter(torch.tensor(5.0), torch.tensor(9.0)).item(), torch.nextafter(torch.tensor(5.0), torch.tensor(0.0)).item()
    vec = torch.tensor([[3.0, 4.0, 0.0], [0.0, -5.0, 0.0], [up, 0.0, 0.0], [0.0, 0.0, down], [0.0, 0.0, 0.0], [1.0, 0.0, 0.0],
                        [float("inf"), 0.0, 0.0], [float("nan"), 1.0, 0.0], [3e38, 3e38, 0.0], [1e-30, 0.0, 0.0]])
    got = luna.distance_buckets(vec.to(DEVICE), boundaries.to(DEVICE)).tolist()
    assert got == [4, 4, 4, 2, 1, 2, 5, 0, 5, 1]
    assert got == oracle.distance_buckets(vec, boundaries).tolist()


def test_shapes_of_vectors():
    vec = torch.randn(4, 5, 3, device=DEVICE)
    boundaries = torch.tensor([0.5, 1.0, 2.0], device=DEVICE)
    flat = luna.distance_buckets(vec.reshape(-1, 3), boundaries)
    assert torch.equal(luna.distance_buckets(vec, boundaries), flat.reshape(4, 5))
    turned = vec.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    assert torch.equal(luna.distance_buckets(turned, boundaries), flat.reshape(4, 5))
    assert luna.distance_buckets(vec[:0], boundaries).shape == (0, 5)
    assert luna.distance_buckets(vec.requires_grad_(True), boundaries).dtype == torch.int32


def indices(edges, buckets, generator):
    """Random buckets, with some that are no row of the table."""
    found = torch.randint(-1, buckets + 1, (edges,), generator=generator)
    if edges > 3:
        found[1], found[2] = 2 ** 31 - 1, -2 ** 31
    return found.to(torch.int32)


CASES = [(1, 1, 1), (5, 3, 2), (1000, 32, 8), (777, 25, 3), (4001, 128, 16), (300, 256, 64), (50, 7, 700), (2000, 1, 1), (999, 16, 33),
         (600, 20000, 1), (500, 9000, 12), (20000, 2, 5)]


@pytest.mark.parametrize("dtype", [F32, F64, BF16, F16])
@pytest.mark.parametrize("edges,buckets,heads", CASES)
def test_values_and_gradient(edges, buckets, heads, dtype):
    generator = torch.Generator().manual_seed(edges)
    table = torch.randn(buckets, heads, generator=generator, dtype=F64).to(dtype)
    g = torch.randn(edges, heads, generator=generator, dtype=F64).to(dtype)
    index = indices(edges, buckets, generator)
    leaf = table.to(DEVICE).requires_grad_(True)
    out = luna.relative_bias(leaf, index.to(DEVICE))
    assert torch.equal(out.detach().cpu(), oracle.relative_bias(table, index))
    got, = torch.autograd.grad(out, leaf, g.to(DEVICE))
    reference = table.double().requires_grad_(True)
    want, = torch.autograd.grad(oracle.relative_bias(reference, index), reference, g.double())
    magnitude, = torch.autograd.grad(oracle.relative_bias(reference, index), reference, g.double().abs())
    # the rounding of the result, and of every addition: one after the other at worst, each of at most the sum of magnitudes
    inside = (index >= 0) & (index < buckets)
    most = int(torch.bincount(index[inside].long(), minlength=1).max()) if inside.any() else 0
    inner = step(F64 if dtype == F64 else F32)
    allowed = step(dtype) * want.abs() + min(most, 200) * inner * magnitude + (2.0 ** -25 if dtype == F16 else 0) + 1e-300
    assert got.dtype == dtype and ((got.cpu().double() - want).abs() <= allowed).all()
    assert torch.equal(got, torch.autograd.grad(luna.relative_bias(leaf, index.to(DEVICE)), leaf, g.to(DEVICE))[0])


def test_shapes_and_memory_orders():
    generator = torch.Generator(device=DEVICE).manual_seed(1)
    table = torch.randn(8, 10, generator=generator, device=DEVICE).t()  # 10 buckets, 8 heads
    index = torch.randint(10, (6, 9), generator=generator, device=DEVICE, dtype=torch.int32)
    want = table[index.long()]
    assert torch.equal(luna.relative_bias(table, index), want)
    assert torch.equal(luna.relative_bias(table, index.t()), want.transpose(0, 1))
    odd = torch.randn(81, generator=generator, device=DEVICE)[1:].reshape(10, 8)
    assert torch.equal(luna.relative_bias(odd, index[0]), odd[index[0].long()])
    assert luna.relative_bias(table, index[:0]).shape == (0, 9, 8)
    leaf = odd.clone().requires_grad_(True)
    empty, = torch.autograd.grad(luna.relative_bias(leaf, index[:0]), leaf, torch.zeros(0, 9, 8, device=DEVICE))
    assert not empty.any()
    g = torch.randn(8, 54, generator=generator, device=DEVICE).t().reshape(6, 9, 8)
    a, = torch.autograd.grad(luna.relative_bias(leaf, index), leaf, g)
    b, = torch.autograd.grad(luna.relative_bias(leaf, index), leaf, g.contiguous())
    assert torch.equal(a, b)
    one, = torch.autograd.grad(luna.relative_bias(leaf, index).sum(), leaf)
    assert torch.equal(one, torch.bincount(index.flatten().long(), minlength=10).float()[:, None].expand(10, 8))


def test_every_order():
    """The gradient is linear in its cotangent: its own derivative is the bias again, and so on."""
    index = torch.tensor([0, 2, 2, 1, -1], dtype=torch.int32, device=DEVICE)
    table = torch.randn(3, 4, dtype=F64, device=DEVICE, requires_grad=True)
    check = lambda t: luna.relative_bias(t, index)  # noqa: E731
    assert torch.autograd.gradcheck(check, (table,)) and torch.autograd.gradgradcheck(check, (table,))
    g = torch.randn(5, 4, dtype=F64, device=DEVICE, requires_grad=True)
    first, = torch.autograd.grad(check(table), table, g, create_graph=True)
    second, = torch.autograd.grad((first ** 3).sum(), g, create_graph=True)
    third, = torch.autograd.grad((second ** 2).sum(), g)
    plain = torch.zeros(3, 4, dtype=F64, device=DEVICE).index_add(0, index[:4].long(), g[:4])
    s, = torch.autograd.grad((plain ** 3).sum(), g, create_graph=True)
    t, = torch.autograd.grad((s ** 2).sum(), g)
    assert torch.allclose(third, t, rtol=1e-12, atol=1e-12)


def test_large_numbers_of_edges():
    """Values beyond 2^31 and a bucket with millions of edges: sums of ones are exact."""
    edges, heads = 5_000_001, 3
    index = torch.zeros(edges, dtype=torch.int32, device=DEVICE)
    index[-1] = 1
    leaf = torch.zeros(2, heads, device=DEVICE, requires_grad=True)
    g, = torch.autograd.grad(luna.relative_bias(leaf, index).sum(), leaf)
    assert torch.equal(g.cpu(), torch.tensor([[5_000_000.0] * 3, [1.0] * 3]))
    wide = torch.arange(2 * 700, device=DEVICE, dtype=BF16).reshape(2, 700)
    many = (1 << 31) // 700 + 3
    index = torch.zeros(many, dtype=torch.int32, device=DEVICE)
    index[-1] = 1
    out = luna.relative_bias(wide, index)
    assert torch.equal(out[-1], wide[1]) and torch.equal(out[-2], wide[0]) and torch.equal(out[0], wide[0])


def test_module_compile_and_capture():
    module = luna.RelativeBias([1.0, 2.0, 3.0], 4, device=DEVICE)
    with torch.no_grad():
        module.weight.normal_()
    vec = 2 * torch.randn(50, 3, device=DEVICE)
    want = module.weight[oracle.distance_buckets(vec.cpu(), torch.tensor([1.0, 2.0, 3.0])).long().to(DEVICE)]
    assert torch.equal(module(vec), want)
    assert torch.equal(module.half().buckets(vec), oracle.distance_buckets(vec.cpu(), torch.tensor([1.0, 2.0, 3.0])).to(DEVICE))
    module.double()
    assert torch.equal(module.buckets(vec.double()).cpu(), oracle.distance_buckets(vec.cpu().double(), torch.tensor([1.0, 2.0, 3.0])))
    table, borders = module.weight.detach().clone().requires_grad_(True), torch.tensor([1.0, 2.0, 3.0], device=DEVICE)

    def gradient(table, vec):
        bias = luna.relative_bias(table, luna.distance_buckets(vec, borders))
        # no graph is left behind: the autograd engine cannot capture a backward pass while an eager graph of the leaf lives
        return bias.detach(), torch.autograd.grad((bias ** 2).sum(), table)[0]

    assert torch.equal(torch.compile(module, fullgraph=True)(vec.double()), module(vec.double()))
    traced = torch.compile(lambda t, v: luna.relative_bias(t, luna.distance_buckets(v, borders)), fullgraph=True)
    eager = gradient(table, vec)
    assert torch.equal(traced(table, vec), eager[0])
    assert torch.equal(torch.autograd.grad((traced(table, vec) ** 2).sum(), table)[0], eager[1])
    torch.library.opcheck(torch.ops.lunaeq.relative_bias_forward.default, (table, luna.distance_buckets(vec, borders)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gradient(table, vec)
    torch.cuda.current_stream().wait_stream(side)
    captured = torch.cuda.CUDAGraph()
    with torch.cuda.graph(captured):
        found = gradient(table, vec)
    vec.mul_(0.7)
    captured.replay()
    assert all(torch.equal(a, b) for a, b in zip(found, gradient(table, vec)))


def test_refusals():
    table, index = torch.zeros(4, 2, device=DEVICE), torch.zeros(3, dtype=torch.int32, device=DEVICE)
    with pytest.raises(TypeError, match="buckets must be Int"):
        luna.relative_bias(table, index.long())
    with pytest.raises(ValueError, match="must be on"):
        luna.relative_bias(table, index.cpu())
    with pytest.raises(TypeError, match="float32"):
        luna.relative_bias(table.int(), index)
    for bad in (table[0], table[:0], table[:, :0]):
        with pytest.raises(ValueError, match="bias table"):
            luna.relative_bias(bad, index)
    vec = torch.zeros(3, 3, device=DEVICE)
    with pytest.raises(TypeError, match="boundaries"):
        luna.distance_buckets(vec, torch.zeros(2, device=DEVICE, dtype=F64))
    with pytest.raises(TypeError, match="float32 or float64"):
        luna.distance_buckets(vec.half(), torch.zeros(2, device=DEVICE).half())
    with pytest.raises(ValueError, match="shape"):
        luna.distance_buckets(vec[:, :2], torch.zeros(2, device=DEVICE))
    with pytest.raises(ValueError, match="one-dimensional"):
        luna.distance_buckets(vec, torch.zeros(2, 2, device=DEVICE))
