"""What the operators of attention over neighbours refuse before a kernel runs, and the oracle's own definitions."""

import pytest
import torch

import lunaequivariance_b200 as luna
from oracle import attention as oracle


def test_layer_norm_configuration():
    config = luna.LayerNormConfig("4x0e+0x1o+3x1o+2x0o")
    assert (config.dim, config.weight_numel, config.bias_numel) == (15, 9, 4)
    assert luna.LayerNormConfig(12).irreps == luna.Irreps("12x0e")
    for bad in ("", "0x0e", 0):
        with pytest.raises(ValueError):
            luna.LayerNormConfig(bad)
    with pytest.raises(ValueError, match="normalization"):
        luna.LayerNormConfig(4, normalization="integral")
    for eps in (-1e-5, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="eps"):
            luna.LayerNormConfig(4, eps)
    with pytest.raises(TypeError, match="irreps"):
        luna.layer_norm(torch.zeros(2, 4))
    with pytest.raises(NotImplementedError, match="32 blocks"):
        luna.LayerNormConfig("+".join(["1x0e+1x1o"] * 17)).holder()
    module = luna.LayerNorm("4x1o", dtype=torch.float64)
    assert module.bias is None and module.weight.dtype == torch.float64
    assert luna.LayerNorm(3, affine=False).weight is None


def test_cuda_is_required():
    graph = luna.make_graph(torch.tensor([0, 1]), torch.tensor([0, 1]))
    for call in (lambda: luna.layer_norm(torch.zeros(2, 4), 4), lambda: luna.relative_bias(torch.zeros(2, 2), torch.zeros(3).int()),
                 lambda: luna.distance_buckets(torch.zeros(2, 3), torch.ones(1)), lambda: luna.graph_softmax(torch.zeros(2), graph)):
        with pytest.raises(RuntimeError, match="CUDA is required"):
            call()


def test_arguments_that_come_together():
    graph = luna.make_graph(torch.tensor([0, 1]), torch.tensor([0, 1]))
    with pytest.raises(TypeError, match="together"):
        luna.graph_softmax(torch.zeros(2), graph, table=torch.zeros(2, 1))
    with pytest.raises(TypeError, match="make_graph"):
        luna.graph_softmax(torch.zeros(2), torch.tensor([0, 1]))
    for boundaries in ([-1.0, 2.0], [2.0, 1.0], [0.0, float("inf")], [float("nan")]):
        with pytest.raises(ValueError, match="boundaries"):
            luna.RelativeBias(boundaries, 4)
    with pytest.raises(ValueError, match="heads"):
        luna.RelativeBias([1.0], 0)
    assert luna.RelativeBias([], 4).weight.shape == (1, 4)


def test_descriptions_are_checked_at_the_entry_points():
    """Bad descriptions end in a status; no launch is reached."""
    import ctypes

    from lunaequivariance_b200 import _native

    lib = _native.library()
    desc = _native.NormDesc(dtype=0, num_blocks=1, normalization=0, eps=1e-5)
    desc.mul[0], desc.components[0], desc.scalar[0] = 4, 1, 1
    some = ctypes.c_void_p(16)

    def forward(**change):
        d = _native.NormDesc.from_buffer_copy(desc)
        for name, value in change.items():
            if name in ("mul", "components", "scalar"):
                getattr(d, name)[0] = value
            else:
                setattr(d, name, value)
        return lib.luna_layer_norm_fwd(ctypes.byref(d), some, None, None, some, None, 1, None)

    for change in (dict(dtype=7), dict(num_blocks=0), dict(mul=0), dict(components=2), dict(components=3), dict(normalization=2),
                   dict(eps=-1.0), dict(eps=float("nan"))):
        assert forward(**change) == _native.LUNA_ERR_INVALID_ARGUMENT, change
    assert forward(num_blocks=33) == forward(mul=16385) == _native.LUNA_ERR_UNSUPPORTED
    assert lib.luna_layer_norm_fwd(ctypes.byref(desc), None, None, None, some, None, 1, None) == _native.LUNA_ERR_INVALID_ARGUMENT
    assert lib.luna_layer_norm_fwd(ctypes.byref(desc), ctypes.c_void_p(2), None, None, some, None, 1, None) == _native.LUNA_ERR_MISALIGNED
    assert lib.luna_layer_norm_bwd(ctypes.byref(desc), some, None, some, some, None, some, None, None, 0, 1, None) == _native.LUNA_ERR_SCRATCH
    assert lib.luna_relative_bias_bwd(0, some, some, some, None, 0, 4, 2, 2, None) == _native.LUNA_ERR_SCRATCH
    assert lib.luna_relative_bias_fwd(0, some, some, some, 4, 0, 2, None) == _native.LUNA_ERR_INVALID_ARGUMENT
    assert lib.luna_distance_buckets(2, some, some, 1, some, 1, None) == _native.LUNA_ERR_INVALID_ARGUMENT
    table = _native.RowTable(2, 4, 0, 0, 16)
    softmax = lambda t, **k: lib.luna_graph_softmax_fwd(  # noqa: E731
        k.get("dtype", 0), ctypes.byref(t), k.get("logits", some), k.get("table"), None, None, some, None, k.get("heads", 1), 0, None, 0, None)
    assert softmax(table, heads=0) == softmax(table, dtype=9) == softmax(table, logits=None) == _native.LUNA_ERR_INVALID_ARGUMENT
    assert softmax(table, table=some) == _native.LUNA_ERR_INVALID_ARGUMENT
    assert softmax(_native.RowTable(2, 4, 0, 0, 18)) == _native.LUNA_ERR_MISALIGNED
    assert softmax(_native.RowTable(2, 4, 0, 0, None)) == _native.LUNA_ERR_INVALID_ARGUMENT
    assert softmax(_native.RowTable(2, 1 << 31, 0, 0, 16)) == _native.LUNA_ERR_OVERFLOW
    assert softmax(_native.RowTable(2, 4, 2, 1, 16, 16, 16)) == _native.LUNA_ERR_INVALID_ARGUMENT
    assert softmax(_native.RowTable(2, 4, 3, 1, 16, 16, 16, 16, 16)) == _native.LUNA_ERR_INVALID_ARGUMENT
    assert softmax(_native.RowTable(2, 4, 2, 1, 16, 16, 16, 16, 16)) == _native.LUNA_ERR_SCRATCH


def test_rows_are_cut():
    """The tables of cut rows, checked against the rows they are made of."""
    from lunaequivariance_b200.graph import _cut_rows

    for degrees in ([3, 20, 0, 8, 9, 0], [17], [0, 16, 16, 33]):
        degree = torch.tensor(degrees, dtype=torch.int32)
        rowptr = torch.cat([torch.zeros(1), degree.cumsum(0)]).to(torch.int32)
        rows, piece_of_row, row_of_piece, cut_of_piece, cut_first = (t.tolist() for t in _cut_rows(rowptr, degree, 8, 4))
        row, piece, cut = 0, 0, 0
        for node, n in enumerate(degrees):
            count = -(-n // 4) if n > 8 else 1
            for j in range(count):
                assert rows[row] == rowptr[node] + 4 * j
                assert piece_of_row[row] == (piece if n > 8 else -1)
                if n > 8:
                    assert (row_of_piece[piece], cut_of_piece[piece]) == (row, cut)
                    piece += 1
                row += 1
            if n > 8:
                cut += 1
                assert cut_first[cut] == piece
        assert rows[row] == sum(degrees) and len(rows) == row + 1 and len(cut_first) == cut + 1 and len(row_of_piece) == piece


def test_the_oracle():
    logits = torch.tensor([1.0, 2.0, 3.0, 5.0], dtype=torch.float64)
    dst = torch.tensor([0, 0, 2, 2])
    alpha = oracle.graph_softmax(logits, dst, 4, mask=torch.tensor([True, True, False, False]))
    assert torch.allclose(alpha, torch.tensor([0.2689414213699951, 0.7310585786300049, 0.0, 0.0], dtype=torch.float64))
    vec = torch.tensor([[3.0, 4.0, 0.0], [0.0, 0.0, 1.0]])
    assert oracle.distance_buckets(vec, torch.tensor([1.0, 5.0, 6.0])).tolist() == [2, 1]
    x = torch.tensor([[1.0, 3.0, 3.0, 4.0, 0.0]], dtype=torch.float64)
    y = oracle.layer_norm(x, "2x0e+1x1o", eps=0.0)
    assert torch.allclose(y, torch.tensor([[-1.0, 1.0, 3.0, 4.0, 0.0]], dtype=torch.float64) / torch.tensor([1, 1, *[(25 / 3) ** 0.5] * 3]))
