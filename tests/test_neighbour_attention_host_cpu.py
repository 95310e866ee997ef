"""What the operators of attention over neighbours do on the host: checks at the entry points, and tables that are made once."""

import ctypes
import threading

import pytest
import torch

import lunaequivariance_b200 as luna
from lunaequivariance_b200 import _native
from lunaequivariance_b200 import graph as graph_mod
from lunaequivariance_b200.conv import edge_output_graph


def test_wide_cotangents_are_checked():
    """The forms for cotangents in float: refused as their counterparts are, and where 16-bit types are not aligned to 16 bytes."""
    lib = _native.library()
    some, odd = ctypes.c_void_p(16), ctypes.c_void_p(20)
    table = _native.RowTable(2, 4, 0, 0, 16)

    def backward(dtype, alpha=some, g=some, heads=1):
        return lib.luna_graph_softmax_bwd_wide(dtype, ctypes.byref(table), alpha, g, None, None, None, heads, 0, None, 0, None)

    def second(dtype, alpha=some, halpha=some, g=None):
        return lib.luna_graph_softmax_dbl_bwd_wide(dtype, ctypes.byref(table), alpha, g, None, None, None, halpha, None, 1, 0, None, 0, None)

    for dtype in (_native.LUNA_BF16, _native.LUNA_F16):
        assert backward(dtype, g=odd) == backward(dtype, alpha=odd) == _native.LUNA_ERR_MISALIGNED
        assert second(dtype, g=some, halpha=odd) == _native.LUNA_ERR_MISALIGNED
    for dtype in range(4):
        # an output, an operand, a head too few
        assert backward(dtype) == backward(dtype, g=None) == backward(dtype, heads=0) == _native.LUNA_ERR_INVALID_ARGUMENT
        assert second(dtype) == second(dtype, alpha=None, g=some) == _native.LUNA_ERR_INVALID_ARGUMENT
    assert backward(9) == second(9) == _native.LUNA_ERR_INVALID_ARGUMENT
    assert backward(_native.LUNA_F32, g=ctypes.c_void_p(18)) == _native.LUNA_ERR_MISALIGNED


def hub_graph(monkeypatch):
    monkeypatch.setattr(graph_mod, "ROW_SPLIT_EDGES", 8)
    monkeypatch.setattr(graph_mod, "ROW_PIECE_EDGES", 4)
    dst = torch.repeat_interleave(torch.arange(5), torch.tensor([3, 20, 0, 9, 30]))
    return luna.make_graph(torch.randint(5, dst.shape, generator=torch.Generator().manual_seed(0)), dst, 5)


# What a graph makes on first use, by the name it is kept under.
DERIVED = {"rows": lambda g: g.row_holder(), "split": lambda g: g.split_rows(), ("range", 1, 4): lambda g: g.destination_range(1, 4),
           "edge_output_graph": edge_output_graph}


@pytest.mark.parametrize("name", list(DERIVED), ids=str)
def test_tables_are_finished_before_anyone_finds_them(name, monkeypatch):
    """Another stream's or thread's call takes what is kept at once: it is kept only after the stream that makes it was waited for."""
    graph, waits = hub_graph(monkeypatch), []

    def wait(device):
        assert name not in graph._tables
        waits.append(device)

    monkeypatch.setattr(graph_mod, "_wait_for_tables", wait)
    first = DERIVED[name](graph)
    assert waits == [graph.src.device] and name in graph._tables
    assert DERIVED[name](graph) is first and len(waits) == 1


@pytest.mark.parametrize("name", list(DERIVED), ids=str)
def test_tables_are_made_once_for_two_threads(name, monkeypatch):
    graph, begun, finished, waits = hub_graph(monkeypatch), threading.Event(), threading.Event(), []

    def wait(device):
        waits.append(device)
        begun.set()
        assert finished.wait(20)

    monkeypatch.setattr(graph_mod, "_wait_for_tables", wait)
    found = [None, None]

    def call(i):
        found[i] = DERIVED[name](graph)

    threads = [threading.Thread(target=call, args=(i,), daemon=True) for i in range(2)]
    threads[0].start()
    assert begun.wait(20)
    threads[1].start()
    threads[1].join(0.2)
    assert found == [None, None]  # neither has tables that are not finished
    finished.set()
    for thread in threads:
        thread.join(20)
    assert found[0] is not None and found[0] is found[1] and len(waits) == 1


@pytest.mark.parametrize("name", list(DERIVED), ids=str)
def test_memory_of_tables_is_kept_for_every_stream(name, monkeypatch):
    """Tables that no caller sees are recorded once with each stream that a call uses them on."""
    graph, recorded = hub_graph(monkeypatch), []
    stream = None
    monkeypatch.setattr(graph_mod, "_stream_in_use", lambda device: stream)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: recorded.append((t.data_ptr(), s)))
    for stream in ("one", "other", "one", "other"):
        DERIVED[name](graph)
    tables = {t.data_ptr() for t in graph._tables[name].tensors}
    assert sorted(recorded) == sorted((t, s) for s in ("one", "other") for t in [t.data_ptr() for t in graph._tables[name].tensors])
    own = {t.data_ptr() for t in graph.tensors() if t.numel()}
    assert len(tables) > 1 and not tables & own


def test_graphs_without_tables_of_their_own_wait_for_nothing(monkeypatch):
    monkeypatch.setattr(graph_mod, "_wait_for_tables", lambda device: pytest.fail("waited"))
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: pytest.fail("recorded"))
    graph = luna.make_graph(torch.tensor([0, 1, 1]), torch.tensor([0, 1, 1]), 2)
    assert graph.split_rows() is None and graph.row_holder() is graph.row_holder()


@pytest.mark.parametrize("known", [True, False])
def test_a_trace_leaves_no_stand_ins_in_a_module(known):
    """Borders of a trace with stand-ins for tensors stay in it: the next trace, and calls with numbers, have their own."""
    from torch.fx.experimental.proxy_tensor import make_fx

    module = luna.RelativeBias([1.0, 2.5], 3)
    if not known:
        module._borders = {}
    before = set(module._borders)
    for mode in ("fake", "symbolic", "fake"):
        traced = make_fx(lambda v: module.buckets(v), tracing_mode=mode)(torch.randn(5, 3))
        assert traced._tensor_constant0.shape == (2,)
        assert set(module._borders) == before
    exported = torch.export.export(_Buckets(module), (torch.randn(5, 3),), strict=False)
    assert "lunaeq.distance_buckets" in str(exported.graph) and set(module._borders) == before
    with torch._subclasses.fake_tensor.FakeTensorMode():
        assert luna.RelativeBias([1.0], 2)._borders == {}
    with torch.inference_mode():
        assert not any(t.is_inference() for t in luna.RelativeBias([1.0], 2)._borders.values())
    for dtype in (torch.float32, torch.float64):
        with pytest.raises(RuntimeError, match="CUDA is required"):  # in the launch, with what is kept for it
            module.buckets(torch.zeros(1, 3, dtype=dtype))
        kept = module._borders[torch.device("cpu"), dtype]
        assert type(kept) is torch.Tensor and kept.dtype == dtype and kept.tolist() == [1.0, 2.5]
    assert all(t.dtype in (torch.float32, torch.float64) for t in module.half()._borders.values()) and len(module._borders) == 2


class _Buckets(torch.nn.Module):
    def __init__(self, module):
        super().__init__()
        self.module = module

    def forward(self, vec):
        return self.module.buckets(vec)


def test_sizes_beyond_the_description():
    """Blocks that a description of 32 bits would hold as others are refused like all that are too long."""
    for irreps in (16385, "1x0e+20000x1o", (1 << 32) + 64):
        with pytest.raises(NotImplementedError, match="16384"):
            luna.LayerNormConfig(irreps).holder()


def test_tables_of_rows_that_launches_could_not_follow():
    rows = _native.binding().Rows
    numbers = torch.arange(8, dtype=torch.int32)
    for bad in (numbers[::2], numbers.reshape(2, 4), numbers[:0]):
        with pytest.raises(ValueError, match="row"):
            rows(bad, 4, None, None, None, None)
    with pytest.raises(ValueError, match="rows"):
        rows(numbers, 4, numbers[::2], numbers, numbers, numbers)
    with pytest.raises(RuntimeError, match="Int"):
        rows(numbers.long(), 4, None, None, None, None)


@pytest.mark.parametrize("name", ["split", ("range", 1, 4), "edge_output_graph"], ids=str)
def test_graphs_are_copied_with_their_tables(name, monkeypatch):
    import copy
    import pickle

    graph = hub_graph(monkeypatch)
    monkeypatch.setattr(graph_mod, "_stream_in_use", lambda device: lambda: None)  # no stream can be copied
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: None)
    DERIVED[name](graph)
    for other in (copy.deepcopy(graph), pickle.loads(pickle.dumps(graph))):
        mine, its = graph._tables[name].tensors, other._tables[name].tensors
        assert len(mine) == len(its) and all(torch.equal(a, b) and a.data_ptr() != b.data_ptr() for a, b in zip(mine, its) if a.numel())
        assert not other._tables[name].streams
