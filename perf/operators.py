"""The operators of attention over a node's neighbours, as cases that can be timed and compared.

Layer norm over irreps, the learned bias by distance buckets, and the softmax over the in-edges of every node: what a
network computes between its features and the ``env=`` of the convolution that sums the messages.  ``prepare`` makes what a
program holds before the call, ``run`` is one pass, in elementary torch operations or, with ``own`` set, through the package.
"""

from __future__ import annotations

import math
import re

import torch

own = False

DTYPES = {"float32": torch.float32, "float64": torch.float64, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZES = {"float32": 4, "float64": 8, "bfloat16": 2, "float16": 2}
EPS = 1e-5
CUTOFF = 5.0  # Angstrom


def listed():
    return [
        # The scalars and vectors of one molecule before a layer, in inference.
        _norm("norm_molecule_24", "forward", 24, "64x0e+64x1o+64x2e"),
        # The hidden layer of a radial network in training: one row per edge of a protein-sized system.
        _norm("norm_radial_86k", "training", 85_876, "64x0e"),
        # Node features of the 128-channel interaction layer in training, 50,000 atoms.
        _norm("norm_nodes_50k", "training", 50_000, "128x0e+128x1o+128x2e"),
        # A radial network in force training, where the norm is differentiated twice: 1.0 M edges in double precision.
        _norm("norm_radial_1m_f64", "force_training", 1_047_038, "64x0e", dtype="float64"),
        # A wide readout in half precision whose rows are no multiple of anything.
        _norm("norm_wide_odd_bf16", "training", 20_011, "1001x0e", dtype="bfloat16"),
        # The bias of every edge of a protein-sized system, and its gradient.
        _bias("bias_86k", "training", 85_876, 32, 8),
        # Learned weights by distance for every channel of a small layer: wide rows, few buckets, inference.
        _bias("bias_weights_200k", "forward", 209_200, 16, 704),
        # The bias of 2.6 M edges with many buckets and heads in training.
        _bias("bias_2600k", "training", 2_614_912, 128, 16),
        # Attention over one molecule in inference: every atom neighbours every other.
        _softmax("softmax_molecule_24", "forward", 24, 552, 4, 32, graph="complete"),
        # Force training of a protein-sized system.
        _softmax("softmax_forces_2k", "force_training", 2_083, 85_876, 8, 32),
        # Training step of a large system: 50,000 atoms with 52 neighbours, an eighth of the edges beyond the cutoff.
        _softmax("softmax_50k", "training", 50_000, 2_614_912, 8, 64, masked=0.125),
        # Virtual nodes and hubs: rows of very different length, the longest of tens of thousands of edges.
        _softmax("softmax_hubs_f64", "training", 5_003, 1_000_003, 3, 0, graph="hubs", dtype="float64"),
    ]


def _norm(name, order, rows, irreps, *, normalization="component", dtype="float32"):
    return _named(name, {"kind": "layer_norm", "order": order, "rows": rows, "irreps": irreps,
                         "normalization": normalization, "dtype": dtype})


def _bias(name, order, edges, buckets, heads, *, dtype="float32"):
    return _named(name, {"kind": "relative_bias", "order": order, "edges": edges, "buckets": buckets, "heads": heads,
                         "dtype": dtype})


def _softmax(name, order, nodes, edges, heads, buckets, *, masked=0.0, graph="radius", dtype="float32"):
    return _named(name, {"kind": "graph_softmax", "order": order, "nodes": nodes, "edges": edges, "heads": heads,
                         "buckets": buckets, "masked": masked, "graph": graph, "dtype": dtype})


def _named(name, case):
    return dict(case, name=name) if name else case


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("layer_norm", "layer_norm", "layer_norm", "relative_bias", "graph_softmax", "graph_softmax", "graph_softmax"))
    order = rng.choice(("forward", "training", "training", "force_training"))
    dtype = rng.choice(("float32", "float32", "float32", "float64"))
    if order != "force_training" and rng.random() < 0.25:
        dtype = rng.choice(("bfloat16", "float16"))
    if kind == "layer_norm":
        if rng.random() < 0.5:
            irreps = f"{_log_uniform(rng, 8, 2_100)}x0e"
        else:
            mul = rng.choice((16, 32, 48, 50, 64, 96, 128))
            irreps = "+".join(f"{mul}x{l}{'o' if l % 2 else 'e'}" for l in range(rng.randint(0, 1), rng.randint(2, 4)))
        most = int(5e7 * 4 / (_dim(irreps) * SIZES[dtype]))
        return _norm(None, order, _log_uniform(rng, 24, min(2_000_000, most)), irreps,
                     normalization=rng.choice(("component", "component", "norm")), dtype=dtype)
    heads = rng.choice((1, 1, 2, 3, 4, 4, 5, 8, 8, 12, 16, 32, 64))
    buckets = rng.choice((16, 25, 32, 64, 100, 128, 256))
    most = int(4e7 * 4 / (heads * SIZES[dtype]))
    if kind == "relative_bias":
        order = "forward" if order == "forward" else "training"
        return _bias(None, order, _log_uniform(rng, 500, min(2_600_000, most)), buckets, heads, dtype=dtype)
    edges = _log_uniform(rng, 500, min(2_600_000, most))
    degree = rng.uniform(4.0, 60.0)
    return _softmax(None, order, max(2, int(edges / degree)), edges, heads, rng.choice((0, buckets, buckets)),
                    masked=rng.choice((0.0, 0.0, 0.1, 0.5)), graph=rng.choice(("radius", "radius", "radius", "hubs")), dtype=dtype)


# ------------------------------------------------------------------------------------------------------- inputs


def _blocks(irreps):
    """(multiplicity, components, whether the block is of scalars) of every block."""
    found = re.findall(r"(\d+)x(\d+)([eo])", irreps)
    return [(int(mul), 2 * int(l) + 1, l == "0" and p == "e") for mul, l, p in found]


def _dim(irreps):
    return sum(mul * d for mul, d, _ in _blocks(irreps))


def _vectors(edges, generator, dtype):
    """Edge vectors of a uniform density, all within 1.1 cutoffs."""
    direction = torch.randn(edges, 3, generator=generator, device="cuda", dtype=torch.float32)
    length = 1.1 * CUTOFF * torch.rand(edges, 1, generator=generator, device="cuda").pow(1.0 / 3.0)
    return (direction * (length / direction.norm(dim=1, keepdim=True))).to(dtype)


def _boundaries(buckets, dtype):
    """Borders whose distances grow from bucket to bucket, as the resolution of a learned bias falls with distance."""
    steps = torch.linspace(math.log(0.5), math.log(CUTOFF), buckets - 1, device="cuda", dtype=torch.float64)
    return steps.exp().to(dtype)


def _destinations(case, generator):
    nodes, edges = case["nodes"], case["edges"]
    if case["graph"] == "complete":
        return torch.arange(nodes, device="cuda").repeat_interleave(nodes - 1)
    place = torch.rand(edges, generator=generator, device="cuda", dtype=torch.float64)
    if case["graph"] == "hubs":
        place = place.pow(3.0)
    return (place * nodes).long().clamp_(max=nodes - 1).sort()[0]


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0):
        # drawn in single precision, so that it costs little, and spread over the bits of the type
        return torch.randn(*shape, generator=generator, device="cuda").to(dtype) * scale + shift

    state = {"case": case}
    second = case["order"] == "force_training"
    if case["kind"] == "layer_norm":
        shape = (case["rows"], _dim(case["irreps"]))
        blocks = _blocks(case["irreps"])
        state["x"] = normal(*shape, scale=1.3, shift=0.2)
        state["weight"] = normal(sum(mul for mul, _, _ in blocks), scale=0.1, shift=1.0)
        state["bias"] = normal(sum(mul for mul, _, scalar in blocks if scalar), scale=0.1)
        if own:
            import lunaequivariance_b200 as luna

            state["irreps"] = luna.Irreps(case["irreps"])
    elif case["kind"] == "relative_bias":
        shape = (case["edges"], case["heads"])
        vectors = dtype if dtype in (torch.float32, torch.float64) else torch.float32
        state["vec"] = _vectors(case["edges"], generator, vectors)
        state["boundaries"] = _boundaries(case["buckets"], vectors)
        state["table"] = normal(case["buckets"], case["heads"], scale=0.5)
    else:
        shape = (case["edges"], case["heads"])
        state["logits"] = normal(*shape, scale=1.5)
        state["dst"] = _destinations(case, generator)
        state["mask"] = state["table"] = state["buckets"] = None
        if case["masked"]:
            state["mask"] = torch.rand(case["edges"], generator=generator, device="cuda") >= case["masked"]
        if case["buckets"]:
            length = _vectors(case["edges"], generator, torch.float32).norm(dim=1)
            state["buckets"] = torch.bucketize(length, _boundaries(case["buckets"], torch.float32), right=True, out_int32=True)
            state["table"] = normal(case["buckets"], case["heads"], scale=0.5)
        if own:
            import lunaequivariance_b200 as luna

            others = torch.Generator(device="cuda").manual_seed(seed + 1)  # the inputs do not depend on the sources
            src = torch.randint(case["nodes"], (case["edges"],), generator=others, device="cuda")
            state["graph"] = luna.make_graph(src, state["dst"], case["nodes"])
    if case["order"] != "forward":
        state["g"] = normal(*shape)
    if second:
        state["r"] = normal(*shape)
    if own and case["order"] != "forward":  # parameters and features of a program that differentiates
        for name in ("x", "weight", "bias", "table", "logits"):
            if state.get(name) is not None:
                state[name].requires_grad_(True)
        if second:
            state["g"].requires_grad_(True)
    return state


# ---------------------------------------------------------------------------------------------------------- run


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"layer_norm": _own_norm, "relative_bias": _own_bias, "graph_softmax": _own_softmax}[kind](state)
    return {"layer_norm": _plain_norm, "relative_bias": _plain_bias, "graph_softmax": _plain_softmax}[kind](state)


def _own_norm(state):
    import lunaequivariance_b200 as luna

    case, x, weight, bias = state["case"], state["x"], state["weight"], state["bias"]
    y = luna.layer_norm(x, state["irreps"], weight, bias, eps=EPS, normalization=case["normalization"])
    if case["order"] == "forward":
        return {"y": y}
    if case["order"] == "training":
        gx, gw, gb = torch.autograd.grad(y, (x, weight, bias), state["g"])
        return {"y": y, "gx": gx, "gw": gw, "gb": gb}
    gx, = torch.autograd.grad(y, x, state["g"], create_graph=True)
    hx, hw, hg = torch.autograd.grad(gx, (x, weight, state["g"]), state["r"])
    return {"y": y, "gx": gx, "hx": hx, "hw": hw, "hg": hg}


def _own_bias(state):
    import lunaequivariance_b200 as luna

    buckets = luna.distance_buckets(state["vec"], state["boundaries"])
    bias = luna.relative_bias(state["table"], buckets)
    if state["case"]["order"] == "forward":
        return {"buckets": buckets, "bias": bias}
    return {"buckets": buckets, "bias": bias, "gtable": torch.autograd.grad(bias, state["table"], state["g"])[0]}


def _own_softmax(state):
    import lunaequivariance_b200 as luna

    order, logits, table = state["case"]["order"], state["logits"], state["table"]
    alpha = luna.graph_softmax(logits, state["graph"], mask=state["mask"], table=table, buckets=state["buckets"])
    if order == "forward":
        return {"alpha": alpha}
    inputs = (logits,) if table is None else (logits, table)
    if order == "training":
        return {"alpha": alpha, "first": torch.autograd.grad(alpha, inputs, state["g"])}
    first = torch.autograd.grad(alpha, inputs, state["g"], create_graph=True)
    second = torch.autograd.grad(first[0], (*inputs, state["g"]), state["r"])
    return {"alpha": alpha, "first": first, "hg": second[-1], "second": second[:-1]}


def _wide(t):
    """The type that the plain forms compute in."""
    return t if t is None or t.dtype == torch.float64 else t.float()


def _plain_norm(state):
    case, dtype = state["case"], state["x"].dtype
    x, weight, bias, g, r = (_wide(state.get(name)) for name in ("x", "weight", "bias", "g", "r"))
    rows = x.shape[0]
    parts = {name: [] for name in ("y", "gx", "gw", "gb", "hx", "hw", "hg")}
    at = wat = bat = 0
    for mul, d, scalar in _blocks(case["irreps"]):
        share = 1.0 / (mul * d if case["normalization"] == "component" else mul)
        block = lambda t: t[:, at:at + mul * d].reshape(rows, mul, d)  # noqa: B023, E731
        total = lambda t: t.sum((1, 2), keepdim=True)  # noqa: E731
        centred = lambda t: t - total(t) / mul if scalar else t  # noqa: B023, E731
        w = weight[wat:wat + mul].reshape(1, mul, 1)
        h = centred(block(x))
        s = 1.0 / (total(h * h) * share + EPS).sqrt()
        h = h * s
        y = h * w
        if scalar:
            y = y + bias[bat:bat + mul].reshape(1, mul, 1)
        found = {"y": y}
        if g is not None:
            e = block(g)
            project = lambda t: centred(t) - h * (total(t * h) * share)  # noqa: B023, E731
            found["gx"] = s * project(e * w)
            parts["gw"].append((e * h).sum((0, 2)))
            if scalar:
                parts["gb"].append(e.sum((0, 2)))
        if r is not None:
            t, c = block(r), e * w
            p, k = project(t), project(c)
            a, b, dot = total(t * h), total(c * h), total(centred(t) * c)
            found["hx"] = -s * s * share * ((dot - share * a * b) * h + b * p + a * k)
            found["hg"] = w * s * p
            parts["hw"].append((s * p * e).sum((0, 2)))
        for name, value in found.items():
            parts[name].append(value.reshape(rows, mul * d))
        at, wat, bat = at + mul * d, wat + mul, bat + (mul if scalar else 0)
    gathered = {}
    for name in {"forward": ("y",), "training": ("y", "gx", "gw", "gb"), "force_training": ("y", "gx", "hx", "hw", "hg")}[case["order"]]:
        gathered[name] = torch.cat(parts[name], -1).to(dtype) if parts[name] else torch.empty(0, dtype=dtype, device=x.device)
    return gathered


def _sum_by(index, values, count):
    """Sums of rows with one index: of very many, so in 64 bits."""
    return values.new_zeros(count, values.shape[1], dtype=torch.float64).index_add_(0, index, values.double())


def _plain_bias(state):
    case, table = state["case"], state["table"]
    vec, boundaries = state["vec"].double(), state["boundaries"].double()
    squared = vec[:, 0] * vec[:, 0] + vec[:, 1] * vec[:, 1] + vec[:, 2] * vec[:, 2]
    buckets = torch.bucketize(squared, boundaries * boundaries, right=True, out_int32=True)
    found = {"buckets": buckets, "bias": table[buckets]}
    if case["order"] == "training":
        found["gtable"] = _sum_by(buckets, state["g"], case["buckets"]).to(table.dtype)
    return found


def _plain_softmax(state):
    case, dst, mask, buckets = state["case"], state["dst"], state["mask"], state["buckets"]
    dtype = state["logits"].dtype
    z, table, g, r = (_wide(state.get(name)) for name in ("logits", "table", "g", "r"))
    nodes, heads = case["nodes"], case["heads"]

    def total(t):
        return t.new_zeros(nodes, heads).index_add_(0, dst, t)[dst]

    if table is not None:
        z = z + table[buckets]
    if mask is not None:
        z = torch.where(mask[:, None], z, -math.inf)
    largest = z.new_full((nodes, heads), -math.inf).index_reduce_(0, dst, z, "amax")
    largest = torch.where(largest == -math.inf, 0.0, largest)
    e = (z - largest[dst]).exp()
    alpha = torch.where(e > 0, e / total(e), e)
    found = {"alpha": alpha.to(dtype)}
    if case["order"] == "forward":
        return found

    def with_table(t):
        return (t.to(dtype),) if table is None else (t.to(dtype), _sum_by(buckets, t, case["buckets"]).to(dtype))

    dot = total(alpha * g)
    found["first"] = with_table(alpha * (g - dot))
    if case["order"] == "force_training":
        other = total(alpha * r)
        found["hg"] = (alpha * (r - other)).to(dtype)
        change = r * (g - dot) - g * other
        found["second"] = with_table(alpha * (change - total(alpha * change)))
    return found


# -------------------------------------------------------------------------------------------------------- floors


def work(case):
    size = SIZES[case["dtype"]]
    # arrays of the operator's shape that a pass reads and writes, and operations for each of their values
    arrays, flops = {"forward": (2, 8), "training": (4, 24), "force_training": (7, 64)}[case["order"]]
    if case["kind"] == "layer_norm":
        values = case["rows"] * _dim(case["irreps"])
        parameters = sum(mul * (2 if scalar else 1) for mul, _, scalar in _blocks(case["irreps"]))
        return {"bytes": size * (arrays * values + parameters * (1 if case["order"] == "forward" else 2)),
                "flops": flops * values}
    values, rows = case["edges"] * case["heads"], case["buckets"] * case["heads"]
    if case["kind"] == "relative_bias":
        training = case["order"] == "training"
        vectors = 8 if case["dtype"] == "float64" else 4
        return {"bytes": case["edges"] * (3 * vectors + 4) + size * (2 if training else 1) * (values + rows),
                "flops": 5 * case["edges"] + (values if training else 0)}
    tables = {"forward": 1, "training": 2, "force_training": 3}[case["order"]]
    per_edge = (4 if case["buckets"] else 0) + (1 if case["masked"] else 0)
    return {"bytes": size * (arrays * values + tables * rows) + per_edge * case["edges"] + 4 * (case["nodes"] + 1),
            "flops": flops * values}


# ------------------------------------------------------------------------------- the definitions, in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    exactly = {"layer_norm": _exact_norm, "relative_bias": _exact_bias, "graph_softmax": _exact_softmax}[case["kind"]]
    with torch.enable_grad():
        found = exactly(case, state)
    detached = lambda v: v.detach() if isinstance(v, torch.Tensor) else tuple(t.detach() for t in v)  # noqa: E731
    return {name: None if v is None else detached(v) for name, v in found.items()}


def _leaf(t):
    return t.detach().double().requires_grad_(True)


def _exact_norm(case, state):
    """Values from the moments of every block; derivatives from those of the values."""
    x, weight, bias = (_leaf(state[name]) for name in ("x", "weight", "bias"))
    pieces, columns = [], 0
    weights, biases = iter(weight.split([mul for mul, _, _ in _blocks(case["irreps"])])), bias
    for mul, d, scalar in _blocks(case["irreps"]):
        piece = x.narrow(1, columns, mul * d).unflatten(1, (mul, d))
        columns += mul * d
        power = piece.square().sum(-1).mean(-1) / (d if case["normalization"] == "component" else 1)
        if scalar:
            centre = piece.mean((1, 2))
            piece, power = piece - centre[:, None, None], power - centre.square()
        piece = torch.einsum("rud,u,r->rud", piece, next(weights), (power + EPS).rsqrt())
        if scalar:
            piece, biases = piece + biases[:mul, None], biases[mul:]
        pieces.append(piece.flatten(1))
    y = torch.cat(pieces, 1)
    if case["order"] == "forward":
        return {"y": y}
    if case["order"] == "training":
        gx, gw, gb = torch.autograd.grad(y, (x, weight, bias), state["g"].double(), allow_unused=True)
        return {"y": y, "gx": gx, "gw": gw, "gb": gb if gb is not None else torch.zeros_like(bias)}
    g = _leaf(state["g"])
    gx, = torch.autograd.grad(y, x, g, create_graph=True)
    hx, hw, hg = torch.autograd.grad(gx, (x, weight, g), state["r"].double())
    return {"y": y, "gx": gx, "hx": hx, "hw": hw, "hg": hg}


def _exact_bias(case, state):
    table = _leaf(state["table"])
    length = torch.linalg.vector_norm(state["vec"].double(), dim=1)
    buckets = torch.searchsorted(state["boundaries"].double(), length, right=True)
    bias = table.index_select(0, buckets)
    found = {"buckets": None, "bias": bias}
    if case["order"] == "training":
        order = buckets.argsort(stable=True)
        ends = torch.bincount(buckets, minlength=case["buckets"]).cumsum(0)
        running = torch.cat([bias.new_zeros(1, case["heads"]), state["g"].double()[order].cumsum(0)])[torch.cat([ends.new_zeros(1), ends])]
        found["gtable"] = running.diff(dim=0)
    return found


def _exact_softmax(case, state):
    """Without the largest logit taken out: the logits are far from the ends of the type's range."""
    logits = _leaf(state["logits"])
    table = None if state["table"] is None else _leaf(state["table"])
    weights = logits.exp()
    if table is not None:
        weights = weights * table.exp().index_select(0, state["buckets"])
    if state["mask"] is not None:
        weights = weights * state["mask"].double()[:, None]
    sums = torch.zeros(case["nodes"], case["heads"], dtype=torch.float64, device=logits.device).index_add(0, state["dst"], weights)
    sums = torch.where(sums == 0, 1.0, sums)
    alpha = weights / sums.index_select(0, state["dst"])
    if case["order"] == "forward":
        return {"alpha": alpha}
    inputs = (logits,) if table is None else (logits, table)
    g = _leaf(state["g"])
    first = torch.autograd.grad(alpha, inputs, g, create_graph=case["order"] == "force_training")
    if case["order"] == "training":
        return {"alpha": alpha, "first": first}
    second = torch.autograd.grad(first[0], (*inputs, g), state["r"].double())
    return {"alpha": alpha, "first": first, "hg": second[-1], "second": second[:-1]}
