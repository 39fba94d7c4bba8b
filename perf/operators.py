"""Workloads of the segmented scan and the segmented matrix product.

Both operators take the packed rows ``values[N, ...]`` and ``offsets[B + 1]``
that the rest of the library takes; segment s holds rows offsets[s] to
offsets[s + 1].

* scan: h[t] = gates[t] * h[t - 1] + values[t] within each segment, column by
  column.  Before a segment's first row the state is initial[s] if initial
  states are given; without them the first row is values[t] itself.  final[s]
  is the state after the segment's last row (the initial one, or zeros, where
  the segment is empty).
* matmul: out[t] = values[t] @ weights[s] for the rows t of segment s.

A case with ``train`` computes the outputs and all gradients for given
gradients of the outputs.  ``run`` computes a case in plain torch operations
(``own`` false) or through the library (``own`` true); ``exact`` computes it
in 64 bits, by another route.
"""
from __future__ import annotations

import math
from pathlib import Path
import sys
import tempfile

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
INDEX = {"i32": torch.int32, "i64": torch.int64}


def listed():
    return [
        # One token of each of 200 sequences that are being generated: the state goes in and comes out.
        dict(name="scan step", op="scan", train=False, dtype="bf16", index="i32", n=200, b=200, d=1024,
             lengths="ones", state=True),
        # Prompts of very different lengths read in one packed batch, some of them empty.
        dict(name="scan prompts", op="scan", train=False, dtype="bf16", index="i64", n=131_072, b=2048, d=256,
             lengths="long_tail", state=True),
        # Features of an odd width over short uneven groups of rows.
        dict(name="scan narrow f32", op="scan", train=False, dtype="f32", index="i64", n=262_001, b=1024, d=100,
             lengths="uniform", state=False),
        # A training step over a packed batch of sequences of a few thousand rows.
        dict(name="scan train", op="scan", train=True, dtype="bf16", index="i32", n=65_536, b=16, d=1024,
             lengths="uniform", state=False),
        # A training step over one long sequence with a carried state.
        dict(name="scan train long f32", op="scan", train=True, dtype="f32", index="i64", n=65_499, b=1, d=128,
             lengths="uniform", state=True),
        # A few tokens, each with its own expert: reading the weights is the work.
        dict(name="matmul few tokens", op="matmul", train=False, dtype="bf16", index="i32", n=32, b=16, k=1024,
             m=2048, lengths="routed"),
        # Narrow per-group projections (adapters) over a batch of many groups.
        dict(name="matmul adapters", op="matmul", train=False, dtype="bf16", index="i32", n=8192, b=256, k=1024,
             m=64, lengths="uniform"),
        # The tokens of a prompt batch through their experts.
        dict(name="matmul prompts", op="matmul", train=False, dtype="bf16", index="i64", n=16_384, b=64, k=1024,
             m=1024, lengths="routed"),
        # Widths whose rows start at odd addresses.
        dict(name="matmul odd widths", op="matmul", train=False, dtype="bf16", index="i64", n=5003, b=12, k=501,
             m=333, lengths="routed"),
        # Full precision, as in a check or a small model.
        dict(name="matmul f32", op="matmul", train=False, dtype="f32", index="i64", n=8192, b=8, k=512, m=512,
             lengths="routed"),
        # A training step of an expert layer.
        dict(name="matmul train", op="matmul", train=True, dtype="bf16", index="i64", n=32_768, b=16, k=1024,
             m=2048, lengths="routed"),
        # A training step of a small layer in full precision, at odd sizes.
        dict(name="matmul train f32", op="matmul", train=True, dtype="f32", index="i32", n=3001, b=5, k=300, m=210,
             lengths="uniform"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("scan", "matmul"))
    case = dict(op=op, train=rng.random() < 0.5, dtype=rng.choice(("f32", "bf16")), index=rng.choice(("i32", "i64")))
    if op == "scan":
        d = _log(rng, 1, 1024)
        if rng.random() < 0.5:
            d = max(8, d // 8 * 8)
        n = _log(rng, 64, min(262_144, 65_536 * 1024 // d))
        case.update(n=n, b=_log(rng, max(1, n // 65_536), n), d=d, state=rng.random() < 0.5,
                    lengths=rng.choice(("uniform", "long_tail")))
        if rng.random() < 0.15:
            case.update(n=case["b"], lengths="ones")
    else:
        k, m = _log(rng, 16, 2048), _log(rng, 16, 2048)
        if rng.random() < 0.6:
            k, m = max(8, k // 8 * 8), max(8, m // 8 * 8)
        most = 32_768 * 1024 * 2048 // (k * m)
        if case["dtype"] == "f32":
            most //= 8
        n = _log(rng, 1, max(64, min(65_536, most)))
        b = _log(rng, 1, 256)
        case.update(n=n, b=min(b, max(1, (1 << 26) // (k * m))), k=k, m=m, lengths=rng.choice(("routed", "uniform")))
    return case


def _lengths(case):
    """Lengths that sum to n, by the case alone; ``prepare`` puts them in the order that its seed gives."""
    n, b = case["n"], case["b"]
    rng = np.random.default_rng(n * 1009 + b)
    if case["lengths"] == "ones":
        return np.ones(b, dtype=np.int64)
    if case["lengths"] == "uniform":
        weights = rng.uniform(0.2, 1.8, b)
    elif case["lengths"] == "long_tail":
        weights = rng.lognormal(3.0, 1.5, b) * (rng.random(b) > 0.05)
        weights[0] = max(weights[0], 1.0)
    else:
        return rng.multinomial(n, rng.dirichlet(np.full(b, 8.0))).astype(np.int64)
    share = weights / weights.sum() * n
    lengths = np.floor(share).astype(np.int64)
    short = n - int(lengths.sum())
    lengths[np.argsort(lengths - share, kind="stable")[:short]] += 1
    return lengths


_cache = []


def _program(case):
    package = str(Path(__file__).resolve().parents[1] / "ragged-mlir_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from ragged import ArtifactCache, Compiler, MatmulSpec, ScanSpec
    if not _cache:
        _cache.append(ArtifactCache(tempfile.mkdtemp(prefix="ragged-operators-"), max_specializations=4096))
    if case["op"] == "scan":
        spec = ScanSpec(case["dtype"], case["d"], case["index"])
    else:
        spec = MatmulSpec(case["dtype"], case["k"], case["m"], case["index"])
    return Compiler().compile(spec, _cache[0])


def prepare(case, seed):
    device = torch.device("cuda")
    generator = torch.Generator(device=device)
    generator.manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=TYPES[case["dtype"]]):
        return (torch.randn(shape, generator=generator, device=device) * scale).to(dtype)

    lengths = np.random.default_rng(seed).permutation(_lengths(case))
    offsets = np.concatenate([[0], np.cumsum(lengths)])
    n, b, train = case["n"], case["b"], case["train"]
    state = dict(case=case, offsets=torch.from_numpy(offsets).to(device, INDEX[case["index"]]),
                 longest=int(lengths.max(initial=0)))
    if case["op"] == "scan":
        d = case["d"]
        state["values"] = normal(n, d)
        # Gates as a model computes them: the logistic function of a score that leans to keeping the state.
        score = torch.randn((n, d), generator=generator, device=device) * 2 + 2
        state["gates"] = torch.sigmoid(score).to(TYPES[case["dtype"]])
        state["initial"] = normal(b, d, dtype=torch.float32) if case["state"] else None
        state["out"] = torch.empty_like(state["values"])
        state["final"] = torch.empty((b, d), dtype=torch.float32, device=device)
        if train:
            state["grad_out"] = normal(n, d)
            state["grad_final"] = normal(b, d, dtype=torch.float32)
        leaves = ("values", "gates", "initial")
    else:
        k, m = case["k"], case["m"]
        state["values"] = normal(n, k)
        state["weights"] = normal(b, k, m, scale=1 / math.sqrt(k))
        state["out"] = torch.empty((n, m), dtype=TYPES[case["dtype"]], device=device)
        if train:
            state["grad_out"] = normal(n, m)
        leaves = ("values", "weights")
    if train:
        for name in leaves:
            if state[name] is not None:
                state[name].requires_grad_()
    if own:
        state["program"] = _program(case)
    return state


def run(state):
    scan, train = state["case"]["op"] == "scan", state["case"]["train"]
    if own:
        return (_own_scan if scan else _own_matmul)(state, train)
    with torch.no_grad():
        return (_plain_scan if scan else _plain_matmul)(state, train)


# ------------------------------------------------------------ the library

def _own_scan(state, train):
    values, gates, offsets, initial = (state[x] for x in ("values", "gates", "offsets", "initial"))
    if not train:
        state["program"].run(values, gates, offsets, state["out"], initial=initial, final=state["final"])
        return {"out": state["out"], "final": state["final"]}
    from ragged import torch_adapter
    out, final = torch_adapter.segment_scan(values, gates, offsets, program=state["program"], initial=initial)
    leaves = [values, gates] + ([initial] if initial is not None else [])
    grads = torch.autograd.grad((out, final), leaves, (state["grad_out"], state["grad_final"]))
    return {"out": out, "final": final, "grads": list(grads)}


def _own_matmul(state, train):
    values, weights, offsets = (state[x] for x in ("values", "weights", "offsets"))
    if not train:
        state["program"].run(values, weights, offsets, state["out"])
        return {"out": state["out"]}
    from ragged import torch_adapter
    out = torch_adapter.segment_matmul(values, weights, offsets, program=state["program"])
    grads = torch.autograd.grad(out, (values, weights), state["grad_out"])
    return {"out": out, "grads": list(grads)}


# --------------------------------------------------------- the plain forms

def _rows(state):
    """(offsets, lengths, segment of each row) on the device."""
    offsets = state["offsets"].long()
    counts = offsets[1:] - offsets[:-1]
    segments = torch.arange(counts.numel(), device=offsets.device)
    return offsets, counts, torch.repeat_interleave(segments, counts, output_size=state["case"]["n"])


def _doubling(gate, value, steps):
    """y[t] = gate[t] * y[t - 1] + value[t] over rows, by recursive doubling (both arguments are overwritten)."""
    for step in range(steps):
        k = 1 << step
        value[k:] += gate[k:] * value[:-k]
        gate[k:] *= gate[:-k].clone()
    return value


def _plain_scan(state, train):
    offsets, counts, segment = _rows(state)
    n, dtype, initial = state["case"]["n"], TYPES[state["case"]["dtype"]], state["initial"]
    steps = max(0, (state["longest"] - 1).bit_length())
    value, gate = state["values"].float(), state["gates"].float()
    row = torch.arange(n, device=value.device)
    first = (row == offsets[segment])[:, None]
    before = initial[segment] if initial is not None else torch.zeros((), device=value.device)
    h = _doubling(gate.masked_fill(first, 0), value + torch.where(first, gate * before, 0), steps)
    empty = (counts == 0)[:, None]
    at_empty = initial if initial is not None else torch.zeros((), device=value.device)
    final = torch.where(empty, at_empty, h[(offsets[1:] - 1).clamp(min=0)])
    out = {"out": h.to(dtype), "final": final}
    if not train:
        return out
    # g[t] = grad_out[t] + gate[t + 1] * g[t + 1], the same recurrence from each segment's last row to its first.
    last = (row + 1 == offsets[segment + 1])[:, None]
    grad = state["grad_out"].float() + torch.where(last, state["grad_final"][segment], 0)
    after = torch.cat([gate[1:], gate[:1]]).masked_fill(last, 0)
    g = _doubling(after.flip(0), grad.flip(0), steps).flip(0)
    previous = torch.where(first, before, torch.cat([h[:1], h[:-1]]))
    grads = [g.to(dtype), (g * previous).to(dtype)]
    if initial is not None:
        at = offsets[:-1].clamp(max=n - 1)
        grads.append(torch.where(empty, state["grad_final"], gate[at] * g[at]))
    return {**out, "grads": grads}


def _plain_matmul(state, train):
    offsets, counts, segment = _rows(state)
    n, dtype = state["case"]["n"], TYPES[state["case"]["dtype"]]
    place = torch.arange(n, device=segment.device) - offsets[segment]

    def padded(rows):
        full = torch.zeros((counts.numel(), state["longest"], rows.shape[1]), device=rows.device)
        full[segment, place] = rows.float()
        return full

    x, w = padded(state["values"]), state["weights"].float()
    out = {"out": torch.bmm(x, w)[segment, place].to(dtype)}
    if not train:
        return out
    grad = padded(state["grad_out"])
    return {**out, "grads": [torch.bmm(grad, w.transpose(1, 2))[segment, place].to(dtype),
                             torch.bmm(x.transpose(1, 2), grad).to(dtype)]}


# ------------------------------------------------------------ in 64 bits

def exact(case, seed):
    if case["op"] == "scan" and _lengths(case).max() > 70_000:
        return None
    state = prepare(case, seed)
    with torch.no_grad():
        return (_exact_scan if case["op"] == "scan" else _exact_matmul)(state, case["train"])


def _exact_scan(state, train):
    """Row by row: step t takes row t of every segment that has one, the longest segments first."""
    bounds = state["offsets"].cpu().numpy().astype(np.int64)
    lengths = np.diff(bounds)
    order = np.argsort(-lengths, kind="stable")
    active = np.searchsorted(-lengths[order], -np.arange(state["longest"]), side="left")
    device = state["values"].device
    order = torch.from_numpy(order).to(device)
    start = state["offsets"].long()[:-1][order]
    value, gate = state["values"].double(), state["gates"].double()
    initial = state["initial"]
    b, d = state["final"].shape
    h0 = initial.double()[order] if initial is not None else torch.zeros((b, d), dtype=torch.float64, device=device)
    h, out, previous = h0.clone(), torch.empty_like(value), torch.empty_like(value)
    for t, count in enumerate(active):
        rows = start[:count] + t
        previous[rows] = h[:count]
        h[:count] = gate[rows] * h[:count] + value[rows]
        out[rows] = h[:count]
    back = torch.argsort(order)
    result = {"out": out, "final": h[back]}
    if not train:
        return result
    grad_out = state["grad_out"].double()
    u, grad = state["grad_final"].double()[order].clone(), torch.empty_like(value)
    for t in range(len(active) - 1, -1, -1):
        rows = start[:active[t]] + t
        step = grad_out[rows] + u[:active[t]]
        grad[rows] = step
        u[:active[t]] = gate[rows] * step
    grads = [grad, grad * previous]
    return {**result, "grads": grads + ([u[back]] if initial is not None else [])}


def _exact_matmul(state, train):
    """Segment by segment."""
    bounds = state["offsets"].tolist()
    x, w = state["values"].double(), state["weights"]
    out = torch.zeros(state["out"].shape, dtype=torch.float64, device=x.device)
    spans = [(s, lo, hi) for s, (lo, hi) in enumerate(zip(bounds[:-1], bounds[1:])) if hi > lo]
    for s, lo, hi in spans:
        out[lo:hi] = x[lo:hi] @ w[s].double()
    if not train:
        return {"out": out}
    grad = state["grad_out"].double()
    gx, gw = torch.zeros_like(x), torch.zeros(w.shape, dtype=torch.float64, device=x.device)
    for s, lo, hi in spans:
        gx[lo:hi] = grad[lo:hi] @ w[s].double().T
        gw[s] = x[lo:hi].T @ grad[lo:hi]
    return {"out": out, "grads": [gx, gw]}


def work(case):
    """Inputs read once and outputs written once; the weights of segments with rows alone."""
    n, b = case["n"], case["b"]
    size = 4 if case["dtype"] == "f32" else 2
    index = (b + 1) * (4 if case["index"] == "i32" else 8)
    if case["op"] == "scan":
        d, state = case["d"], 4 * b * case["d"]
        traffic, flops = 3 * n * d * size + state * (2 if case["state"] else 1) + index, 2 * n * d
        if case["train"]:  # the backward pass reads values, gates and gradients and writes two gradients
            traffic += 5 * n * d * size + state * (3 if case["state"] else 1) + index
            flops += 5 * n * d
    else:
        k, m = case["k"], case["m"]
        used = int((_lengths(case) > 0).sum()) * k * m * size
        traffic, flops = n * (k + m) * size + used + index, 2 * n * k * m
        if case["train"]:  # reads the weights, the values and the gradient; writes a gradient of each input
            traffic += n * (2 * k + m) * size + used + b * k * m * size + index
            flops += 4 * n * k * m
    return {"bytes": traffic, "flops": flops}
