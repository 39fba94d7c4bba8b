"""The segmented matrix product on the GPU against 64-bit products: lengths,
widths, alignments, gradients, and what a caller may do with it."""
from __future__ import annotations

import functools

import numpy as np
import pytest

import matmul_reference as ref
from helpers import _cache_dir, offsets_of, prepared

pytestmark = pytest.mark.gpu

SENTINEL = -64.0


@functools.lru_cache(maxsize=256)
def matmul_program(dtype, k, m, index="i64"):
    from ragged import ArtifactCache, Compiler, MatmulSpec
    return Compiler().compile(MatmulSpec(dtype, k, m, index), ArtifactCache(_cache_dir(), max_specializations=4096))


def make_case(lengths, k, m, dtype, seed=0):
    rng = np.random.default_rng(seed)
    offsets = offsets_of(np.asarray(lengths, dtype=np.int64))
    n, b = int(offsets[-1]), len(lengths)
    return dict(values=prepared(rng.normal(size=(n, k)), dtype), offsets=offsets,
                weights=prepared(rng.normal(size=(b, k, m)) / np.sqrt(k), dtype),
                grad_out=prepared(rng.normal(size=(n, m)), dtype))


def device(torch, case, dtype, index="i64"):
    tdtype = torch.float32 if dtype == "f32" else torch.bfloat16
    kinds = dict(values=tdtype, weights=tdtype, grad_out=tdtype,
                 offsets=torch.int32 if index == "i32" else torch.int64)
    return {k: torch.from_numpy(np.ascontiguousarray(case[k])).to("cuda").to(t) for k, t in kinds.items()}


def host(tensor):
    return tensor.detach().float().cpu().numpy().astype(np.float64)


def run(torch, case, dtype, index="i64", stream=None):
    t = device(torch, case, dtype, index)
    (n, k), m = t["values"].shape, t["weights"].shape[2]
    program = matmul_program(dtype, k, m, index)
    made = {}
    for name, shape in dict(out=(n, m), grad_values=(n, k), grad_weights=tuple(t["weights"].shape)).items():
        buffer = torch.full((int(np.prod(shape)) + 128,), SENTINEL, device="cuda", dtype=t["values"].dtype)
        made[name] = (buffer[64:buffer.numel() - 64].view(shape), buffer)
    o = {name: pair[0] for name, pair in made.items()}
    if stream is not None:
        stream.wait_stream(torch.cuda.current_stream())
    program.run(t["values"], t["weights"], t["offsets"], o["out"], stream)
    program.run_backward(t["values"], t["weights"], t["offsets"], t["grad_out"], stream, grad_values=o["grad_values"],
                         grad_weights=o["grad_weights"])
    torch.cuda.synchronize()
    for name, (_, buffer) in made.items():
        assert torch.all(buffer[:64] == SENTINEL).item() and torch.all(buffer[-64:] == SENTINEL).item(), name
    return {name: host(x) for name, x in o.items()}


def check(case, got, dtype):
    wide = [case[k].astype(np.float64) for k in ("values", "weights")]
    want = ref.products(*wide, case["offsets"], case["grad_out"].astype(np.float64))
    for name, pair in want.items():
        if name in got:
            ref.close(got[name], pair, dtype)


LENGTHS = {
    "one": [1],
    "ones": [1] * 40,
    "edges": [127, 1, 128, 129, 0, 15, 16, 17, 63, 64, 65, 31, 0],
    "empties": [0, 0, 5, 0, 200, 0, 0, 0, 1, 0],
    "long": [1500],
    "many": [3, 0, 40, 7] * 30,
}


@pytest.mark.parametrize("lengths", sorted(LENGTHS))
@pytest.mark.parametrize("dtype,k,m", [("f32", 72, 136), ("bf16", 72, 136), ("bf16", 256, 64), ("bf16", 64, 320)])
def test_lengths(cuda, dtype, k, m, lengths):
    case = make_case(LENGTHS[lengths], k, m, dtype)
    check(case, run(cuda, case, dtype), dtype)


@pytest.mark.parametrize("k,m", [(1, 1), (1, 64), (7, 13), (8, 8), (16, 16), (31, 33), (64, 64), (65, 129), (100, 260),
                                 (200, 72), (333, 501), (264, 520), (1000, 24)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_widths(cuda, dtype, k, m):
    case = make_case([70, 0, 1, 150, 33], k, m, dtype, seed=k)
    check(case, run(cuda, case, dtype, "i32"), dtype)


@pytest.mark.parametrize("k,m,lengths", [
    (512, 2048, "routed 9000 8"), (2048, 512, "routed 9000 8"), (1024, 1024, "routed 20000 40"),
    (520, 1544, "routed 9100 8"), (1544, 520, "routed 9100 8"), (777, 1290, "routed 6500 4"),
    (1024, 1536, [0, 1, 129, 255, 257, 4000, 5000, 0, 300, 3000, 0]), (1536, 1024, [128, 6000, 0, 31, 256, 4097]),
    (136, 4160, [5000, 16, 15, 17, 48, 0, 2500])])
def test_wide_tiles(cuda, k, m, lengths):
    """Enough tiles for the widest ones and for pairs of SMs, several a CTA."""
    if isinstance(lengths, str):
        n, b = map(int, lengths.split()[1:])
        lengths = np.random.default_rng(n).multinomial(n, np.random.default_rng(b).dirichlet(np.full(b, 4.0)))
    lengths = np.asarray(lengths)
    n, b = int(lengths.sum()), len(lengths)
    torch = cuda
    generator = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.randn(s, generator=generator, device="cuda").bfloat16()  # noqa: E731
    values, weights, grad = rand(n, k), rand(b, k, m) / k ** 0.5, rand(n, m)
    offsets = torch.from_numpy(offsets_of(lengths)).to("cuda")
    program = matmul_program("bf16", k, m)
    out, gv, gw = (torch.full_like(x, SENTINEL) for x in (grad, values, weights))
    program.run(values, weights, offsets, out)
    program.run_backward(values, weights, offsets, grad, grad_values=gv, grad_weights=gw)
    bounds = offsets.tolist()
    for s in range(b):
        rows = slice(bounds[s], bounds[s + 1])
        x, w, g = values[rows].double(), weights[s].double(), grad[rows].double()
        for got, left, right in ((out[rows], x, w), (gv[rows], g, w.T), (gw[s], x.T, g)):
            want, size = left @ right, left.abs() @ right.abs()
            limit = 2 * (left.shape[1] + 1) * 2.0 ** -24 * size
            limit = limit + 2.0 ** -8 * (want.abs() + limit)
            assert ((got.double() - want).abs() <= limit).all().item(), s


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("k,m,lengths", [(64, 64, [20_000]), (33, 100, [9000, 0, 5, 3001]), (200, 72, [64 * 40, 64 * 41 + 1]),
                                         (1, 8, [100_000]), (256, 64, [0, 6000, 0, 7777]),
                                         (40, 30, [9000]), (136, 257, [5000])])
def test_gradients_of_small_weights_of_long_segments(cuda, dtype, k, m, lengths):
    """Few tiles: the sums over a segment's rows are taken in parts."""
    torch = cuda
    case = make_case(lengths, k, m, dtype, seed=k)
    check(case, run(torch, case, dtype), dtype)
    t = device(torch, case, dtype)
    report = matmul_program(dtype, k, m).run_backward(t["values"], t["weights"], t["offsets"], t["grad_out"],
                                                      grad_weights=torch.empty_like(t["weights"]))
    assert "matmul_parts" in report.kernel_names


@pytest.mark.parametrize("k,m", [(8, 8), (7, 64), (100, 136), (1024, 264), (2500, 40)])
@pytest.mark.parametrize("lengths", [[1], [3], [8, 1], [0, 1, 2, 0, 4, 0, 5], [1] * 30, [0] * 60 + [100, 9, 16, 17] + [0] * 40])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_few_rows_a_segment(cuda, dtype, lengths, k, m):
    """Calls of few rows a segment on average, however they fall."""
    torch = cuda
    case = make_case(lengths, k, m, dtype, seed=m)
    check(case, run(torch, case, dtype), dtype)
    t = device(torch, case, dtype)
    report = matmul_program(dtype, k, m).run(t["values"], t["weights"], t["offsets"], torch.empty_like(t["grad_out"]))
    assert report.kernel_names == ("matmul_few",) or sum(lengths) > (16 if dtype == "f32" else 2) * len(lengths)


@pytest.mark.parametrize("shifts", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (3, 5, 7)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_unaligned_views(cuda, dtype, shifts):
    torch = cuda
    case = make_case([30, 0, 140], 40, 56, dtype)
    t = device(torch, case, dtype)

    def shifted(x, by):
        return torch.empty(x.numel() + by, dtype=x.dtype, device="cuda")[by:].view_as(x).copy_(x)

    values, weights, grad = (shifted(t[k], by) for k, by in zip(("values", "weights", "grad_out"), shifts))
    o = dict(out=shifted(torch.empty_like(t["grad_out"]), shifts[0]),
             grad_values=shifted(torch.empty_like(t["values"]), shifts[1]),
             grad_weights=shifted(torch.empty_like(t["weights"]), shifts[2]))
    program = matmul_program(dtype, 40, 56)
    program.run(values, weights, t["offsets"], o["out"])
    program.run_backward(values, weights, t["offsets"], grad, grad_values=o["grad_values"], grad_weights=o["grad_weights"])
    check(case, {k: host(v) for k, v in o.items()}, dtype)


@pytest.mark.parametrize("lengths", [[], [0], [0, 0, 0]])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_no_rows(cuda, dtype, lengths):
    case = make_case(lengths, 24, 40, dtype)
    got = run(cuda, case, dtype)
    assert not got["grad_weights"].any()


@pytest.mark.parametrize("k,m", [(40, 72), (33, 9)])
@pytest.mark.parametrize("lengths,behind", [([3, 0, 9], 20), ([300, 0, 700, 0], 5), ([0, 0], 90)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_behind_the_last_segment_stay(cuda, dtype, lengths, behind, k, m):
    """Neither read nor written: NaN in the inputs there reaches nothing."""
    torch = cuda
    case = make_case(lengths, k, m, dtype, seed=behind)
    t = device(torch, case, dtype)
    used = case["offsets"][-1]
    for name in ("values", "grad_out"):
        t[name] = torch.cat([t[name], torch.full((behind, t[name].shape[1]), float("nan"), device="cuda",
                                                 dtype=t[name].dtype)])
    program = matmul_program(dtype, k, m)
    o = dict(out=torch.full_like(t["grad_out"], SENTINEL), grad_values=torch.full_like(t["values"], SENTINEL),
             grad_weights=torch.full_like(t["weights"], SENTINEL))
    program.run(t["values"], t["weights"], t["offsets"], o["out"])
    program.run_backward(t["values"], t["weights"], t["offsets"], t["grad_out"], grad_values=o["grad_values"],
                         grad_weights=o["grad_weights"])
    for name in ("out", "grad_values"):
        assert torch.all(o[name][used:] == SENTINEL).item(), name
        o[name] = o[name][:used]
    check(case, {name: host(x) for name, x in o.items()}, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_nothing_crosses_segments(cuda, dtype, bad):
    """Rows and weights of one segment that are not finite leave the others
    alone: neighbouring rows in one tile, widths that end inside one."""
    lengths = [20, 30, 0, 40, 100]
    case = make_case(lengths, 72, 88, dtype)
    clean = run(cuda, case, dtype)
    for name, index in (("values", slice(20, 50)), ("weights", 1), ("grad_out", slice(20, 50))):
        dirty_case = dict(case, **{name: case[name].copy()})
        dirty_case[name][index] = bad
        dirty = run(cuda, dirty_case, dtype)
        rows = np.r_[0:20, 50:190]
        for key in ("out", "grad_values"):
            assert np.array_equal(clean[key][rows], dirty[key][rows]), (name, key)
        others = [0, 2, 3, 4]
        assert np.array_equal(clean["grad_weights"][others], dirty["grad_weights"][others]), name
        assert not np.isfinite(dirty["out" if name != "grad_out" else "grad_values"][20:50]).all()


def test_weights_of_empty_segments_are_not_read(cuda):
    case = make_case([5, 0, 6], 64, 64, "bf16")
    case["weights"][1] = np.nan
    got = run(cuda, case, "bf16")
    assert all(np.isfinite(x).all() for x in got.values())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_equal_calls_give_equal_bits(cuda, dtype):
    case = make_case([300, 1, 77, 500], 200, 264, dtype)
    first = run(cuda, case, dtype)
    for _ in range(3):
        again = run(cuda, case, dtype)
        assert all(np.array_equal(first[k], again[k]) for k in first)


def test_other_stream(cuda):
    torch = cuda
    case = make_case([300, 1, 77], 64, 96, "bf16")
    check(case, run(torch, case, "bf16", stream=torch.cuda.Stream()), "bf16")


def test_checked_mode(cuda):
    torch = cuda
    from ragged import ValidationError
    program = matmul_program("bf16", 8, 16)
    values = torch.ones((6, 8), device="cuda", dtype=torch.bfloat16)
    out = torch.full((6, 16), SENTINEL, device="cuda", dtype=torch.bfloat16)
    for offsets in ([0, 4, 3, 6], [1, 6], [0, 5], [0, -1, 6]):
        weights = torch.ones((len(offsets) - 1, 8, 16), device="cuda", dtype=torch.bfloat16)
        with pytest.raises(ValidationError, match="offsets validation failed"):
            program.run(values, weights, torch.tensor(offsets, device="cuda"), out, mode="checked")
    assert torch.all(out == SENTINEL).item()
    weights = torch.ones((1, 8, 16), device="cuda", dtype=torch.bfloat16)
    report = program.run(values, weights, torch.tensor([0, 6], device="cuda"), out, mode="checked")
    assert report.kernel_names == ("offsets_init", "offsets_check", "matmul_tensor") and torch.all(out == 8).item()


def test_captured_calls_replay_on_new_inputs(cuda):
    torch = cuda
    program = matmul_program("bf16", 65, 96)
    cases = [make_case([200, 0, 130, 1], 65, 96, "bf16", seed=s) for s in (1, 2, 3)]
    t = device(torch, cases[0], "bf16")
    o = dict(out=torch.empty_like(t["grad_out"]), grad_values=torch.empty_like(t["values"]),
             grad_weights=torch.empty_like(t["weights"]))

    def step():
        program.run(t["values"], t["weights"], t["offsets"], o["out"])
        program.run_backward(t["values"], t["weights"], t["offsets"], t["grad_out"], grad_values=o["grad_values"],
                             grad_weights=o["grad_weights"])

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for case in cases:
        for name, x in device(torch, case, "bf16").items():
            t[name].copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        check(case, {k: host(v) for k, v in o.items()}, "bf16")
    del graph


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_autograd(cuda, dtype):
    """All gradients, one at a time, of expanded and transposed tensors."""
    torch = cuda
    from ragged import ValidationError, torch_adapter
    case = make_case(LENGTHS["edges"], 40, 24, dtype)
    program = matmul_program(dtype, 40, 24)
    t = device(torch, case, dtype)
    values, weights = t["values"].requires_grad_(), t["weights"].requires_grad_()
    out = torch_adapter.segment_matmul(values, weights, t["offsets"], program=program)
    gv, gw = torch.autograd.grad(out, (values, weights), t["grad_out"], retain_graph=True)
    check(case, dict(out=host(out), grad_values=host(gv), grad_weights=host(gw)), dtype)
    (only,) = torch.autograd.grad(out, weights, t["grad_out"], retain_graph=True)
    assert torch.equal(only, gw)
    case["grad_out"] = np.ones_like(case["grad_out"])
    gv, gw = torch.autograd.grad(out.float().sum(), (values, weights), retain_graph=True)
    check(case, dict(grad_values=host(gv), grad_weights=host(gw)), dtype)
    turned = t["weights"].detach().transpose(1, 2).contiguous().transpose(1, 2).requires_grad_()
    out2 = torch_adapter.segment_matmul(values, turned, t["offsets"], program=program)
    assert torch.equal(out, out2) and torch.equal(torch.autograd.grad(out2.float().sum(), turned)[0], gw)
    with pytest.raises((ValidationError, RuntimeError), match="second derivatives"):
        torch.autograd.grad(out.float().sum(), values, create_graph=True)


def test_gradients_are_the_differences_of_the_outputs(cuda):
    """<grad_out, out> is linear in values and in weights: its differences over
    steps of any size are the gradients, but for the rounding of the outputs."""
    torch = cuda
    rng = np.random.default_rng(3)
    case = make_case([30, 0, 77, 1], 33, 20, "f32")
    got = run(torch, case, "f32")
    weight = case["grad_out"].astype(np.float64)

    def loss(case):
        r = ref.products(*(case[k].astype(np.float64) for k in ("values", "weights")), case["offsets"])["out"]
        noise = (np.abs(weight) * (r[1] + 2.0 ** -24 * np.abs(r[0]))).sum()
        return (weight * run(torch, case, "f32")["out"]).sum(), noise

    base, noise = loss(case)
    for name, grad in (("values", "grad_values"), ("weights", "grad_weights")):
        moved = dict(case, **{name: case[name] + rng.normal(size=case[name].shape).astype(np.float32)})
        step = moved[name].astype(np.float64) - case[name]
        there, more = loss(moved)
        exact = ref.products(*(case[k].astype(np.float64) for k in ("values", "weights")), case["offsets"], weight)[grad]
        slack = (np.abs(step) * (exact[1] + 2.0 ** -24 * np.abs(exact[0]))).sum()
        assert abs(there - base - (got[grad] * step).sum()) <= noise + more + slack, name


@pytest.mark.parametrize("compiled", [False, True])
def test_operator_in_a_graph(cuda, compiled):
    """The operator below the eager call, alone and in a compiled full graph."""
    torch = cuda
    from ragged import torch_adapter
    case = make_case([5, 0, 130, 2], 32, 48, "bf16")
    t = device(torch, case, "bf16")
    token = torch_adapter.register_program(matmul_program("bf16", 32, 48))
    torch_adapter.register_torch_ops()

    def model(values, weights, offsets):
        return torch.ops.ragged_mlir.segment_matmul(values, weights, offsets, token)

    if compiled:
        model = torch.compile(model, backend="aot_eager", fullgraph=True)
    leaves = [t[k].requires_grad_() for k in ("values", "weights")]
    out = model(*leaves, t["offsets"])
    gv, gw = torch.autograd.grad(out, leaves, t["grad_out"])
    check(case, dict(out=host(out), grad_values=host(gv), grad_weights=host(gw)), "bf16")


def test_jagged_tensors(cuda):
    torch = cuda
    from ragged import torch_adapter
    case = make_case([5, 0, 130, 2], 32, 48, "bf16")
    t = device(torch, case, "bf16")
    nt = torch.nested.nested_tensor_from_jagged(t["values"], t["offsets"])
    out = torch_adapter.njt_matmul(nt, t["weights"], program=matmul_program("bf16", 32, 48))
    assert out.offsets().data_ptr() == t["offsets"].data_ptr()
    check(case, dict(out=host(out.values())), "bf16")


def test_operands_beyond_32_bits_of_elements(cuda):
    """values and weights of more than 2^32 elements: the last rows and the
    last segment are reached by 64-bit addresses."""
    torch = cuda
    k, m, b = 4096, 1024, 1030
    n = 1_049_600
    program = matmul_program("bf16", k, m)
    weights = torch.zeros((b, k, m), dtype=torch.bfloat16, device="cuda")
    weights[-1, :, 5] = 0.5
    values = torch.zeros((n, k), dtype=torch.bfloat16, device="cuda")
    values[-3:] = 1
    lengths = np.full(b, 1)
    lengths[0] = n - b + 1 - 2
    lengths[-1] = 3
    out = torch.empty((n, m), dtype=torch.bfloat16, device="cuda")
    program.run(values, weights, torch.from_numpy(offsets_of(lengths)).to("cuda"), out)
    assert torch.all(out[-3:, 5] == k / 2).item() and out.count_nonzero().item() == 3


def test_a_captured_training_step(cuda):
    """Projection, recurrence and their gradients by autograd, inside one graph,
    replayed on new inputs; no eager graph of the leaves is alive."""
    torch = cuda
    from ragged import ArtifactCache, Compiler, ScanSpec, torch_adapter
    offsets = torch.from_numpy(offsets_of([300, 0, 41, 700])).to("cuda")
    n, k, d = 1041, 40, 64
    scan = Compiler().compile(ScanSpec("bf16", d), ArtifactCache(_cache_dir(), max_specializations=4096))
    project = matmul_program("bf16", k, d)
    generator = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(s, generator=generator, device="cuda").bfloat16()  # noqa: E731
    x, w, gates, grad = rand(n, k), rand(4, k, d), torch.sigmoid(rand(n, d)), rand(n, d)
    leaves = [t.requires_grad_() for t in (x, w, gates)]

    def step():
        h, _ = torch_adapter.segment_scan(torch_adapter.segment_matmul(x, w, offsets, program=project), gates, offsets,
                                          program=scan)
        return torch.autograd.grad(h, leaves, grad)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(2):
        with torch.no_grad():
            x.copy_(rand(n, k))
            w.copy_(rand(4, k, d))
            grad.copy_(rand(n, d))
        graph.replay()
        torch.cuda.synchronize()
        kept = [g.clone() for g in captured]
        for a, b in zip(kept, step()):
            assert torch.equal(a, b)
    del graph


def test_a_run_of_the_operators_together(cuda):
    """Packed sequences through a gated recurrence: projections per group of
    sequences make the inputs and the gates, the states are projected back and
    pooled over each sequence; forward and all gradients against autograd in
    64 bits."""
    torch = cuda
    from ragged import ArtifactCache, Compiler, ProgramSpec, ScanSpec, torch_adapter
    rng = np.random.default_rng(7)
    lengths = rng.integers(0, 90, size=24)
    sequences = offsets_of(lengths)
    groups = sequences[[0, 5, 5, 14, 24]]  # whole sequences of one task each, one task without any
    n, k, d = int(sequences[-1]), 48, 80
    to = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to("cuda")  # noqa: E731
    by_sequence, by_group = to(sequences), to(groups)
    tokens = to(rng.normal(size=(n, k))).float()
    w_in, w_gate, w_out = (to(rng.normal(size=s) / np.sqrt(s[1])).float() for s in ((4, k, d), (4, k, d), (4, d, k)))
    leaves = [x.requires_grad_() for x in (tokens, w_in, w_gate, w_out)]
    cache = ArtifactCache(_cache_dir(), max_specializations=4096)
    scan = Compiler().compile(ScanSpec("f32", d), cache)
    into, back = matmul_program("f32", k, d), matmul_program("f32", d, k)
    x = torch_adapter.segment_matmul(tokens, w_in, by_group, program=into)
    gate = torch.sigmoid(torch_adapter.segment_matmul(tokens, w_gate, by_group, program=into))
    h, _ = torch_adapter.segment_scan(x * (1 - gate), gate, by_sequence, program=scan)
    y = torch_adapter.segment_matmul(h, w_out, by_group, program=back)
    pooled = torch_adapter.segment_reduce(y.detach(), by_sequence, "sum",
                                          program=Compiler().compile(ProgramSpec("sum", "f32", k), cache))
    grad = to(rng.normal(size=(n, k))).float()
    grads = torch.autograd.grad(y, leaves, grad)

    wide = [v.detach().double().requires_grad_() for v in leaves]
    rows = [slice(groups[i], groups[i + 1]) for i in range(4)]
    project = lambda v, w: torch.cat([v[r] @ w[i] for i, r in enumerate(rows)])  # noqa: E731
    x64, g64 = project(wide[0], wide[1]), torch.sigmoid(project(wide[0], wide[2]))
    states = []
    for s in range(24):
        state = None
        for t in range(sequences[s], sequences[s + 1]):
            new = x64[t] * (1 - g64[t])
            state = new if state is None else g64[t] * state + new
            states.append(state)
    y64 = project(torch.stack(states), wide[3])
    # Each of the four steps is off by no more than its own bound of a few
    # hundred roundings of 2^-24 of its majorant: 1e-3 of the largest value is
    # over ten times the chain of them (90 rows, widths of 80, factors below 4).
    def near(a, e):
        assert (a.double() - e).abs().max().item() <= 1e-3 * e.abs().max().item()
    near(y, y64)
    for a, e in zip(grads, torch.autograd.grad(y64, wide, grad.double())):
        near(a, e)
    sums = torch.zeros((24, k), dtype=torch.float64, device="cuda")
    sums.index_add_(0, torch.repeat_interleave(torch.arange(24, device="cuda"), by_sequence.diff()), y.detach().double())
    near(pooled, sums)


@pytest.mark.parametrize("captured", [False, True])
def test_chained_calls_of_unaligned_rows(cuda, captured):
    """Each call packs what the one before it wrote, back to back and in a
    replayed graph: the same bits as with a synchronisation after each."""
    torch = cuda
    torch.manual_seed(5)
    offsets = torch.tensor([0, 700, 701, 701, 1500, 2111], device="cuda")
    x = torch.randn(2111, 77, device="cuda").bfloat16()
    widths = [77, 131, 64, 201, 77]
    weights = [(torch.randn(5, k, m, device="cuda") / k ** 0.5).bfloat16() for k, m in zip(widths, widths[1:])]
    rows = [torch.empty(2111, m, device="cuda", dtype=torch.bfloat16) for m in widths[1:]]
    grads = [torch.empty_like(w) for w in weights]
    programs = [matmul_program("bf16", k, m) for k, m in zip(widths, widths[1:])]

    def chain(wait):
        source = x
        for program, w, out, grad in zip(programs, weights, rows, grads):
            program.run(source, w, offsets, out)
            if wait:
                torch.cuda.synchronize()
            program.run_backward(source, w, offsets, out, grad_weights=grad)
            if wait:
                torch.cuda.synchronize()
            source = out

    results = lambda: [t.clone() for t in rows + grads]  # noqa: E731
    graph = None
    if captured:
        graph = torch.cuda.CUDAGraph()
        chain(True)
        with torch.cuda.graph(graph):
            chain(False)
    for turn in range(4):
        x.copy_(torch.randn(2111, 77, device="cuda").bfloat16())
        chain(True)
        want = results()
        for t in rows + grads:
            t.fill_(SENTINEL)
        if graph is not None:
            graph.replay()
        else:
            chain(False)
        torch.cuda.synchronize()
        for got, expected in zip(results(), want):
            assert torch.equal(got, expected), turn


def test_calls_on_two_streams_at_once(cuda):
    """One program from two streams: scratch is a call's own."""
    torch = cuda
    torch.manual_seed(6)
    offsets = torch.tensor([0, 900, 1700, 3001], device="cuda")
    program = matmul_program("bf16", 75, 131)
    cases = [(torch.randn(3001, 75, device="cuda").bfloat16(), torch.randn(3, 75, 131, device="cuda").bfloat16())
             for _ in range(2)]
    want = []
    for x, w in cases:
        out = torch.empty(3001, 131, device="cuda", dtype=torch.bfloat16)
        program.run(x, w, offsets, out)
        torch.cuda.synchronize()
        want.append(out)
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [[torch.empty_like(want[0]) for _ in range(10)] for _ in cases]
    torch.cuda.synchronize()
    for i in range(10):
        for s, stream in enumerate(streams):
            program.run(*cases[s], offsets, outs[s][i], stream)
    torch.cuda.synchronize()
    for s in range(2):
        assert all(torch.equal(out, want[s]) for out in outs[s])


def dirty_allocator(torch, *byte_counts):
    """Leaves NaN (and, as 64-bit words, nonzero values) in the memory that the
    next allocations of these sizes get."""
    for count in byte_counts:
        blocks = [torch.full((-(-count // 4),), float("nan"), device="cuda") for _ in range(3)]
        torch.cuda.synchronize()
        del blocks


@pytest.mark.parametrize("mode", ["validated", "checked"])
@pytest.mark.parametrize("shift", range(1, 8))
@pytest.mark.parametrize("k,m", [(7, 64), (33, 8), (100, 64), (64, 40), (1100, 136)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_few_rows_with_weights_inside_a_buffer(cuda, dtype, k, m, shift, mode):
    """Calls of few rows a segment whose weights start anywhere in a flat buffer
    of parameters; the columns fill 16-byte vectors, the rows of values do not."""
    torch = cuda
    program = matmul_program(dtype, k, m)
    for lengths in ([1, 1, 1, 1], [2, 0, 3, 1], [0, 7, 0, 0, 0, 1]):
        case = make_case(lengths, k, m, dtype, seed=shift)
        t = device(torch, case, dtype)
        weights = torch.zeros(t["weights"].numel() + shift, dtype=t["weights"].dtype, device="cuda")[shift:]
        weights = weights.view_as(t["weights"]).copy_(t["weights"])
        out = torch.full_like(t["grad_out"], SENTINEL)
        dirty_allocator(torch, 8192 + 2 * (k + 8) * (len(out) + len(lengths) * (m + 8)))
        program.run(t["values"], weights, t["offsets"], out, mode=mode)
        check(case, dict(out=host(out)), dtype)


@pytest.mark.parametrize("route", ["call", "operator"])
@pytest.mark.parametrize("dtype,k,m,lengths,behind", [
    ("f32", 40, 72, [3, 0, 9], 20), ("bf16", 40, 72, [3, 0, 9], 20),              # few rows and tiles
    ("f32", 33, 9, [300, 0, 700, 0], 5), ("bf16", 33, 9, [300, 0, 700, 0], 5),    # rows off 16-byte boundaries
    ("f32", 16, 8, [1, 0, 1, 2], 60), ("bf16", 16, 8, [1, 0, 0, 0, 0, 0, 0, 0], 13),  # few rows a segment, padded
    ("f32", 24, 200, [0, 0], 700), ("bf16", 24, 200, [0, 0], 700),                # no rows at all
    ("bf16", 512, 2048, [4000, 100, 6000], 9000), ("f32", 512, 512, [4000, 100, 3000], 999)])  # wide tiles, pairs
def test_padded_rows_of_results_are_zero(cuda, dtype, k, m, lengths, behind, route):
    """Rows behind the last offset, NaN in the inputs: zeros in what the call
    allocates, in fresh memory that holds NaN, and no gradient of the weights."""
    torch = cuda
    from ragged import torch_adapter
    generator = torch.Generator(device="cuda").manual_seed(behind)
    offsets = torch.from_numpy(offsets_of(np.asarray(lengths))).to("cuda")
    used, n, b = sum(lengths), sum(lengths) + behind, len(lengths)
    kind = torch.float32 if dtype == "f32" else torch.bfloat16
    rand = lambda *s: torch.randn(s, generator=generator, device="cuda").to(kind)  # noqa: E731
    values, grad, weights = rand(n, k), rand(n, m), rand(b, k, m)
    values[used:], grad[used:] = float("nan"), float("nan")
    program = matmul_program(dtype, k, m)
    want = dict(out=torch.zeros_like(grad), grad_values=torch.zeros_like(values), grad_weights=torch.empty_like(weights))
    program.run(values, weights, offsets, want["out"])
    program.run_backward(values, weights, offsets, grad, grad_values=want["grad_values"],
                         grad_weights=want["grad_weights"])
    leaves = [values.requires_grad_(), weights.requires_grad_()]
    size = kind.itemsize
    dirty_allocator(torch, n * m * size, n * k * size)
    if route == "call":
        out = torch_adapter.segment_matmul(*leaves, offsets, program=program)
    else:
        torch_adapter.register_torch_ops()
        out = torch.ops.ragged_mlir.segment_matmul(*leaves, offsets, torch_adapter.register_program(program))
    dirty_allocator(torch, n * k * size)
    gv, gw = torch.autograd.grad(out, leaves, grad)
    assert torch.equal(out, want["out"]) and torch.equal(gv, want["grad_values"]) and torch.equal(gw, want["grad_weights"])


@pytest.mark.parametrize("call", ["forward", "backward", "autograd"])
def test_the_first_call_of_a_thread(cuda, call):
    """A new thread whose first use of the GPU is a product that another thread
    has made before: a serving thread, or autograd's own."""
    import threading
    torch = cuda
    from ragged import torch_adapter
    case = make_case([300, 0, 41], 72, 136, "bf16")
    t = device(torch, case, "bf16")
    program = matmul_program("bf16", 72, 136)
    leaves = [t["values"].requires_grad_(), t["weights"].requires_grad_()]
    grads = [torch.empty_like(x) for x in leaves]
    out = torch.empty_like(t["grad_out"])

    def forward():
        with torch.no_grad():
            program.run(*leaves, t["offsets"], out)

    def backward():
        program.run_backward(*leaves, t["offsets"], t["grad_out"], grad_values=grads[0], grad_weights=grads[1])

    forward()
    backward()
    want = [x.clone() for x in (out, *grads)]
    graph = torch_adapter.segment_matmul(*leaves, t["offsets"], program=program)
    for x in (out, *grads):
        x.fill_(SENTINEL)
    torch.cuda.synchronize()
    raised = []

    def work():
        try:
            if call == "autograd":
                grads[:] = torch.autograd.grad(graph, leaves, t["grad_out"])
            else:
                (forward if call == "forward" else backward)()
        except BaseException as error:  # noqa: BLE001 - shown by the assertion below
            raised.append(error)

    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert not raised, raised
    if call == "forward":
        assert torch.equal(out, want[0])
    else:
        assert torch.equal(grads[0], want[1]) and torch.equal(grads[1], want[2])


@pytest.mark.parametrize("k,m,lengths", [(64, 64, [20_000]), (33, 100, [9000, 0, 5, 3001]), (136, 257, [5000]),
                                         (72, 136, [3, 0, 200]), (1024, 1544, [9000, 0, 700])])
def test_checked_backward(cuda, k, m, lengths):
    """The offsets are validated first; parts of sums and packed operands in the
    scratch are not taken for words of waits that gave up."""
    torch = cuda
    from ragged import ValidationError
    case = make_case(lengths, k, m, "bf16", seed=k)
    t = device(torch, case, "bf16")
    program = matmul_program("bf16", k, m)
    plain, checked = ([torch.full_like(t[name], SENTINEL) for name in ("values", "weights")] for _ in range(2))
    for mode, (gv, gw) in (("validated", plain), ("checked", checked)):
        dirty_allocator(torch, 1 << 20, 1 << 22)
        report = program.run_backward(t["values"], t["weights"], t["offsets"], t["grad_out"], mode=mode,
                                      grad_values=gv, grad_weights=gw)
    assert report.mode == "checked" and report.kernel_names[:2] == ("offsets_init", "offsets_check")
    assert all(torch.equal(a, b) for a, b in zip(plain, checked))
    wrong = t["offsets"].clone()
    wrong[-1] -= 1
    with pytest.raises(ValidationError, match="offsets validation failed"):
        program.run_backward(t["values"], t["weights"], wrong, t["grad_out"], mode="checked", grad_values=plain[0])
    with pytest.raises(ValidationError, match="mode"):
        program.run_backward(t["values"], t["weights"], t["offsets"], t["grad_out"], mode="unsafe", grad_values=plain[0])


@pytest.mark.parametrize("route", ["run", "call", "operator"])
@pytest.mark.parametrize("kind,k,m,lengths,kernel", [
    ("grad_values", 72, 136, [300, 0, 41], "matmul_tensor"), ("grad_values", 1024, 1544, [9000, 0, 700], "matmul_pair"),
    ("grad_weights", 72, 136, [300, 0, 41], "matmul_tensor"), ("grad_weights", 64, 64, [20_000], "matmul_tensor")])
def test_a_wait_that_gave_up_in_a_gradient_is_reported(cuda, monkeypatch, kind, k, m, lengths, kernel, route):
    """A launch that reports a wait that gave up (its words are written here, by
    the host, after the launch: the last CTA's) raises in checked mode alone."""
    torch = cuda
    from ragged import _native, torch_adapter
    case = make_case(lengths, k, m, "bf16")
    t = device(torch, case, "bf16")
    program = matmul_program("bf16", k, m)
    scratch, empty, launch = [], torch.empty, _native.matmul

    def remember(*args, **options):
        made = empty(*args, **options)
        if options.get("dtype") == torch.uint8:
            scratch.append(made)
        return made

    def give_up(which, *args, **options):
        report = _native.Report()
        launch(which, *args[:-2], report, args[-1])
        if args[-2] is not None:
            import ctypes
            ctypes.memmove(ctypes.byref(args[-2]), ctypes.byref(report), ctypes.sizeof(report))
        if which == kind:
            names = [_native.kernel_name(report.kernel_ids[i]) for i in range(report.num_launches)]
            scratch[-1].view(torch.int64)[report.grid[names.index(kernel)][0] - 1] = 1

    monkeypatch.setattr(torch, "empty", remember)
    monkeypatch.setattr(_native, "matmul", give_up)
    leaves = [t["values"].requires_grad_(), t["weights"].requires_grad_()]
    names = ("grad_values", "grad_weights")

    def gradients(mode):
        if route == "run":
            grads = {name: torch.empty_like(x) for name, x in zip(names, leaves) if name == kind}
            program.run_backward(t["values"], t["weights"], t["offsets"], t["grad_out"], mode=mode, **grads)
            return
        if route == "call":
            out = torch_adapter.segment_matmul(*leaves, t["offsets"], program=program, mode=mode)
        else:
            torch_adapter.register_torch_ops()
            out = torch.ops.ragged_mlir.segment_matmul(*leaves, t["offsets"], torch_adapter.register_program(program), mode)
        torch.autograd.grad(out, leaves[names.index(kind)], t["grad_out"])

    gradients("validated")
    with pytest.raises(RuntimeError, match="bounded wait"):
        gradients("checked")


@pytest.mark.parametrize("compiled", [False, True])
def test_bound_programs_give_what_the_calls_give(cuda, compiled):
    torch = cuda
    from ragged import ArtifactCache, Compiler, ScanSpec, torch_adapter
    case = make_case([5, 0, 130, 2], 32, 48, "bf16")
    t = device(torch, case, "bf16")
    scan = Compiler().compile(ScanSpec("bf16", 48), ArtifactCache(_cache_dir(), max_specializations=4096))
    product = matmul_program("bf16", 32, 48)
    project, recur = torch_adapter.bind(product), torch_adapter.bind(scan)
    leaves = [t["values"].requires_grad_(), t["weights"].requires_grad_(),
              torch.rand_like(t["grad_out"]).requires_grad_(), torch.randn(4, 48, device="cuda", requires_grad=True)]

    def model(values, weights, gates, initial, offsets):
        out, final = recur(project(values, weights, offsets), gates, offsets, initial)
        return recur(out, gates, offsets)[0], final

    if compiled:
        model = torch.compile(model, backend="aot_eager", fullgraph=True)
    got = model(*leaves, t["offsets"])
    x = torch_adapter.segment_matmul(*leaves[:2], t["offsets"], program=product)
    out, final = torch_adapter.segment_scan(x, leaves[2], t["offsets"], program=scan, initial=leaves[3])
    want = torch_adapter.segment_scan(out, leaves[2], t["offsets"], program=scan)[0], final
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    grads = [torch.autograd.grad((y.float().sum(), f.sum()), leaves) for y, f in (got, want)]
    assert all(torch.equal(a, b) for a, b in zip(*grads))
