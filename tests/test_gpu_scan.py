"""The segmented scan on the GPU against the 64-bit recurrence: every vector
width, column tile and chunk edge, states in and out, gradients, and what a
caller may do with it (streams, captured calls, other layouts of gradients)."""
from __future__ import annotations

import functools

import numpy as np
import pytest

import scan_reference as ref
from helpers import _cache_dir, offsets_of, prepared

pytestmark = pytest.mark.gpu

SENTINEL = -64.0


@functools.lru_cache(maxsize=256)
def scan_program(dtype, d, index="i64"):
    from ragged import ArtifactCache, Compiler, ScanSpec
    return Compiler().compile(ScanSpec(dtype, d, index),
                              ArtifactCache(_cache_dir(), max_specializations=4096))


def make_case(lengths, d, dtype, initial, seed=0, gate="keep"):
    rng = np.random.default_rng(seed)
    offsets = offsets_of(np.asarray(lengths, dtype=np.int64))
    n, b = int(offsets[-1]), len(lengths)
    values = prepared(rng.normal(size=(n, d)), dtype)
    if gate == "keep":
        gates = 1 / (1 + np.exp(-(rng.normal(size=(n, d)) * 2 + 2)))
    else:
        gates = rng.uniform(-1, 1, size=(n, d)) * (rng.random((n, d)) > 0.1)
    gates = prepared(gates, dtype)
    f32 = lambda *s: rng.normal(size=s).astype(np.float32)  # noqa: E731
    return dict(values=values, gates=gates, offsets=offsets, initial=f32(b, d) if initial else None,
                grad_out=prepared(rng.normal(size=(n, d)), dtype), grad_final=f32(b, d))


def guarded(torch, shape, dtype):
    """A tensor of ``shape`` in the middle of a buffer of sentinels."""
    count = int(np.prod(shape))
    buffer = torch.full((count + 128,), SENTINEL, device="cuda", dtype=dtype)
    return buffer[64:64 + count].view(shape), buffer


def untouched(buffer, count):
    flat = buffer.float().cpu().numpy()
    return np.all(flat[:64] == SENTINEL) and np.all(flat[64 + count:] == SENTINEL)


def device(torch, case, dtype, index):
    tdtype = torch.float32 if dtype == "f32" else torch.bfloat16
    to = lambda x, t: None if x is None else torch.from_numpy(np.ascontiguousarray(x)).to("cuda").to(t)  # noqa: E731
    kinds = dict(values=tdtype, gates=tdtype, grad_out=tdtype, initial=torch.float32, grad_final=torch.float32,
                 offsets=torch.int32 if index == "i32" else torch.int64)
    return {name: to(case[name], kind) for name, kind in kinds.items()}


def host(tensor):
    return None if tensor is None else tensor.float().cpu().numpy().astype(np.float64)


def run(torch, case, dtype, index="i64", backward=True, stream=None):
    """Forward and backward through the public calls; guarded outputs."""
    t = device(torch, case, dtype, index)
    n, d = t["values"].shape
    b = t["offsets"].numel() - 1
    program = scan_program(dtype, d, index)
    kind = t["values"].dtype
    shapes = dict(out=((n, d), kind), final=((b, d), torch.float32), carries=((program.carry_rows(n), d), torch.float32),
                  grad_values=((n, d), kind), grad_gates=((n, d), kind), grad_initial=((b, d), torch.float32))
    made = {name: guarded(torch, *spec) for name, spec in shapes.items()}
    o = {name: pair[0] for name, pair in made.items()}
    program.run(t["values"], t["gates"], t["offsets"], o["out"], stream, initial=t["initial"], final=o["final"],
                carries=o["carries"])
    if backward:
        gi = o["grad_initial"] if t["initial"] is not None else None
        program.run_backward(t["values"], t["gates"], t["offsets"], o["carries"], t["grad_out"], stream,
                             initial=t["initial"], grad_final=t["grad_final"], grad_values=o["grad_values"],
                             grad_gates=o["grad_gates"], grad_initial=gi)
    torch.cuda.synchronize()
    for name, (view, buffer) in made.items():
        assert untouched(buffer, view.numel()), f"write outside {name}"
    return {name: host(x) for name, x in o.items()}


def check(case, got, dtype, backward=True):
    wide = {k: None if v is None else v.astype(np.float64) for k, v in case.items() if k != "offsets"}
    r = ref.backward(wide["values"], wide["gates"], case["offsets"], wide["grad_out"], wide["grad_final"],
                     wide["initial"])
    ref.check_forward(r, got["out"], got["final"], dtype)
    if backward:
        ref.check_backward(r, got["grad_values"], got["grad_gates"],
                           got["grad_initial"] if case["initial"] is not None else None, dtype)


LENGTHS = {
    "one": [1],
    "ones": [1] * 300,
    "edges": [127, 1, 128, 129, 0, 255, 256, 257, 3, 0, 0, 31],
    "empties": [0, 0, 5, 0, 200, 0, 0, 0, 1, 0],
    "long": [5000],
    "mixed": [700, 1, 2100, 0, 13, 260, 2],
}


@pytest.mark.parametrize("initial", [False, True])
@pytest.mark.parametrize("lengths", sorted(LENGTHS))
@pytest.mark.parametrize("dtype,d", [("f32", 128), ("bf16", 64)])
def test_lengths(cuda, dtype, d, lengths, initial):
    case = make_case(LENGTHS[lengths], d, dtype, initial)
    check(case, run(cuda, case, dtype), dtype)


@pytest.mark.parametrize("d", [1, 2, 3, 4, 6, 7, 8, 13, 31, 36, 72, 100, 130, 200, 264])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_widths(cuda, dtype, d):
    case = make_case([300, 0, 1, 1500, 17, 64], d, dtype, True, seed=d, gate="signed")
    check(case, run(cuda, case, dtype, "i32"), dtype)


@pytest.mark.parametrize("d", [16, 96])
@pytest.mark.parametrize("shifts", [(1, 1, 1), (1, 0, 0), (0, 0, 1), (2, 4, 0)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_unaligned_views(cuda, dtype, shifts, d):
    """Views that start anywhere in their storage, states among them; the
    recorded states serve a backward pass of other alignment."""
    torch = cuda
    case = make_case([200, 3, 0, 390], d, dtype, True)
    t = device(torch, case, dtype, "i64")

    def shifted(x, by):
        view = torch.empty(x.numel() + by, dtype=x.dtype, device="cuda")[by:].view_as(x)
        return view.copy_(x)

    values, gates, initial = (shifted(t[k], by) for k, by in zip(("values", "gates", "initial"), shifts))
    program = scan_program(dtype, d)
    empty = lambda x: torch.empty_like(x)  # noqa: E731
    o = dict(out=shifted(empty(t["values"]), shifts[2]), final=empty(initial), grad_values=empty(t["values"]),
             grad_gates=empty(t["values"]), grad_initial=empty(initial))
    carries = torch.empty((program.carry_rows(593), d), device="cuda")
    program.run(values, gates, t["offsets"], o["out"], initial=initial, final=o["final"], carries=carries)
    program.run_backward(t["values"], t["gates"], t["offsets"], carries, t["grad_out"], initial=t["initial"],
                         grad_final=t["grad_final"], grad_values=o["grad_values"], grad_gates=o["grad_gates"],
                         grad_initial=o["grad_initial"])
    check(case, {k: host(v) for k, v in o.items()}, dtype)


@pytest.mark.parametrize("dtype,d,rows", [("f32", 32, 80_000), ("bf16", 66, 40_000)])
def test_one_long_segment_passes_every_level_of_the_fold(cuda, dtype, d, rows):
    """More than 256 chunks of 128 rows, in one segment and with a start in the
    middle; gates near one carry states over many chunks."""
    for lengths in ([rows], [rows // 3, rows - rows // 3]):
        case = make_case(lengths, d, dtype, True, seed=5)
        case["gates"] = prepared(1 - (1 - case["gates"]) * 1e-3, dtype)
        check(case, run(cuda, case, dtype), dtype)


def test_equal_calls_give_equal_bits(cuda):
    case = make_case([9000, 1, 7000, 333], 128, "bf16", True)
    first = run(cuda, case, "bf16")
    for _ in range(5):
        again = run(cuda, case, "bf16")
        for name in ("out", "final", "grad_values", "grad_gates", "grad_initial"):
            assert np.array_equal(first[name], again[name]), name


@pytest.mark.parametrize("lengths", [[], [0], [0] * 9000])
def test_no_rows(cuda, lengths):
    case = make_case(lengths, 24, "f32", True)
    got = run(cuda, case, "f32")
    if lengths:
        assert np.array_equal(got["final"], case["initial"]) and np.array_equal(got["grad_initial"], case["grad_final"])


def test_few_rows_among_many_empty_segments(cuda):
    lengths = np.zeros(50_000, dtype=np.int64)
    lengths[[0, 17, 4096, 30_000, 49_999]] = [3, 200, 1, 129, 2]
    case = make_case(lengths, 16, "f32", True)
    check(case, run(cuda, case, "f32", "i32"), "f32")


@pytest.mark.parametrize("initial", [False, True])
@pytest.mark.parametrize("lengths,behind", [([3, 0, 9], 20), ([300, 0, 700, 0], 5), ([65, 2000, 1], 1500), ([0, 0], 900)])
@pytest.mark.parametrize("dtype,d", [("f32", 12), ("bf16", 128)])
def test_rows_behind_the_last_segment_stay(cuda, dtype, d, lengths, behind, initial):
    """Neither read nor written: NaN in the inputs there reaches nothing."""
    torch = cuda
    case = make_case(lengths, d, dtype, initial, seed=behind)
    t = device(torch, case, dtype, "i64")
    used, b = case["offsets"][-1], len(lengths)
    for name in ("values", "gates", "grad_out"):
        t[name] = torch.cat([t[name], torch.full((behind, d), float("nan"), device="cuda", dtype=t[name].dtype)])
    program = scan_program(dtype, d)
    o = {name: torch.full_like(t["values"], SENTINEL) for name in ("out", "grad_values", "grad_gates")}
    o["final"], o["grad_initial"] = (torch.full((b, d), SENTINEL, device="cuda") for _ in range(2))
    carries = torch.empty((program.carry_rows(used + behind), d), device="cuda")
    program.run(t["values"], t["gates"], t["offsets"], o["out"], initial=t["initial"], final=o["final"], carries=carries)
    program.run_backward(t["values"], t["gates"], t["offsets"], carries, t["grad_out"], initial=t["initial"],
                         grad_final=t["grad_final"], grad_values=o["grad_values"], grad_gates=o["grad_gates"],
                         grad_initial=o["grad_initial"] if initial else None)
    for name in ("out", "grad_values", "grad_gates"):
        assert torch.all(o[name][used:] == SENTINEL).item(), name
        o[name] = o[name][:used]
    check(case, {name: host(x) for name, x in o.items()}, dtype)


def test_many_empty_segments_in_the_middle_of_a_slab(cuda):
    lengths = [3] + [0] * 9000 + [5] + [0] * 40 + [600, 0, 1] + [0] * 70 + [2]
    for d in (8, 100):
        case = make_case(lengths, d, "f32", True)
        check(case, run(cuda, case, "f32"), "f32")


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("where", ["values", "initial", "grad_out", "grad_final"])
def test_nothing_crosses_segments(cuda, where, bad):
    """A non-finite input changes its own segment (and column) alone."""
    if where == "initial" or where == "grad_final":
        index = (2, 5)
    else:
        index = (400, 5)
    case = make_case([100, 200, 300, 400, 0, 50], 32, "f32", True)
    clean = run(cuda, case, "f32")
    case[where] = case[where].copy()
    case[where][index] = bad
    dirty = run(cuda, case, "f32")
    rows = np.r_[0:300, 600:1050]
    for name in ("out", "grad_values", "grad_gates"):
        assert np.array_equal(clean[name][rows], dirty[name][rows]), name
        others = np.delete(np.arange(32), 5)
        assert np.array_equal(clean[name][:, others], dirty[name][:, others]), name
    changed = "out" if where in ("values", "initial") else "grad_values"
    assert not np.isfinite(dirty[changed][300:600, 5]).all()


def test_first_gates_do_not_count_without_a_state(cuda):
    case = make_case([40, 1, 600], 32, "f32", False)
    case["gates"][[0, 40, 41]] = np.nan
    got = run(cuda, case, "f32")
    assert np.isfinite(got["out"]).all() and np.isfinite(got["grad_values"]).all()
    assert np.array_equal(got["grad_gates"][[0, 40, 41]], np.zeros((3, 32)))


def test_growing_gates_over_states_that_are_zero(cuda):
    """The product of the gates overflows where the state is still zero."""
    case = make_case([1000], 32, "f32", False)
    case["gates"][:600], case["values"][:600] = 1e4, 0.0
    case["gates"][600:] = 0.5
    got = run(cuda, case, "f32", backward=False)
    check(case, got, "f32", backward=False)


def test_other_stream(cuda):
    torch = cuda
    case = make_case(LENGTHS["mixed"], 64, "bf16", True)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    check(case, run(torch, case, "bf16", stream=stream), "bf16")


def test_checked_mode_refuses_bad_offsets(cuda):
    torch = cuda
    from ragged import ValidationError
    program = scan_program("f32", 8)
    values = torch.ones((6, 8), device="cuda")
    out = torch.full_like(values, SENTINEL)
    for offsets in ([0, 4, 3, 6], [1, 6], [0, 5], [0, -1, 6]):
        with pytest.raises(ValidationError, match="offsets validation failed"):
            program.run(values, values, torch.tensor(offsets, device="cuda"), out, mode="checked")
    assert torch.all(out == SENTINEL).item()
    report = program.run(values, values, torch.tensor([0, 4, 6], device="cuda"), out, mode="checked")
    assert report.mode == "checked" and report.kernel_names == ("offsets_init", "offsets_check", "scan")
    big = torch.ones((5000, 8), device="cuda")
    program.run(big, big, torch.tensor([0, 5000], device="cuda"), torch.empty_like(big), mode="checked")


def test_captured_calls_replay_on_new_inputs(cuda):
    """Forward and backward in one graph; scratch is reset inside it, and two
    graphs of the same program do not share it."""
    torch = cuda
    program = scan_program("f32", 64)
    cases = [make_case([3000, 5, 2000], 64, "f32", True, seed=s) for s in (1, 2, 3)]
    statics, graphs, outs = [], [], []
    for _ in range(2):
        t = device(torch, cases[0], "f32", "i64")
        o = dict(out=torch.empty_like(t["values"]), final=torch.empty_like(t["initial"]),
                 carries=torch.empty((program.carry_rows(5005), 64), device="cuda"),
                 grad_values=torch.empty_like(t["values"]), grad_gates=torch.empty_like(t["values"]),
                 grad_initial=torch.empty_like(t["initial"]))

        def step(t=t, o=o):
            program.run(t["values"], t["gates"], t["offsets"], o["out"], initial=t["initial"], final=o["final"],
                        carries=o["carries"])
            program.run_backward(t["values"], t["gates"], t["offsets"], o["carries"], t["grad_out"],
                                 initial=t["initial"], grad_final=t["grad_final"], grad_values=o["grad_values"],
                                 grad_gates=o["grad_gates"], grad_initial=o["grad_initial"])

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        statics.append(t)
        graphs.append(graph)
        outs.append(o)
    for case in cases:
        fresh = device(torch, case, "f32", "i64")
        for t in statics:
            for name, tensor in t.items():
                tensor.copy_(fresh[name])
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for o in outs:
            check(case, {k: host(v) for k, v in o.items()}, "f32")
    del graphs


@pytest.mark.parametrize("route", ["call", "operator", "compiled"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_autograd(cuda, dtype, route):
    """The eager call, the operator below it, and a compiled full graph."""
    torch = cuda
    from ragged import torch_adapter
    case = make_case(LENGTHS["mixed"], 40, dtype, True)
    t = device(torch, case, dtype, "i64")
    leaves = [t[k].requires_grad_() for k in ("values", "gates", "initial")]
    program = scan_program(dtype, 40)
    if route == "call":
        out, final = torch_adapter.segment_scan(leaves[0], leaves[1], t["offsets"], program=program, initial=leaves[2])
    else:
        token = torch_adapter.register_program(program)
        torch_adapter.register_torch_ops()

        def model(values, gates, initial, offsets):
            return torch.ops.ragged_mlir.segment_scan(values, gates, offsets, initial, token)[:2]

        if route == "compiled":
            model = torch.compile(model, backend="aot_eager", fullgraph=True)
        out, final = model(*leaves, t["offsets"])
    grads = torch.autograd.grad((out, final), leaves, (t["grad_out"], t["grad_final"]))
    got = dict(out=out, final=final, grad_values=grads[0], grad_gates=grads[1], grad_initial=grads[2])
    check(case, {k: host(v.detach()) for k, v in got.items()}, dtype)


def test_autograd_layouts_and_missing_gradients(cuda):
    """Expanded and transposed gradients, one output's gradient alone, inputs
    that are views, leaves without a gradient."""
    torch = cuda
    from ragged import ValidationError, torch_adapter
    program = scan_program("f32", 40)
    case = make_case(LENGTHS["mixed"], 40, "f32", False)
    t = device(torch, case, "f32", "i64")
    case["grad_out"], case["grad_final"] = np.ones_like(case["grad_out"]), np.zeros_like(case["grad_final"])
    values = t["values"].t().contiguous().t().requires_grad_()
    out, final = torch_adapter.segment_scan(values, t["gates"].requires_grad_(), t["offsets"], program=program)
    gv, gg = torch.autograd.grad(out.sum(), (values, t["gates"]), retain_graph=True)
    check(case, dict(out=host(out.detach()), final=host(final.detach()), grad_values=host(gv), grad_gates=host(gg)), "f32")
    case["grad_out"], case["grad_final"] = np.zeros_like(case["grad_out"]), np.ones_like(case["grad_final"])
    gv, gg = torch.autograd.grad(final.sum(), (values, t["gates"]), retain_graph=True)
    check(case, dict(out=host(out.detach()), final=host(final.detach()), grad_values=host(gv), grad_gates=host(gg)), "f32")
    with pytest.raises((ValidationError, RuntimeError), match="second derivatives"):
        torch.autograd.grad(out.sum(), values, create_graph=True)
    with torch.no_grad():
        out, _ = torch_adapter.segment_scan(values, t["gates"], t["offsets"], program=program)
    assert not out.requires_grad


@pytest.mark.parametrize("wanted", [(0,), (1,), (2,), (0, 2)])
def test_gradients_of_some_inputs(cuda, wanted):
    """Gradients that no one asks for are not computed; the others are the same."""
    torch = cuda
    from ragged import torch_adapter
    case = make_case(LENGTHS["mixed"], 48, "bf16", True)
    all_of_them = run(torch, case, "bf16")
    t = device(torch, case, "bf16", "i64")
    names = ("values", "gates", "initial")
    leaves = [t[names[i]].requires_grad_() for i in wanted]
    out, final = torch_adapter.segment_scan(t["values"], t["gates"], t["offsets"], program=scan_program("bf16", 48),
                                            initial=t["initial"])
    grads = torch.autograd.grad((out, final), leaves, (t["grad_out"], t["grad_final"]))
    for i, grad in zip(wanted, grads):
        assert np.array_equal(host(grad), all_of_them["grad_" + names[i]]), names[i]


_FIRST_CALL = """
import sys
sys.path[:0] = {paths!r}
import tempfile, torch
from ragged import ArtifactCache, Compiler, MatmulSpec, ScanSpec
cache = ArtifactCache(tempfile.mkdtemp())
scan = Compiler().compile(ScanSpec("f32", 32), cache)
product = Compiler().compile(MatmulSpec("bf16", 64, 64), cache)
v, g = torch.ones(3000, 32, device="cuda"), torch.full((3000, 32), 0.5, device="cuda")
o, out = torch.tensor([0, 1, 3000], device="cuda"), torch.empty(3000, 32, device="cuda")
x, w = torch.ones(3000, 64, device="cuda").bfloat16(), torch.ones(2, 64, 64, device="cuda").bfloat16()
y = torch.empty_like(x)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    scan.run(v, g, o, out)
    product.run(x, w, o, y)
graph.replay()
torch.cuda.synchronize()
assert out[0, 0].item() == 1 and abs(out[2999, 5].item() - 2) < 1e-6 and torch.all(y == 64).item()
print("captured")
"""


def test_the_first_call_may_be_captured(cuda):
    """A process whose first calls are inside a graph capture."""
    import subprocess
    import sys
    from conftest import PACKAGE, REPO
    code = _FIRST_CALL.format(paths=[str(REPO), str(PACKAGE)])
    result = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert result.returncode == 0 and "captured" in result.stdout, result.stderr[-2000:]


def test_gradients_are_the_differences_of_the_outputs(cuda):
    """The loss <grad_out, out> + <grad_final, final> is linear in values and
    initial, and in each single row of the gates, so its differences over
    steps of any size are the gradients, but for the rounding of the losses
    (f32 outputs, summed in 64 bits)."""
    torch = cuda
    rng = np.random.default_rng(3)
    case = make_case([300, 0, 77, 1], 16, "f32", True)
    got = run(torch, case, "f32")

    def loss(case):
        o = run(torch, case, "f32", backward=False)
        weight = [case["grad_out"].astype(np.float64), case["grad_final"].astype(np.float64)]
        r = ref.forward(*(case[k].astype(np.float64) for k in ("values", "gates")), case["offsets"],
                        case["initial"].astype(np.float64))
        noise = sum((np.abs(w) * m).sum() for w, m in zip(weight, (r["major"], r["final_major"]))) * (2 * 300 + 128) * ref.STEP
        return (weight[0] * o["out"]).sum() + (weight[1] * o["final"]).sum(), noise

    base, noise = loss(case)
    for name, grad in (("values", "grad_values"), ("initial", "grad_initial")):
        step = rng.normal(size=case[name].shape).astype(np.float32)
        moved = dict(case, **{name: case[name] + step})
        step = moved[name].astype(np.float64) - case[name]
        there, more = loss(moved)
        slack = (np.abs(got[grad]) * np.abs(step)).sum() * (2 * 300 + 128) * ref.STEP * 10
        assert abs(there - base - (got[grad] * step).sum()) <= noise + more + slack, name
    for row in (0, 1, 150, 299, 300, 377):
        gates = case["gates"].copy()
        gates[row] = rng.uniform(0, 1, 16)
        step = gates[row].astype(np.float64) - case["gates"][row]
        there, more = loss(dict(case, gates=gates))
        assert abs(there - base - (got["grad_gates"][row] * step).sum()) <= noise + more, row


def test_jagged_tensors(cuda):
    torch = cuda
    from ragged import torch_adapter
    case = make_case([5, 0, 300, 2], 32, "f32", False)
    t = device(torch, case, "f32", "i64")
    nt = torch.nested.nested_tensor_from_jagged(t["values"], t["offsets"])
    gates = torch.nested.nested_tensor_from_jagged(t["gates"], t["offsets"])
    out, final = torch_adapter.njt_scan(nt, gates, program=scan_program("f32", 32))
    wide = [case[k].astype(np.float64) for k in ("values", "gates")]
    ref.check_forward(ref.forward(*wide, case["offsets"]), host(out.values()), host(final), "f32")


def test_offsets_beyond_32_bits_of_elements(cuda):
    """N * D passes 2^32: the last rows are found by 64-bit offsets."""
    torch = cuda
    n, d = 4_300_000, 1024
    program = scan_program("bf16", d)
    values = torch.zeros((n, d), dtype=torch.bfloat16, device="cuda")
    gates = torch.ones_like(values)
    values[-3:] = 1
    out = torch.empty_like(values)
    offsets = torch.tensor([0, n - 2, n], device="cuda")
    final = torch.empty((2, d), device="cuda")
    program.run(values, gates, offsets, out, final=final)
    tail = out[-4:].float()
    assert torch.equal(tail, torch.tensor([[0.0], [1.0], [1.0], [2.0]], device="cuda").expand(4, d))
    assert torch.equal(final, torch.tensor([[1.0], [2.0]], device="cuda").expand(2, d))
    assert not out[:-3].any().item()


def test_chained_calls_and_two_streams_at_once(cuda):
    """Calls whose launches may overlap, back to back on the rows before and
    from two streams: the same bits as with a synchronisation after each."""
    torch = cuda
    torch.manual_seed(7)
    offsets = torch.tensor([0, 900, 901, 5000, 20_011], device="cuda")
    program = scan_program("bf16", 200)
    gates = torch.rand(20_011, 200, device="cuda").bfloat16()
    streams = [torch.cuda.Stream() for _ in range(2)]
    first = [torch.randn(20_011, 200, device="cuda").bfloat16() for _ in streams]
    rows = [[torch.empty_like(x) for _ in range(6)] for x in first]

    def chain(s, wait):
        source = first[s]
        for out in rows[s]:
            program.run(source, gates, offsets, out, streams[s])
            if wait:
                torch.cuda.synchronize()
            source = out

    torch.cuda.synchronize()
    for s in range(2):
        chain(s, True)
    want = [[t.clone() for t in row] for row in rows]
    for _ in range(5):
        for row in rows:
            for t in row:
                t.fill_(SENTINEL)
        torch.cuda.synchronize()
        for s in range(2):
            chain(s, False)
        torch.cuda.synchronize()
        for s in range(2):
            assert all(torch.equal(a, b) for a, b in zip(rows[s], want[s]))


@pytest.mark.parametrize("route", ["call", "operator"])
@pytest.mark.parametrize("initial", [False, True])
@pytest.mark.parametrize("lengths,behind", [([3, 0, 9], 20), ([300, 0, 700, 0], 5), ([65, 2000, 1], 1500), ([0, 0], 900),
                                            ([1] * 60, 200), ([64, 64], 64)])
@pytest.mark.parametrize("dtype,d", [("f32", 12), ("f32", 100), ("bf16", 128), ("bf16", 7)])
def test_padded_rows_of_results_are_zero(cuda, dtype, d, lengths, behind, initial, route):
    """Rows behind the last offset, NaN in the inputs: zeros in what the call
    allocates, in fresh memory that holds NaN; the rest is what run() writes."""
    torch = cuda
    from ragged import torch_adapter
    case = make_case(lengths, d, dtype, initial, seed=behind)
    t = device(torch, case, dtype, "i64")
    used = int(case["offsets"][-1])
    for name in ("values", "gates", "grad_out"):
        t[name] = torch.cat([t[name], torch.full((behind, d), float("nan"), device="cuda", dtype=t[name].dtype)])
    program = scan_program(dtype, d)
    want = {name: torch.zeros_like(t["values"]) for name in ("out", "grad_values", "grad_gates")}
    want["final"] = torch.empty((len(lengths), d), device="cuda")
    want["grad_initial"] = torch.empty_like(want["final"]) if initial else None
    carries = torch.empty((program.carry_rows(used + behind), d), device="cuda")
    program.run(t["values"], t["gates"], t["offsets"], want["out"], initial=t["initial"], final=want["final"],
                carries=carries)
    program.run_backward(t["values"], t["gates"], t["offsets"], carries, t["grad_out"], initial=t["initial"],
                         grad_final=t["grad_final"], grad_values=want["grad_values"], grad_gates=want["grad_gates"],
                         grad_initial=want["grad_initial"])
    names = ["values", "gates"] + (["initial"] if initial else [])
    leaves = [t[name].requires_grad_() for name in names]

    def dirty():
        blocks = [torch.full(t["values"].shape, float("nan"), device="cuda", dtype=t["values"].dtype) for _ in range(4)]
        torch.cuda.synchronize()
        del blocks

    dirty()
    if route == "call":
        out, final = torch_adapter.segment_scan(*leaves[:2], t["offsets"], program=program, initial=t["initial"])
    else:
        torch_adapter.register_torch_ops()
        out, final, _ = torch.ops.ragged_mlir.segment_scan(*leaves[:2], t["offsets"], t["initial"],
                                                           torch_adapter.register_program(program))
    dirty()
    grads = torch.autograd.grad((out, final), leaves, (t["grad_out"], t["grad_final"]))
    for got, name in zip((out, final, *grads), ("out", "final", "grad_values", "grad_gates", "grad_initial")):
        assert torch.equal(got, want[name]), name


def test_checked_backward_validates_the_offsets(cuda):
    torch = cuda
    from ragged import ValidationError, torch_adapter
    program = scan_program("f32", 8)
    case = make_case([700, 0, 301], 8, "f32", False)
    t = device(torch, case, "f32", "i64")
    carries = torch.empty((program.carry_rows(1001), 8), device="cuda")
    program.run(t["values"], t["gates"], t["offsets"], torch.empty_like(t["values"]), carries=carries)
    grads = []
    for mode in ("validated", "checked"):
        grads.append(torch.empty_like(t["values"]))
        report = program.run_backward(t["values"], t["gates"], t["offsets"], carries, t["grad_out"], mode=mode,
                                      grad_values=grads[-1])
    assert report.kernel_names[:2] == ("offsets_init", "offsets_check") and torch.equal(*grads)
    for mode, wrong in (("checked", t["offsets"] + 1), ("unsafe", t["offsets"])):
        with pytest.raises(ValidationError, match="offsets validation failed|mode"):
            program.run_backward(t["values"], t["gates"], wrong, carries, t["grad_out"], mode=mode, grad_values=grads[0])
    out, _ = torch_adapter.segment_scan(t["values"].requires_grad_(), t["gates"], t["offsets"], program=program,
                                        mode="checked")
    assert torch.equal(torch.autograd.grad(out, t["values"], t["grad_out"])[0], grads[0])
