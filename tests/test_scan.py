"""The segmented scan without a GPU: specifications, the C ABI's checks of
arguments, shape inference, refusals, and the 64-bit recurrence that the GPU
tests go by."""
from __future__ import annotations

import ctypes
from types import SimpleNamespace

import numpy as np
import pytest

import scan_reference as ref

torch = pytest.importorskip("torch")


@pytest.fixture
def program(native_library, tmp_path):
    from ragged import ArtifactCache, Compiler, ScanSpec
    return Compiler().compile(ScanSpec("f32", 8), ArtifactCache(tmp_path))


def test_spec_round_trip_and_refusals():
    from ragged import Hints, MatmulSpec, ProgramSpec, ScanSpec, ValidationError
    spec = ScanSpec("bf16", 256, "i32", hints=Hints(max_len=9))
    assert ScanSpec.from_dict(spec.to_dict()) == spec and spec.op == "scan"
    assert len({spec.ir_hash, ScanSpec("bf16", 256, "i32").ir_hash, ProgramSpec("sum", "bf16", 256, "i32").ir_hash,
                MatmulSpec("bf16", 256, 256, "i32").ir_hash}) == 4
    for bad in (dict(dtype="f16"), dict(feature_dim=0), dict(feature_dim=65537), dict(feature_dim=2.0),
                dict(offsets_dtype="i16"), dict(hints=None), dict(chip="sm_90")):
        with pytest.raises(ValidationError):
            ScanSpec(**bad)
    with pytest.raises(ValidationError):
        ScanSpec.from_dict(MatmulSpec().to_dict())


def test_compile_caches_the_program(native_library, tmp_path):
    from ragged import ArtifactCache, CompiledScan, Compiler, ScanSpec
    cache = ArtifactCache(tmp_path)
    first, second = (Compiler().compile(ScanSpec("f32", 8), cache) for _ in range(2))
    assert isinstance(first, CompiledScan) and not first.cache_hit and second.cache_hit
    assert first.schedules == ("scan",)


def test_abi_refuses_bad_arguments(native_library):
    from ragged import _native
    lib = native_library
    one = ctypes.c_int64()

    def sizes(dtype=0, index=1, d=8, n=4, b=1):
        return lib.rg_scan_workspace_bytes(dtype, index, d, n, b, ctypes.byref(one))

    assert sizes() == 0
    for bad in (dict(dtype=2), dict(index=5), dict(d=0), dict(d=65537), dict(n=-1), dict(b=-1), dict(b=0),
                dict(n=2**31, index=0), dict(b=2**31), dict(n=2**62)):
        assert sizes(**bad) == _native.RG_ERR_INVALID_ARGUMENT, bad
    assert lib.rg_scan_workspace_bytes(0, 1, 8, 4, 1, None) == _native.RG_ERR_INVALID_ARGUMENT
    buffer = (ctypes.c_char * 4096)()
    base = (ctypes.addressof(buffer) + 255) // 256 * 256
    v, g, o, out = base, base + 128, base + 256, base + 512

    def scan(values=v, gates=g, offsets=o, initial=None, out=out, final=None, carries=None):
        return lib.rg_scan(0, 1, 8, 4, 1, values, gates, offsets, initial, out, final, carries, None, 0, None, None)

    for bad in (dict(values=None), dict(gates=None), dict(offsets=None), dict(out=None), dict(values=v + 2),
                dict(out=v), dict(out=g + 16), dict(final=v), dict(final=out + 4), dict(carries=out),
                dict(out=o - 64), dict(initial=base + 1024 + 2)):
        assert scan(**bad) == _native.RG_ERR_INVALID_ARGUMENT, bad
    assert lib.rg_scan(0, 1, 8, 0, 0, *[None] * 8, 0, None, None) == 0  # no segments: nothing to do
    grads = dict(values=v, gates=g, offsets=o, initial=None, carries=base + 768, grad_out=base + 896, grad_final=None,
                 grad_values=base + 1024, grad_gates=base + 1152, grad_initial=None)

    def backward(**change):
        return lib.rg_scan_backward(0, 1, 8, 4, 1, *dict(grads, **change).values(), None, 0, None, None)

    for bad in (dict(carries=None), dict(grad_out=None), dict(grad_values=base + 896), dict(grad_gates=base + 1024),
                dict(grad_initial=base + 1280), dict(grad_values=v)):
        assert backward(**bad) == _native.RG_ERR_INVALID_ARGUMENT, bad


def test_host_tensors_are_refused(program):
    from ragged import RuntimeUnavailable, ValidationError
    values, offsets = torch.ones((6, 8)), torch.tensor([0, 2, 6])
    out = torch.full((6, 8), -1.0)
    with pytest.raises(RuntimeUnavailable, match="no CPU execution fallback"):
        program.run(values, values, offsets, out)
    with pytest.raises(RuntimeUnavailable, match="no CPU execution fallback"):
        program.run_backward(values, values, offsets, torch.ones((1, 8)), values)
    with pytest.raises(ValidationError, match="mode"):
        program.run(values, values, offsets, out, mode="unsafe")
    with pytest.raises(ValidationError, match="grad_initial"):
        program.run_backward(values, values, offsets, torch.ones((1, 8)), values, grad_initial=torch.ones((2, 8)))
    for bad in (torch.ones(()), None, torch.ones((2, 2))):
        with pytest.raises(ValidationError):
            program.run(values, values, bad, out)
    with pytest.raises(ValidationError):
        program.run(torch.ones(8), values, offsets, out)
    assert torch.all(out == -1).item()


def _registered(monkeypatch, dtype, d):
    from ragged import ScanSpec, torch_adapter
    monkeypatch.setattr(torch_adapter, "_table", torch_adapter.ProgramTable())
    program = SimpleNamespace(spec=ScanSpec(dtype, d), artifact=SimpleNamespace(key=SimpleNamespace(digest=f"scan-{d}")))
    return program


def test_fake_shapes_and_refusals(monkeypatch):
    from ragged import ValidationError, torch_adapter
    program = _registered(monkeypatch, "bf16", 24)
    meta = dict(device="meta")
    values, offsets = torch.empty((700, 24), dtype=torch.bfloat16, **meta), torch.empty((5,), dtype=torch.int32, **meta)
    out, final = torch_adapter.segment_scan(values, values, offsets, program=program)
    assert out.shape == (700, 24) and out.dtype == torch.bfloat16
    assert final.shape == (4, 24) and final.dtype == torch.float32
    ops = torch.ops.ragged_mlir
    assert ops.segment_scan(values, values, offsets, None, "scan-24")[2].shape == (88, 24)
    assert ops.segment_scan(values, values, offsets, None, "scan-24", "validated", False)[2].shape == (0, 24)
    initial = torch.empty((4, 24), **meta)
    for bad in (dict(gates=values.float()), dict(gates=values[:5]), dict(initial=initial.bfloat16()),
                dict(initial=initial[:3]), dict(offsets=offsets.float()), dict(values=values.double()),
                dict(values=values[0])):
        call = dict(dict(values=values, gates=values, offsets=offsets, initial=None), **bad)
        with pytest.raises((ValidationError, RuntimeError)):
            ops.segment_scan(call["values"], call["gates"], call["offsets"], call["initial"], "scan-24")


def test_full_graph_capture_with_gradients(monkeypatch):
    from ragged import torch_adapter
    program = _registered(monkeypatch, "f32", 8)
    token = torch_adapter.register_program(program)
    torch_adapter.register_torch_ops()

    def loss(values, gates, offsets):
        out, final, _ = torch.ops.ragged_mlir.segment_scan(values * 2, gates, offsets, None, token)
        return out.sum() + final.sum()

    values, gates = (torch.empty((30, 8), device="meta", requires_grad=True) for _ in range(2))
    offsets = torch.empty((4,), dtype=torch.int64, device="meta")
    torch.compile(loss, backend="aot_eager", fullgraph=True)(values, gates, offsets).backward()
    assert values.grad.shape == values.shape and gates.grad.shape == gates.shape


def test_reference_gradients_are_differences():
    """The 64-bit gradients against central differences of the 64-bit outputs."""
    rng = np.random.default_rng(0)
    offsets, d = np.array([0, 3, 3, 9, 10]), 2
    values, gates, grad = (rng.normal(size=(10, d)) for _ in range(3))
    initial, grad_final = rng.normal(size=(4, d)), rng.normal(size=(4, d))
    for state in (None, initial):
        r = ref.backward(values, gates, offsets, grad, grad_final, state)

        def loss(v, a, s):
            f = ref.forward(v, a, offsets, s)
            return (f["out"] * grad).sum() + (f["final"] * grad_final).sum()

        inputs = [values, gates] + ([initial] if state is not None else [])
        for k, (x, name) in enumerate(zip(inputs, ("grad_values", "grad_gates", "grad_initial"))):
            for at in np.ndindex(x.shape):
                moved = []
                for sign in (1, -1):
                    y = [z.copy() for z in inputs] + ([None] if state is None else [])
                    y[k][at] += sign * 1e-5
                    moved.append(loss(*y))
                assert abs((moved[0] - moved[1]) / 2e-5 - r[name][at]) < 1e-7, (name, at)
