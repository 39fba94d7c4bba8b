"""The segmented matrix product without a GPU: specifications, the C ABI's
checks of arguments, shape inference, refusals, and the 64-bit products that
the GPU tests go by."""
from __future__ import annotations

import ctypes
from types import SimpleNamespace

import numpy as np
import pytest

import matmul_reference as ref

torch = pytest.importorskip("torch")


def test_spec_round_trip_and_refusals():
    from ragged import MatmulSpec, ScanSpec, ValidationError
    spec = MatmulSpec("bf16", 256, 512, "i32")
    assert MatmulSpec.from_dict(spec.to_dict()) == spec and spec.op == "matmul"
    assert spec.ir_hash != MatmulSpec("bf16", 512, 256, "i32").ir_hash
    for bad in (dict(dtype="f16"), dict(feature_dim=0), dict(out_dim=0), dict(out_dim=65537), dict(out_dim="8"),
                dict(offsets_dtype="u32"), dict(hints=3), dict(chip="sm_90")):
        with pytest.raises(ValidationError):
            MatmulSpec(**bad)
    with pytest.raises(ValidationError):
        MatmulSpec.from_dict(ScanSpec().to_dict())


def test_compile(native_library, tmp_path):
    from ragged import ArtifactCache, CompilationError, CompiledMatmul, Compiler, MatmulSpec
    program = Compiler().compile(MatmulSpec("f32", 8, 4), ArtifactCache(tmp_path))
    assert isinstance(program, CompiledMatmul) and program.schedules == ("matmul",)
    with pytest.raises(CompilationError):
        Compiler().compile(object(), ArtifactCache(tmp_path))


def test_abi_refuses_bad_arguments(native_library):
    from ragged import _native
    lib = native_library
    one = ctypes.c_int64()

    def sizes(kind=0, dtype=1, index=1, k=8, m=8, n=64, b=1, left=4096, right=4096):
        return lib.rg_matmul_workspace_bytes(kind, dtype, index, k, m, n, b, left, right, ctypes.byref(one))

    assert sizes() == 0
    aligned = one.value
    assert sizes(left=4098) == 0 and one.value > aligned  # a copy at aligned rows
    assert sizes(k=9) == 0 and one.value > aligned
    assert sizes(dtype=0) == 0 and one.value == 0
    for bad in (dict(kind=3), dict(kind=-1), dict(dtype=2), dict(index=2), dict(k=0), dict(m=65537), dict(n=-1),
                dict(b=-1), dict(b=0), dict(n=2**31), dict(b=2**31)):
        assert sizes(**bad) == _native.RG_ERR_INVALID_ARGUMENT, bad
    assert lib.rg_matmul_workspace_bytes(0, 1, 1, 8, 8, 4, 1, None, None, None) == _native.RG_ERR_INVALID_ARGUMENT
    buffer = (ctypes.c_char * 8192)()
    base = (ctypes.addressof(buffer) + 255) // 256 * 256

    def matmul(kind=0, left=base, right=base + 1024, offsets=base + 2048, out=base + 4096):
        return lib.rg_matmul(kind, 0, 1, 8, 8, 4, 1, left, right, offsets, out, None, 0, None, None)

    for kind in range(3):
        for bad in (dict(left=None), dict(right=None), dict(offsets=None), dict(out=None), dict(left=base + 2),
                    dict(out=base), dict(out=base + 1000), dict(out=base + 2048)):
            assert matmul(kind, **bad) == _native.RG_ERR_INVALID_ARGUMENT, (kind, bad)
    for kind in range(3):  # no rows and no segments: nothing to do
        assert lib.rg_matmul(kind, 0, 1, 8, 8, 0, 0, *[None] * 5, 0, None, None) == 0


def test_host_tensors_are_refused(native_library, tmp_path):
    from ragged import ArtifactCache, Compiler, MatmulSpec, RuntimeUnavailable, ValidationError
    program = Compiler().compile(MatmulSpec("f32", 8, 4), ArtifactCache(tmp_path))
    values, weights, offsets = torch.ones((6, 8)), torch.ones((2, 8, 4)), torch.tensor([0, 2, 6])
    out = torch.full((6, 4), -1.0)
    with pytest.raises(RuntimeUnavailable, match="no CPU execution fallback"):
        program.run(values, weights, offsets, out)
    with pytest.raises(RuntimeUnavailable, match="no CPU execution fallback"):
        program.run_backward(values, weights, offsets, out, grad_values=torch.empty_like(values))
    with pytest.raises(ValidationError, match="mode"):
        program.run(values, weights, offsets, out, mode="unsafe")
    with pytest.raises(ValidationError):
        program.run(torch.ones(8), weights, offsets, out)
    assert torch.all(out == -1).item()


def test_fake_shapes_and_refusals(monkeypatch):
    from ragged import MatmulSpec, ValidationError, torch_adapter
    monkeypatch.setattr(torch_adapter, "_table", torch_adapter.ProgramTable())
    program = SimpleNamespace(spec=MatmulSpec("bf16", 24, 40),
                              artifact=SimpleNamespace(key=SimpleNamespace(digest="matmul-meta")))
    meta = dict(device="meta", dtype=torch.bfloat16)
    values, weights = torch.empty((70, 24), **meta), torch.empty((4, 24, 40), **meta)
    offsets = torch.empty((5,), dtype=torch.int32, device="meta")
    out = torch_adapter.segment_matmul(values, weights, offsets, program=program)
    assert out.shape == (70, 40) and out.dtype == torch.bfloat16
    for bad in (dict(weights=weights[:3]), dict(weights=weights.float()), dict(weights=weights[0]),
                dict(weights=weights.transpose(1, 2)), dict(values=values.half()), dict(offsets=offsets.float())):
        call = dict(dict(values=values, weights=weights, offsets=offsets), **bad)
        with pytest.raises((ValidationError, RuntimeError)):
            torch.ops.ragged_mlir.segment_matmul(call["values"], call["weights"], call["offsets"], "matmul-meta")


def test_full_graph_capture_with_gradients():
    from ragged import torch_adapter
    torch_adapter.register_torch_ops()

    def loss(values, weights, offsets):
        return torch.ops.ragged_mlir.segment_matmul(values * 2, weights, offsets, "shape-only-no-program").sum()

    values = torch.empty((30, 8), device="meta", requires_grad=True)
    weights = torch.empty((3, 8, 4), device="meta", requires_grad=True)
    offsets = torch.empty((4,), dtype=torch.int64, device="meta")
    torch.compile(loss, backend="aot_eager", fullgraph=True)(values, weights, offsets).backward()
    assert values.grad.shape == values.shape and weights.grad.shape == weights.shape


def test_reference_gradients_are_differences():
    rng = np.random.default_rng(0)
    offsets = np.array([0, 3, 3, 7])
    values, weights, grad = rng.normal(size=(7, 4)), rng.normal(size=(3, 4, 5)), rng.normal(size=(7, 5))
    found = ref.products(values, weights, offsets, grad)
    for x, name, other in ((values, "grad_values", lambda v: (v, weights)), (weights, "grad_weights", lambda w: (values, w))):
        for at in np.ndindex(x.shape):
            moved = []
            for sign in (1, -1):
                y = x.copy()
                y[at] += sign * 0.5
                moved.append((ref.products(*other(y), offsets)["out"][0] * grad).sum())
            assert abs(moved[0] - moved[1] - found[name][0][at]) < 1e-9


def test_forward_mode_is_refused(native_library, tmp_path):
    from ragged import ArtifactCache, Compiler, MatmulSpec, ScanSpec, ValidationError, torch_adapter
    cache, offsets = ArtifactCache(tmp_path), torch.tensor([0, 4])
    scan, product = (Compiler().compile(spec, cache) for spec in (ScanSpec("f32", 8), MatmulSpec("f32", 8, 8)))
    x, w = torch.ones(4, 8), torch.ones(1, 8, 8)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, x)
        with pytest.raises(ValidationError, match="forward-mode"):
            torch_adapter.segment_scan(x, dual, offsets, program=scan)
        with pytest.raises(ValidationError, match="forward-mode"):
            torch_adapter.segment_matmul(dual, w, offsets, program=product)


def test_clear_rest_is_a_flag_of_the_calls_alone(native_library):
    """RG_CLEAR_REST goes with a dtype of rg_scan, rg_scan_backward and rg_matmul,
    changes no check of theirs, and is none of a size's."""
    from conftest import REPO
    from ragged import _native
    lib, one, flag = native_library, ctypes.c_int64(), _native.CLEAR_REST
    assert f"RG_CLEAR_REST = {flag} " in (REPO / "include" / "ragged_b200.h").read_text()
    for dtype in (0, 1):
        assert lib.rg_matmul(0, dtype | flag, 1, 8, 8, 0, 0, *[None] * 5, 0, None, None) == 0
        assert lib.rg_scan(dtype | flag, 1, 8, 0, 0, *[None] * 8, 0, None, None) == 0
        assert lib.rg_scan_backward(dtype | flag, 1, 8, 0, 0, *[None] * 11, 0, None, None) == 0
        assert lib.rg_matmul(0, dtype | flag, 1, 8, 8, 4, 1, *[None] * 5, 0, None, None) == _native.RG_ERR_INVALID_ARGUMENT
        assert lib.rg_matmul_workspace_bytes(0, dtype | flag, 1, 8, 8, 4, 1, None, None,
                                             ctypes.byref(one)) == _native.RG_ERR_INVALID_ARGUMENT
        assert lib.rg_scan_workspace_bytes(dtype | flag, 1, 8, 4, 1, ctypes.byref(one)) == _native.RG_ERR_INVALID_ARGUMENT
    for dtype in (2 | flag, flag * 2, -1):
        assert lib.rg_scan(dtype, 1, 8, 0, 0, *[None] * 8, 0, None, None) == _native.RG_ERR_INVALID_ARGUMENT, dtype
        assert lib.rg_matmul(0, dtype, 1, 8, 8, 0, 0, *[None] * 5, 0, None, None) == _native.RG_ERR_INVALID_ARGUMENT, dtype
