"""torch integration: custom operators over compiled programs, and NJT helpers.

Importing ``ragged`` never imports torch; ``register_torch_ops()`` defines
the operators once per process.  Their names and schemas are the
reference's interface (``ragged_mlir::segment_reduce`` and
``ragged_mlir::segment_softmax``, python/ragged/torch_adapter.py:51-86 of
the reference) so graphs written against the reference keep working.
Behind them:

* ``ProgramTable`` maps a string token (the program's artifact digest) to a
  ``CompiledProgram``.  The operators take only the token, which
  torch.compile keeps as a graph constant, so a traced graph holds no Python
  object and the operator stays opaque.
* ``OpContract`` states the operators' tensor contract once; the fake
  (meta) kernels and the real ones share it and share ``output_shape``, so
  shape inference under torch.compile cannot drift from what the real call
  allocates.
* The operators live in a ``torch.library`` fragment: a CPU and a CUDA
  kernel that hand the call to ``CompiledProgram.run`` (which refuses CPU
  tensors: there is no CPU fallback) and a registered fake for tracing.
"""
from __future__ import annotations

from dataclasses import dataclass
import threading
from typing import Any

from .errors import ValidationError
from .layers import CARRY_ROWS, CompiledMatmul, CompiledScan
from .runtime import CompiledProgram, _torch

MODES = ("validated", "checked")
REDUCTIONS = ("sum", "max")
MISMATCH = "custom op does not match compiled program semantics"
SCHEMAS = {
    "segment_reduce": 'segment_reduce(Tensor values, Tensor offsets, str kind, str program, '
                      'str mode="validated") -> Tensor',
    "segment_softmax": 'segment_softmax(Tensor values, Tensor offsets, str program, str mode="validated", '
                       'Tensor? mask=None) -> Tensor',
    # The learned operators (no counterpart in the reference).  `record` keeps
    # the states that the backward operator needs.
    "segment_scan": 'segment_scan(Tensor values, Tensor gates, Tensor offsets, Tensor? initial, str program, '
                    'str mode="validated", bool record=True) -> (Tensor, Tensor, Tensor)',
    "segment_scan_backward": 'segment_scan_backward(Tensor values, Tensor gates, Tensor offsets, Tensor? initial, '
                             'Tensor carries, Tensor grad_out, Tensor? grad_final, str program, '
                             'str mode="validated") '
                             '-> (Tensor, Tensor, Tensor)',
    "segment_matmul": 'segment_matmul(Tensor values, Tensor weights, Tensor offsets, str program, '
                      'str mode="validated") -> Tensor',
    "segment_matmul_backward": 'segment_matmul_backward(Tensor values, Tensor weights, Tensor offsets, '
                               'Tensor grad_out, str program, bool[2] wanted, str mode="validated") '
                               '-> (Tensor, Tensor)',
}


def _same_op(program, op: str) -> None:
    if program.spec.op != op:
        raise ValidationError(MISMATCH)


class ProgramTable:
    """Process-wide token -> program map behind the custom operators."""

    def __init__(self):
        self._lock = threading.Lock()
        self._programs: dict[str, CompiledProgram] = {}

    def enter(self, program) -> str:
        if getattr(program.spec, "alias", "none") != "none":
            raise ValidationError("functional custom ops require an out-of-place specialization")
        token = program.artifact.key.digest
        with self._lock:
            self._programs[token] = program
        return token

    def lookup(self, token: str, op: str):
        with self._lock:
            program = self._programs.get(token)
        if program is None:
            raise ValidationError("compiled program token is not registered in this process")
        _same_op(program, op)
        return program


_table = ProgramTable()
_operators: dict[str, Any] = {}
_define_lock = threading.Lock()
_library = None  # the torch.library fragment; kept alive with the operators


def register_program(program) -> str:
    """Enter ``program`` in the operators' table; returns its token."""
    return _table.enter(program)


@dataclass(frozen=True)
class OpContract:
    """The operators' tensor contract (the reference's docs/abi.md and
    docs/mask-abi.md), checked on fake tensors during tracing; the real
    call's CompiledProgram.run checks the same rules on device tensors."""

    torch: Any

    def mode(self, mode: str) -> None:
        if mode not in MODES:
            raise ValidationError("mode must be validated or checked")

    def kind(self, kind: str) -> None:
        if kind not in REDUCTIONS:
            raise ValidationError("segment_reduce kind must be sum or max")

    def inputs(self, values, offsets) -> None:
        torch = self.torch
        if values.ndim != 2 or offsets.ndim != 1:
            raise ValidationError("expected values[N,D] and offsets[B+1]")
        torch._check(offsets.shape[0] >= 1)
        torch._check(values.shape[1] >= 1)
        torch._check(values.shape[1] <= 1024)
        if values.dtype not in (torch.float32, torch.bfloat16):
            raise ValidationError("values must be f32 or bf16")
        if offsets.dtype not in (torch.int32, torch.int64):
            raise ValidationError("offsets must be i32 or i64")
        if not (values.is_contiguous() and offsets.is_contiguous()):
            raise ValidationError("values and offsets must be contiguous")
        if values.device != offsets.device:
            raise ValidationError("values and offsets must use the same device")

    def mask(self, values, mask) -> None:
        if mask is None:
            return
        if mask.dtype != self.torch.float32:
            raise ValidationError("mask must be f32")
        if tuple(mask.shape) != tuple(values.shape):
            raise ValidationError("mask must have exactly values shape [N,D]; broadcasting is unsupported")
        if not mask.is_contiguous():
            raise ValidationError("mask must be contiguous")
        if mask.device != values.device:
            raise ValidationError("mask must use the values device")
        if mask.requires_grad:
            raise ValidationError("autograd is outside the supported forward-only contract")


    def scan(self, values, gates, offsets, initial) -> None:
        self.inputs_of("scan", values, offsets)
        if gates.shape != values.shape or gates.dtype != values.dtype or gates.device != values.device:
            raise ValidationError("gates must have the shape, dtype and device of values")
        if initial is not None and (tuple(initial.shape) != (offsets.shape[0] - 1, values.shape[1])
                                    or initial.dtype != self.torch.float32 or initial.device != values.device):
            raise ValidationError("initial must be f32 [B, D] on the values device")

    def matmul(self, values, weights, offsets) -> None:
        self.inputs_of("matmul", values, offsets)
        if (weights.ndim != 3 or weights.shape[0] != offsets.shape[0] - 1 or weights.shape[1] != values.shape[1]
                or weights.dtype != values.dtype or weights.device != values.device):
            raise ValidationError("weights must be [B, D, out] with the dtype and device of values")

    def inputs_of(self, op: str, values, offsets) -> None:
        """What the learned operators ask of values and offsets."""
        torch = self.torch
        if values.ndim != 2 or offsets.ndim != 1:
            raise ValidationError("expected values[N,D] and offsets[B+1]")
        torch._check(offsets.shape[0] >= 1)
        if values.dtype not in (torch.float32, torch.bfloat16):
            raise ValidationError("values must be f32 or bf16")
        if offsets.dtype not in (torch.int32, torch.int64):
            raise ValidationError("offsets must be i32 or i64")
        if values.device != offsets.device:
            raise ValidationError("values and offsets must use the same device")


def output_shape(op: str, values, offsets) -> tuple:
    """[B, D] for sum and max, [N, D] for softmax."""
    rows = values.shape[0] if op == "softmax" else offsets.shape[0] - 1
    return (rows, values.shape[1])


def _mask_presence(program, mask) -> None:
    if not hasattr(program.spec, "mask"):  # a scan or a product
        raise ValidationError(MISMATCH)
    if program.spec.mask != (mask is not None):
        raise ValidationError("mask presence must match the compiled specialization")


def _call(values, offsets, token: str, op: str, mode: str, mask=None):
    """The real kernel of both operators: look the program up, allocate the
    output, run it on the current stream."""
    if mode not in MODES:
        raise ValidationError("mode must be validated or checked")
    program = _table.lookup(token, op)
    _mask_presence(program, mask)
    output = values.new_empty(output_shape(op, values, offsets))
    options = {"mode": mode} if mask is None else {"mode": mode, "mask": mask}
    program.run(values, offsets, output, **options)
    return output


def _dense(*tensors):
    """The tensors, contiguous: a gradient arrives in whatever layout autograd
    made of it (an expanded sum, a transposed view)."""
    return [t if t is None or t.is_contiguous() else t.contiguous() for t in tensors]


def _scan_shapes(values, offsets, record: bool) -> tuple:
    """Shapes of out, final and carries."""
    n, d = values.shape
    return (n, d), (offsets.shape[0] - 1, d), ((n + CARRY_ROWS - 1) // CARRY_ROWS if record else 0, d)


def _scan_call(values, gates, offsets, initial, program, mode: str, record: bool):
    """(out, final, carries) of segment_scan, on the GPU."""
    torch = _torch()
    values, gates, initial = _dense(values, gates, initial)
    shapes = _scan_shapes(values, offsets, record)
    out = torch.empty_like(values)
    final, carries = (torch.empty(shape, dtype=torch.float32, device=values.device) for shape in shapes[1:])
    program._run(values, gates, offsets, out, initial, final, carries if record else None, None, mode, False, True)
    return out, final, carries


def _scan_backward_call(values, gates, offsets, initial, carries, grad_out, grad_final, program, mode, known=None):
    """The gradients of values, gates and initial, on the GPU.  ``known``: the
    tensors are those of a forward call and the gradients autograd made of its
    outputs, so that they fit, and these gradients are wanted."""
    torch = _torch()
    values, gates, initial, grad_out, grad_final = _dense(values, gates, initial, grad_out, grad_final)
    wanted = known or (True, True, initial is not None)
    grad_values, grad_gates, grad_initial = (torch.empty_like(t) if want else None
                                             for t, want in zip((values, values, initial), wanted))
    if known:
        program._gradients(torch, values, gates, offsets, carries, grad_out, None, mode, initial, grad_final,
                           grad_values, grad_gates, grad_initial, True)
    else:
        program._run_backward(values, gates, offsets, carries, grad_out, None, mode, initial, grad_final, grad_values,
                              grad_gates, grad_initial, True)
    return grad_values, grad_gates, grad_initial


def _no_tangents(torch, *tensors) -> None:
    """Refuses forward-mode derivatives, which a call would drop unnoticed."""
    forward = torch.autograd.forward_ad
    if forward._current_level >= 0 and any(t is not None and forward.unpack_dual(t).tangent is not None
                                           for t in tensors):
        raise ValidationError("forward-mode derivatives are not supported")


def _records(torch, *tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _first_derivative(torch) -> None:
    if torch.is_grad_enabled():
        raise ValidationError("second derivatives are not supported (create_graph)")


def _register_scan(torch, library, contract) -> None:
    def scan_kernel(values, gates, offsets, initial, program, mode="validated", record=True):
        return _scan_call(values, gates, offsets, initial, _table.lookup(program, "scan"), mode, record)

    def scan_backward_kernel(values, gates, offsets, initial, carries, grad_out, grad_final, program, mode="validated"):
        grads = _scan_backward_call(values, gates, offsets, initial, carries, grad_out, grad_final,
                                    _table.lookup(program, "scan"), mode)
        return grads if initial is not None else (*grads[:2], carries.new_empty((0,)))

    for key in ("CPU", "CUDA"):
        library.impl("segment_scan", scan_kernel, key)
        library.impl("segment_scan_backward", scan_backward_kernel, key)

    @torch.library.register_fake("ragged_mlir::segment_scan", lib=library)
    def scan_fake(values, gates, offsets, initial, program, mode="validated", record=True):
        contract.mode(mode)
        contract.scan(values, gates, offsets, initial)
        out, final, carries = _scan_shapes(values, offsets, record)
        state = dict(dtype=torch.float32, device=values.device)
        return (torch.empty(out, dtype=values.dtype, device=values.device), torch.empty(final, **state),
                torch.empty(carries, **state))

    @torch.library.register_fake("ragged_mlir::segment_scan_backward", lib=library)
    def scan_backward_fake(values, gates, offsets, initial, carries, grad_out, grad_final, program, mode="validated"):
        contract.mode(mode)
        grad = torch.empty(values.shape, dtype=values.dtype, device=values.device)
        state = torch.empty(initial.shape if initial is not None else (0,), dtype=torch.float32, device=values.device)
        return grad, torch.empty_like(grad), state

    def setup(ctx, inputs, output):
        values, gates, offsets, initial, program, mode, record = inputs
        ctx.record, ctx.program, ctx.mode, ctx.has_initial = record, program, mode, initial is not None
        ctx.save_for_backward(values, gates, offsets, output[2], *([initial] if initial is not None else []))
        ctx.mark_non_differentiable(output[2])
        ctx.set_materialize_grads(False)

    def backward(ctx, grad_out, grad_final, _):
        if not ctx.record:
            raise ValidationError("the scan recorded no states (record=False): it has no backward pass")
        _first_derivative(torch)
        if grad_out is None and grad_final is None:
            return (None,) * 7
        values, gates, offsets, carries, *initial = ctx.saved_tensors
        if grad_out is None:
            grad_out = torch.zeros_like(values)
        grads = torch.ops.ragged_mlir.segment_scan_backward(
            values, gates, offsets, initial[0] if ctx.has_initial else None, carries, grad_out, grad_final,
            ctx.program, ctx.mode)
        return grads[0], grads[1], None, grads[2] if ctx.has_initial else None, None, None, None

    torch.library.register_autograd("ragged_mlir::segment_scan", backward, setup_context=setup, lib=library)


def _matmul_call(values, weights, offsets, program, mode: str):
    """The output of segment_matmul, on the GPU."""
    values, weights = _dense(values, weights)
    out = _torch().empty((values.shape[0], program.spec.out_dim), dtype=values.dtype, device=values.device)
    program._run(values, weights, offsets, out, None, mode, False, True)
    return out


def _matmul_backward_call(values, weights, offsets, grad_out, program, wanted, mode, known=False):
    """The gradients of values and weights (None: not wanted), on the GPU;
    ``known`` as for the scan."""
    torch = _torch()
    values, weights, grad_out = _dense(values, weights, grad_out)
    grads = [torch.empty_like(t) if want else None for t, want in zip((values, weights), wanted)]
    if known:
        program._gradients(torch, values, weights, offsets, grad_out, None, mode, *grads, True)
    else:
        program._run_backward(values, weights, offsets, grad_out, None, mode, *grads, True)
    return grads


def _plain(torch, *tensors) -> bool:
    """Whether a call can go to the GPU as it is: CUDA tensors, and nothing
    that traces, fakes or wraps calls.  It then skips the operator's dispatch,
    which costs several times what its launches do; everything else (tracing,
    meta and wrapped tensors) takes the operator."""
    return (all(t is None or (type(t) in (torch.Tensor, torch.nn.Parameter) and t.is_cuda) for t in tensors)
            and not torch.compiler.is_compiling() and not torch._C._len_torch_dispatch_stack()
            and not torch._C._functorch.peek_interpreter_stack())


_functions: dict[str, Any] = {}


def _autograd_functions(torch) -> dict[str, Any]:
    """The operators' differentiable forms for plain calls."""
    if _functions:
        return _functions

    class Scan(torch.autograd.Function):
        @staticmethod
        def forward(ctx, values, gates, offsets, initial, program, mode):
            out, final, carries = _scan_call(values, gates, offsets, initial, program, mode, True)
            ctx.save_for_backward(values, gates, offsets, carries, initial)
            ctx.program, ctx.mode = program, mode
            ctx.set_materialize_grads(False)
            return out, final

        @staticmethod
        def backward(ctx, grad_out, grad_final):
            _first_derivative(torch)
            if grad_out is None and grad_final is None:
                return (None,) * 6
            values, gates, offsets, carries, initial = ctx.saved_tensors
            if grad_out is None:
                grad_out = torch.zeros_like(values)
            wanted = ctx.needs_input_grad
            grads = _scan_backward_call(values, gates, offsets, initial, carries, grad_out, grad_final, ctx.program,
                                        ctx.mode, (wanted[0], wanted[1], wanted[3]))
            return grads[0], grads[1], None, grads[2], None, None

    class Matmul(torch.autograd.Function):
        @staticmethod
        def forward(ctx, values, weights, offsets, program, mode):
            ctx.save_for_backward(values, weights, offsets)
            ctx.program, ctx.mode = program, mode
            ctx.set_materialize_grads(False)
            return _matmul_call(values, weights, offsets, program, mode)

        @staticmethod
        def backward(ctx, grad_out):
            _first_derivative(torch)
            wanted = ctx.needs_input_grad[:2]
            if grad_out is None or not any(wanted):
                return (None,) * 5
            values, weights, offsets = ctx.saved_tensors
            return (*_matmul_backward_call(values, weights, offsets, grad_out, ctx.program, wanted, ctx.mode, True),
                    None, None, None)

    _functions.update(scan=Scan, matmul=Matmul)
    return _functions


def _register_matmul(torch, library, contract) -> None:
    def matmul_kernel(values, weights, offsets, program, mode="validated"):
        return _matmul_call(values, weights, offsets, _table.lookup(program, "matmul"), mode)

    def matmul_backward_kernel(values, weights, offsets, grad_out, program, wanted, mode="validated"):
        grads = _matmul_backward_call(values, weights, offsets, grad_out, _table.lookup(program, "matmul"), wanted, mode)
        return tuple(values.new_empty((0,)) if g is None else g for g in grads)

    for key in ("CPU", "CUDA"):
        library.impl("segment_matmul", matmul_kernel, key)
        library.impl("segment_matmul_backward", matmul_backward_kernel, key)

    @torch.library.register_fake("ragged_mlir::segment_matmul", lib=library)
    def matmul_fake(values, weights, offsets, program, mode="validated"):
        contract.mode(mode)
        contract.matmul(values, weights, offsets)
        return values.new_empty((values.shape[0], weights.shape[2]))

    @torch.library.register_fake("ragged_mlir::segment_matmul_backward", lib=library)
    def matmul_backward_fake(values, weights, offsets, grad_out, program, wanted, mode="validated"):
        contract.mode(mode)
        return tuple(t.new_empty(t.shape if want else (0,)) for t, want in zip((values, weights), wanted))

    def setup(ctx, inputs, output):
        values, weights, offsets, ctx.program, ctx.mode = inputs
        ctx.save_for_backward(values, weights, offsets)
        ctx.set_materialize_grads(False)

    def backward(ctx, grad_out):
        _first_derivative(torch)
        wanted = list(ctx.needs_input_grad[:2])
        if grad_out is None or not any(wanted):
            return (None,) * 5
        values, weights, offsets = ctx.saved_tensors
        grads = torch.ops.ragged_mlir.segment_matmul_backward(values, weights, offsets, grad_out, ctx.program, wanted,
                                                              ctx.mode)
        return grads[0] if wanted[0] else None, grads[1] if wanted[1] else None, None, None, None

    torch.library.register_autograd("ragged_mlir::segment_matmul", backward, setup_context=setup, lib=library)


def register_torch_ops() -> dict[str, Any]:
    """Define the ``ragged_mlir`` operators (once); returns name -> operator of
    segment_reduce and segment_softmax, as the reference's function does
    (``torch.ops.ragged_mlir`` holds them all)."""
    global _library
    with _define_lock:
        if _operators:
            return dict(_operators)
        torch = _torch()
        contract = OpContract(torch)
        library = torch.library.Library("ragged_mlir", "FRAGMENT")
        for schema in SCHEMAS.values():
            library.define(schema)

        def reduce_kernel(values, offsets, kind, program, mode="validated"):
            contract.kind(kind)
            return _call(values, offsets, program, kind, mode)

        def softmax_kernel(values, offsets, program, mode="validated", mask=None):
            return _call(values, offsets, program, "softmax", mode, mask)

        for key in ("CPU", "CUDA"):
            library.impl("segment_reduce", reduce_kernel, key)
            library.impl("segment_softmax", softmax_kernel, key)

        @torch.library.register_fake("ragged_mlir::segment_reduce", lib=library)
        def reduce_fake(values, offsets, kind, program, mode="validated"):
            contract.mode(mode)
            contract.inputs(values, offsets)
            contract.kind(kind)
            return values.new_empty(output_shape(kind, values, offsets))

        @torch.library.register_fake("ragged_mlir::segment_softmax", lib=library)
        def softmax_fake(values, offsets, program, mode="validated", mask=None):
            contract.mode(mode)
            contract.inputs(values, offsets)
            contract.mask(values, mask)
            return values.new_empty(output_shape("softmax", values, offsets))

        _register_scan(torch, library, contract)
        _register_matmul(torch, library, contract)
        _library = library
        namespace = torch.ops.ragged_mlir
        _operators.update(segment_reduce=namespace.segment_reduce, segment_softmax=namespace.segment_softmax)
        return dict(_operators)


def segment_reduce(values, offsets, kind: str, *, program: CompiledProgram, mode: str = "validated"):
    """Segmented sum or max of ``program`` through the custom operator."""
    return register_torch_ops()["segment_reduce"](values, offsets, kind, register_program(program), mode)


def segment_softmax(values, offsets, *, program: CompiledProgram, mode: str = "validated", mask=None):
    """Segmented softmax of ``program`` through the custom operator."""
    _mask_presence(program, mask)
    return register_torch_ops()["segment_softmax"](values, offsets, register_program(program), mode, mask)


def segment_scan(values, gates, offsets, *, program: CompiledScan, initial=None, mode: str = "validated"):
    """(out [N, D], final f32 [B, D]) of the recurrence out[t] = gates[t] *
    out[t - 1] + values[t] within each segment, differentiable (once) in
    values, gates and initial.  Rows behind the last offset (a padded batch) are
    zero in out and in the gradients, whatever the inputs hold there.

    Under a CUDA graph capture of a backward pass (``torch.autograd.grad``
    included) autograd must not have an eager graph of the same leaves alive:
    its accumulation nodes stay on the stream they were first used on, and the
    capture fails, as with torch's own operations.  Drop earlier graphs first."""
    torch = _torch()
    _same_op(program, "scan")
    record = _records(torch, values, gates, initial)
    _no_tangents(torch, values, gates, initial)
    if _plain(torch, values, gates, offsets, initial):
        if record:
            return _autograd_functions(torch)["scan"].apply(values, gates, offsets, initial, program, mode)
        return _scan_call(values, gates, offsets, initial, program, mode, False)[:2]
    register_torch_ops()
    out, final, _ = torch.ops.ragged_mlir.segment_scan(values, gates, offsets, initial, register_program(program),
                                                       mode, record)
    return out, final


def segment_matmul(values, weights, offsets, *, program: CompiledMatmul, mode: str = "validated"):
    """[N, out] of values[t] @ weights[s] for the rows t of segment s,
    differentiable (once) in values and weights.  Rows behind the last offset
    are zero, as are the gradients of those values.  (On captured backward
    passes: see ``segment_scan``.)"""
    torch = _torch()
    _same_op(program, "matmul")
    _no_tangents(torch, values, weights)
    if _plain(torch, values, weights, offsets):
        if _records(torch, values, weights):
            return _autograd_functions(torch)["matmul"].apply(values, weights, offsets, program, mode)
        return _matmul_call(values, weights, offsets, program, mode)
    register_torch_ops()
    return torch.ops.ragged_mlir.segment_matmul(values, weights, offsets, register_program(program), mode)


def bind(program: CompiledProgram, *, mode: str = "validated"):
    """A callable that only invokes the opaque operator with this program's
    token, so torch.compile can capture it in a full graph: ``f(values,
    offsets[, mask])``, for a scan ``f(values, gates, offsets[, initial])`` ->
    (out, final) and for a product ``f(values, weights, offsets)``, both
    differentiable.  The program is registered here, once."""
    if mode not in MODES:
        raise ValidationError("mode must be validated or checked")
    torch = _torch()
    operators = register_torch_ops()
    token = register_program(program)
    if program.spec.op == "scan":
        scan_op = torch.ops.ragged_mlir.segment_scan

        def scan(values, gates, offsets, initial=None):
            return scan_op(values, gates, offsets, initial, token, mode, _records(torch, values, gates, initial))[:2]

        return scan
    if program.spec.op == "matmul":
        matmul_op = torch.ops.ragged_mlir.segment_matmul
        return lambda values, weights, offsets: matmul_op(values, weights, offsets, token, mode)
    if program.spec.op != "softmax":
        reduce_op, kind = operators["segment_reduce"], program.spec.op
        return lambda values, offsets: reduce_op(values, offsets, kind, token, mode)
    softmax_op = operators["segment_softmax"]

    def softmax(values, offsets, mask=None):
        _mask_presence(program, mask)
        return softmax_op(values, offsets, token, mode, mask)

    return softmax


def jagged_components(nt):
    """(values[N, D], offsets[B+1]) of a contiguous ``torch.jagged`` nested
    tensor of shape [B, jagged, D], without copies."""
    torch = _torch()
    if not getattr(nt, "is_nested", False) or nt.layout != torch.jagged:
        raise ValidationError("expected a torch.jagged nested tensor")
    if nt.dim() != 3:
        raise ValidationError("expected NJT shape [B, jagged, D]")
    if nt.lengths() is not None:
        raise ValidationError("NJT with explicit lengths/holes is outside the contiguous offsets contract")
    if nt._ragged_idx != 1:
        raise ValidationError("only the first non-batch NJT dimension may be ragged")
    values, offsets = nt.values(), nt.offsets()
    if values.ndim != 2 or not (values.is_contiguous() and offsets.is_contiguous()):
        raise ValidationError("NJT values[N,D] and offsets must be contiguous")
    return values, offsets


def njt_reduce(nt, kind: str, *, program: CompiledProgram, mode: str = "validated"):
    """Segmented sum or max over the ragged dimension of an NJT: [B, D]."""
    values, offsets = jagged_components(nt)
    return segment_reduce(values, offsets, kind, program=program, mode=mode)


def njt_scan(nt, gates, *, program: CompiledScan, initial=None, mode: str = "validated"):
    """(NJT of the outputs, final) of ``segment_scan`` over the ragged
    dimension of an NJT; ``gates`` is an NJT on the same offsets."""
    values, offsets = jagged_components(nt)
    gate_values, gate_offsets = jagged_components(gates)
    if gate_offsets is not offsets and gate_offsets.data_ptr() != offsets.data_ptr():
        raise ValidationError("gates must share the offsets of the values")
    out, final = segment_scan(values, gate_values, offsets, program=program, initial=initial, mode=mode)
    return _torch().nested.nested_tensor_from_jagged(out, offsets=offsets), final


def njt_matmul(nt, weights, *, program: CompiledMatmul, mode: str = "validated"):
    """``segment_matmul`` over the ragged dimension of an NJT, returned as an
    NJT on the same offsets."""
    values, offsets = jagged_components(nt)
    out = segment_matmul(values, weights, offsets, program=program, mode=mode)
    return _torch().nested.nested_tensor_from_jagged(out, offsets=offsets)


def njt_softmax(nt, *, program: CompiledProgram, mode: str = "validated", mask=None):
    """Softmax over the ragged dimension of an NJT, returned as an NJT on the
    same offsets."""
    values, offsets = jagged_components(nt)
    output = segment_softmax(values, offsets, program=program, mode=mode, mask=mask)
    return _torch().nested.nested_tensor_from_jagged(output, offsets=offsets)
