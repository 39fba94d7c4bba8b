"""Programs of the learned operators: the segmented scan and the segmented
matrix product.

``Compiler().compile(ScanSpec(...), cache)`` gives a ``CompiledScan`` and a
``MatmulSpec`` a ``CompiledMatmul``.  Both follow ``CompiledProgram.run``: CUDA
tensors on one device, outputs that the caller allocates, the current stream
unless ``stream`` is given, no synchronisation in validated mode, and
``mode="checked"`` to validate the offsets on the device first and to raise
where a bounded wait inside a launch gave up.  ``run`` records no gradient;
``run_backward`` computes the gradients of a call, and
``torch_adapter.segment_scan`` / ``segment_matmul`` put both behind autograd, the
gradients in the mode of the call.
Rows behind the last offset reach no result, so N may stay fixed while the
offsets change (in validated mode; checked mode asks for offsets that end at N).
``run`` and ``run_backward`` leave those rows of what they write as they are;
the functions of ``torch_adapter``, which allocate their results, give zeros.

Neither operation exists in the reference, whose programs end at sums, maxima
and softmaxes of packed rows.
"""
from __future__ import annotations

from contextlib import nullcontext
import time

from . import _native
from .cache import Artifact
from .errors import CacheMismatch, RuntimeUnavailable, ValidationError
from .model import ExecutionReport, MatmulSpec, ScanSpec, runs_on
from .runtime import CompiledProgram, _checked_devices, _torch
from .validation import STATUS_BYTES


CARRY_ROWS = 8  # rows per state that a scan records for its backward pass


class _LayerProgram:
    """Checks and launch steps that both programs share."""

    kind: type

    def __init__(self, spec, artifact: Artifact, *, cache_hit: bool = False):
        if not isinstance(spec, self.kind):
            raise ValidationError(f"spec must be a {self.kind.__name__}")
        if artifact.key.ir_hash != spec.ir_hash:
            raise CacheMismatch("artifact was recorded for a different specialization")
        self.spec, self.artifact, self.cache_hit = spec, artifact, cache_hit
        self._digest = artifact.key.digest
        self._dtypes = None
        self._sizes: dict[tuple, int] = {}
        self._launches: dict[tuple, _Launch] = {}
        self._reports: dict[tuple, dict] = {}

    schedules = property(lambda self: (self.spec.op,))
    _check_offsets = CompiledProgram._check_offsets

    def close(self) -> None:
        """Nothing to unload: kernels live in the shared library."""

    def _cached(self, key, compute):
        found = self._sizes.get(key)
        if found is None:
            if len(self._sizes) >= 256:
                self._sizes.clear()
            found = self._sizes[key] = compute()
        return found

    def _tensors(self, torch, tensors, offsets, mode, gradless):
        """Checks the offsets and each (name, tensor, shape, dtype)."""
        if mode not in ("validated", "checked"):
            raise ValidationError("mode must be validated or checked")
        if self._dtypes is None:
            self._dtypes = ({"f32": torch.float32, "bf16": torch.bfloat16}[self.spec.dtype],
                            {"i32": torch.int32, "i64": torch.int64}[self.spec.offsets_dtype])
        if not isinstance(offsets, torch.Tensor):
            raise ValidationError("offsets must be a torch.Tensor")
        if not offsets.is_cuda:
            raise RuntimeUnavailable(f"offsets must be on a CUDA device that runs {self.spec.chip} code; "
                                     "no CPU execution fallback exists")
        if offsets.dtype != self._dtypes[1]:
            raise ValidationError("tensor dtype differs from compiled dtype/offsets specialization")
        if not offsets.is_contiguous():
            raise ValidationError("offsets must be row-major contiguous")
        device, recording = offsets.device, gradless and torch.is_grad_enabled()
        for name, tensor, shape, dtype in tensors:
            if not isinstance(tensor, torch.Tensor):
                raise ValidationError(f"{name} must be a torch.Tensor")
            if tensor.device != device:
                if not tensor.is_cuda:
                    raise RuntimeUnavailable(f"{name} must be on a CUDA device that runs {self.spec.chip} code; "
                                             "no CPU execution fallback exists")
                raise ValidationError(f"{name} must use the CUDA device of offsets")
            if tensor.dtype != dtype:
                raise ValidationError(f"{name} must have dtype {dtype}: tensor dtype differs from compiled "
                                      "dtype/offsets specialization")
            if tensor.shape != shape:
                raise ValidationError(f"{name} must have shape {tuple(shape)}")
            if not tensor.is_contiguous():
                raise ValidationError(f"{name} must be row-major contiguous")
            if recording and tensor.requires_grad:
                raise ValidationError(f"{name} requires a gradient, which run() does not record: use "
                                      "torch_adapter, or torch.no_grad()")

    def _segments(self, torch, offsets) -> int:
        if not isinstance(offsets, torch.Tensor) or offsets.ndim != 1 or offsets.numel() < 1:
            raise ValidationError("offsets must have shape [B+1], including [0] when B=0")
        return offsets.numel() - 1

    def _rows(self, values, torch, name="values") -> int:
        if not isinstance(values, torch.Tensor) or values.ndim != 2:
            raise ValidationError(f"{name} must have shape [N, static D]")
        return values.shape[0]

    def _launch(self, torch, offsets, n, b, stream, mode, used, work) -> ExecutionReport:
        """For each (key, scratch bytes, call) of ``work``: ``call(scratch
        address, bytes, stream, report)`` on the execution stream.  What a call
        launches goes by its key, and is asked for once for each."""
        started = time.perf_counter()
        checked = mode == "checked"
        if b == 0 and n != 0 and not checked:  # checked mode reports it from the device
            raise ValidationError("B=0 requires N=0; values cannot exist without segments")
        if self.spec.offsets_dtype == "i32" and n > 2**31 - 1:
            raise ValidationError("N exceeds the i32 offsets range")
        device = offsets.device
        if torch.cuda.current_device() != device.index:
            with torch.cuda.device(device):
                return self._launch(torch, offsets, n, b, stream, mode, used, work)
        if device.index not in _checked_devices:
            capability = tuple(torch.cuda.get_device_capability(device))
            if not runs_on(self.spec.chip, capability):
                raise RuntimeUnavailable(f"compiled target {self.spec.chip} does not run on the current device "
                                         f"(sm_{capability[0]}{capability[1]})")
            _checked_devices.add(device.index)
        if stream is not None and (not isinstance(stream, torch.cuda.Stream) or stream.device != device):
            raise ValidationError("stream must be a torch.cuda.Stream on the values device")
        validation, active = None, stream
        if checked:
            active = stream if stream is not None else torch.cuda.current_stream()
            validation = self._check_offsets(offsets, offsets, n, b, active, torch)
        launches, total = (), 0
        if b:
            # (the current stream's handle alone: a Stream object costs as much as a launch)
            on = stream.cuda_stream if stream is not None else torch._C._cuda_getCurrentRawStream(device.index)
            if stream is not None:
                for tensor in used:
                    tensor.record_stream(stream)
            for key, nbytes, call in work:
                address = 0
                if nbytes:
                    # Scratch comes from the caching allocator on the execution
                    # stream, so reuse is ordered after this call's kernels.
                    with torch.cuda.stream(stream) if stream is not None else nullcontext():
                        scratch = torch.empty((nbytes,), dtype=torch.uint8, device=device)
                    address = scratch.data_ptr()
                    if nbytes > total:
                        total = nbytes
                launch = self._launches.get(key)
                if launch is None:
                    report = _native.Report()
                    call(address, nbytes, on, report)
                    if len(self._launches) >= 256:
                        self._launches.clear()
                    launch = self._launches[key] = _Launch(report)
                else:
                    call(address, nbytes, on, None)
                launches += (launch,)
                if checked and launch.status_offset >= 0:
                    self._check_status_words(scratch, launch, active, torch)
        return self._report(started, launches, total, validation)

    def _status_words(self, launch) -> int:
        """Words at a report's status_offset (CompiledProgram's: one)."""
        return 1

    def _check_status_words(self, scratch, launch, active, torch):
        """Checked mode, after the launch: the words in which a bounded wait
        that gave up says so."""
        with torch.cuda.stream(active):
            words = scratch.narrow(0, launch.status_offset, 8 * self._status_words(launch)).view(torch.int64).cpu()
        if words.any():
            raise RuntimeError("a bounded wait inside the kernel gave up; the call's results are undefined")

    def _report(self, started, launches, nbytes, validation) -> ExecutionReport:
        """The call's report: what depends on its launches alone is kept, as
        filling all the fields costs a good part of a small call."""
        template = self._reports.get(launches) if validation is None else None
        if template is None:
            check, check_ms = validation if validation is not None else (None, None)
            parts = (_Launch(check),) + launches if check is not None else launches
            checked_bytes = STATUS_BYTES if check is not None else 0
            last = launches[-1] if launches else None
            template = ExecutionReport(("rows",) if launches else (), (), sum((x.grids for x in parts), ()),
                                       nbytes + checked_bytes, self._digest, None,
                                       "checked" if check is not None else "validated",
                                       sum((x.names for x in parts), ()), cache_hit=self.cache_hit,
                                       validation_workspace_bytes=checked_bytes, validation_host_ms=check_ms,
                                       d_tile=last.d_tile if last else None, d_vector=last.d_vector if last else 1,
                                       selected=self.spec.op).__dict__
            if check is None:
                if len(self._reports) >= 256:
                    self._reports.clear()
                self._reports[launches] = template
        report = object.__new__(ExecutionReport)
        report.__dict__.update(template, workspace_bytes=nbytes + template["validation_workspace_bytes"],
                               host_enqueue_ms=(time.perf_counter() - started) * 1000)
        return report


class _Launch:
    """What a call launched, from the library's report."""

    __slots__ = ("names", "grids", "d_tile", "d_vector", "status_offset")

    def __init__(self, report):
        count = report.num_launches
        self.names = tuple(_native.kernel_name(report.kernel_ids[i]) for i in range(count))
        self.grids = tuple(tuple(report.grid[i]) for i in range(count))
        self.d_tile, self.d_vector = int(report.d_tile), int(report.d_vector)
        self.status_offset = int(report.status_offset)


def _address(tensor) -> int:
    return 0 if tensor is None else tensor.data_ptr()


def _alignment(pointers) -> tuple:
    """What of the addresses decides how a call runs."""
    return tuple(p % 16 for p in pointers)


class CompiledScan(_LayerProgram):
    """out[t] = gates[t] * out[t - 1] + values[t] within each segment."""

    kind = ScanSpec

    def carry_rows(self, n: int) -> int:
        """Rows of the ``carries`` that a call over ``n`` rows records."""
        return (n + CARRY_ROWS - 1) // CARRY_ROWS

    def _scratch(self, n, b) -> int:
        return self._cached((n, b), lambda: _native.scan_workspace_bytes(
            self.spec.dtype, self.spec.offsets_dtype, self.spec.feature_dim, n, b))

    def run(self, values, gates, offsets, out, stream=None, mode: str = "validated", *, initial=None, final=None,
            carries=None) -> ExecutionReport:
        """Writes ``out`` [N, D] and, where given, ``final`` (f32 [B, D], the
        state after each segment) and ``carries`` (f32 [carry_rows(N), D],
        what ``run_backward`` needs).  ``initial`` (f32 [B, D]) is the state
        before each segment; without it a segment's first row is its first
        value.  ``values``, ``gates`` and ``out`` have the program's dtype;
        outputs overlap nothing."""
        return self._run(values, gates, offsets, out, initial, final, carries, stream, mode, True)

    def _run(self, values, gates, offsets, out, initial, final, carries, stream, mode, gradless, clear_rest=False):
        torch = _torch()
        spec, d = self.spec, self.spec.feature_dim
        b, n = self._segments(torch, offsets), self._rows(values, torch)
        dtype = torch.float32 if spec.dtype == "f32" else torch.bfloat16
        tensors = [("values", values, (n, d), dtype), ("gates", gates, (n, d), dtype), ("out", out, (n, d), dtype)]
        if initial is not None:
            tensors.append(("initial", initial, (b, d), torch.float32))
        if final is not None:
            tensors.append(("final", final, (b, d), torch.float32))
        if carries is not None:
            tensors.append(("carries", carries, (self.carry_rows(n), d), torch.float32))
        self._tensors(torch, tensors, offsets, mode, gradless)
        pointers = (values.data_ptr(), gates.data_ptr(), offsets.data_ptr(), _address(initial), out.data_ptr(),
                    _address(final), _address(carries))

        def call(scratch, nbytes, on, report):
            _native.scan(spec.dtype, spec.offsets_dtype, d, n, b, pointers, scratch, nbytes, on, report, clear_rest)

        return self._launch(torch, offsets, n, b, stream, mode, [t[1] for t in tensors] + [offsets],
                            (((False, n, b) + _alignment(pointers), self._scratch(n, b), call),))

    def run_backward(self, values, gates, offsets, carries, grad_out, stream=None, mode: str = "validated", *,
                     initial=None, grad_final=None, grad_values=None, grad_gates=None,
                     grad_initial=None) -> ExecutionReport:
        """Gradients of a ``run`` that recorded ``carries``, from those of its
        outputs (``grad_final`` f32 [B, D]; None: zero).  Writes those of
        ``grad_values``, ``grad_gates`` [N, D] and ``grad_initial`` (f32
        [B, D], with ``initial``) that are given."""
        return self._run_backward(values, gates, offsets, carries, grad_out, stream, mode, initial, grad_final,
                                  grad_values, grad_gates, grad_initial)

    def _run_backward(self, values, gates, offsets, carries, grad_out, stream, mode, initial, grad_final, grad_values,
                      grad_gates, grad_initial, clear_rest=False):
        torch = _torch()
        spec, d = self.spec, self.spec.feature_dim
        b, n = self._segments(torch, offsets), self._rows(values, torch)
        dtype = torch.float32 if spec.dtype == "f32" else torch.bfloat16
        if grad_initial is not None and initial is None:
            raise ValidationError("grad_initial needs initial")
        rows = [("values", values, (n, d), dtype), ("gates", gates, (n, d), dtype),
                ("carries", carries, (self.carry_rows(n), d), torch.float32), ("grad_out", grad_out, (n, d), dtype),
                ("initial", initial, (b, d), torch.float32), ("grad_final", grad_final, (b, d), torch.float32),
                ("grad_values", grad_values, (n, d), dtype), ("grad_gates", grad_gates, (n, d), dtype),
                ("grad_initial", grad_initial, (b, d), torch.float32)]
        tensors = rows[:4] + [row for row in rows[4:] if row[1] is not None]
        self._tensors(torch, tensors, offsets, mode, False)
        return self._gradients(torch, values, gates, offsets, carries, grad_out, stream, mode, initial, grad_final,
                               grad_values, grad_gates, grad_initial, clear_rest)

    def _gradients(self, torch, values, gates, offsets, carries, grad_out, stream, mode, initial, grad_final,
                   grad_values, grad_gates, grad_initial, clear_rest):
        """``run_backward`` of tensors that are known to fit."""
        spec, d, n, b = self.spec, self.spec.feature_dim, values.shape[0], offsets.numel() - 1
        pointers = (values.data_ptr(), gates.data_ptr(), offsets.data_ptr(), _address(initial), carries.data_ptr(),
                    grad_out.data_ptr(), _address(grad_final), _address(grad_values), _address(grad_gates),
                    _address(grad_initial))

        def call(scratch, nbytes, on, report):
            _native.scan_backward(spec.dtype, spec.offsets_dtype, d, n, b, pointers, scratch, nbytes, on, report,
                                  clear_rest)

        used = [t for t in (values, gates, offsets, carries, grad_out, initial, grad_final, grad_values, grad_gates,
                            grad_initial) if t is not None] if stream is not None else ()
        return self._launch(torch, offsets, n, b, stream, mode, used,
                            (((True, n, b) + _alignment(pointers), self._scratch(n, b), call),))


class CompiledMatmul(_LayerProgram):
    """out[t] = values[t] @ weights[s] for the rows t of segment s."""

    kind = MatmulSpec

    def _status_words(self, launch) -> int:
        """One for each CTA of the tensor-core launch (before it operands may be
        packed, after it parts be summed)."""
        return next(grid[0] for name, grid in zip(launch.names, launch.grids)
                    if name in ("matmul_tensor", "matmul_pair"))

    def _product(self, kind, left, right, offsets, out, n, b, clear_rest):
        """(key, scratch bytes, call) of one product."""
        spec = self.spec
        shape = (kind, spec.dtype, spec.offsets_dtype, spec.feature_dim, spec.out_dim, n, b)
        left, right = left.data_ptr(), right.data_ptr()
        pointers = (left, right, offsets.data_ptr(), out.data_ptr())
        key = (kind, n, b) + _alignment(pointers)
        nbytes = self._cached(key, lambda: _native.matmul_workspace_bytes(*shape, left, right))
        return key, nbytes, lambda scratch, size, on, report: _native.matmul(*shape, *pointers, scratch, size, on,
                                                                             report, clear_rest)

    def run(self, values, weights, offsets, out, stream=None, mode: str = "validated") -> ExecutionReport:
        """Writes ``out`` [N, out_dim] from ``values`` [N, feature_dim] and
        ``weights`` [B, feature_dim, out_dim]; all of the program's dtype and
        contiguous.  ``out`` overlaps nothing."""
        return self._run(values, weights, offsets, out, stream, mode, True)

    def _run(self, values, weights, offsets, out, stream, mode, gradless, clear_rest=False):
        torch = _torch()
        k, m = self.spec.feature_dim, self.spec.out_dim
        b, n = self._segments(torch, offsets), self._rows(values, torch)
        dtype = torch.float32 if self.spec.dtype == "f32" else torch.bfloat16
        tensors = (("values", values, (n, k), dtype), ("weights", weights, (b, k, m), dtype), ("out", out, (n, m), dtype))
        self._tensors(torch, tensors, offsets, mode, gradless)
        return self._launch(torch, offsets, n, b, stream, mode, (values, weights, offsets, out),
                            (self._product("forward", values, weights, offsets, out, n, b, clear_rest),))

    def run_backward(self, values, weights, offsets, grad_out, stream=None, mode: str = "validated", *,
                     grad_values=None, grad_weights=None) -> ExecutionReport:
        """Gradients of ``run`` from that of ``out``: those of ``grad_values``
        and ``grad_weights`` that are given (zero for the weights of a segment
        without rows)."""
        return self._run_backward(values, weights, offsets, grad_out, stream, mode, grad_values, grad_weights)

    def _run_backward(self, values, weights, offsets, grad_out, stream, mode, grad_values, grad_weights,
                      clear_rest=False):
        torch = _torch()
        k, m = self.spec.feature_dim, self.spec.out_dim
        b, n = self._segments(torch, offsets), self._rows(values, torch)
        dtype = torch.float32 if self.spec.dtype == "f32" else torch.bfloat16
        tensors = [("values", values, (n, k), dtype), ("weights", weights, (b, k, m), dtype),
                   ("grad_out", grad_out, (n, m), dtype)]
        if grad_values is not None:
            tensors.append(("grad_values", grad_values, (n, k), dtype))
        if grad_weights is not None:
            tensors.append(("grad_weights", grad_weights, (b, k, m), dtype))
        self._tensors(torch, tensors, offsets, mode, False)
        return self._gradients(torch, values, weights, offsets, grad_out, stream, mode, grad_values, grad_weights,
                               clear_rest)

    def _gradients(self, torch, values, weights, offsets, grad_out, stream, mode, grad_values, grad_weights, clear_rest):
        """``run_backward`` of tensors that are known to fit."""
        n, b = values.shape[0], offsets.numel() - 1
        work = []
        if grad_values is not None:
            work.append(self._product("grad_values", grad_out, weights, offsets, grad_values, n, b, clear_rest))
        if grad_weights is not None:
            work.append(self._product("grad_weights", values, grad_out, offsets, grad_weights, n, b, False))
        used = [t for t in (values, weights, offsets, grad_out, grad_values, grad_weights) if t is not None]
        return self._launch(torch, offsets, n, b, stream, mode, used, work)
