"""8-bit integer linear: row quantisation, RMS norm with an 8-bit output, and
the product of the codes.

A quantised matrix is a pair of 8-bit codes and FP32 scales, one for each row:
a token of the activations, an output channel of the weight.  The value of a
code is ``code * scale``; codes are symmetric, ``round(127 x / max|x|)``.

* ``quantize_rows(x)`` -- codes and scales of BF16, FP16 or FP32 rows;
* ``rms_norm_int8(x, weight, residual, eps)`` -- adds the residual, normalises
  and quantises in one pass, and returns the new residual;
* ``linear_int8(codes, scales, weight_codes, weight_scales, bias)`` -- the
  linear, exact 32-bit sums scaled once;
* ``Int8Plan`` -- a plan in the manner of ``runtime.Rank7Plan``: packs a
  weight once, keeps a workspace, runs ``x -> codes -> product`` and
  ``x, residual -> norm -> codes -> product``;
* ``torch.ops.rdna3_fastmm.{quantize_rows_int8, rms_norm_int8, linear_int8}``.

Code rows start on 16-byte boundaries: a ``[rows, K]`` tensor of codes made
here is a view of ``[rows, round_up(K, 16)]`` storage.  Calls are queued on the
current stream of the operands' device; with buffers given for their outputs
they allocate nothing and capture into CUDA graphs; autograd sees such buffers as
changed in place.  The operators do not support autograd themselves: an operand
that requires a gradient is refused while gradients are enabled, one with a
forward-mode tangent always, and ``torch.func`` transforms are refused too.  The
reference has no quantised operator.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import NamedTuple, Optional

import torch
from torch._functorch import eager_transforms
from torch.autograd import forward_ad

from . import _native
from .runtime import _LinearPlan, _round_up

__all__ = [
    "Int8Rows",
    "NormedInt8Rows",
    "Int8PackedWeight",
    "Int8Workspace",
    "Int8Plan",
    "quantize_rows",
    "rms_norm_int8",
    "linear_int8",
    "empty_codes",
]

CODE_ALIGNMENT = 16
_INF = float("inf")
MAX_INNER = 131071  # 2^14 a product of two codes of -128, sums below 2^31
_HALF_TYPES = (torch.bfloat16, torch.float16)


class Int8Rows(NamedTuple):
    codes: torch.Tensor  # int8, [..., K]
    scales: torch.Tensor  # float32, [...]


class NormedInt8Rows(NamedTuple):
    codes: torch.Tensor
    scales: torch.Tensor
    residual: torch.Tensor | None  # x + residual in x's type; None without a residual


def empty_codes(shape: tuple[int, ...], device: torch.device) -> torch.Tensor:
    """Uninitialised codes of ``shape`` whose rows start on 16-byte boundaries."""
    inner = shape[-1]
    pitch = _round_up(inner, CODE_ALIGNMENT)
    storage = torch.empty((*shape[:-1], pitch), device=device, dtype=torch.int8)
    return storage if pitch == inner else storage[..., :inner]


# ---------------------------------------------------------------- operands
# A call between two single tokens is a few microseconds of GPU time, so the
# checks below read each tensor's attributes once and pass plain integers on.
_BF16, _FP16, _FP32, _INT8 = torch.bfloat16, torch.float16, torch.float32, torch.int8
_grad_enabled = torch.is_grad_enabled
_current_device = torch._C._cuda_getDevice
_current_stream = torch._C._cuda_getCurrentRawStream
_mark_written = torch._C._increment_version  # of buffers given, as by any operator that writes in place
_ROW_TYPES = {torch.bfloat16: _native.FMM_DTYPE_BF16, torch.float16: _native.FMM_DTYPE_F16,
              torch.float32: _native.FMM_DTYPE_F32}


# A tensor as rows: (address, count, length and step in elements, element size)
_Rows = tuple[int, int, int, int, int]


def _flat(tensor: torch.Tensor) -> tuple[int, int, int] | None:
    """(rows, inner, pitch) where the leading dimensions are rows a constant
    step apart and the last dimension is dense, else None."""
    shape = tensor.shape
    inner = shape[-1]
    if inner and tensor.is_contiguous():
        rows = shape[0] if len(shape) == 2 else tensor.numel() // inner
        # a single row has no second one to reach
        return rows, inner, inner if rows > 1 else (inner + 15) & -16
    rows, pitch, step = 1, None, None
    for size, stride in zip(reversed(shape[:-1]), reversed(tensor.stride()[:-1])):
        if size == 1:
            continue
        if pitch is None:
            pitch = stride
        elif stride != step:
            return None
        rows *= size
        step = stride * size
    if inner > 1 and tensor.stride(-1) != 1:
        return None
    if rows <= 1:
        pitch = (inner + 15) & -16
    elif pitch < inner:
        return None
    return rows, inner, pitch


def _input_rows(tensor: torch.Tensor) -> tuple[torch.Tensor, _Rows]:
    """The rows, and the tensor that holds them (a copy where they had to be made dense)."""
    flat = _flat(tensor)
    if flat is None:
        tensor = tensor.contiguous()
        flat = _flat(tensor)
    return tensor, (tensor.data_ptr(), *flat, tensor.element_size())


def _touched_rows(tensor: torch.Tensor) -> _Rows:
    """The rows of a tensor where it lies, for checks of overlap: of one whose
    rows are not dense, rows that hold its elements (no copy is made)."""
    flat = _flat(tensor)
    if flat is None:
        *inside, (pitch, rows) = sorted((stride, size) for size, stride in zip(tensor.shape, tensor.stride()) if size != 1)
        inner = 1 + sum(stride * (size - 1) for stride, size in inside)
        if pitch < inner:
            rows, inner = min(rows, 1), inner + pitch * (rows - 1)
            pitch = inner
        flat = rows if tensor.numel() else 0, inner, pitch
    return tensor.data_ptr(), *flat, tensor.element_size()


def _output_rows(tensor: torch.Tensor, shape: torch.Size, dtype: torch.dtype, device: int, name: str,
                 like: _Rows | None = None) -> _Rows:
    if tensor.shape != shape:
        raise ValueError(f"{name} has shape {tuple(tensor.shape)}, expected {tuple(shape)}")
    if tensor.get_device() != device or tensor.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype} on cuda:{device}")
    if like is not None and tensor.is_contiguous():
        _, rows, inner, _, _ = like
        return tensor.data_ptr(), rows, inner, inner if rows > 1 else (inner + 15) & -16, dtype.itemsize
    flat = _flat(tensor)
    if flat is None:
        raise ValueError(f"{name} must have dense rows a constant step apart")
    return tensor.data_ptr(), *flat, dtype.itemsize


def _like(tensor: torch.Tensor, rows: _Rows) -> _Rows | None:
    """Rows of a dense tensor with the shape of an operand whose rows are known."""
    if not tensor.is_contiguous():
        return None
    _, count, inner, _, _ = rows
    return tensor.data_ptr(), count, inner, inner if count > 1 else (inner + 15) & -16, tensor.element_size()


def _input_scales(tensor: torch.Tensor, shape: torch.Size, device: int, name: str) -> torch.Tensor:
    if tensor.shape != shape:
        raise ValueError(f"{name} has shape {tuple(tensor.shape)}, expected {tuple(shape)}")
    if tensor.get_device() != device or tensor.dtype is not _FP32:
        raise ValueError(f"{name} must be float32 on cuda:{device}")
    return tensor if tensor.is_contiguous() else tensor.contiguous()


def _output_scales(tensor: torch.Tensor, shape: torch.Size, device: int) -> None:
    if tensor.shape != shape:
        raise ValueError(f"scales has shape {tuple(tensor.shape)}, expected {tuple(shape)}")
    if tensor.get_device() != device or tensor.dtype is not _FP32 or not tensor.is_contiguous():
        raise ValueError(f"scales must be contiguous float32 on cuda:{device}")


def _refuse_unread(*tensors: torch.Tensor | None) -> None:
    """Refuse what the storage alone does not hold: a gradient to come, a
    forward-mode tangent, the other sign of a lazily negated view (``z.conj().imag``)."""
    grad = _grad_enabled()
    for tensor in tensors:
        if tensor is not None:
            if grad and tensor.requires_grad:
                raise ValueError("the B200 8-bit operators do not support autograd")
            if tensor.is_neg():
                raise ValueError("lazily negated views must be resolved (torch.resolve_neg) first")
    if forward_ad._current_level >= 0:
        for tensor in tensors:
            if tensor is not None and forward_ad.unpack_dual(tensor).tangent is not None:
                raise ValueError("the B200 8-bit operators do not support autograd")


def _refuse_transforms() -> None:
    """Of the torch operators: ``torch.func.jvp`` takes the tangents off before they get here."""
    if eager_transforms.JVP_NESTING > 0:
        raise ValueError("the B200 8-bit operators do not support torch.func.jvp")


def _require_cuda(tensor: torch.Tensor, name: str) -> int:
    device = tensor.get_device()
    if device < 0 or not tensor.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    return device


def _rows_overlap(a: _Rows, b: _Rows) -> bool:
    """Whether two row operands share a byte."""
    ptr_a, rows_a, inner_a, pitch_a, size_a = a
    ptr_b, rows_b, inner_b, pitch_b, size_b = b
    if rows_a == 0 or rows_b == 0:
        return False
    width_a, width_b = inner_a * size_a, inner_b * size_b
    step_a, step_b = pitch_a * size_a, pitch_b * size_b
    if ptr_a >= ptr_b + (rows_b - 1) * step_b + width_b or ptr_b >= ptr_a + (rows_a - 1) * step_a + width_a:
        return False
    if rows_a > 1 and rows_b > 1 and step_a == step_b:
        # columns of one buffer: apart if their byte ranges within a step are
        offset = (ptr_b - ptr_a) % step_a
        return offset < width_a or offset + width_b > step_a
    return True


def _row_vector(tensor: torch.Tensor) -> _Rows:
    n = tensor.numel()
    return tensor.data_ptr(), 1 if n else 0, n, n, tensor.element_size()


def _same_rows(a: _Rows, b: _Rows) -> bool:
    return a[0] == b[0] and a[3] == b[3]


def _all_apart(operands: list[_Rows]) -> bool:
    """Whether no operand's address range touches another's: the common case, decided by one sort."""
    operands.sort()
    reach = 0
    for ptr, rows, inner, pitch, itemsize in operands:
        if ptr < reach:
            return False
        if rows:
            reach = ptr + ((rows - 1) * pitch + inner) * itemsize
    return True


def _refuse_overlap(outputs: list[_Rows], inputs: list[_Rows]) -> None:
    if _all_apart(outputs + inputs):
        return
    for i, out in enumerate(outputs):
        for other in outputs[i + 1:] + inputs:
            if _rows_overlap(out, other):
                raise ValueError("output storage must not overlap inputs or other outputs")


_entry_points: dict = {}


def _entry_point(name: str):
    return _entry_points.setdefault(name, _native.entry_point(name))


def _launch(device: int, name: str, *args) -> None:
    """Call the C entry point with ``device`` current, on its current stream."""
    function = _entry_points.get(name) or _entry_point(name)
    if device == _current_device():
        code = function(*args, _current_stream(device))
    else:
        with torch.cuda.device(device):
            code = function(*args, _current_stream(device))
    if code:
        _native.check(code, name)


# ---------------------------------------------------------------- operators
def quantize_rows(x: torch.Tensor, *, codes: torch.Tensor | None = None,
                  scales: torch.Tensor | None = None) -> Int8Rows:
    """8-bit codes and scales of the rows ``x[..., K]`` (BF16, FP16 or FP32).

    ``codes[..., k] = round_half_even(127 x[..., k] / a)`` and ``scales = a / 127``
    with ``a`` the row's largest magnitude.  A row of zeros has scale 0; a row
    with an infinity or a NaN has codes 0 and scale NaN.  ``codes`` and
    ``scales`` are written and returned where given."""
    device = _require_cuda(x, "x")
    dtype = _ROW_TYPES.get(x.dtype)
    if dtype is None:
        raise ValueError(f"the 8-bit operators take BF16, FP16 or FP32 rows, not {x.dtype}")
    shape = x.shape
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError("x must have a last dimension of at least one element")
    _refuse_unread(x, codes, scales)
    held, source = _input_rows(x)
    leading = shape[:-1]
    given = ()
    if codes is None:
        codes = empty_codes(shape, x.device)
    else:
        given = (codes,)
    if scales is None:
        scales = torch.empty(leading, device=x.device, dtype=torch.float32)
    else:
        given += (scales,)
    q = _output_rows(codes, shape, _INT8, device, "codes", source)
    _output_scales(scales, leading, device)
    rows = source[1]
    s = scales.data_ptr(), 1 if rows else 0, rows, rows, 4
    _refuse_overlap([q, s], [source])
    if rows:
        _launch(device, "fmm_quantize_rows", dtype, *source[:4], q[0], q[3], s[0])
        if given:
            _mark_written(given)
    return Int8Rows(codes, scales)


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-6, *,
                  codes: torch.Tensor | None = None, scales: torch.Tensor | None = None,
                  residual_out: torch.Tensor | None = None) -> NormedInt8Rows:
    """RMS norm of ``h = x + residual`` with an 8-bit output.

    ``h`` is rounded to ``x``'s type (BF16 or FP16), returned as the new
    residual, and read by the norm; ``y = h * weight / sqrt(mean(h^2) + eps)``
    is quantised unrounded as by ``quantize_rows``.  A row has codes 0 and scale
    NaN where a value, its square or its gain is not finite in FP32, or the
    scale is beyond FP32.  ``weight[K]`` has ``x``'s type or FP32.  ``residual_out`` may be ``residual`` or ``x`` itself, which
    updates the stream in place."""
    device = _require_cuda(x, "x")
    kind = x.dtype
    if kind is not _BF16 and kind is not _FP16:
        raise ValueError(f"rms_norm_int8 takes BF16 or FP16 rows, not {kind}")
    shape = x.shape
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError("x must have a last dimension of at least one element")
    if weight.shape != shape[-1:]:
        raise ValueError(f"weight has shape {tuple(weight.shape)}, expected {tuple(shape[-1:])}")
    gain_kind = weight.dtype
    if weight.get_device() != device or (gain_kind is not kind and gain_kind is not _FP32):
        raise ValueError("weight must have x's dtype or float32, on x's device")
    if not 0.0 <= eps < _INF:
        raise ValueError("eps must be finite and not negative")
    if residual is None and residual_out is not None:
        raise ValueError("residual_out needs a residual")
    _refuse_unread(x, weight, residual, codes, scales, residual_out)
    held, source = _input_rows(x)
    if not weight.is_contiguous():
        weight = weight.contiguous()
    ptr, rows, inner, pitch, _ = source
    gain = weight.data_ptr(), 1, inner, inner, 4 if gain_kind is _FP32 else 2
    leading = shape[:-1]
    given = () if residual_out is None else (residual_out,)
    if codes is None:
        codes = empty_codes(shape, x.device)
    else:
        given += (codes,)
    if scales is None:
        scales = torch.empty(leading, device=x.device, dtype=torch.float32)
    else:
        given += (scales,)
    q = _output_rows(codes, shape, _INT8, device, "codes", source)
    _output_scales(scales, leading, device)
    s = scales.data_ptr(), 1 if rows else 0, rows, rows, 4
    if residual is None:
        _refuse_overlap([q, s], [source, gain])
        if rows:
            _launch(device, "fmm_rms_norm_int8", _ROW_TYPES[kind], _ROW_TYPES[gain_kind], ptr, pitch, None, 0, gain[0],
                    rows, inner, eps, None, 0, q[0], q[3], s[0])
            if given:
                _mark_written(given)
        return NormedInt8Rows(codes, scales, None)
    if residual.shape != shape or residual.dtype is not kind or residual.get_device() != device:
        raise ValueError("residual must have x's shape, dtype and device")
    held_residual, added = residual, _like(residual, source)
    if added is None:
        held_residual, added = _input_rows(residual)
    if residual_out is None:
        residual_out = torch.empty(shape, device=x.device, dtype=kind)
    stream = _output_rows(residual_out, shape, kind, device, "residual_out", source)
    if not _all_apart([q, s, stream, source, gain, added]):
        for other in (source, added):
            if not _same_rows(stream, other) and _rows_overlap(stream, other):
                raise ValueError("residual_out must be residual, x or storage of its own")
        _refuse_overlap([stream], [gain, q, s])
        _refuse_overlap([q, s], [source, gain, added])
    if rows:
        _launch(device, "fmm_rms_norm_int8", _ROW_TYPES[kind], _ROW_TYPES[gain_kind], ptr, pitch, added[0], added[3],
                gain[0], rows, inner, eps, stream[0], stream[3], q[0], q[3], s[0])
        if given:
            _mark_written(given)
    return NormedInt8Rows(codes, scales, residual_out)


def linear_int8(codes: torch.Tensor, scales: torch.Tensor, weight_codes: torch.Tensor, weight_scales: torch.Tensor,
                bias: torch.Tensor | None = None, *, dtype: torch.dtype | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """``(codes * scales) @ (weight_codes * weight_scales).T + bias``.

    ``codes[..., K]`` with ``scales[...]``, ``weight_codes[N, K]`` with
    ``weight_scales[N]``; the output ``[..., N]`` is BF16 or FP16 (``dtype``,
    or ``out``'s or ``bias``'s; BF16 where none says).  Products are summed
    exactly in 32-bit integers (``K`` up to 131071), scaled and biased in FP32
    and rounded once.  Code rows must start on 16-byte boundaries, as
    ``quantize_rows``, ``rms_norm_int8`` and ``empty_codes`` make them."""
    device = _require_cuda(codes, "codes")
    if (codes.dtype is not _INT8 or weight_codes.dtype is not _INT8
            or weight_codes.get_device() != device):
        raise ValueError("codes and weight_codes must be int8 tensors of one device")
    token_shape, weight_shape = codes.shape, weight_codes.shape
    if len(token_shape) < 1 or len(weight_shape) != 2 or token_shape[-1] != weight_shape[1]:
        raise ValueError("codes and weight_codes shapes do not form a linear")
    columns, inner = weight_shape
    if columns < 1 or inner < 1:
        raise ValueError("matrix dimensions must be positive")
    if inner > MAX_INNER:
        raise ValueError(f"K = {inner} could leave the 32-bit sum (at most {MAX_INNER})")
    if dtype is None:
        dtype = out.dtype if out is not None else bias.dtype if bias is not None else torch.bfloat16
    if dtype is not _BF16 and dtype is not _FP16:
        raise ValueError(f"linear_int8 writes BF16 or FP16, not {dtype}")
    _refuse_unread(codes, scales, weight_codes, weight_scales, bias, out)
    q, w = _flat(codes), _flat(weight_codes)
    if q is None or w is None:
        raise ValueError("codes must have dense rows a constant step apart")
    leading = token_shape[:-1]
    scales = _input_scales(scales, leading, device, "scales")
    weight_scales = _input_scales(weight_scales, weight_shape[:1], device, "weight_scales")
    if bias is not None:
        if bias.shape != weight_shape[:1] or bias.dtype is not dtype or bias.get_device() != device:
            raise ValueError(f"bias must be {dtype} [N] on the codes' device")
        if not bias.is_contiguous():
            bias = bias.contiguous()
    rows, _, pitch = q
    ptr, weight_ptr, bias_ptr = codes.data_ptr(), weight_codes.data_ptr(), None if bias is None else bias.data_ptr()
    scales_ptr, weight_scales_ptr = scales.data_ptr(), weight_scales.data_ptr()
    given = out
    if out is None:
        out = torch.empty((*leading, columns), device=codes.device, dtype=dtype)
        result_ptr, result_pitch = out.data_ptr(), columns if rows > 1 else (columns + 15) & -16
    else:
        result = _output_rows(out, torch.Size((*leading, columns)), dtype, device, "out")
        result_ptr, result_pitch = result[0], result[3]
        inputs = [(ptr, *q, 1), (weight_ptr, *w, 1), (scales_ptr, 1, rows, rows, 4),
                  (weight_scales_ptr, 1, columns, columns, 4)]
        if bias_ptr is not None:
            inputs.append((bias_ptr, 1, columns, columns, 2))
        if rows and not _all_apart([result, *inputs]):
            _refuse_overlap([result], inputs)
    if rows:
        _launch(device, "fmm_linear_int8", _ROW_TYPES[dtype], ptr, pitch, scales_ptr, weight_ptr, w[2],
                weight_scales_ptr, bias_ptr, result_ptr, result_pitch, rows, inner, columns)
        if given is not None:
            _mark_written((given,))
    return out


# ---------------------------------------------------------------- plan
@dataclass
class Int8Workspace:
    algorithm: str
    output_dtype: torch.dtype
    codes: torch.Tensor  # [rows, K] of 16-byte aligned rows
    scales: torch.Tensor  # [rows]


@dataclass(frozen=True)
class Int8PackedWeight:
    algorithm: str
    source_dtype: torch.dtype
    codes: torch.Tensor  # [N, K] of 16-byte aligned rows
    scales: torch.Tensor  # [N]
    source_shape: tuple[int, int]


class Int8Plan:
    """8-bit linear of ``rows x inner`` inputs and a ``columns x inner`` weight,
    used as the reduced-rank plans are: pack the weight once, keep a workspace,
    run.  A packed weight serves plans of any row count; two streams (or two
    captured graphs that may run together) need a workspace each."""

    algorithm = "int8-v1"
    _ensure_memory_budget = _LinearPlan._ensure_memory_budget

    def __init__(self, rows: int, inner: int, columns: int, device: torch.device,
                 dtype: torch.dtype = torch.bfloat16) -> None:
        device = torch.device(device)
        if device.type != "cuda" or torch.version.cuda is None or not torch.cuda.is_available():
            raise ValueError("the B200 backend requires a CUDA sm_100 device")
        if dtype not in _HALF_TYPES:
            raise ValueError(f"{self.algorithm} does not support {dtype} inputs")
        if min(rows, inner, columns) < 1:
            raise ValueError("matrix dimensions must be positive")
        if inner > MAX_INNER:
            raise ValueError(f"K = {inner} could leave the 32-bit sum (at most {MAX_INNER})")
        index = torch.cuda.current_device() if device.index is None else device.index
        self.device = torch.device("cuda", index)
        self.dtype = dtype
        self.rows, self.inner, self.columns = rows, inner, columns

    @property
    def workspace_bytes(self) -> int:
        return self.rows * (_round_up(self.inner, CODE_ALIGNMENT) + 4)

    @property
    def packed_weight_bytes(self) -> int:
        return self.columns * (_round_up(self.inner, CODE_ALIGNMENT) + 4)

    def allocate_workspace(self, max_free_memory_fraction: float = 0.75) -> Int8Workspace:
        self._ensure_memory_budget(self.workspace_bytes, max_free_memory_fraction, f"{self.algorithm} workspace")
        return Int8Workspace(self.algorithm, self.dtype, empty_codes((self.rows, self.inner), self.device),
                             torch.empty((self.rows,), device=self.device, dtype=torch.float32))

    def pack_weight(self, weight: torch.Tensor, max_free_memory_fraction: float = 0.75) -> Int8PackedWeight:
        """Quantise ``weight[N, K]`` (the plan's type or FP32) once, a scale for
        each output channel, into an immutable snapshot."""
        if tuple(weight.shape) != (self.columns, self.inner):
            raise ValueError(f"weight matrix has shape {tuple(weight.shape)}, "
                             f"expected {(self.columns, self.inner)}")
        if weight.device != self.device or weight.dtype not in (self.dtype, torch.float32):
            raise ValueError("weight matrix device or dtype does not match the plan")
        self._ensure_memory_budget(self.packed_weight_bytes, max_free_memory_fraction,
                                   f"{self.algorithm} packed Linear weight")
        codes, scales = quantize_rows(weight)
        return Int8PackedWeight(self.algorithm, self.dtype, codes, scales, (self.columns, self.inner))

    def run_linear_packed(self, input_tensor: torch.Tensor, weight: Int8PackedWeight, workspace: Int8Workspace,
                          bias: torch.Tensor | None = None, output: torch.Tensor | None = None) -> torch.Tensor:
        """``F.linear(input, weight, bias)``: tokens to codes, codes to output."""
        self._validate_input(input_tensor)
        self._validate_packed(weight)
        self._validate_workspace(workspace)
        self._validate_product(workspace, weight, bias, output)
        self._refuse_output(output, input_tensor)
        quantize_rows(input_tensor, codes=workspace.codes, scales=workspace.scales)
        return linear_int8(workspace.codes, workspace.scales, weight.codes, weight.scales, bias, dtype=self.dtype,
                           out=output)

    def run_norm_linear_packed(self, input_tensor: torch.Tensor, norm_weight: torch.Tensor, weight: Int8PackedWeight,
                               workspace: Int8Workspace, residual: torch.Tensor | None = None, eps: float = 1e-6,
                               bias: torch.Tensor | None = None, output: torch.Tensor | None = None,
                               residual_output: torch.Tensor | None = None,
                               ) -> tuple[torch.Tensor, torch.Tensor | None]:
        """``F.linear(rms_norm(input + residual), weight, bias)`` and the new
        residual (``None`` without one)."""
        self._validate_input(input_tensor)
        self._validate_packed(weight)
        self._validate_workspace(workspace)
        self._validate_product(workspace, weight, bias, output)
        self._refuse_output(output, input_tensor, norm_weight, residual, residual_output)
        self._refuse_output(residual_output, weight.codes, weight.scales, bias)
        stream = rms_norm_int8(input_tensor, norm_weight, residual, eps, codes=workspace.codes,
                               scales=workspace.scales, residual_out=residual_output).residual
        result = linear_int8(workspace.codes, workspace.scales, weight.codes, weight.scales, bias, dtype=self.dtype,
                             out=output)
        return result, stream

    # ------------------------------------------------------------------ checks
    def _validate_input(self, tensor: torch.Tensor) -> None:
        if tuple(tensor.shape) != (self.rows, self.inner):
            raise ValueError(f"left matrix has shape {tuple(tensor.shape)}, expected {(self.rows, self.inner)}")
        if tensor.device != self.device or tensor.dtype != self.dtype:
            raise ValueError("left matrix device or dtype does not match the plan")

    def _validate_packed(self, packed: Int8PackedWeight) -> None:
        if (not isinstance(packed, Int8PackedWeight) or packed.algorithm != self.algorithm
                or packed.source_dtype != self.dtype or packed.codes.device != self.device):
            raise ValueError("packed Linear weight does not match the plan")
        if packed.source_shape != (self.columns, self.inner) or tuple(packed.codes.shape) != packed.source_shape:
            raise ValueError("packed Linear weight shape does not match the plan")

    def _validate_workspace(self, workspace: Int8Workspace) -> None:
        if (not isinstance(workspace, Int8Workspace) or workspace.algorithm != self.algorithm
                or workspace.output_dtype != self.dtype or workspace.codes.device != self.device
                or tuple(workspace.codes.shape) != (self.rows, self.inner)):
            raise ValueError("workspace does not match the plan")

    def _validate_product(self, workspace: Int8Workspace, weight: Int8PackedWeight, bias: torch.Tensor | None,
                          output: torch.Tensor | None) -> None:
        """What the product would refuse, before the first kernel has changed anything."""
        buffers = [_touched_rows(buffer) for buffer in (workspace.codes, workspace.scales)]
        read = [_touched_rows(tensor) for tensor in (weight.codes, weight.scales)]
        _refuse_unread(bias, output)
        if bias is not None:
            if tuple(bias.shape) != (self.columns,):
                raise ValueError(f"bias matrix has shape {tuple(bias.shape)}, expected {(self.columns,)}")
            if bias.device != self.device or bias.dtype != self.dtype:
                raise ValueError("bias matrix device or dtype does not match the plan")
            read.append(_touched_rows(bias))
        # the first kernel writes the buffers before the product reads the others
        if any(_rows_overlap(buffer, tensor) for buffer in buffers for tensor in read):
            raise ValueError("work buffers must not overlap")
        if output is not None:
            rows = _output_rows(output, torch.Size((self.rows, self.columns)), self.dtype, self.device.index, "output")
            if any(_rows_overlap(rows, tensor) for tensor in buffers + read):
                raise ValueError("output storage must not overlap inputs or workspace")

    @staticmethod
    def _refuse_output(output: torch.Tensor | None, *tensors: torch.Tensor | None) -> None:
        """What the first kernel reads or writes must outlive the second's output."""
        if output is None or _flat(output) is None:
            return  # a malformed output is refused where it is used
        rows = _touched_rows(output)
        for tensor in tensors:
            if tensor is not None and _rows_overlap(rows, _touched_rows(tensor)):
                raise ValueError("output storage must not overlap inputs or workspace")


# ---------------------------------------------------------------- torch.library
@torch.library.custom_op("rdna3_fastmm::quantize_rows_int8", mutates_args=(), device_types="cuda")
def quantize_rows_int8_op(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    _refuse_transforms()
    codes, scales = quantize_rows(x)
    return codes, scales


@torch.library.custom_op("rdna3_fastmm::rms_norm_int8", mutates_args=(), device_types="cuda")
def rms_norm_int8_op(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None,
                     eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    _refuse_transforms()
    codes, scales, stream = rms_norm_int8(x, weight, residual, eps)
    # without a residual there is no new one: an operator cannot return None
    return codes, scales, x.new_empty((0,)) if stream is None else stream


@torch.library.custom_op("rdna3_fastmm::linear_int8", mutates_args=(), device_types="cuda")
def linear_int8_op(codes: torch.Tensor, scales: torch.Tensor, weight_codes: torch.Tensor,
                   weight_scales: torch.Tensor, bias: Optional[torch.Tensor] = None,
                   dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    _refuse_transforms()
    return linear_int8(codes, scales, weight_codes, weight_scales, bias, dtype=dtype)


@quantize_rows_int8_op.register_fake
def _(x):
    return empty_codes(x.shape, x.device), x.new_empty(x.shape[:-1], dtype=torch.float32)


@rms_norm_int8_op.register_fake
def _(x, weight, residual=None, eps=1e-6):
    stream = x.new_empty((0,)) if residual is None else x.new_empty(x.shape)
    return empty_codes(x.shape, x.device), x.new_empty(x.shape[:-1], dtype=torch.float32), stream


@linear_int8_op.register_fake
def _(codes, scales, weight_codes, weight_scales, bias=None, dtype=torch.bfloat16):
    return codes.new_empty((*codes.shape[:-1], weight_codes.shape[0]), dtype=dtype)
