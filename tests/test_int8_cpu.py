"""Host side of the 8-bit operators without a GPU: refusals of the C ABI, the
row arithmetic, and the fake forms of the torch operators."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from rdna3_fastmm import _native, int8
from rdna3_fastmm.int8 import _flat, _row_vector, _rows_overlap

P = ctypes.c_void_p
FAKE, ODD = P(0x10000), P(0x10001)


def _quantize(dtype=0, x=FAKE, rows=4, cols=64, ldx=64, codes=FAKE, ldq=64, scales=FAKE):
    return _native.library().fmm_quantize_rows(dtype, x, rows, cols, ldx, codes, ldq, scales, None)


def _norm(dtype=0, gain_dtype=0, x=FAKE, ldx=64, residual=None, ldr=0, gain=FAKE, rows=4, cols=64, eps=1e-6, out=None,
          ldo=0, codes=FAKE, ldq=64, scales=FAKE):
    return _native.library().fmm_rms_norm_int8(dtype, gain_dtype, x, ldx, residual, ldr, gain, rows, cols, eps, out,
                                               ldo, codes, ldq, scales, None)


def _linear(dtype=0, codes=FAKE, ldq=64, scales=FAKE, w=FAKE, ldw=64, ws=FAKE, bias=None, out=FAKE, ldc=32, M=4, K=64,
            N=32):
    return _native.library().fmm_linear_int8(dtype, codes, ldq, scales, w, ldw, ws, bias, out, ldc, M, K, N, None)


INVALID, MISALIGNED, UNSUPPORTED, TOO_LARGE = (_native.FMM_ERR_INVALID_ARGUMENT, _native.FMM_ERR_MISALIGNED,
                                               _native.FMM_ERR_UNSUPPORTED, _native.FMM_ERR_TOO_LARGE)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=2), UNSUPPORTED), (dict(dtype=9), UNSUPPORTED), (dict(rows=-1), INVALID), (dict(cols=0), INVALID),
    (dict(cols=2**31, ldx=2**31, ldq=2**31), TOO_LARGE), (dict(x=None), INVALID), (dict(codes=None), INVALID),
    (dict(scales=None), INVALID), (dict(ldx=63), INVALID), (dict(ldq=63), INVALID), (dict(x=ODD), MISALIGNED),
    (dict(scales=ODD), MISALIGNED), (dict(rows=0), 0), (dict(rows=0, x=None, codes=None, scales=None), 0),
])
def test_quantize_rows_refusals(change, code):
    assert _quantize(**change) == code


@pytest.mark.parametrize("change,code", [
    (dict(dtype=3), UNSUPPORTED), (dict(gain_dtype=1), UNSUPPORTED), (dict(dtype=2, gain_dtype=2), UNSUPPORTED),
    (dict(rows=-1), INVALID), (dict(cols=0), INVALID), (dict(eps=-1.0), INVALID), (dict(eps=float("nan")), INVALID),
    (dict(eps=float("inf")), INVALID), (dict(x=None), INVALID), (dict(gain=None), INVALID),
    (dict(residual=FAKE, ldr=64), INVALID), (dict(residual=FAKE, ldr=63, out=FAKE, ldo=64), INVALID),
    (dict(residual=FAKE, ldr=64, out=FAKE, ldo=63), INVALID), (dict(ldq=63), INVALID), (dict(gain=ODD), MISALIGNED),
    (dict(gain=P(0x10002), gain_dtype=3), MISALIGNED), (dict(rows=0), 0),
])
def test_rms_norm_int8_refusals(change, code):
    assert _norm(**change) == code


@pytest.mark.parametrize("change,code", [
    (dict(dtype=3), UNSUPPORTED), (dict(M=-1), INVALID), (dict(K=0), INVALID), (dict(N=0), INVALID),
    (dict(K=131072, ldq=131072, ldw=131072), TOO_LARGE), (dict(M=2**31), TOO_LARGE), (dict(N=2**31, ldc=2**31), TOO_LARGE),
    (dict(ldq=48), INVALID), (dict(ldw=48), INVALID), (dict(ldc=31), INVALID), (dict(codes=None), INVALID),
    (dict(ws=None), INVALID), (dict(out=None), INVALID), (dict(codes=P(0x10008)), MISALIGNED), (dict(w=ODD), MISALIGNED),
    (dict(ldq=72), MISALIGNED), (dict(ldw=65), MISALIGNED), (dict(bias=ODD), MISALIGNED), (dict(out=ODD), MISALIGNED),
    (dict(M=0), 0),
])
def test_linear_int8_refusals(change, code):
    assert _linear(**change) == code


def test_refusals_reach_python_as_value_errors():
    with pytest.raises(ValueError, match="16-byte"):
        _native.check(_linear(codes=ODD), "fmm_linear_int8")


def test_rows_of_views():
    x = torch.zeros((2, 3, 4, 10))
    assert _flat(x) == (24, 10, 10)
    assert _flat(x[..., :7]) == (24, 7, 10)
    assert _flat(x[:, :, 1]) == (6, 10, 40)
    assert _flat(x[:, 1:, :2]) is None
    assert _flat(x.transpose(0, 1)) is None
    assert _flat(x[..., ::2]) is None
    assert _flat(x[:1, :, 0]) == (3, 10, 40)
    assert _flat(torch.zeros((1, 10)).expand(5, 10)) is None
    assert _flat(torch.zeros(10)) == (1, 10, 16)
    assert _flat(torch.zeros((0, 10)))[0] == 0
    assert _flat(torch.zeros((6, 1))[::2]) == (3, 1, 2)


def _cut(buffer, first, width):
    part = buffer[:, first:first + width]
    return part.data_ptr(), *_flat(part), part.element_size()


def test_overlap_of_rows():
    buffer = torch.zeros((4, 100), dtype=torch.int16)
    assert not _rows_overlap(_cut(buffer, 0, 50), _cut(buffer, 50, 50))
    assert not _rows_overlap(_cut(buffer, 50, 50), _cut(buffer, 0, 50))
    assert _rows_overlap(_cut(buffer, 0, 51), _cut(buffer, 50, 50))
    assert _rows_overlap(_cut(buffer, 50, 50), _cut(buffer, 0, 51))
    assert _rows_overlap(_cut(buffer, 3, 5), _cut(buffer, 3, 5))
    assert _rows_overlap(_cut(buffer[1:], 0, 5), _cut(buffer, 4, 9))
    assert not _rows_overlap(_cut(buffer[:2], 0, 100), _cut(buffer[2:], 0, 100))
    assert _rows_overlap(_row_vector(buffer.view(-1)[150:160]), _cut(buffer, 0, 50))
    assert not _rows_overlap(_row_vector(buffer.view(-1)[:0]), _cut(buffer, 0, 50))


def test_operands_apart_by_one_sort():
    buffer = torch.zeros((4, 100), dtype=torch.int16)
    apart = int8._all_apart
    assert apart([_cut(buffer[2:], 0, 100), _cut(buffer[:2], 0, 100)])
    assert apart([_cut(buffer[:2], 0, 100), _row_vector(buffer.view(-1)[200:]), _row_vector(buffer.view(-1)[:0])])
    assert not apart([_cut(buffer, 0, 50), _cut(buffer, 50, 50)])  # beside each other: for the closer look
    assert not apart([_cut(buffer[:3], 0, 100), _row_vector(buffer.view(-1)[299:])])
    int8._refuse_overlap([_cut(buffer, 0, 50)], [_cut(buffer, 50, 50)])
    with pytest.raises(ValueError, match="overlap"):
        int8._refuse_overlap([_cut(buffer, 0, 50)], [_cut(buffer, 49, 50)])


def test_cpu_tensors_and_plans_are_refused():
    x = torch.ones((2, 16), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        int8.quantize_rows(x)
    with pytest.raises(ValueError, match="CUDA"):
        int8.rms_norm_int8(x, x[0])
    with pytest.raises(ValueError, match="CUDA"):
        int8.linear_int8(x.to(torch.int8), x[:, 0].float(), x.to(torch.int8), x[:, 0].float())
    with pytest.raises(ValueError, match="CUDA sm_100"):
        int8.Int8Plan(2, 16, 2, torch.device("cpu"))


@pytest.mark.parametrize("change,match", [
    (dict(rows=0), "positive"), (dict(inner=0), "positive"), (dict(columns=-1), "positive"),
    (dict(inner=131072), "32-bit sum"), (dict(dtype=torch.float32), "does not support"),
])
def test_plan_arguments(monkeypatch, change, match):
    monkeypatch.setattr(torch.version, "cuda", "12.8")
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    arguments = dict(rows=3, inner=70, columns=5, device=torch.device("cuda"))
    plan = int8.Int8Plan(**arguments)
    assert (plan.workspace_bytes, plan.packed_weight_bytes) == (3 * 84, 5 * 84)
    with pytest.raises(ValueError, match=match):
        int8.Int8Plan(**{**arguments, **change})


def test_fake_forms_have_the_real_shapes_and_strides():
    with FakeTensorMode():
        x = torch.empty((2, 3, 100), dtype=torch.bfloat16, device="cuda")
        codes, scales = torch.ops.rdna3_fastmm.quantize_rows_int8(x)
        assert codes.shape == (2, 3, 100) and codes.stride() == (336, 112, 1) and codes.dtype == torch.int8
        assert scales.shape == (2, 3) and scales.dtype == torch.float32
        weight = torch.empty(100, dtype=torch.bfloat16, device="cuda")
        codes, scales, stream = torch.ops.rdna3_fastmm.rms_norm_int8(x, weight, x)
        assert stream.shape == x.shape and stream.dtype == x.dtype
        assert torch.ops.rdna3_fastmm.rms_norm_int8(x, weight)[2].shape == (0,)
        w, ws = torch.ops.rdna3_fastmm.quantize_rows_int8(torch.empty((7, 100), device="cuda"))
        y = torch.ops.rdna3_fastmm.linear_int8(codes, scales, w, ws, None, torch.float16)
        assert y.shape == (2, 3, 7) and y.dtype == torch.float16
