"""What the 8-bit operators tell autograd, and what they refuse of it."""

import pytest
import torch
from torch.autograd import forward_ad

from rdna3_fastmm.int8 import Int8Plan, empty_codes, linear_int8, quantize_rows, rms_norm_int8

pytestmark = pytest.mark.gpu
DEVICE = torch.device("cuda", 0)
BF16 = torch.bfloat16


def _randn(*shape):
    return torch.randn(shape, device=DEVICE).to(BF16)


@torch.enable_grad()  # whatever the mode that a test before left behind
@pytest.mark.parametrize("target", ["residual", "x"])
def test_backward_notices_a_stream_that_was_updated_in_place(target):
    """A trainable linear saved the stream; an in-place norm of it, without a gradient of its own, came after."""
    x, residual, gain = _randn(5, 64), _randn(5, 64), torch.ones(64, device=DEVICE)
    stream = residual if target == "residual" else x
    weight = _randn(8, 64).requires_grad_(True)
    loss = (stream @ weight.t()).sum()
    rms_norm_int8(x, gain, residual)  # into storage of its own: the saved values stay
    loss.backward(retain_graph=True)
    rms_norm_int8(x, gain, residual, residual_out=stream)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def _versions(*tensors):
    return [tensor._version for tensor in tensors]


def test_buffers_that_are_written_count_as_written():
    x, gain = _randn(5, 64), torch.ones(64, device=DEVICE)
    codes, scales, stream = empty_codes((5, 64), DEVICE), torch.empty(5, device=DEVICE), _randn(5, 64)
    w, ws = quantize_rows(_randn(8, 64))
    out = torch.empty((5, 8), dtype=BF16, device=DEVICE)
    inputs = x, gain, w, ws
    before = _versions(*inputs)
    quantize_rows(x, codes=codes)
    assert _versions(codes, scales, stream, out) == [1, 0, 0, 0]
    quantize_rows(x, codes=codes, scales=scales)
    assert _versions(codes, scales, stream, out) == [2, 1, 0, 0]
    rms_norm_int8(x, gain, codes=codes, scales=scales)
    assert _versions(codes, scales, stream, out) == [3, 2, 0, 0]
    rms_norm_int8(x, gain, x, codes=codes, scales=scales, residual_out=stream)
    assert _versions(codes, scales, stream, out) == [4, 3, 1, 0]
    linear_int8(codes, scales, w, ws, out=out)
    assert _versions(codes, scales, stream, out) == [4, 3, 1, 1]
    # a call that is refused, and one of no rows, write nothing
    with pytest.raises(ValueError):
        linear_int8(codes, scales, w, ws, out=out[:, :4])
    with pytest.raises(ValueError):
        rms_norm_int8(x, gain, eps=-1.0, codes=codes, scales=scales)
    quantize_rows(x[:0], codes=codes[:0], scales=scales[:0])
    assert _versions(codes, scales, stream, out) == [4, 3, 1, 1]
    assert _versions(*inputs) == before


def test_a_plan_marks_its_buffers_too():
    plan = Int8Plan(5, 64, 8, DEVICE)
    packed, ws = plan.pack_weight(_randn(8, 64), 0.1), plan.allocate_workspace(0.1)
    x, r, out = _randn(5, 64), _randn(5, 64), torch.empty((5, 8), dtype=BF16, device=DEVICE)
    plan.run_linear_packed(x, packed, ws, output=out)
    assert _versions(ws.codes, ws.scales, out, x, packed.codes) == [1, 1, 1, 0, 0]
    plan.run_norm_linear_packed(x, torch.ones(64, device=DEVICE), packed, ws, r, output=out, residual_output=r)
    assert _versions(ws.codes, ws.scales, out, x, r) == [2, 2, 2, 0, 1]


def test_buffers_of_inference_mode():
    with torch.inference_mode():
        x, codes, scales = _randn(5, 64), empty_codes((5, 64), DEVICE), torch.empty(5, device=DEVICE)
        got = quantize_rows(x, codes=codes, scales=scales)
    again = quantize_rows(x, codes=codes, scales=scales)
    assert again.codes is codes and torch.equal(got.codes, again.codes)


def test_tangents_are_refused():
    """A dual tensor does not require a gradient, and its tangent would be lost without a word."""
    x, gain, tangent = _randn(5, 64), torch.ones(64, device=DEVICE), _randn(5, 64)
    codes, scales = quantize_rows(x)
    w, ws = quantize_rows(_randn(8, 64))
    bias, out = _randn(8), torch.zeros((5, 8), dtype=BF16, device=DEVICE)
    plan = Int8Plan(5, 64, 8, DEVICE)
    packed, workspace = plan.pack_weight(_randn(8, 64), 0.1), plan.allocate_workspace(0.1)
    operators = torch.ops.rdna3_fastmm
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: quantize_rows(dual(x)),
                     lambda: rms_norm_int8(dual(x), gain),
                     lambda: rms_norm_int8(x, dual(gain)),
                     lambda: rms_norm_int8(x, gain, dual(x)),
                     lambda: linear_int8(codes, dual(scales), w, ws),
                     lambda: linear_int8(codes, scales, w, dual(ws)),
                     lambda: linear_int8(codes, scales, w, ws, dual(bias)),
                     lambda: linear_int8(codes, scales, w, ws, out=dual(out)),
                     lambda: plan.run_linear_packed(dual(x), packed, workspace),
                     lambda: plan.run_linear_packed(x, packed, workspace, dual(bias)),
                     lambda: plan.run_norm_linear_packed(x, dual(gain), packed, workspace),
                     lambda: operators.quantize_rows_int8(dual(x)),
                     lambda: operators.rms_norm_int8(dual(x), gain),
                     lambda: operators.linear_int8(codes, dual(scales), w, ws)):
            with torch.no_grad(), pytest.raises(ValueError, match="autograd"):
                call()
        rms_norm_int8(x, gain)  # operands without one
        operators.linear_int8(codes, scales, w, ws)
    for function in (quantize_rows, operators.quantize_rows_int8, lambda x: rms_norm_int8(x, gain),
                     lambda x: operators.rms_norm_int8(x, gain)):
        with pytest.raises((ValueError, RuntimeError)):
            torch.func.jvp(lambda x: function(x)[1], (x,), (tangent,))
    assert not out.any()
