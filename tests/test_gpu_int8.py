"""8-bit integer operators on the GPU against their formulas in 64 bits.

Codes are compared for equality: the kernels round the exact quotient.  The
other tolerances count roundings (half a step each, ``eps / 2`` relative)."""

import pytest
import torch

from rdna3_fastmm import _native
from rdna3_fastmm.int8 import (Int8Plan, empty_codes, linear_int8, quantize_rows, rms_norm_int8)

pytestmark = pytest.mark.gpu
DEVICE = torch.device("cuda", 0)
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
HALF = [BF16, FP16]
U32 = 2.0**-24  # half a step of FP32


def _randn(shape, seed, dtype=FP32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(shape, generator=g)).to(dtype)


def _codes(p):
    """Exact codes and peaks of rows in 64 bits."""
    peak = p.abs().amax(dim=-1, keepdim=True)
    return torch.round(127.0 * p / torch.where(peak > 0, peak, 1.0)), peak[..., 0]


def _check_rows(codes, scales, p, scale_factor, scale_roundings):
    expected, peak = _codes(p)
    assert torch.equal(codes.cpu().double(), expected)
    reference = peak * scale_factor / 127.0
    error = (scales.cpu().double() - reference).abs()
    assert bool((error <= scale_roundings * U32 * reference).all())


# rows and widths around a lane's vector, a warp's row (1024), a block's
# (4096, 8192, 16384, 32768) and beyond
WIDTHS = [(1, 1), (1, 7), (3, 8), (5, 127), (9, 256), (6, 504), (4, 1024), (7, 1025), (3, 4096), (2, 4104),
          (2, 4607), (2, 8200), (1, 16384), (2, 16392), (2, 20001), (2, 32768), (2, 32776), (1, 50003)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,inner", WIDTHS)
def test_quantize_rows_gives_the_exact_codes(rows, inner, dtype):
    x = _randn((rows, inner), rows * 7 + inner, dtype, 3.0)
    x[0, inner // 2] = -20.0
    codes, scales = quantize_rows(x.to(DEVICE))
    # one rounding: the peak is exact
    _check_rows(codes, scales, x.double(), 1.0, 1)


def _norm_reference(x, weight, residual, eps):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    p = h.double() * weight.double()
    return h, p, torch.rsqrt(h.double().square().mean(dim=-1) + eps)


def _norm_roundings(inner):
    # a thread adds at most 96 squares one after another (12 vectors of 8 of a
    # streamed row; 8 V = 32 of a row in registers; of a longer row 8 a pass of
    # 1024 threads), then up to 12 joins (two chains, 5 in the warp, up to 32
    # warps in 5 or, one after another, 16 warps that share fewer squares); the
    # root halves what the mean is off, four roundings follow (mean and epsilon,
    # root, two quotients; the peak is exact or one rounding more)
    mine = max(96, 8 * -(-inner // 8192))
    return (mine + 12) / 2 + 5


@pytest.mark.parametrize("gain", ["same", "fp32"])
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows,inner", WIDTHS)
def test_rms_norm_int8_gives_the_exact_codes(rows, inner, dtype, with_residual, gain):
    x = _randn((rows, inner), inner, dtype)
    residual = _randn((rows, inner), inner + 1, dtype, 2.0) if with_residual else None
    weight = (1 + 0.3 * _randn((inner,), inner + 2)).to(FP32 if gain == "fp32" else dtype)
    codes, scales, stream = rms_norm_int8(x.to(DEVICE), weight.to(DEVICE),
                                          None if residual is None else residual.to(DEVICE), 1e-5)
    h, p, rstd = _norm_reference(x, weight, residual, 1e-5)
    _check_rows(codes, scales, p, rstd, _norm_roundings(inner))
    assert (stream is None) == (residual is None)
    if residual is not None:
        assert torch.equal(stream.cpu(), h)


def test_ties_go_to_the_even_code():
    # the peak 127 makes every quotient the value itself
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 62.5, 63.5, -126.5, 126.5, 0.4990234375, 0.5009765625]])
    expected = [127, 0, 2, 2, 0, -2, 62, 64, -126, 126, 0, 1]
    for dtype in (FP16, FP32):
        codes, scales = quantize_rows(x.to(dtype).to(DEVICE))
        assert codes.cpu().tolist() == [expected]
        assert scales.item() == 1.0


@pytest.mark.parametrize("gain_dtype", [BF16, FP32])
def test_codes_next_to_a_border_are_exact(gain_dtype):
    """Products a step of their type on either side of a half code."""
    inner = 2048
    k = torch.arange(inner, dtype=torch.float64)
    target = ((k % 127) + 0.5) / 127.0
    x = target.to(BF16)
    # the gain brings x * gain as near to the half as its type allows, +- one step
    gain = (target / x.double()).to(gain_dtype)
    gain = torch.where(k % 3 == 0, torch.nextafter(gain.float(), torch.tensor(2.0)),
                       gain.float()).to(gain_dtype)
    x[0] = 1.0
    gain[0] = 1.0
    codes, _, _ = rms_norm_int8(x[None].to(DEVICE), gain.to(DEVICE))
    assert torch.equal(codes.cpu().double(), _codes((x.double() * gain.double())[None])[0])


@pytest.mark.parametrize("inner", [5, 600, 5000, 40000])
def test_rows_of_zeros_infinities_and_nans(inner):
    x = _randn((5, inner), 3, BF16)
    x[1] = 0
    x[2, inner - 1] = float("inf")
    x[3, inner // 3] = float("nan")
    weight = torch.ones(inner, dtype=BF16)
    for codes, scales in (quantize_rows(x.to(DEVICE)),
                          rms_norm_int8(x.to(DEVICE), weight.to(DEVICE))[:2]):
        codes, scales = codes.cpu(), scales.cpu()
        assert not codes[1:4].any()
        assert scales[1] == 0
        assert scales[2:4].isnan().all()
        assert torch.equal(codes[[0, 4]].double(), _codes(x[[0, 4]].double())[0])
        w = torch.ones((3, inner))
        wc, ws = quantize_rows(w.to(DEVICE))
        y = linear_int8(codes.to(DEVICE) if inner % 16 == 0 else empty_codes(codes.shape, DEVICE).copy_(codes),
                        scales.to(DEVICE), wc, ws).cpu()
        assert not y[1].any()
        assert y[2:4].isnan().all()


@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("gain", ["same", "fp32"])
@pytest.mark.parametrize("rows,inner", [(12001, 512), (11003, 1024), (4097, 1032), (1201, 4608), (700, 8200), (401, 16384),
                                        (330, 24576), (310, 32768), (3100, 4607), (9000, 1031), (1300, 9001),
                                        (20000, 259)])
def test_many_rows_stream_through(rows, inner, gain, with_residual):
    """More rows than resident blocks take at once; padding rows among them."""
    x = _randn((rows, inner), 1, BF16).to(DEVICE)
    x[rows // 2:rows // 2 + 40] = 0
    residual = _randn((rows, inner), 2, BF16).to(DEVICE) if with_residual else None
    if with_residual:
        residual[rows // 2:rows // 2 + 40] = 0
    weight = (1 + 0.3 * _randn((inner,), 3)).to(FP32 if gain == "fp32" else BF16).to(DEVICE)
    codes, scales, stream = rms_norm_int8(x, weight, residual, 1e-5)
    h, p, rstd = _norm_reference(x, weight, residual, 1e-5)
    expected, peak = _codes(p)
    assert torch.equal(codes, expected.to(torch.int8))
    reference = peak * rstd / 127.0
    assert bool(((scales.double() - reference).abs() <= _norm_roundings(inner) * U32 * reference).all())
    if with_residual:
        assert torch.equal(stream, h)
    codes, scales = quantize_rows(x)
    expected, peak = _codes(x.double())
    assert torch.equal(codes, expected.to(torch.int8))
    assert bool(((scales.double() - peak / 127.0).abs() <= U32 * peak / 127.0).all())


@pytest.mark.parametrize("rows", [2, 5000])
def test_zeros_without_an_epsilon(rows):
    x = torch.zeros((rows, 1024), dtype=BF16, device=DEVICE)
    x[1] = 1
    codes, scales, _ = rms_norm_int8(x, torch.ones(1024, device=DEVICE), eps=0.0)
    assert not codes[0].any() and scales[0] == 0 and bool((codes[1] == 127).all())
    assert bool((scales[2:] == 0).all()) and abs(scales[1].item() - 1 / 127) <= 4 * U32


def test_offsets_beyond_32_bits():
    """More than 2^32 bytes and 2^31 elements; the last rows come out as alone."""
    rows, inner = 70000, 32768
    x = torch.zeros((rows, inner), dtype=BF16, device=DEVICE)
    x[-3:] = _randn((3, inner), 1, BF16).to(DEVICE)
    codes, scales = quantize_rows(x)
    alone = quantize_rows(x[-3:].clone())
    assert torch.equal(codes[-3:], alone.codes) and torch.equal(scales[-3:], alone.scales)
    weight = torch.ones(inner, device=DEVICE)
    got = rms_norm_int8(x, weight, x, codes=codes, scales=scales, residual_out=x)
    again = rms_norm_int8(got.residual[-3:].clone() / 2, weight, got.residual[-3:].clone() / 2)
    assert torch.equal(got.codes[-3:], again.codes) and torch.equal(got.residual[-3:], again.residual)
    del x, got
    w, ws = quantize_rows(_randn((40, inner), 2).to(DEVICE))
    y = linear_int8(codes, scales, w, ws)
    assert torch.equal(y[-3:], linear_int8(codes[-3:], scales[-3:], w, ws))
    del codes, y
    q, s = quantize_rows(_randn((300000, 64), 3).to(DEVICE))
    w, ws = quantize_rows(_randn((8200, 64), 4).to(DEVICE))
    y = linear_int8(q, s, w, ws)
    assert torch.equal(y[-5:], linear_int8(q[-5:], s[-5:], w, ws))


@pytest.mark.parametrize("scale", [2.0**-130, 2.0**-110, 2.0**100])
def test_rows_of_extreme_magnitude(scale):
    x = (_randn((3, 700), 5).to(BF16).double() * scale).to(FP32)
    codes, _ = quantize_rows(x.to(DEVICE))
    assert torch.equal(codes.cpu().double(), _codes(x.double())[0])


def test_squares_beyond_fp32_are_not_finite():
    x = torch.full((1, 64), 1e30, dtype=BF16, device=DEVICE)
    codes, scales, _ = rms_norm_int8(x, torch.ones(64, device=DEVICE))
    assert not codes.any() and scales.isnan().all()


@pytest.mark.parametrize("offset,pitch", [(0, 640), (8, 640), (1, 640), (0, 601), (3, 777)])
@pytest.mark.parametrize("inner", [600, 5001])
def test_rows_in_larger_buffers(offset, pitch, inner):
    """Any step and alignment; what lies beside the rows stays as it was."""
    rows, pitch = 5, pitch - 600 + inner
    x_buf = _randn((rows + 1, pitch), 1, BF16).to(DEVICE)
    r_buf = _randn((rows + 1, pitch), 2, BF16).to(DEVICE)
    o_buf = torch.full((rows + 1, pitch), 9.0, dtype=BF16, device=DEVICE)
    q_buf = torch.full((rows + 1, pitch), 99, dtype=torch.int8, device=DEVICE)
    cut = lambda b: b.view(-1)[offset:offset + rows * pitch].view(rows, pitch)[:, :inner]  # noqa: E731
    weight = (1 + 0.1 * _randn((inner,), 4)).to(BF16).to(DEVICE)
    x, r, o, q = cut(x_buf), cut(r_buf), cut(o_buf), cut(q_buf)
    scales = torch.empty(rows, device=DEVICE)
    got = rms_norm_int8(x, weight, r, codes=q, scales=scales, residual_out=o)
    assert got.codes.data_ptr() == q.data_ptr() and got.residual.data_ptr() == o.data_ptr()
    h, p, rstd = _norm_reference(x.cpu(), weight.cpu(), r.cpu(), 1e-6)
    _check_rows(q, scales, p, rstd, _norm_roundings(inner))
    assert torch.equal(o.cpu(), h)
    o.fill_(9.0)
    q.fill_(99)
    assert bool((o_buf == 9.0).all()) and bool((q_buf == 99).all())


@pytest.mark.parametrize("offset,pitch,code_pitch", [(1, 2003, 2000), (3, 2001, 2003), (8, 2008, 2008), (4, 2004, 2016),
                                                     (5, 2008, 2001)])
@pytest.mark.parametrize("dtype", [FP16, FP32])
def test_many_rows_in_larger_buffers(offset, pitch, code_pitch, dtype):
    """The streamed form at any step and alignment; what lies beside the rows stays."""
    rows, inner = 6000, 2000
    cut = lambda b, p: b.view(-1)[offset:offset + rows * p].view(rows, p)[:, :inner]  # noqa: E731
    x_buf = _randn((rows + 1, pitch), 1, dtype).to(DEVICE)
    q_buf = torch.full((rows + 1, code_pitch), 99, dtype=torch.int8, device=DEVICE)
    x, q = cut(x_buf, pitch), cut(q_buf, code_pitch)
    scales = torch.empty(rows, device=DEVICE)
    quantize_rows(x, codes=q, scales=scales)
    expected, peak = _codes(x.double())
    assert torch.equal(q, expected.to(torch.int8))
    assert bool(((scales.double() - peak / 127.0).abs() <= U32 * peak / 127.0).all())
    if dtype != FP32:
        r_buf = _randn((rows + 1, pitch + 2), 2, dtype).to(DEVICE)
        o_buf = torch.full((rows + 1, pitch + 1), 9.0, dtype=dtype, device=DEVICE)
        r, o = cut(r_buf, pitch + 2), cut(o_buf, pitch + 1)
        weight = (1 + 0.1 * _randn((inner,), 4)).to(DEVICE)
        rms_norm_int8(x, weight, r, codes=q, scales=scales, residual_out=o)
        h, p, rstd = _norm_reference(x, weight, r, 1e-6)
        expected, peak = _codes(p)
        assert torch.equal(q, expected.to(torch.int8)) and torch.equal(o, h)
        reference = peak * rstd / 127.0
        assert bool(((scales.double() - reference).abs() <= _norm_roundings(inner) * U32 * reference).all())
        expected_stream = o.clone()
        rms_norm_int8(x, weight, r, codes=q, scales=scales, residual_out=r)  # in place
        assert torch.equal(r, expected_stream) and torch.equal(q, expected.to(torch.int8))
        o.fill_(9.0)
        assert bool((o_buf == 9.0).all())
    q.fill_(99)
    assert bool((q_buf == 99).all())


@pytest.mark.parametrize("rows,inner,dtype", [(20000, 300, FP32), (3100, 4612, FP32), (9000, 1004, FP32), (5, 4612, FP32),
                                              (20000, 132, FP32), (12000, 260, BF16), (9000, 1001, FP16)])
def test_aligned_rows_that_are_not_whole_vectors(rows, inner, dtype):
    """FP32 rows of 4 n elements, and 16-bit rows of any length at an aligned step."""
    pitch = inner if dtype == FP32 else -(-inner // 8) * 8
    x = _randn((rows, pitch), 1, dtype).to(DEVICE)[:, :inner]
    codes, scales = quantize_rows(x)
    expected, peak = _codes(x.double())
    assert torch.equal(codes, expected.to(torch.int8))
    assert bool(((scales.double() - peak / 127.0).abs() <= U32 * peak / 127.0).all())
    if dtype != FP32:
        weight = (1 + 0.1 * _randn((inner,), 4)).to(dtype).to(DEVICE)
        codes, scales, h = rms_norm_int8(x, weight, x)
        reference, p, _ = _norm_reference(x, weight, x, 1e-6)
        assert torch.equal(codes, _codes(p)[0].to(torch.int8)) and torch.equal(h, reference)


@pytest.mark.parametrize("rows", [6, 4000])
@pytest.mark.parametrize("inner", [96, 4608, 40000])
def test_the_stream_is_updated_in_place(inner, rows):
    x, r = _randn((rows, inner), 1, FP16).to(DEVICE), _randn((rows, inner), 2, FP16).to(DEVICE)
    weight = torch.ones(inner, device=DEVICE)
    expected = rms_norm_int8(x, weight, r)
    for target in ("residual", "x"):
        a, b = x.clone(), r.clone()
        got = rms_norm_int8(a, weight, b, residual_out=b if target == "residual" else a)
        assert torch.equal(got.codes, expected.codes) and torch.equal(got.scales, expected.scales)
        assert torch.equal(got.residual, expected.residual)
        assert torch.equal(a if target == "x" else b, expected.residual)


def test_leading_dimensions_and_strided_inputs():
    x = _randn((2, 3, 5, 40), 1, BF16).to(DEVICE)
    codes, scales = quantize_rows(x)
    assert codes.shape == x.shape and scales.shape == (2, 3, 5)
    flat = quantize_rows(x.view(-1, 40))
    assert torch.equal(codes.reshape(-1, 40), flat.codes) and torch.equal(scales.view(-1), flat.scales)
    for view in (x.transpose(1, 2), x.transpose(-1, -2), x[:, 1:2, ::2], x[:1, :1].expand(4, 3, 5, 40), x[0, 0, 0]):
        codes, scales = quantize_rows(view)
        expected = quantize_rows(view.contiguous())
        assert torch.equal(codes, expected.codes) and torch.equal(scales, expected.scales)
    w, ws = quantize_rows(_randn((24, 40), 2).to(DEVICE))
    codes, scales = quantize_rows(x)
    y = linear_int8(codes, scales, w, ws)
    assert y.shape == (2, 3, 5, 24)
    assert torch.equal(y.view(-1, 24), linear_int8(flat.codes, flat.scales, w, ws))
    one = linear_int8(*quantize_rows(x[0, 0, 0]), w, ws)
    assert one.shape == (24,) and torch.equal(one, y[0, 0, 0])


def test_empty_batches():
    weight = torch.ones(64, device=DEVICE)
    x = torch.empty((0, 64), dtype=BF16, device=DEVICE)
    codes, scales, stream = rms_norm_int8(x, weight, x.clone())
    assert codes.shape == (0, 64) and scales.shape == (0,) and stream.shape == (0, 64)
    codes, scales = quantize_rows(x)
    w, ws = quantize_rows(torch.ones((8, 64), device=DEVICE))
    assert linear_int8(codes, scales, w, ws).shape == (0, 8)


# ---------------------------------------------------------------- product
def _int_rows(rows, inner, seed, low=-127):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(low, 128, (rows, inner), generator=g, dtype=torch.int8)


def _to_device(codes):
    return empty_codes(tuple(codes.shape), DEVICE).copy_(codes)


def _linear_reference(codes, scales, w, ws, bias):
    """The value, and the magnitude that FP32 roundings go by."""
    y = (codes.double() @ w.double().T) * scales.double()[:, None] * ws.double()
    size = y.abs()
    if bias is not None:
        y = y + bias.double()
        size = size + bias.double().abs()
    return y, size


def _check_linear(got, reference, size, dtype):
    # FP32: the sum, the scales' product, theirs, the bias; then one rounding
    # to dtype (of a value 4 roundings off), which below the normal range is
    # half a subnormal step
    info = torch.finfo(dtype)
    fp32 = 4 * U32 * size
    allowed = fp32 + (reference.abs() + fp32) * info.eps / 2 + info.smallest_normal * info.eps / 2
    assert bool(((got.cpu().double() - reference).abs() <= allowed).all())


def _linear_case(rows, inner, columns, dtype, with_bias, seed=0):
    codes, w = _int_rows(rows, inner, seed, -128), _int_rows(columns, inner, seed + 1, -128)
    scales = 0.01 * (0.5 + torch.rand(rows, generator=torch.Generator().manual_seed(seed + 2)))
    ws = 0.002 * (0.5 + torch.rand(columns, generator=torch.Generator().manual_seed(seed + 3)))
    bias = _randn((columns,), seed + 4, dtype) if with_bias else None
    return codes, scales, w, ws, bias


def _run_linear(codes, scales, w, ws, bias, dtype, **kw):
    return linear_int8(_to_device(codes), scales.to(DEVICE), _to_device(w), ws.to(DEVICE),
                       None if bias is None else bias.to(DEVICE), dtype=dtype, **kw)


SHAPES = [(1, 1, 1), (1, 128, 128), (2, 17, 31), (7, 129, 300), (15, 16, 129), (16, 4097, 127), (17, 300, 257),
          (31, 1000, 33), (33, 640, 1000), (64, 2048, 512), (80, 513, 640), (100, 96, 2000), (128, 4096, 256),
          (129, 384, 385), (255, 256, 130), (256, 128, 512), (257, 263, 269), (520, 776, 392), (1000, 200, 1),
          (1025, 1152, 2049), (2050, 64, 300), (1, 16384, 4096), (3, 70000, 40),
          # each kernel, its widths and its ends: few tokens by 1, 2 and 4 channels, tiles of 64 and
          # 128 channels, pairs of SMs with whole and ragged token tiles
          (1, 1040, 500), (2, 2063, 4001), (4, 1025, 3600), (4, 4096, 131), (1, 4609, 8001), (2, 1024, 7300),
          (5, 300, 9000), (48, 1100, 8200), (200, 2000, 4100), (700, 515, 9001), (600, 4096, 9472),
          (1300, 1031, 4999), (300, 1024, 37889),
          # a short K with many outputs: tokens in the lanes where rows of 8 outputs are aligned
          (3000, 64, 1000), (20003, 100, 304), (2500, 33, 72), (5000, 257, 520), (9000, 16, 8), (4001, 128, 1001)]


@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("shape", SHAPES)
def test_linear_int8_matches_the_formula(shape, dtype, with_bias):
    case = _linear_case(*shape, dtype, with_bias)
    got = _run_linear(*case, dtype)
    assert got.dtype == dtype and got.shape == (shape[0], shape[2])
    _check_linear(got, *_linear_reference(*case), dtype)


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_sums_are_exact_at_the_largest_inner_length(rows):
    inner = 131071
    codes = torch.full((rows, inner), -128, dtype=torch.int8)
    w = torch.full((130, inner), -128, dtype=torch.int8)
    w[1::2] = 127
    one = torch.ones
    y = _run_linear(codes, one(rows), w, one(130) * 2.0**-20, None, BF16)
    reference, size = _linear_reference(codes[:1], one(1), w, one(130) * 2.0**-20, None)
    _check_linear(y, reference.expand(rows, -1), size.expand(rows, -1), BF16)


@pytest.mark.parametrize("rows,columns", [(3, 200), (70, 129), (300, 515)])
def test_linear_writes_its_output_only(rows, columns):
    inner = 200
    case = _linear_case(rows, inner, columns, BF16, True)
    expected = _run_linear(*case, BF16)
    for offset, pitch in ((0, columns + 8), (1, columns + 3)):
        buf = torch.full((rows + 2, pitch), 7.0, dtype=BF16, device=DEVICE)
        out = buf.view(-1)[offset:offset + rows * pitch].view(rows, pitch)[:, :columns]
        got = _run_linear(*case, BF16, out=out)
        assert got.data_ptr() == out.data_ptr()
        assert torch.equal(out, expected)
        out.fill_(7.0)
        assert bool((buf == 7.0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,columns,pitch", [(1167, 329, 352), (14595, 9, 16), (2083, 2574, 2592), (113, 13975, 13984),
                                                (2610, 1, 16), (5389, 13, 32), (464, 6271, 6272), (2083, 2568, 2592)])
def test_linear_writes_columns_of_a_larger_buffer(rows, columns, pitch, dtype):
    """Aligned rows, whose last 16 bytes hold columns of somebody else."""
    a, w = (torch.randint(-127, 128, (n, 48), device=DEVICE, dtype=torch.int8) for n in (rows, columns))
    sa = torch.rand(rows, device=DEVICE) * 0.01 + 1e-3
    sw = torch.rand(columns, device=DEVICE) * 1e-3 + 1e-4
    buffer = torch.full((rows, pitch), 7.0, device=DEVICE, dtype=dtype)
    linear_int8(a, sa, w, sw, out=buffer[:, :columns])
    assert torch.equal(buffer[:, :columns], linear_int8(a, sa, w, sw, dtype=dtype))
    assert (buffer[:, columns:] == 7.0).all()


def test_linear_reads_code_rows_of_any_pitch():
    rows, inner, columns = 20, 200, 150
    case = _linear_case(rows, inner, columns, FP16, False)
    expected = _run_linear(*case, FP16)
    codes = torch.full((rows, 320), 77, dtype=torch.int8, device=DEVICE)
    w = torch.full((columns, 512), 77, dtype=torch.int8, device=DEVICE)
    codes[:, 16:16 + inner] = case[0].to(DEVICE)
    w[:, :inner] = case[2].to(DEVICE)
    got = linear_int8(codes[:, 16:16 + inner], case[1].to(DEVICE), w[:, :inner], case[3].to(DEVICE), dtype=FP16)
    assert torch.equal(got, expected)


def test_repeated_calls_give_the_same_bits():
    case = _linear_case(37, 5000, 700, BF16, True)
    first = _run_linear(*case, BF16)
    for _ in range(5):
        assert torch.equal(_run_linear(*case, BF16), first)


@pytest.mark.parametrize("sms", [2, 36])
def test_the_sm_budget_keeps_results(sms):
    case = _linear_case(300, 700, 2100, BF16, False)
    few = _linear_case(9, 3000, 2100, BF16, False)
    x = _randn((4000, 1500), 1, BF16).to(DEVICE)
    expected = _run_linear(*case, BF16), _run_linear(*few, BF16), quantize_rows(x)
    try:
        _native.set_sm_budget(sms)
        got = _run_linear(*case, BF16), _run_linear(*few, BF16), quantize_rows(x)
        torch.cuda.synchronize()
    finally:
        _native.set_sm_budget(0)
    assert torch.equal(got[0], expected[0]) and torch.equal(got[1], expected[1])
    assert torch.equal(got[2].codes, expected[2].codes) and torch.equal(got[2].scales, expected[2].scales)


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("rows", [1, 8, 33, 300])
@pytest.mark.parametrize("dtype", HALF)
def test_plan_runs_the_operators_together(rows, dtype):
    """norm -> product against the float layer: what is lost is the rounding to codes."""
    inner, columns = 1032, 640
    x, r = _randn((rows, inner), 1, dtype).to(DEVICE), _randn((rows, inner), 2, dtype).to(DEVICE)
    norm_weight = (1 + 0.1 * _randn((inner,), 3)).to(dtype).to(DEVICE)
    weight = _randn((columns, inner), 4, dtype, 0.03).to(DEVICE)
    bias = _randn((columns,), 5, dtype).to(DEVICE)
    plan = Int8Plan(rows, inner, columns, DEVICE, dtype=dtype)
    ws = plan.allocate_workspace(0.1)
    packed = plan.pack_weight(weight, 0.1)
    y, stream = plan.run_norm_linear_packed(x, norm_weight, packed, ws, r, 1e-6, bias)
    codes, scales, h = rms_norm_int8(x, norm_weight, r, 1e-6)
    wc, wscale = quantize_rows(weight)
    assert torch.equal(stream, h)
    assert torch.equal(y, linear_int8(codes, scales, wc, wscale, bias))
    reference, size = _linear_reference(codes.cpu(), scales.cpu(), wc.cpu(), wscale.cpu(), bias.cpu())
    _check_linear(y, reference, size, dtype)
    # against the layer without 8 bits: each code is at most half a step off
    norm = h.double() * torch.rsqrt(h.double().square().mean(-1, keepdim=True) + 1e-6) * norm_weight.double()
    full = norm @ weight.double().T + bias.double()
    step = (scales.double()[:, None] / 2) * weight.double().abs().sum(1) \
        + (norm.abs().sum(1) + inner * scales.double() / 2)[:, None] * wscale.double() / 2
    # and the roundings of the sums and of the output
    rounding = (full.abs() + step) * torch.finfo(dtype).eps + 1e-3 * step
    assert bool(((y.double() - full).abs() <= step + rounding).all())
    z = plan.run_linear_packed(x, packed, ws, bias)
    assert torch.equal(z, linear_int8(*quantize_rows(x), wc, wscale, bias))
    out = torch.empty_like(z)
    assert plan.run_linear_packed(x, packed, ws, bias, out).data_ptr() == out.data_ptr()
    assert torch.equal(out, z)


@pytest.mark.parametrize("rows", [1, 70, 600])
def test_calls_capture_and_replay(rows):
    inner, columns = 640, 392
    plan = Int8Plan(rows, inner, columns, DEVICE)
    packed = plan.pack_weight(_randn((columns, inner), 1, BF16).to(DEVICE), 0.1)
    norm_weight = torch.ones(inner, device=DEVICE)
    graphs, runs = [], []
    for k in range(2):  # two graphs with a workspace each
        ws = plan.allocate_workspace(0.1)
        x, r = _randn((rows, inner), 2 + k, BF16).to(DEVICE), _randn((rows, inner), 4 + k, BF16).to(DEVICE)
        out = torch.empty((rows, columns), dtype=BF16, device=DEVICE)
        stream_out = torch.empty_like(x)
        run = lambda x=x, r=r, ws=ws, out=out, s=stream_out: plan.run_norm_linear_packed(  # noqa: E731
            x, norm_weight, packed, ws, r, output=out, residual_output=s)
        run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        graphs.append(graph)
        runs.append((x, r, out, stream_out))
    for k, (x, r, out, stream_out) in enumerate(runs):
        x.copy_(_randn((rows, inner), 10 + k, BF16))
        out.zero_()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graphs[1].replay()
    graphs[0].replay()
    torch.cuda.synchronize()
    for x, r, out, stream_out in runs:
        codes, scales, h = rms_norm_int8(x, norm_weight, r)
        assert torch.equal(out, linear_int8(codes, scales, packed.codes, packed.scales))
        assert torch.equal(stream_out, h)


def test_calls_follow_the_current_stream():
    x = _randn((512, 4096), 1, BF16).to(DEVICE)
    w, ws = quantize_rows(_randn((1024, 4096), 2).to(DEVICE))
    expected = linear_int8(*quantize_rows(x), w, ws)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    y = torch.zeros_like(x)
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        y.copy_(x)
        got = linear_int8(*quantize_rows(y), w, ws)
    side.synchronize()
    assert torch.equal(got, expected)


@pytest.mark.parametrize("rows", [1, 3, 40, 700])
def test_back_to_back_calls_wait_for_each_other(rows):
    """Launches overlap the kernel before them; every buffer here is written by
    one call and read, then overwritten, by the next ones."""
    inner = 2048
    plan = Int8Plan(rows, inner, inner, DEVICE)
    packed = [plan.pack_weight(_randn((inner, inner), k, BF16, 0.05).to(DEVICE), 0.1) for k in range(3)]
    gain = (1 + 0.1 * _randn((inner,), 9)).to(BF16).to(DEVICE)

    def run(wait):
        ws = plan.allocate_workspace(0.1)
        weight, x = torch.empty((inner, inner), device=DEVICE), _randn((rows, inner), 7, BF16).to(DEVICE)
        stream = torch.zeros_like(x)
        wc, wscale = empty_codes((inner, inner), DEVICE), torch.empty(inner, device=DEVICE)
        for k in range(30):
            if k % 5:
                rms_norm_int8(x, gain, stream, codes=ws.codes, scales=ws.scales, residual_out=stream)
            else:
                quantize_rows(x, codes=ws.codes, scales=ws.scales)
            wait()
            linear_int8(ws.codes, ws.scales, packed[k % 3].codes, packed[k % 3].scales, out=x)
            wait()
            weight.fill_(0.001 * k)  # a kernel of another library in between
            weight.diagonal().add_(x[0].float())
            quantize_rows(weight, codes=wc, scales=wscale)  # a weight that the next call reads at once
            wait()
            linear_int8(ws.codes, ws.scales, wc, wscale, out=x)
            wait()
        return x.clone(), stream.clone()

    expected = run(torch.cuda.synchronize)
    for _ in range(3):
        got = run(lambda: None)
        assert torch.equal(got[0], expected[0]) and torch.equal(got[1], expected[1])


def test_torch_operators_match_and_compile():
    x, r = _randn((2, 9, 100), 1, BF16).to(DEVICE), _randn((2, 9, 100), 2, BF16).to(DEVICE)
    weight = torch.ones(100, dtype=BF16, device=DEVICE)
    w, ws = torch.ops.rdna3_fastmm.quantize_rows_int8(_randn((48, 100), 3).to(DEVICE))
    codes, scales, h = torch.ops.rdna3_fastmm.rms_norm_int8(x, weight, r, 1e-6)
    expected = rms_norm_int8(x, weight, r, 1e-6)
    assert torch.equal(codes, expected.codes) and torch.equal(scales, expected.scales)
    assert torch.equal(h, expected.residual)
    assert torch.ops.rdna3_fastmm.rms_norm_int8(x, weight)[2].shape == (0,)
    y = torch.ops.rdna3_fastmm.linear_int8(codes, scales, w, ws)
    assert torch.equal(y, linear_int8(codes, scales, w, ws))

    def layer(x, r):
        codes, scales, h = torch.ops.rdna3_fastmm.rms_norm_int8(x, weight, r, 1e-6)
        return torch.ops.rdna3_fastmm.linear_int8(codes, scales, w, ws), h

    with torch.no_grad():
        compiled = torch.compile(layer, backend="aot_eager", fullgraph=True)
        got = compiled(x, r)
    assert torch.equal(got[0], y) and torch.equal(got[1], h)


# ---------------------------------------------------------------- refusals
def test_refusals():
    x = torch.ones((4, 64), dtype=BF16, device=DEVICE)
    gain = torch.ones(64, device=DEVICE)
    codes, scales = quantize_rows(x)
    w, ws = quantize_rows(torch.ones((8, 64), device=DEVICE))
    with pytest.raises(ValueError, match="autograd"):
        quantize_rows(x.clone().requires_grad_(True))
    with torch.no_grad():
        quantize_rows(x.clone().requires_grad_(True))
    with pytest.raises(ValueError, match="8-bit operators take"):
        quantize_rows(x.double())
    with pytest.raises(ValueError, match="at least one element"):
        quantize_rows(x[:, :0])
    with pytest.raises(ValueError, match="codes has shape"):
        quantize_rows(x, codes=codes[:3])
    with pytest.raises(ValueError, match="scales must be contiguous"):
        quantize_rows(x, scales=torch.empty((8,), device=DEVICE)[::2])
    with pytest.raises(ValueError, match="overlap"):
        quantize_rows(x, codes=x.view(torch.int8)[:, :64])
    with pytest.raises(ValueError, match="dense rows"):
        quantize_rows(x, codes=torch.empty((64, 4), dtype=torch.int8, device=DEVICE).t())
    with pytest.raises(ValueError, match="BF16 or FP16"):
        rms_norm_int8(x.float(), gain)
    with pytest.raises(ValueError, match="weight has shape"):
        rms_norm_int8(x, gain[:32])
    with pytest.raises(ValueError, match="weight must have"):
        rms_norm_int8(x, gain.half())
    with pytest.raises(ValueError, match="eps"):
        rms_norm_int8(x, gain, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        rms_norm_int8(x, gain, eps=float("nan"))
    with pytest.raises(ValueError, match="residual must have"):
        rms_norm_int8(x, gain, x[:2])
    with pytest.raises(ValueError, match="needs a residual"):
        rms_norm_int8(x, gain, residual_out=x.clone())
    wide = torch.ones((4, 96), dtype=BF16, device=DEVICE)
    with pytest.raises(ValueError, match="residual_out must be"):
        rms_norm_int8(wide[:, :64], gain, x, residual_out=wide[:, 16:80])
    # columns of one buffer beside each other are apart
    beside = torch.ones((4, 128), dtype=BF16, device=DEVICE)
    rms_norm_int8(beside[:, :64], gain, x, residual_out=beside[:, 64:])
    with pytest.raises(ValueError, match="do not form a linear"):
        linear_int8(codes, scales, w[:, :32], ws)
    with pytest.raises(ValueError, match="int8 tensors"):
        linear_int8(x, scales, w, ws)
    with pytest.raises(ValueError, match="scales has shape"):
        linear_int8(codes, scales[:2], w, ws)
    with pytest.raises(ValueError, match="weight_scales must be float32"):
        linear_int8(codes, scales, w, ws.half())
    with pytest.raises(ValueError, match="writes BF16 or FP16"):
        linear_int8(codes, scales, w, ws, dtype=FP32)
    with pytest.raises(ValueError, match="bias must be"):
        linear_int8(codes, scales, w, ws, torch.ones(8, device=DEVICE), dtype=BF16)
    with pytest.raises(ValueError, match="16-byte"):
        linear_int8(torch.zeros((4, 65), dtype=torch.int8, device=DEVICE)[:, :64], scales, w, ws)
    with pytest.raises(ValueError, match="16-byte"):
        linear_int8(torch.zeros((4, 80), dtype=torch.int8, device=DEVICE)[:, 1:65], scales, w, ws)
    with pytest.raises(ValueError, match="overlap"):
        linear_int8(codes, scales, w, ws, out=codes.view(BF16)[:, :8])
    big = torch.zeros((1, 131072), dtype=torch.int8, device=DEVICE)
    with pytest.raises(ValueError, match="32-bit sum"):
        linear_int8(big, scales[:1], big, ws[:1])
    with pytest.raises(ValueError, match="CUDA"):
        quantize_rows(x.cpu())
    with pytest.raises(ValueError, match="one device"):
        linear_int8(codes, scales, w.cpu(), ws)


def test_plan_refusals():
    plan = Int8Plan(4, 64, 8, DEVICE)
    weight = torch.ones((8, 64), dtype=BF16, device=DEVICE)
    packed, ws = plan.pack_weight(weight, 0.1), plan.allocate_workspace(0.1)
    x = torch.ones((4, 64), dtype=BF16, device=DEVICE)
    with pytest.raises(MemoryError):
        Int8Plan(2**30, 65536, 8, DEVICE).allocate_workspace()
    with pytest.raises(ValueError, match="weight matrix has shape"):
        plan.pack_weight(weight[:4])
    with pytest.raises(ValueError, match="device or dtype"):
        plan.pack_weight(weight.half())
    with pytest.raises(ValueError, match="left matrix has shape"):
        plan.run_linear_packed(x[:2], packed, ws)
    with pytest.raises(ValueError, match="workspace does not match"):
        plan.run_linear_packed(x, packed, Int8Plan(5, 64, 8, DEVICE).allocate_workspace(0.1))
    with pytest.raises(ValueError, match="shape does not match"):
        plan.run_linear_packed(x, Int8Plan(4, 64, 9, DEVICE).pack_weight(torch.ones((9, 64), device=DEVICE)), ws)
    with pytest.raises(ValueError, match="does not match the plan"):
        plan.run_linear_packed(x, Int8Plan(4, 64, 8, DEVICE, FP16).pack_weight(weight.half()), ws)
    with pytest.raises(ValueError, match="overlap"):
        plan.run_linear_packed(x, packed, ws, output=x[:, :8])
    r = x.clone()
    with pytest.raises(ValueError, match="overlap"):
        plan.run_norm_linear_packed(x, torch.ones(64, device=DEVICE), packed, ws, r, output=r[:, :8],
                                    residual_output=r)
    # a product that is refused leaves the stream as it was
    before = r.clone()
    for wrong in (dict(bias=torch.ones(8, device=DEVICE)), dict(bias=torch.ones(9, dtype=BF16, device=DEVICE)),
                  dict(output=torch.empty((4, 9), dtype=BF16, device=DEVICE)),
                  dict(output=torch.empty((4, 8), dtype=FP16, device=DEVICE)),
                  dict(output=ws.codes.view(BF16)[:, :8])):
        with pytest.raises(ValueError):
            plan.run_norm_linear_packed(x, torch.ones(64, device=DEVICE), packed, ws, r, residual_output=r, **wrong)
    assert torch.equal(r, before)
    other = Int8Plan(6, 64, 8, DEVICE)
    out = other.run_linear_packed(torch.ones((6, 64), dtype=BF16, device=DEVICE), packed,
                                  other.allocate_workspace(0.1))
    assert out.shape == (6, 8)  # a packed weight serves other row counts


def test_negated_views_are_refused():
    """Their storage holds the other sign; the torch operators are given resolved ones."""
    z = torch.randn(5, 64, device=DEVICE, dtype=torch.complex64)
    x = z.conj().imag
    assert x.is_neg()
    rows = x.resolve_neg()
    codes, scales = quantize_rows(rows)
    assert torch.equal(torch.ops.rdna3_fastmm.quantize_rows_int8(x)[0], codes)
    half = rows.to(FP16)
    gain, neg = torch.ones(64, device=DEVICE, dtype=FP16), torch._neg_view
    w, ws = quantize_rows(torch.randn(24, 64, device=DEVICE))
    bias, out = torch.ones(24, device=DEVICE, dtype=FP16), torch.zeros(5, 24, device=DEVICE, dtype=FP16)
    plan = Int8Plan(5, 64, 24, torch.device(DEVICE), FP16)
    packed, workspace = plan.pack_weight(rows.new_ones(24, 64)), plan.allocate_workspace()
    workspace.codes.fill_(3)
    for call in (lambda: quantize_rows(x),
                 lambda: quantize_rows(rows, scales=neg(scales.clone())),
                 lambda: rms_norm_int8(neg(half), gain),
                 lambda: rms_norm_int8(half, neg(gain)),
                 lambda: rms_norm_int8(half, gain, neg(half)),
                 lambda: rms_norm_int8(half, gain, half, residual_out=neg(half.clone())),
                 lambda: linear_int8(codes, neg(scales), w, ws),
                 lambda: linear_int8(codes, scales, w, neg(ws)),
                 lambda: linear_int8(codes, scales, w, ws, neg(bias)),
                 lambda: linear_int8(codes, scales, w, ws, out=neg(out)),
                 lambda: plan.run_linear_packed(neg(half), packed, workspace),
                 lambda: plan.run_linear_packed(half, packed, workspace, neg(bias)),
                 lambda: plan.run_linear_packed(half, packed, workspace, output=neg(out))):
        with pytest.raises(ValueError, match="negated"):
            call()
    assert (workspace.codes == 3).all()
    assert (out == 0).all()
