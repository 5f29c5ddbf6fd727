"""Every kernel of the 8-bit operators, by name, against the formulas in 64
bits at the sizes where its tiles, its groups and its ends differ."""

import pytest
import torch

from int8_kernels import kernels_of
from rdna3_fastmm.int8 import empty_codes, linear_int8, quantize_rows, rms_norm_int8

pytestmark = pytest.mark.gpu
DEVICE = torch.device("cuda", 0)
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
U32 = 2.0**-24  # half a step of FP32
FEW, SINGLE, PAIR = "int8_linear_few_kernel", "int8_linear_kernel", "int8_linear_pair_kernel"


def _codes(rows, inner, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    codes = torch.randint(-128, 128, (rows, inner), generator=g, dtype=torch.int8, device=DEVICE)
    return empty_codes((rows, inner), DEVICE).copy_(codes)


def _positive(count, seed, scale):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    return scale * (0.5 + torch.rand(count, generator=g, device=DEVICE))


def _check_linear(rows, inner, columns, dtype, with_bias, kernel, pitch=None):
    codes, w = _codes(rows, inner, 1), _codes(columns, inner, 2)
    scales, ws = _positive(rows, 3, 0.01), _positive(columns, 4, 0.002)
    bias = torch.randn(columns, device=DEVICE).to(dtype) if with_bias else None
    buffer = torch.full((rows + 1, pitch or columns), 7.0, dtype=dtype, device=DEVICE)
    out = buffer[:rows, :columns]
    linear_int8(codes, scales, w, ws, bias, out=out)
    # FP64 holds the sums; FP32: the sum, the scales' product, theirs, the
    # bias, then one rounding to dtype of a value 4 roundings off
    y = (codes.double() @ w.double().t()) * scales.double()[:, None] * ws.double()
    size = y.abs()
    if with_bias:
        y += bias.double()
        size += bias.double().abs()
    info = torch.finfo(dtype)
    fp32 = 4 * U32 * size
    allowed = fp32 + (y.abs() + fp32) * info.eps / 2 + info.smallest_normal * info.eps / 2
    assert bool(((out.double() - y).abs() <= allowed).all())
    out.fill_(7.0)
    assert bool((buffer == 7.0).all())
    assert kernels_of(lambda: linear_int8(codes, scales, w, ws, bias, out=out)) == [kernel]


# Two SMs a tile: whole and ragged tiles of tokens (a last one of 1, of 16, of
# 17 and of 255 of 256), channels that end in the first or the second SM's
# half, K that ends in the first or the second half of a 256-deep stage, or
# inside 16 codes, and K on either side of 2048, where the epilogue's warps change
PAIRS = [(2048, 2048, 8192), (1281, 2100, 8193), (1283, 2305, 8320), (5000, 1030, 2500), (5008, 1153, 2433),
         (5119, 2049, 2600), (5000, 2047, 2496), (9473, 1000, 1100), (9472, 2100, 1025), (2033, 4097, 4000),
         (2064, 2176, 8191)]


@pytest.mark.parametrize("dtype,with_bias", [(BF16, True), (FP16, False)])
@pytest.mark.parametrize("rows,inner,columns", PAIRS)
def test_two_sms_a_tile(rows, inner, columns, dtype, with_bias):
    _check_linear(rows, inner, columns, dtype, with_bias, PAIR)


@pytest.mark.parametrize("rows,inner,columns,pitch", [(1283, 2100, 8193, 8200), (5000, 1030, 2500, 2501)])
def test_two_sms_a_tile_write_their_outputs_only(rows, inner, columns, pitch):
    _check_linear(rows, inner, columns, FP16, True, PAIR, pitch)


@pytest.mark.parametrize("rows,inner,columns,kernel", [
    (1, 4608, 12289, FEW), (2, 1000, 4000, FEW), (4, 4096, 500, FEW), (3, 4609, 8001, SINGLE), (33, 4096, 16383, SINGLE),
    (300, 1024, 37889, SINGLE), (600, 4096, 9472, SINGLE), (20003, 100, 304, SINGLE)])
def test_other_products_by_name(rows, inner, columns, kernel):
    _check_linear(rows, inner, columns, BF16, True, kernel)


# ---------------------------------------------------------------- rows
def _roundings(inner):
    # as many squares one after another as a thread of any form adds, then the
    # joins; the root halves what the mean is off, five roundings follow
    return (max(144, 8 * -(-inner // 8192)) + 17) / 2 + 5


def _check_rows(codes, scales, p, factor, roundings):
    peak = p.abs().amax(dim=1)
    expected = torch.round(127.0 * p / torch.where(peak > 0, peak, 1.0)[:, None])
    assert torch.equal(codes, expected.to(torch.int8))
    reference = peak * factor / 127.0
    assert bool(((scales.double() - reference).abs() <= roundings * U32 * reference).all())


def _rows(rows, inner, seed, dtype, offset, pitch):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    x = torch.randn(offset + rows * pitch, generator=g, device=DEVICE).to(dtype)
    x = x[offset:].view(rows, pitch)[:, :inner]
    x[rows // 2:rows // 2 + 40] = 0
    return x


# rows of one warp, of several, of a block; more of them than two for each of
# an SM's groups, which is where rows are streamed
STREAMED = [(9900, 264), (9700, 1032), (9000, 1800), (8100, 2048), (3700, 4608), (2000, 8200), (1000, 16384), (700, 24576)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("offset,more", [(0, 0), (0, 8), (1, 0), (3, 5), (4, 0)])
@pytest.mark.parametrize("rows,inner", STREAMED)
def test_streamed_quantisation(rows, inner, offset, more, dtype):
    inner -= offset == 3  # a width that is not whole vectors either
    if dtype == FP32 and inner > 24000:
        if offset % 4:
            pytest.skip("two stages of such a row and its codes do not fit")
        rows = 400
    x = _rows(rows, inner, 1, dtype, offset, inner + more)
    codes, scales = quantize_rows(x)
    _check_rows(codes, scales, x.double(), 1.0, 1)
    assert kernels_of(lambda: quantize_rows(x)) == ["int8_rows_streamed_kernel"]


@pytest.mark.parametrize("gain_type", ["same", "fp32"])
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("offset,more", [(0, 0), (1, 2)])
@pytest.mark.parametrize("rows,inner", [shape for shape in STREAMED if shape[1] < 24576] + [(400, 24576)])
def test_streamed_norms(rows, inner, offset, more, dtype, with_residual, gain_type):
    if inner == 24576 and (offset or with_residual):
        pytest.skip("two stages of such a row do not fit")
    x = _rows(rows, inner, 1, dtype, offset, inner + more)
    residual = _rows(rows, inner, 2, dtype, offset, inner + 2 * more) if with_residual else None
    gain = (1 + 0.3 * torch.randn(inner, generator=torch.Generator(device=DEVICE).manual_seed(3), device=DEVICE))
    gain = gain.to(FP32 if gain_type == "fp32" else dtype)
    h = x if residual is None else (x.float() + residual.float()).to(dtype)
    p, rstd = h.double() * gain.double(), torch.rsqrt(h.double().square().mean(dim=1) + 1e-5)
    codes, scales, stream = rms_norm_int8(x, gain, residual, 1e-5)
    _check_rows(codes, scales, p, rstd, _roundings(inner))
    assert kernels_of(lambda: rms_norm_int8(x, gain, residual, 1e-5)) == ["int8_rows_streamed_kernel"]
    if residual is not None:
        assert torch.equal(stream, h)
        x, residual = x.clone(), residual.clone()
        again = rms_norm_int8(x, gain, residual, 1e-5, residual_out=residual)  # in place
        assert torch.equal(residual, h)
        _check_rows(again.codes, again.scales, p, rstd, _roundings(inner))


# ---------------------------------------------------------------- compiled
@pytest.mark.parametrize("inner", [100, 112])
def test_operators_compile_with_inductor(inner):
    """Codes of a width that is not 16's multiple are views with a step of their own."""
    g = torch.Generator(device=DEVICE).manual_seed(1)
    x, r = (torch.randn((2, 9, inner), generator=g, device=DEVICE).to(BF16) for _ in range(2))
    gain = torch.ones(inner, dtype=BF16, device=DEVICE)
    w, ws = torch.ops.rdna3_fastmm.quantize_rows_int8(torch.randn((48, inner), generator=g, device=DEVICE))

    def layer(x, r):
        codes, scales, h = torch.ops.rdna3_fastmm.rms_norm_int8(x, gain, r, 1e-6)
        y = torch.ops.rdna3_fastmm.linear_int8(codes, scales, w, ws)
        codes, scales = torch.ops.rdna3_fastmm.quantize_rows_int8(x)
        return y, h, torch.ops.rdna3_fastmm.linear_int8(codes, scales, w, ws), codes

    with torch.no_grad():
        expected = layer(x, r)
        got = torch.compile(layer, fullgraph=True)(x, r)
    for a, b in zip(got, expected):
        assert torch.equal(a, b) and a.stride() == b.stride()
