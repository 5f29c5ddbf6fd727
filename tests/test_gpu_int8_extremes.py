"""Rows of the 8-bit operators whose FP32 totals say too little, in every form
of the row kernels: against their formulas in 64 bits, codes by equality."""

import pytest
import torch

from int8_kernels import kernels_of
from rdna3_fastmm.int8 import quantize_rows, rms_norm_int8

pytestmark = pytest.mark.gpu
DEVICE = torch.device("cuda", 0)
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
U32 = 2.0**-24  # half a step of FP32

# rows of a warp or a block in registers, vectors and elements; rows read
# twice; streamed rows of one warp and of several, vectors and elements
REGISTERS = [(25, 40), (24, 301), (26, 700), (25, 1001), (24, 5001), (23, 8200), (23, 40000)]
STREAMED = [(9700, 600), (9700, 601), (3700, 4608), (2700, 4607)]
FORMS = [(*shape, "int8_rows_kernel") for shape in REGISTERS] + [(*shape, "int8_rows_streamed_kernel")
                                                                 for shape in STREAMED]


def _randn(shape, seed, dtype=FP32, scale=1.0):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, device=DEVICE)).to(dtype)


def _special(x, values):
    """Every third row takes the next of `values`, a factor or a function of the row."""
    for n, row in enumerate(range(1, x.shape[0], 3)):
        value = values[n % len(values)]
        x[row] = value(x[row].clone()) if callable(value) else x[row] * value
    return x


def _last(value):
    def change(row):
        row[-1] = value
        return row
    return change


def _roundings(inner):
    # a thread adds at most 96 squares one after another (12 vectors of 8 of a
    # streamed row, or 144 elements of one that is not aligned; 32 of a row in
    # registers; 8 a pass of 1024 threads of a longer one), then up to 12 joins
    # or 17; the root halves what the mean is off, five roundings follow
    return (max(144, 8 * -(-inner // 8192)) + 17) / 2 + 5


def _check(got, p, h, eps, inner):
    """Codes and scales against rows p (64 bits) of the stream h; h None: no norm."""
    codes, scales = got
    finite = p.isfinite().all(dim=1)
    if h is not None:
        finite &= h.float().square().isfinite().all(dim=1)
    p = torch.where(finite[:, None], p, 0.0)
    peak = p.abs().amax(dim=1)
    expected = torch.round(127.0 * p / torch.where(peak > 0, peak, 1.0)[:, None])
    assert torch.equal(codes, expected.to(torch.int8))
    scale = peak / 127.0
    if h is not None:
        mean = torch.where(finite[:, None], h.double(), 0.0).square().mean(dim=1) + eps
        scale = torch.where(peak > 0, scale * torch.rsqrt(mean), 0.0)
    finite &= scale < torch.finfo(FP32).max
    assert bool((scales[~finite].isnan()).all()) and not codes[~finite].any()
    roundings = 1 if h is None else _roundings(inner)
    error = (scales.double() - scale).abs()[finite]
    # and half a step of FP32's subnormals
    assert bool((error <= roundings * U32 * scale[finite] + 2.0**-150).all())


def _check_norm(x, gain, residual, eps, kernel):
    got = rms_norm_int8(x, gain, residual, eps)
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    if residual is not None:
        assert bool(((got.residual == h) | (got.residual.isnan() & h.isnan())).all())
    _check(got[:2], h.double() * gain.double(), h, eps, x.shape[1])
    assert kernels_of(lambda: rms_norm_int8(x, gain, residual, eps)) == [kernel]


EACH = [pytest.mark.parametrize("rows,inner,kernel", FORMS), pytest.mark.parametrize("gain_type", ["same", "fp32"]),
        pytest.mark.parametrize("with_residual", [False, True])]


def each(function):
    for mark in EACH:
        function = mark(function)
    return function


@each
def test_rows_without_a_code_and_rows_of_small_values(rows, inner, kernel, gain_type, with_residual):
    """Zeros, infinities, NaN, squares beyond FP32, and values next to nothing beside the epsilon."""
    values = [0.0, _last(float("inf")), 2.0**-112, _last(float("nan")), _last(2.0**70), _last(-2.0**-124), 2.0**-118]
    x = _special(_randn((rows, inner), 1, BF16), values)
    residual = x.clone() if with_residual else None  # x + x is exact
    gain = (1 + 0.2 * _randn((inner,), 2)).to(FP32 if gain_type == "fp32" else BF16)
    _check_norm(x, gain, residual, 1e-5, kernel)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows,inner,kernel", FORMS)
def test_quantised_rows_of_extreme_magnitude(rows, inner, kernel, dtype):
    values = [0.0, _last(float("inf")), 2.0**-130, _last(float("nan")), 2.0**120, 2.0**-110, _last(-2.0**-133)]
    x = _special(_randn((rows, inner), 1, dtype), values)
    _check(quantize_rows(x), x.double(), None, 0.0, inner)
    assert kernels_of(lambda: quantize_rows(x)) == [kernel]


@each
def test_products_below_the_normal_range(rows, inner, kernel, gain_type, with_residual):
    """Rows whose products are subnormal numbers of FP32, or less than those."""
    x = _special(_randn((rows, inner), 3, BF16), [2.0**-70, 2.0**-50, 2.0**-90, 0.0, 2.0**-71, _last(2.0**-60)])
    residual = x.clone() if with_residual else None
    gain = ((1 + 0.2 * _randn((inner,), 4)) * 2.0**-77).to(FP32 if gain_type == "fp32" else BF16)
    _check_norm(x, gain, residual, 1e-6, kernel)


@each
def test_squares_outside_the_range_of_fp32(rows, inner, kernel, gain_type, with_residual):
    """Squares that underflow with no epsilon to cover it, and sums of finite squares that overflow."""
    x = _special(_randn((rows, inner), 5, BF16), [2.0**-76, 2.0**-66, 0.0, 2.0**60, 2.0**-61, 2.0**-100, 2.0**-120])
    residual = x.clone() if with_residual else None
    gain = (1 + 0.2 * _randn((inner,), 6)).to(FP32 if gain_type == "fp32" else BF16)
    _check_norm(x, gain, residual, 0.0, kernel)
    _check_norm(x, gain, residual, 2.0**-140, kernel)


@each
def test_products_beyond_the_range_of_fp32(rows, inner, kernel, gain_type, with_residual):
    """Finite values times a finite gain, whose norm is finite again."""
    x = _special(_randn((rows, inner), 7, BF16), [16.0, 0.0, 2.0**-30, 2.0**60, _last(float("inf"))])
    residual = x.clone() if with_residual else None
    gain = ((1 + 0.1 * _randn((inner,), 8)).clamp(0.5, 1.5) * 2.0**125).to(FP32 if gain_type == "fp32" else BF16)
    _check_norm(x, gain, residual, 1e-6, kernel)


def test_a_scale_beyond_fp32_is_nan():
    x = torch.zeros((3, 40000), dtype=BF16, device=DEVICE)
    x[0, 7], x[1, 3], x[2] = 1.0, -5.0, 1.0
    gain = torch.full((40000,), torch.finfo(FP32).max, device=DEVICE)
    codes, scales, _ = rms_norm_int8(x, gain, eps=0.0)  # 200 times the gain, over 127
    assert scales[:2].isnan().all() and not codes[:2].any()
    assert bool((codes[2] == 127).all()) and abs(scales[2].item() * 127.0 / torch.finfo(FP32).max - 1) < 4 * U32


@pytest.mark.parametrize("gain", [0.0, float("inf"), float("nan")])
@pytest.mark.parametrize("rows,inner", [(4, 300), (4, 5000), (9700, 600)])
def test_gains_without_a_value(rows, inner, gain):
    """A gain of zeros gives zeros; one that is not finite gives rows that are not."""
    x = _special(_randn((rows, inner), 9, BF16), [0.0, 2.0**-100])
    weight = torch.zeros(inner, dtype=BF16, device=DEVICE)
    weight[inner // 2] = gain
    for eps in (1e-6, 0.0):
        codes, scales, _ = rms_norm_int8(x, weight, eps=eps)
        assert not codes.any()
        assert bool((scales == 0).all()) if gain == 0.0 else bool(scales.isnan().all())
