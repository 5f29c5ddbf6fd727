"""Cases of the 8-bit integer operators: row quantisation, RMS norm with an
8-bit output, the 8-bit linear, and a norm with the linear that reads it.

The plain forms (``own`` false) are elementary torch operations; with ``own``
true the same inputs go through ``rdna3_fastmm.int8``.  Codes are symmetric
8-bit integers with one FP32 scale for each row (token or output channel) and
come back as the values that they stand for, code times scale.
"""

import math
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parent.parent
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

# the largest listed product and the largest listed row operator
MOST_PRODUCT = 65536 * 4608 * 12288
MOST_ROWS_INNER = 65536 * 4608


def _quant(name, rows, inner, dtype):
    return {"name": name, "op": "quant", "rows": rows, "inner": inner, "dtype": dtype}


def _norm(name, rows, inner, dtype, gain, residual):
    return {"name": name, "op": "norm", "rows": rows, "inner": inner, "dtype": dtype, "gain": gain,
            "residual": residual}


def _linear(name, rows, inner, columns, dtype, bias):
    return {"name": name, "op": "linear", "rows": rows, "inner": inner, "columns": columns, "dtype": dtype,
            "bias": bias}


def _layer(name, rows, inner, columns, dtype, bias):
    return {"name": name, "op": "layer", "rows": rows, "inner": inner, "columns": columns, "dtype": dtype,
            "gain": dtype, "residual": True, "bias": bias}


def listed():
    return [
        # one token's input of an MLP-down projection: latency alone
        _quant("quant-token", 1, 12288, "bf16"),
        # the MLP-down input of a whole video latent
        _quant("quant-4992x16384", 4992, 16384, "bf16"),
        # an FP32 master weight being packed, odd width
        _quant("quant-weight-fp32", 12288, 4607, "fp32"),
        # one token's norm before an MLP
        _norm("norm-token", 1, 4608, "bf16", "bf16", True),
        # a prompt's norm with an FP32 gain and no residual, rows not a multiple of anything
        _norm("norm-8214", 8214, 4608, "fp16", "fp32", False),
        # the residual stream of the largest batch
        _norm("norm-65536", 65536, 4608, "bf16", "bf16", True),
        # one token through an MLP-up projection: the weight's bytes alone
        _linear("linear-token", 1, 4608, 12288, "bf16", False),
        # an odd decode batch with bias, odd number of outputs
        _linear("linear-batch-33", 33, 4096, 16383, "fp16", True),
        # a short prompt: few tiles for 148 SMs
        _linear("linear-720", 720, 4096, 16384, "bf16", True),
        # the headline product
        _linear("linear-65536", 65536, 4608, 12288, "bf16", False),
        # norm and MLP-up of one decode step of eight sequences
        _layer("layer-8", 8, 4096, 12288, "bf16", False),
        # norm and MLP-up of a prompt
        _layer("layer-8214", 8214, 4608, 12288, "bf16", True),
    ]


def _spread(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(("quant", "norm", "linear", "linear", "layer"))
    while True:
        rows, inner, columns = _spread(rng, 1, 65536), _spread(rng, 64, 16384), _spread(rng, 64, 16384)
        # widths are odd at times, and multiples of 64 most of the time
        if rng.random() < 0.7:
            inner = -(-inner // 64) * 64
        if rng.random() < 0.7:
            columns = -(-columns // 64) * 64
        if rows * inner <= MOST_ROWS_INNER and (op in ("quant", "norm") or rows * inner * columns <= MOST_PRODUCT):
            break
    dtype = rng.choice(("bf16", "fp16"))
    if op == "quant":
        case = _quant("", rows, inner, rng.choice(("bf16", "fp16", "fp32")))
    elif op == "norm":
        case = _norm("", rows, inner, dtype, rng.choice((dtype, "fp32")), rng.random() < 0.7)
    elif op == "linear":
        case = _linear("", rows, inner, columns, dtype, rng.random() < 0.5)
    else:
        case = _layer("", rows, inner, columns, dtype, rng.random() < 0.5)
    del case["name"]
    return case


def _activations(rows, inner, g, dtype):
    """Gaussian tokens with a few loud channels, as residual streams have them,
    and a padded tail of empty tokens."""
    x = torch.randn((rows, inner), generator=g, device="cuda", dtype=torch.float32)
    loud = torch.exp(0.6 * torch.randn((inner,), generator=g, device="cuda"))
    x *= loud
    if rows >= 64:
        x[rows - rows // 64:] = 0
    return x.to(dtype)


def _codes(rows, inner, g):
    """8-bit codes and scales of Gaussian rows; code rows start on 16-byte
    boundaries, as the product reads them."""
    x = torch.randn((rows, inner), generator=g, device="cuda", dtype=torch.float32)
    peak = x.abs().amax(dim=1, keepdim=True)
    codes = torch.zeros((rows, -(-inner // 16) * 16), device="cuda", dtype=torch.int8)
    codes[:, :inner] = torch.round(x * (127.0 / peak)).to(torch.int8)
    scales = (peak[:, 0] / 127.0) * torch.exp(0.3 * torch.randn((rows,), generator=g, device="cuda"))
    return codes[:, :inner], scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, inner, dtype = case["rows"], case["inner"], DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] != "linear":
        s["x"] = _activations(rows, inner, g, dtype)
        # what a serving loop keeps for the codes of its tokens
        s["codes"] = torch.empty((rows, -(-inner // 16) * 16), device="cuda", dtype=torch.int8)[:, :inner]
        s["scales"] = torch.empty((rows,), device="cuda", dtype=torch.float32)
    if case["op"] in ("norm", "layer"):
        s["gain"] = (1 + 0.2 * torch.randn((inner,), generator=g, device="cuda")).to(DTYPES[case["gain"]])
        s["residual"] = _activations(rows, inner, g, dtype) if case["residual"] else None
        s["residual_out"] = torch.empty_like(s["x"]) if case["residual"] else None
    if case["op"] in ("quant", "norm"):
        s["values"] = torch.empty((rows, inner), device="cuda", dtype=dtype)
    if case["op"] == "linear":
        s["codes"], s["scales"] = _codes(rows, inner, g)
    if case["op"] in ("linear", "layer"):
        columns = case["columns"]
        s["weight_codes"], s["weight_scales"] = _codes(columns, inner, g)
        s["weight_scales"] *= 1 / math.sqrt(inner)
        s["bias"] = torch.randn((columns,), generator=g, device="cuda").to(dtype) if case["bias"] else None
        s["out"] = torch.empty((rows, columns), device="cuda", dtype=dtype)
    return s


# ------------------------------------------------------------------ plain forms
def _plain_rows(p):
    """(codes, FP32 peak) of rows given in 64 bits: codes next to a rounding
    border need the exact quotient."""
    peak = p.abs().amax(dim=1, keepdim=True)
    codes = torch.round(p * 127.0 / torch.where(peak > 0, peak, 1.0))
    return codes, peak[:, 0]


def _plain_quant(s):
    codes, peak = _plain_rows(s["x"].double())
    return codes, (peak / 127.0).float()


def _plain_norm(s):
    h = s["x"]
    if s["residual"] is not None:
        h = (h.float() + s["residual"].float()).to(h.dtype)
    codes, peak = _plain_rows(h.double() * s["gain"].double())
    mean = h.float().square().mean(dim=1)
    scales = (peak * torch.rsqrt(mean.double() + EPS) / 127.0).float()
    return codes, scales, h if s["residual"] is not None else None


def _plain_linear(s, codes, scales):
    total = codes.float() @ s["weight_codes"].float().t()
    out = total * (scales[:, None] * s["weight_scales"][None, :])
    if s["bias"] is not None:
        out = out + s["bias"].float()
    return out.to(s["out"].dtype)


def _plain_values(s, codes, scales):
    return (codes.float() * scales[:, None]).to(s["values"].dtype)


def _run_plain(s):
    op = s["case"]["op"]
    if op == "quant":
        codes, scales = _plain_quant(s)
        return {"values": _plain_values(s, codes, scales), "scales": scales}
    if op == "norm":
        codes, scales, residual = _plain_norm(s)
        return {"values": _plain_values(s, codes, scales), "scales": scales, "residual": residual}
    if op == "linear":
        return {"out": _plain_linear(s, s["codes"], s["scales"])}
    codes, scales, residual = _plain_norm(s)
    return {"out": _plain_linear(s, codes, scales), "residual": residual}


# ------------------------------------------------------------------ the framework
def _ops():
    path = str(ROOT / "rdna3-fastmm_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from rdna3_fastmm import int8

    return int8


def _run_own(s):
    ops = _ops()
    op = s["case"]["op"]
    if op == "quant":
        codes, scales = ops.quantize_rows(s["x"], codes=s["codes"], scales=s["scales"])
        return {"values": torch.mul(codes, scales[:, None], out=s["values"]), "scales": scales}
    if op == "linear":
        return {"out": ops.linear_int8(s["codes"], s["scales"], s["weight_codes"], s["weight_scales"], s["bias"],
                                       out=s["out"])}
    codes, scales, residual = ops.rms_norm_int8(s["x"], s["gain"], s["residual"], EPS, codes=s["codes"],
                                                scales=s["scales"], residual_out=s["residual_out"])
    if op == "norm":
        return {"values": torch.mul(codes, scales[:, None], out=s["values"]), "scales": scales,
                "residual": residual}
    return {"out": ops.linear_int8(codes, scales, s["weight_codes"], s["weight_scales"], s["bias"], out=s["out"]),
            "residual": residual}


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    rows, inner, size = case["rows"], case["inner"], DTYPES[case["dtype"]].itemsize
    columns = case.get("columns", 0)
    total, flops = 0, 0
    if case["op"] != "linear":
        total += rows * inner * size  # the tokens
        if case.get("residual"):
            total += 2 * rows * inner * size  # the residual in and out
        if "gain" in case:
            total += inner * DTYPES[case["gain"]].itemsize
        flops += rows * inner * (6 if "gain" in case else 3)
    if case["op"] != "layer":
        total += rows * inner + 4 * rows  # the codes and their scales, written or read
    if columns:
        total += columns * inner + 4 * columns + rows * columns * size + (columns * size if case["bias"] else 0)
        flops += 2 * rows * inner * columns
    return {"bytes": total, "flops": flops}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    result = {}
    if case["op"] == "linear":
        q, scale = s["codes"].double(), s["scales"].double()
    else:
        v = s["x"].double()
        gain = 1.0
        rstd = 1.0
        if case["op"] in ("norm", "layer"):
            if s["residual"] is not None:
                # the stream is kept in the tokens' type: rounded once, then read
                v += s["residual"].double()
                result["residual"] = v
                v = v.to(s["x"].dtype).double()
            else:
                result["residual"] = None
            gain = s["gain"].double()
            rstd = torch.pow(torch.linalg.vector_norm(v, dim=1).square() / case["inner"] + EPS, -0.5)
        v = v * gain
        top = torch.maximum(v.amax(dim=1), -v.amin(dim=1))
        q = torch.nan_to_num(torch.div(v * 127.0, top[:, None]), nan=0.0).round_()
        scale = top * rstd / 127.0
    if case["op"] in ("quant", "norm"):
        result["values"], result["scales"] = q * scale[:, None], scale
        return result
    out = torch.matmul(q, s["weight_codes"].double().t())
    out *= scale[:, None]
    out *= s["weight_scales"].double()
    if s["bias"] is not None:
        out += s["bias"].double()
    result["out"] = out
    return result
