"""FP64 reference of the fused operators: plain restatements of their formulas, for the tests."""
from __future__ import annotations

import math

import numpy as np
import torch

import mxfp6_b200 as lib

DTYPE = {lib.OutType.F32: torch.float32, lib.OutType.F16: torch.float16, lib.OutType.BF16: torch.bfloat16}
# Steepest slope of each activation: an error e of its input becomes at most slope * e.
SLOPE = {lib.Act.NONE: 1.0, lib.Act.RELU: 1.0, lib.Act.GELU: 1.13, lib.Act.GELU_TANH: 1.13, lib.Act.SILU: 1.1}


def act64(act, v):
    if act == lib.Act.RELU:
        return torch.where(v < 0, torch.zeros_like(v), v)
    if act == lib.Act.GELU:
        return v * 0.5 * torch.special.erfc(-v * math.sqrt(0.5))
    if act == lib.Act.GELU_TANH:
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    if act == lib.Act.SILU:
        return v / (1 + torch.exp(-v))
    return v


def values(packed: np.ndarray, scales: np.ndarray, rows: int, cols: int) -> torch.Tensor:
    """Packed codes and raw scales -> FP64 values on the GPU (every one exact in FP32)."""
    q = lib.QuantizedMatrix(np.ascontiguousarray(packed[:, :cols * 3 // 4]), np.ascontiguousarray(scales), rows, cols)
    return torch.from_numpy(lib.dequantize_mxfp6(q)).cuda().double()


class Operand:
    """A quantised [rows][K] matrix: host packed / raw scales, device packed / tiled scales, FP64 values.
    row_bytes: the packed stride (0.75*kpad(K) by default; the compact 0.75*K is allowed for A)."""

    def __init__(self, rows, K, std, seed, row_bytes=None):
        self.rows, self.K, self.Kp = rows, K, lib.kpad(K)
        x = np.random.default_rng(seed).standard_normal((rows, K), dtype=np.float32) * np.float32(std)
        q = lib.quantize_to_mxfp6(x)
        self.row_bytes = row_bytes or self.Kp * 3 // 4
        host = np.zeros((rows, self.row_bytes), np.uint8)
        host[:, :K * 3 // 4] = q.packed_data
        self.packed = torch.from_numpy(host).cuda()
        self.scales = torch.from_numpy(lib.preprocess_scale(lib.pad_scales_k(q.scales, rows, K), rows, self.Kp)).cuda()
        self.values = values(q.packed_data, q.scales, rows, K)


def fused64(A: Operand, B: Operand, act, bias, aux, aux_op):
    """(op(act(A·B^T + bias), aux) in FP64, a bound on the kernel's error before its output rounding).

    The accumulator is within 1e-5 of max|A·B^T| (the library's FP32 tolerance); bias, the activation's
    exponential and quotient and the aux operation round in FP32 a few times: 2^-20 of the largest
    magnitude on the way covers them (each is at most 2^-24 * 4)."""
    acc = A.values @ B.values.T
    v = acc if bias is None else acc + bias.double()
    tol = 1e-5 * acc.abs().max() + 2.0 ** -22 * v.abs()
    h = act64(act, v)
    tol = SLOPE[act] * tol + 2.0 ** -20 * v.abs()
    if aux_op == lib.AuxOp.ADD:
        return h + aux.double(), tol + 2.0 ** -23 * (h.abs() + aux.double().abs())
    if aux_op == lib.AuxOp.MUL:
        return h * aux.double(), (tol + 2.0 ** -23 * h.abs()) * aux.double().abs()
    return h, tol


def check_rounded(got, ref, tol, ot, label=""):
    """got: ref rounded to the output type, within tol plus half a step of that type."""
    eps = torch.finfo(DTYPE[ot]).eps
    tiny = torch.finfo(DTYPE[ot]).smallest_normal * eps
    err = (got.double() - ref).abs()
    bad = ~(err <= tol + eps / 2 * (ref.abs() + tol) + tiny)
    assert not bad.any(), f"{label}: {int(bad.sum())} of {bad.numel()} off, worst {float((err - tol).max()):.3e}"


def check_quantised(packed, raw, ref, tol, label=""):
    """MXFP6 rows of values within tol of ref: each scale is the smallest power of two >= max / 7.5 for
    some maximum within tol of ref's, each code within half a step of its binade of the value."""
    rows, cols = ref.shape
    s = torch.from_numpy(raw.astype(np.int32)).cuda().double() - 127
    top, slack = ref.abs().view(rows, -1, 32).amax(-1), tol.expand_as(ref).reshape(rows, -1, 32).amax(-1)
    lo = torch.ceil(torch.log2((top - slack).clamp(min=1e-300) / 7.5))
    hi = torch.ceil(torch.log2((top + slack).clamp(min=1e-300) / 7.5))
    zero = (top <= slack) & (s == 0)  # a block of zeros has code 127
    assert (zero | ((s >= lo) & (s <= hi))).all(), f"{label}: scales off"
    got = values(packed, raw, rows, cols)
    scale = torch.exp2(s).repeat_interleave(32, 1)
    m = (got / scale).abs()
    step = torch.where(m < 2, 0.125, torch.where(m < 4, 0.25, 0.5)) * scale
    err = (got - ref).abs()
    assert (err <= step / 2 + tol).all(), f"{label}: codes off by {float((err - step / 2 - tol).max()):.3e}"
