"""Expired waits in the fused GEMM kernels and the mixture-of-experts layer: with a wait budget of one clock cycle
(mxfp6_set_wait_budget) a kernel gives up, reports MXFP6_DEV_* bits and returns, clusters included; the next call with
the default budget is right."""
from __future__ import annotations

import pytest
import torch

import mxfp6_b200 as lib
from fused_ref import Operand, check_rounded, fused64
from mxfp6_b200 import Act, AuxOp, OutType
from test_moe_gpu import Layer, _moe, _randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _expire(call):
    assert lib.device_status() == 0
    prev = lib.set_wait_budget(1)
    try:
        assert call() == lib.OK
        status = lib.device_status()
    finally:
        lib.set_wait_budget(prev)
    assert status != -1 and status & 0x7, hex(status)


# few rows over clusters of 8; the single-CTA tile; the pair; the column layout; long K so that no wait is met at once
@pytest.mark.parametrize("M,N,K", [(5, 2048, 12288), (300, 512, 12288), (2048, 4096, 8192), (300, 513, 12288)])
def test_fused(M, N, K):
    A, B = Operand(M, K, 1.0, 1), Operand(N, K, K ** -0.5, 2)
    bias = _randn(N, seed=3)
    ep = lib.Epilogue(bias, OutType.F32, Act.SILU)
    D = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    call = lambda: lib.gemm_fused(OutType.BF16, M, N, A.Kp, A.packed, B.packed, A.scales, B.scales, D, A.row_bytes,  # noqa: E731
                                  B.row_bytes, ep)
    _expire(call)
    assert call() == lib.OK
    torch.cuda.synchronize()
    assert lib.device_status() == 0
    check_rounded(D, *fused64(A, B, Act.SILU, bias, None, AuxOp.NONE), OutType.BF16)


@pytest.mark.parametrize("gated", [True, False])
def test_moe(gated):
    layer = Layer(8, 4096, 1024, gated)
    T, k = 20, 2
    x = _randn(T, 4096, seed=4, dtype=torch.bfloat16)
    ids = torch.arange(T * k, device="cuda").view(T, k).int() % 8
    w = _randn(T, k, seed=5)
    n = lib.moe_workspace_size(layer.layer, T, k)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    out = torch.empty(T, 4096, device="cuda")
    _expire(lambda: lib.moe(layer.layer, OutType.F32, T, k, x, OutType.BF16, out, ws, n, ids=ids, weights=w))
    check_rounded(_moe(layer, OutType.F32, x, OutType.BF16, k, ids=ids, weights=w), *layer.reference(x, ids, w), OutType.F32)


def test_moe_long_inter():
    """The down product in segments (FP32 output, inter above 12288)."""
    layer = Layer(2, 1024, 24704)
    T, k = 20, 1
    x = _randn(T, 1024, seed=6, dtype=torch.bfloat16)
    ids = torch.arange(T, device="cuda").view(T, 1).int() % 2
    w = _randn(T, k, seed=7)
    n = lib.moe_workspace_size(layer.layer, T, k)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    out = torch.empty(T, 1024, device="cuda")
    _expire(lambda: lib.moe(layer.layer, OutType.F32, T, k, x, OutType.BF16, out, ws, n, ids=ids, weights=w))
    check_rounded(_moe(layer, OutType.F32, x, OutType.BF16, k, ids=ids, weights=w), *layer.reference(x, ids, w), OutType.F32)
