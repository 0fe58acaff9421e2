"""Fused-epilogue GEMM (mxfp6_gemm_fused, mxfp6_gemm_fused_quant) and the typed quantiser against FP64
restatements of their formulas, over routes, odd sizes, strides, types and activations."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import mxfp6_b200 as lib
from fused_ref import DTYPE, Operand, act64, check_quantised, check_rounded, fused64, values
from mxfp6_b200 import Act, AuxOp, OutType

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _workspace(A, N, poison=True):
    n = lib.gemm_fused_workspace_size(A.rows, N, A.Kp, A.row_bytes)
    return (torch.full((n,), 0x5A, dtype=torch.uint8, device="cuda") if n else None), n


def _finish():
    torch.cuda.synchronize()
    assert lib.device_status() == 0


def _randn(*shape, seed, std=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def _fused(A, B, ot, act=Act.NONE, bias=None, bias_type=OutType.F32, aux=None, aux_type=OutType.F32, aux_op=AuxOp.NONE,
           ldd=None, offset=0, ws=True, stream=None):
    """Runs the call into a poisoned buffer with rows ldd apart, `offset` elements past an aligned base,
    and checks that nothing outside D was written."""
    M, N = A.rows, B.rows
    ldd = ldd or N
    buf = torch.full((offset + (M + 1) * ldd,), 1234.0, dtype=DTYPE[ot], device="cuda")
    D = buf[offset:offset + M * ldd].view(M, ldd)
    w, n = _workspace(A, N) if ws else (None, 0)
    ep = lib.Epilogue(bias, bias_type, act, aux, aux_type, aux_op)
    rc = lib.gemm_fused(ot, M, N, A.Kp, A.packed, B.packed, A.scales, B.scales, D, A.row_bytes, B.row_bytes, ep, w, n,
                        ldd=ldd, stream=stream)
    assert rc == lib.OK, lib.last_error_string()
    _finish()
    assert (buf[:offset] == 1234.0).all() and (D[:, N:] == 1234.0).all() and (buf[offset + M * ldd:] == 1234.0).all()
    return D[:, :N]


# Sizes that end inside tiles, chunks and scale atoms, on every tile and on split K; F32 rounds nothing.
@pytest.mark.parametrize("M,N,K", [(1, 1, 128), (1, 4096, 4096), (3, 33, 160), (5, 1000, 2080), (127, 129, 512),
                                   (129, 31, 96), (200, 264, 1024), (257, 513, 384), (1000, 2056, 768),
                                   (1, 128, 8192), (300, 2500, 512), (2049, 2500, 256)])
@pytest.mark.parametrize("ot", list(OutType))
def test_sizes(M, N, K, ot):
    A, B = Operand(M, K, 1.0, M + K), Operand(N, K, K ** -0.5, N + K)
    bias = _randn(N, seed=1)
    got = _fused(A, B, ot, Act.SILU, bias)
    check_rounded(got, *fused64(A, B, Act.SILU, bias, None, AuxOp.NONE), ot, f"{M}x{N}x{K}")


@pytest.mark.parametrize("act", list(Act))
@pytest.mark.parametrize("aux_op", list(AuxOp))
def test_activations_and_aux(act, aux_op):
    M, N, K = 70, 200, 256
    A, B = Operand(M, K, 2.0, 3), Operand(N, K, 0.1, 4)
    for ot, bt, at in ((OutType.F32, OutType.BF16, OutType.F16), (OutType.F16, OutType.F32, OutType.BF16),
                       (OutType.BF16, OutType.F16, OutType.F32)):
        bias, aux = _randn(N, seed=5, dtype=DTYPE[bt]), _randn(M, N + 9, seed=6, dtype=DTYPE[at])[:, 4:N + 4]
        got = _fused(A, B, ot, act, bias, bt, aux, at, aux_op)
        check_rounded(got, *fused64(A, B, act, bias, aux, aux_op), ot, f"{act.name} {aux_op.name} {ot.name}")


# Row and column layouts of the epilogue with an aux operand, whole and partial tiles, on the single-CTA tiles and the pair.
@pytest.mark.parametrize("M,N,K", [(100, 264, 512), (257, 777, 256), (2500, 1544, 256), (3000, 3001, 128)])
@pytest.mark.parametrize("ot,at", [(OutType.F32, OutType.F32), (OutType.F32, OutType.BF16), (OutType.BF16, OutType.BF16),
                                   (OutType.F16, OutType.F32)])
@pytest.mark.parametrize("pad", [0, 7])
def test_aux_layouts(M, N, K, ot, at, pad):
    A, B = Operand(M, K, 1.0, 41), Operand(N, K, K ** -0.5, 42)
    bias, aux = _randn(N, seed=43), _randn(M, N + pad, seed=44, dtype=DTYPE[at])[:, :N]
    got = _fused(A, B, ot, Act.SILU, bias, OutType.F32, aux, at, AuxOp.MUL)
    check_rounded(got, *fused64(A, B, Act.SILU, bias, aux, AuxOp.MUL), ot, f"{M}x{N}")


# Pitches and bases that allow wide accesses, 16-byte ones only by chance, or none.
@pytest.mark.parametrize("ldd,offset", [(256, 0), (264, 8), (257, 0), (300, 1), (256, 3)])
@pytest.mark.parametrize("ot", list(OutType))
def test_output_strides(ldd, offset, ot):
    A, B = Operand(140, 256, 1.0, 7), Operand(256, 256, 0.06, 8)
    got = _fused(A, B, ot, ldd=ldd, offset=offset)
    check_rounded(got, *fused64(A, B, Act.NONE, None, None, AuxOp.NONE), ot)


def _route_of(ot, M, N, K):
    return lib.route(ot, M, N, lib.kpad(K))


# One shape for each schedule: whole tiles on the pair, split K, stream-K tail, banded split.
@pytest.mark.parametrize("M,N,K,want", [(4096, 4700, 256, "pair"), (256, 250, 8192, "splits"),
                                        (4090, 3570, 6144, "stream_k"), (1500, 2040, 24576, "banded")])
def test_schedules(M, N, K, want):
    r = _route_of(OutType.BF16, M, N, K)
    assert (r["MT"] == 256 if want == "pair" else r["splits"] > 1 if want == "splits" else r[want]), r
    A, B = Operand(M, K, 1.0, 9), Operand(N, K, K ** -0.5, 10)
    bias, aux = _randn(N, seed=11), _randn(M, N, seed=12, dtype=torch.bfloat16)
    ref = fused64(A, B, Act.GELU, bias, aux, AuxOp.ADD)
    got = _fused(A, B, OutType.BF16, Act.GELU, bias, OutType.F32, aux, OutType.BF16, AuxOp.ADD)
    check_rounded(got, *ref, OutType.BF16, want)
    again = _fused(A, B, OutType.BF16, Act.GELU, bias, OutType.F32, aux, OutType.BF16, AuxOp.ADD)
    assert torch.equal(got, again)
    # without a workspace: whole tiles, the same tolerance
    got = _fused(A, B, OutType.BF16, Act.GELU, bias, OutType.F32, aux, OutType.BF16, AuxOp.ADD, ws=False)
    check_rounded(got, *ref, OutType.BF16, want + " without workspace")


def test_stream_k_flags_are_used_up():
    """A stream-K launch replayed from a graph has the tag of the capture: no flag of one replay may be left for the next,
    which would take over accumulators that are not written yet."""
    M, N, K = 4090, 3570, 6144
    assert _route_of(OutType.BF16, M, N, K)["stream_k"]
    A, B = Operand(M, K, 1.0, 9), Operand(N, K, K ** -0.5, 10)
    n = lib.gemm_fused_workspace_size(M, N, A.Kp, A.row_bytes)
    ws = torch.zeros(n, dtype=torch.uint8, device="cuda")
    D = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    s = torch.cuda.Stream()

    def call():
        assert lib.gemm_fused(OutType.BF16, M, N, A.Kp, A.packed, B.packed, A.scales, B.scales, D, A.row_bytes, B.row_bytes,
                              None, ws, n, stream=s) == lib.OK

    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        call()
    ref = fused64(A, B, Act.NONE, None, None, AuxOp.NONE)
    pairs = lib.stream_k_bytes() // (256 * 256 * 4 + 16)
    for _ in range(2):
        D.fill_(0)
        g.replay()
        _finish()
        check_rounded(D, *ref, OutType.BF16)
        flags = ws[pairs * 256 * 256 * 4:pairs * (256 * 256 * 4 + 16)].view(torch.int64)
        assert (flags == 0).all()
        assert ws[:pairs * 256 * 256 * 4].any()  # accumulators were handed over


@pytest.mark.parametrize("M,N,K,want", [(1, 128, 128, None), (33, 384, 160, None), (130, 512, 2048, None),
                                        (17, 2048, 4096, None), (64, 128, 256, None), (128, 640, 384, None), (200, 2048, 4096, "splits"), (2050, 6144, 512, None), (1500, 2048, 24576, "banded")])
def test_quantised_output(M, N, K, want):
    if want:
        r = _route_of(OutType.F16, M, N, K)
        assert r["splits"] > 1 and (want == "splits" or r[want]), r
    A, B = Operand(M, K, 1.0, 13), Operand(N, K, K ** -0.5, 14)
    bias, aux = _randn(N, seed=15), _randn(M, N, seed=16)
    bias[32:64] = -1e4  # a block that ReLU makes all zero: scale code 127
    rb = N * 3 // 4 + 32
    packed = torch.full((M + 1, rb), 0x5A, dtype=torch.uint8, device="cuda")
    scales = torch.full((lib.tiled_scale_bytes(M, N),), 0x5A, dtype=torch.uint8, device="cuda")
    w, n = _workspace(A, N)
    ep = lib.Epilogue(bias, OutType.F32, Act.RELU, aux, OutType.F32, AuxOp.MUL)
    rc = lib.gemm_fused_quant(M, N, A.Kp, A.packed, B.packed, A.scales, B.scales, packed, scales, A.row_bytes,
                              B.row_bytes, ep, w, n, packed_row_bytes=rb)
    assert rc == lib.OK, lib.last_error_string()
    _finish()
    host = packed.cpu().numpy()
    assert (host[:, N * 3 // 4:] == 0x5A).all() and (host[M] == 0x5A).all()
    tiled = scales.cpu().numpy()
    raw = lib.untile_scales(tiled, M, N)
    filled = tiled.copy()
    lib_rows = (M + 127) // 128 * 128  # rows past M in the last atom keep what they held
    if lib_rows > M:
        rest = lib.untile_scales(filled, lib_rows, N)[M:]
        assert (rest == 0x5A).all()
    ref, tol = fused64(A, B, Act.RELU, bias, aux, AuxOp.MUL)
    if N > 32:
        assert (raw[:, 1] == 127).all()
    check_quantised(host[:M], raw, ref, tol, f"{M}x{N}x{K}")


# The compact strides of A (0.75*K with K % 128 != 0): re-padded into the workspace, or loaded in place.
@pytest.mark.parametrize("M,N,K", [(5, 70, 96), (130, 300, 2080), (300, 2056, 480), (513, 520, 800), (1500, 2056, 480),
                                   (1500, 2003, 480), (1300, 1537, 288)])
@pytest.mark.parametrize("ws", [True, False])
def test_compact_a(M, N, K, ws):
    A, B = Operand(M, K, 1.0, 17, row_bytes=K * 3 // 4), Operand(N, K, K ** -0.5, 18)
    got = _fused(A, B, OutType.F16, Act.GELU_TANH, ws=ws)
    check_rounded(got, *fused64(A, B, Act.GELU_TANH, None, None, AuxOp.NONE), OutType.F16)


def test_compact_a_in_place_on_the_pair():
    """The loader warps under the pair's fused epilogue: scratch off, no workspace, both epilogue layouts."""
    prev = lib.set_repad_scratch(0)
    try:
        for N in (4704, 4699):
            M, K = 4096, 224
            assert _route_of(OutType.F16, M, N, K)["MT"] == 256
            A, B = Operand(M, K, 1.0, 45, row_bytes=K * 3 // 4), Operand(N, K, K ** -0.5, 46)
            bias, aux = _randn(N, seed=47), _randn(M, N, seed=48, dtype=torch.float16)
            got = _fused(A, B, OutType.F16, Act.RELU, bias, OutType.F32, aux, OutType.F16, AuxOp.ADD, ws=False)
            check_rounded(got, *fused64(A, B, Act.RELU, bias, aux, AuxOp.ADD), OutType.F16)
    finally:
        lib.set_repad_scratch(prev)


def test_residual_in_place_and_null_epilogue():
    A, B = Operand(100, 256, 1.0, 19), Operand(192, 256, 0.06, 20)
    D = _randn(100, 192, seed=21, dtype=torch.bfloat16)
    ref, tol = fused64(A, B, Act.NONE, None, D.clone(), AuxOp.ADD)
    ep = lib.Epilogue(aux=D, aux_type=OutType.BF16, aux_op=AuxOp.ADD)
    assert lib.gemm_fused(OutType.BF16, 100, 192, 256, A.packed, B.packed, A.scales, B.scales, D, 192, 192, ep) == lib.OK
    _finish()
    check_rounded(D, ref, tol, OutType.BF16)
    plain = torch.empty(128, 256, device="cuda")
    A, B = Operand(128, 256, 1.0, 22), Operand(256, 256, 0.06, 23)
    assert lib.gemm_fused(OutType.F32, 128, 256, 256, A.packed, B.packed, A.scales, B.scales, plain, 192, 192) == lib.OK
    want = torch.empty_like(plain)
    lib.gemm(OutType.F32, 128, 256, 256, A.packed, B.packed, A.scales, B.scales, want, 192, 192)
    _finish()
    assert torch.equal(plain, want)  # a null epilogue is gemm()


def test_special_values():
    A, B = Operand(64, 128, 1.0, 24), Operand(96, 128, 0.1, 25)
    bias, aux = torch.zeros(96, device="cuda"), torch.zeros(64, 96, device="cuda")
    bias[0], bias[1], bias[2] = float("inf"), float("-inf"), float("nan")
    bias[3], bias[4] = 3e38, -3e38
    aux[5, 10], aux[6, 11] = float("nan"), float("inf")
    for act in Act:
        got = _fused(A, B, OutType.F32, act, bias, OutType.F32, aux, OutType.F32, AuxOp.ADD)
        ref = fused64(A, B, act, bias, aux, AuxOp.ADD)[0]
        assert got[:, 2].isnan().all() and got[5, 10].isnan() and got[6, 11].isinf()
        assert (got[:, 0] == float("inf")).all()
        assert (got[:, 3] > 2e38).all()
        if act in (Act.RELU,):
            assert (got[:, 1] == 0).all() and (got[:, 4] == 0).all()
        fine = ref.isfinite() & (ref.abs() < 1e30)
        fine[:, 4] = False
        assert (got[fine].double() - ref[fine]).abs().max() < 1e-4


@pytest.mark.parametrize("M", [1, 5, 20, 130, 1030])
@pytest.mark.parametrize("N", [256, 257])
def test_values_beside_each_other(M, N):
    """Every ordered pair of extreme values in neighbouring columns: two values share a reciprocal."""
    inf, nan = float("inf"), float("nan")
    some = torch.tensor([0.0, -0.0, 1e-30, 0.7, -0.7, 6.5, -6.5, -8.0, 20.0, -44.0, 60.0, -90.0, 3e38, -3e38, inf, -inf])
    pairs = torch.stack([some[:, None].expand(16, 16), some[None].expand(16, 16)], -1)
    A, B = Operand(M, 128, 0.0, 40), Operand(N, 128, 1.0, 41)
    for first, poison in ((0, False), (1, False), (0, True)):
        v = torch.cat([pairs[:, 0:8], pairs[:, 8:16]])[16 * first:16 * first + 16].reshape(-1)
        v = torch.cat([v, torch.zeros(N - 256)])
        if poison:
            v[::2] = nan
        v = v.cuda()
        for act in Act:
            got = _fused(A, B, OutType.F32, act, v)
            assert (got == got[0]).logical_or(got.isnan()).all()
            got, x = got[0].double(), v.double()
            assert (got.isnan() == x.isnan()).all()
            low = x == -inf if act != Act.NONE else torch.zeros_like(x, dtype=torch.bool)
            fine = x.isfinite() & (x.abs() < 1e9)
            assert (got[low].abs() < 1e-16).all() and (got[x == inf] == inf).all()
            assert (got[x == 3e38] > 2.9e38).all() and (act == Act.NONE or (got[x == -3e38].abs() < 1e-16).all())
            # 2^-20 of the value as in fused64, and the 1e-17 that the negative tails end at
            assert ((got - act64(act, x)).abs() <= 2.0 ** -20 * x.abs() + 1e-17)[fine].all(), act


@pytest.mark.parametrize("M,N", [(6, 33), (20, 33), (40, 128), (200, 260), (300, 513)])
def test_rows_do_not_depend_on_each_other(M, N):
    A, B = Operand(M, 256, 2.0, 42), Operand(N, 256, 0.2, 43)
    order = torch.from_numpy(np.random.default_rng(44).permutation(M))
    P = Operand(M, 256, 2.0, 42)
    P.packed = A.packed[order.cuda()].contiguous()
    x = np.random.default_rng(42).standard_normal((M, 256), dtype=np.float32) * np.float32(2.0)
    q = lib.quantize_to_mxfp6(x[order.numpy()])
    P.scales = torch.from_numpy(lib.preprocess_scale(lib.pad_scales_k(q.scales, M, 256), M, 256)).cuda()
    for act in Act:
        assert torch.equal(_fused(P, B, OutType.F32, act), _fused(A, B, OutType.F32, act)[order.cuda()]), act


# Around the rows where the few-row kernel hands over, with a last chunk that ends inside a lane's four columns or not.
@pytest.mark.parametrize("M", [1, 2, 15, 17, 40, 41, 64, 65])
@pytest.mark.parametrize("N,K", [(1608, 2560), (1606, 640), (100, 12416)])
@pytest.mark.parametrize("ot", list(OutType))
def test_few_rows(M, N, K, ot):
    A, B = Operand(M, K, 1.0, 50), Operand(N, K, K ** -0.5, 51)
    bias, aux = _randn(N, seed=52), _randn(M, N, seed=53, dtype=DTYPE[ot])
    for act, op in ((Act.GELU, AuxOp.ADD), (Act.SILU, AuxOp.MUL), (Act.NONE, AuxOp.NONE)):
        a = None if op == AuxOp.NONE else aux
        got = _fused(A, B, ot, act, bias, aux=a, aux_type=ot, aux_op=op)
        check_rounded(got, *fused64(A, B, act, bias, a, op), ot, f"{M}x{N}x{K}")


def test_empty_and_stream():
    A, B = Operand(40, 256, 1.0, 26), Operand(64, 256, 0.06, 27)
    n0 = lib.launch_count()
    assert lib.gemm_fused(OutType.F16, 0, 64, 256, 0, 0, 0, 0, 0, 192, 192) == lib.OK
    assert lib.quantize_device_typed(0, OutType.BF16, 0, 32, 32, 32, 0, 0) == lib.OK
    assert lib.launch_count() == n0
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = _fused(A, B, OutType.F16, stream=s)
    check_rounded(got, *fused64(A, B, Act.NONE, None, None, AuxOp.NONE), OutType.F16)


@pytest.mark.parametrize("rows,cols,ld,padded,offset", [(1, 32, 32, 32, 0), (7, 96, 96, 128, 0), (130, 512, 513, 512, 0),
                                                        (33, 2080, 2080, 2176, 1), (300, 4160, 4168, 4224, 8),
                                                        (70000, 32, 32, 128, 0), (30001, 64, 72, 64, 0), (3003, 4160, 4161, 4224, 1)])
@pytest.mark.parametrize("ot", list(OutType))
@pytest.mark.parametrize("tiled", [False, True])
def test_typed_quantiser(rows, cols, ld, padded, offset, ot, tiled):
    if tiled and padded % 128:
        padded = lib.kpad(padded)
    buf = (_randn(offset + rows * ld, seed=rows + cols) * torch.exp(_randn(offset + rows * ld, seed=2) * 3)).to(DTYPE[ot])
    x = buf[offset:].view(rows, ld)[:, :cols]
    x[0, :32] = 0
    if rows > 4:
        x[1, 3], x[2, 4], x[3, 5] = float("nan"), float("inf"), float("-inf")
    full = torch.zeros(rows, padded)
    full[:, :cols] = x.float().cpu()
    want = lib.quantize_to_mxfp6(full.numpy())
    want.scales[:, cols // 32:] = 127
    packed = torch.full((rows, padded * 3 // 4), 0x5A, dtype=torch.uint8, device="cuda")
    scales = torch.full((lib.tiled_scale_bytes(rows, padded) if tiled else rows * padded // 32,), 0x5A, dtype=torch.uint8,
                        device="cuda")
    assert lib.quantize_device_typed(x, ot, rows, cols, ld, padded, packed, scales, tiled=tiled) == lib.OK
    torch.cuda.synchronize()
    assert np.array_equal(packed.cpu().numpy(), want.packed_data)
    raw = scales.cpu().numpy()
    raw = lib.untile_scales(raw, rows, padded) if tiled else raw.reshape(rows, -1)
    assert np.array_equal(raw, want.scales)


def _mlp(x, B1, B2, b1, b2, buffers, stream=None):
    """A feed-forward block as a user runs it: quantise, up with activation to MXFP6, down with residual."""
    T, H, I = x.shape[0], B1.K, B1.rows
    xq, sx, hq, sh, y, ws, n = buffers
    ot = OutType.BF16
    up = lib.Epilogue(b1, OutType.F32, Act.GELU)
    down = lib.Epilogue(b2, OutType.F32, aux=x, aux_type=ot, aux_op=AuxOp.ADD)
    assert lib.quantize_device_typed(x, ot, T, H, H, H, xq, sx, tiled=True, stream=stream) == lib.OK
    assert lib.gemm_fused_quant(T, I, H, xq, B1.packed, sx, B1.scales, hq, sh, H * 3 // 4, H * 3 // 4, up, ws, n,
                                stream=stream) == lib.OK
    assert lib.gemm_fused(ot, T, H, I, hq, B2.packed, sh, B2.scales, y, I * 3 // 4, I * 3 // 4, down, ws, n,
                          stream=stream) == lib.OK


@pytest.mark.parametrize("T,H,I", [(1, 256, 1024), (19, 1024, 4096), (300, 512, 2048)])
def test_feed_forward_block(T, H, I):
    """The block's intermediate codes are read back, so each GEMM is held to its own formula; then the
    block is captured in a graph and replayed on new inputs."""
    B1, B2 = Operand(I, H, H ** -0.5, 30), Operand(H, I, I ** -0.5, 31)
    b1, b2 = _randn(I, seed=32, std=0.2), _randn(H, seed=33, std=0.2)
    x = _randn(T, H, seed=34, dtype=torch.bfloat16)
    byte = lambda n: torch.zeros(n, dtype=torch.uint8, device="cuda")  # noqa: E731
    n = max(lib.gemm_fused_workspace_size(T, I, H), lib.gemm_fused_workspace_size(T, H, I))
    buffers = (byte(T * H * 3 // 4), byte(lib.tiled_scale_bytes(T, H)), byte(T * I * 3 // 4),
               byte(lib.tiled_scale_bytes(T, I)), torch.empty(T, H, dtype=torch.bfloat16, device="cuda"), byte(n), n)

    def check():
        _finish()
        q = lib.quantize_to_mxfp6(x.float().cpu().numpy())
        a = lib.dequantize_mxfp6(q)
        A = type("A", (), {"values": torch.from_numpy(a).cuda().double()})
        packed, raw = buffers[2].cpu().numpy().reshape(T, -1), lib.untile_scales(buffers[3].cpu().numpy(), T, I)
        check_quantised(packed, raw, *fused64(A, B1, Act.GELU, b1, None, AuxOp.NONE), "hidden")
        h = lib.QuantizedMatrix(packed, raw, T, I)
        Hm = type("H", (), {"values": torch.from_numpy(lib.dequantize_mxfp6(h)).cuda().double()})
        check_rounded(buffers[4], *fused64(Hm, B2, Act.NONE, b2, x, AuxOp.ADD), OutType.BF16, "output")

    _mlp(x, B1, B2, b1, b2, buffers)
    check()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        _mlp(x, B1, B2, b1, b2, buffers, stream=s)
    x.copy_(_randn(T, H, seed=35, dtype=torch.bfloat16))
    g.replay()
    check()


@pytest.mark.parametrize("M,N,K", [(130, 300, 2080), (1500, 2056, 2080), (4096, 4704, 2016)])
def test_compact_a_in_place_repeats(M, N, K):
    """The loader warps refill each stage many times: every call gives the bits of the tensor load's A."""
    prev = lib.set_repad_scratch(0)
    try:
        A, B = Operand(M, K, 1.0, 60, row_bytes=K * 3 // 4), Operand(N, K, K ** -0.5, 61)
        P = Operand(M, K, 1.0, 60)
        want = _fused(P, B, OutType.F32, Act.RELU, ws=False)
        first = _fused(A, B, OutType.F32, Act.RELU, ws=False)
        check_rounded(first, *fused64(A, B, Act.RELU, None, None, AuxOp.NONE), OutType.F32)
        assert torch.equal(first, want)
        ep = lib.Epilogue(act=Act.RELU)
        outs = [torch.empty(M, N, device="cuda") for _ in range(8)]
        for _ in range(10):
            for D in outs:
                assert lib.gemm_fused(OutType.F32, M, N, A.Kp, A.packed, B.packed, A.scales, B.scales, D, A.row_bytes,
                                      B.row_bytes, ep) == lib.OK
            _finish()
            assert all(torch.equal(D, first) for D in outs)
    finally:
        lib.set_repad_scratch(prev)


def test_types_and_strides_of_tensors():
    """Operands given as tensors alone: their element types and row strides are the call's."""
    M, N, K = 33, 200, 256
    A, B = Operand(M, K, 1.0, 70), Operand(N, K, 0.06, 71)
    bias, aux = _randn(N, seed=72, dtype=torch.bfloat16), _randn(M, N + 16, seed=73, dtype=torch.float16)[:, 8:N + 8]
    D = torch.full((M, N + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    ep = lib.Epilogue(bias, act=Act.SILU, aux=aux, aux_op=AuxOp.MUL)
    assert lib.gemm_fused(OutType.BF16, M, N, A.Kp, A.packed, B.packed, A.scales, B.scales, D[:, :N], A.row_bytes,
                          B.row_bytes, ep) == lib.OK
    _finish()
    assert (D[:, N:] == 7.0).all()
    check_rounded(D[:, :N], *fused64(A, B, Act.SILU, bias, aux, AuxOp.MUL), OutType.BF16)


def _activation_bound(act, v):
    """Relative error of an activation on FP32 values: roundings of the exponent, which grow with its size, and 2^-20 or
    2^-19 for the reciprocal (with a shared one t is off by five half steps), the exponential (two ulp) and the rest."""
    if act == Act.GELU:
        return 2.0 ** -19 + 2.0 ** -23 * v ** 2
    return 2.0 ** -20 + (2.0 ** -23 * v.abs() if act == Act.SILU else 2.0 ** -21 * v.abs() * (1 + 0.0447 * v ** 2))


# one row, few rows by columns and in fours, one tile in both layouts, split K, the pair
@pytest.mark.parametrize("M,N,K", [(1, 4096, 128), (3, 4095, 128), (40, 4095, 128), (40, 4096, 128), (300, 4096, 128),
                                   (300, 4095, 128), (200, 2048, 4096), (2050, 6144, 128)])
@pytest.mark.parametrize("act,low", [(Act.GELU, -12.9), (Act.GELU_TANH, -7.5), (Act.SILU, -43.0)])
def test_activations_relative_error(M, N, K, act, low):
    """Zero operands: the activation of the bias alone, relative to its value, down to where it ends."""
    A, B = Operand(M, K, 0.0, 80), Operand(N, K, 0.0, 81)
    rng = np.random.default_rng(82)
    for v in (rng.uniform(low, 6.0, N), rng.uniform(-3.0, 3.0, N), rng.choice([-1.0, 1.0], N) * 10.0 ** rng.uniform(-30, 0.4, N)):
        v = torch.from_numpy(v.astype(np.float32)).cuda()
        got, x = _fused(A, B, OutType.F32, act, v), v.double()
        assert (got == got[0]).all()
        ref = x * torch.special.erfc(-x * np.sqrt(0.5)) / 2 if act == Act.GELU else x * torch.sigmoid(
            x if act == Act.SILU else 2 * np.sqrt(2 / np.pi) * (x + 0.044715 * x ** 3))
        off = (got[0].double() / ref - 1).abs()
        worst = (off - _activation_bound(act, x)).argmax()
        assert (off <= _activation_bound(act, x)).all(), (act, float(x[worst]), float(off[worst]))


# Few rows of a matrix too wide for tiles of 128 columns at two per SM, and just narrow enough for tiles of 256 at one.
@pytest.mark.parametrize("M,K", [(1, 1280), (3, 160), (16, 480)])
def test_few_rows_of_wide_matrices(M, K):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    first, last = (2 * sms - 4) * 128 + 1, sms * 256
    A, B = Operand(M, K, 1.0, 90), Operand(last, K, K ** -0.5, 91)
    whole = B.values
    for N in (first, first + 6, last - 100, last):
        B.rows, B.values = N, whole[:N]
        bias = _randn(N, seed=92)
        for ot, act, op in ((OutType.F32, Act.GELU, AuxOp.ADD), (OutType.BF16, Act.SILU, AuxOp.MUL), (OutType.F16, Act.NONE, AuxOp.NONE)):
            aux = None if op == AuxOp.NONE else _randn(M, N, seed=93, dtype=DTYPE[ot])
            got = _fused(A, B, ot, act, bias, aux=aux, aux_op=op, aux_type=ot)
            check_rounded(got, *fused64(A, B, act, bias, aux, op), ot, f"{M}x{N}x{K}")


@pytest.mark.parametrize("M", [1, 16])
def test_few_rows_of_wide_matrices_quantised(M):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    N, K = sms * 256 - 128, 640
    A, B = Operand(M, K, 1.0, 94), Operand(N, K, K ** -0.5, 95)
    bias = _randn(N, seed=96)
    packed = torch.full((M + 1, N * 3 // 4), 0x5A, dtype=torch.uint8, device="cuda")
    scales = torch.full((lib.tiled_scale_bytes(M, N),), 0x5A, dtype=torch.uint8, device="cuda")
    assert lib.gemm_fused_quant(M, N, A.Kp, A.packed, B.packed, A.scales, B.scales, packed, scales, A.row_bytes, B.row_bytes,
                                lib.Epilogue(bias, act=Act.SILU)) == lib.OK
    _finish()
    assert (packed[M] == 0x5A).all()
    raw = lib.untile_scales(scales.cpu().numpy(), M, N)
    check_quantised(packed[:M].cpu().numpy(), raw, *fused64(A, B, Act.SILU, bias, None, AuxOp.NONE), f"{M}x{N}")


@pytest.mark.parametrize("T,H,I", [(1, 256, 512), (19, 1024, 1408), (300, 512, 2048)])
def test_gated_feed_forward_block(T, H, I):
    """A gated block: the up half first, then the gate with it as the multiplied aux, to MXFP6, then the down product."""
    Bg, Bu, Bd = Operand(I, H, H ** -0.5, 100), Operand(I, H, H ** -0.5, 101), Operand(H, I, I ** -0.5, 102)
    x = _randn(T, H, seed=103, dtype=torch.bfloat16)
    byte = lambda n: torch.zeros(n, dtype=torch.uint8, device="cuda")  # noqa: E731
    n = max(lib.gemm_fused_workspace_size(T, I, H), lib.gemm_fused_workspace_size(T, H, I))
    ws, xq, sx = byte(n), byte(T * H * 3 // 4), byte(lib.tiled_scale_bytes(T, H))
    hq, sh = byte(T * I * 3 // 4), byte(lib.tiled_scale_bytes(T, I))
    up, y = torch.empty(T, I, dtype=torch.bfloat16, device="cuda"), torch.empty(T, H, dtype=torch.bfloat16, device="cuda")
    ot, rh, ri = OutType.BF16, H * 3 // 4, I * 3 // 4
    gate, down = lib.Epilogue(act=Act.SILU, aux=up, aux_op=AuxOp.MUL), lib.Epilogue(aux=x, aux_op=AuxOp.ADD)
    assert lib.quantize_device_typed(x, ot, T, H, H, H, xq, sx, tiled=True) == lib.OK
    assert lib.gemm_fused(ot, T, I, H, xq, Bu.packed, sx, Bu.scales, up, rh, rh, None, ws, n) == lib.OK
    assert lib.gemm_fused_quant(T, I, H, xq, Bg.packed, sx, Bg.scales, hq, sh, rh, rh, gate, ws, n) == lib.OK
    assert lib.gemm_fused(ot, T, H, I, hq, Bd.packed, sh, Bd.scales, y, ri, ri, down, ws, n) == lib.OK
    _finish()
    q = lib.quantize_to_mxfp6(x.float().cpu().numpy())
    A = type("A", (), {"values": values(q.packed_data, q.scales, T, H)})
    check_rounded(up, *fused64(A, Bu, Act.NONE, None, None, AuxOp.NONE), ot, "up")
    packed, raw = hq.cpu().numpy().reshape(T, -1), lib.untile_scales(sh.cpu().numpy(), T, I)
    check_quantised(packed, raw, *fused64(A, Bg, Act.SILU, None, up, AuxOp.MUL), "hidden")
    Hm = type("H", (), {"values": values(packed, raw, T, I)})
    check_rounded(y, *fused64(Hm, Bd, Act.NONE, None, x, AuxOp.ADD), ot, "output")


# D and aux of more than 2^31 elements: in place in the row layout, and the column layout.
@pytest.mark.parametrize("N", [33024, 33023])
def test_offsets_beyond_32_bits(N):
    M, K = 66000, 128
    A, B = Operand(M, K, 1.0, 110), Operand(N, K, K ** -0.5, 111)
    D = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
    last = _randn(64, N, seed=112, dtype=torch.bfloat16)
    D[-64:] = last
    ep = lib.Epilogue(act=Act.RELU, aux=D, aux_op=AuxOp.ADD)
    assert lib.gemm_fused(OutType.BF16, M, N, A.Kp, A.packed, B.packed, A.scales, B.scales, D, A.row_bytes, B.row_bytes, ep) == lib.OK
    _finish()
    for rows, aux in ((slice(0, 64), torch.zeros_like(last)), (slice(M - 64, M), last)):
        part = type("A", (), {"values": A.values[rows]})
        check_rounded(D[rows], *fused64(part, B, Act.RELU, None, aux, AuxOp.ADD), OutType.BF16, f"{N}")


def test_quantiser_offsets_beyond_32_bits():
    rows, cols = 66000, 33024
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[-3:] = _randn(3, cols, seed=113, dtype=torch.bfloat16)
    packed = torch.full((rows, cols * 3 // 4), 0x5A, dtype=torch.uint8, device="cuda")
    scales = torch.full((lib.tiled_scale_bytes(rows, cols),), 0x5A, dtype=torch.uint8, device="cuda")
    assert lib.quantize_device_typed(x, OutType.BF16, rows, cols, cols, cols, packed, scales, tiled=True) == lib.OK
    torch.cuda.synchronize()
    want = lib.quantize_to_mxfp6(x[-3:].float().cpu().numpy())
    assert np.array_equal(packed[-3:].cpu().numpy(), want.packed_data) and (packed[:-3] == 0).all()
    atoms = cols // 128 * 512  # bytes of a block of 128 rows
    first = rows // 128 * 128
    raw = lib.untile_scales(scales[-atoms:].cpu().numpy(), rows - first, cols)
    assert np.array_equal(raw[-3:], want.scales) and (raw[:-3] == 127).all() and (scales[:-atoms] == 127).all()


@pytest.mark.parametrize("M,N,K,what", [(100, 2560, 2048, "split-K"), (4090, 3570, 6144, "stream-K")])
def test_skipped_workspace_names_the_query(capfd, M, N, K, what):
    """A workspace of the size that the message's query gives is enough; gemm()'s own may not be."""
    A, B = Operand(M, K, 1.0, 120), Operand(N, K, K ** -0.5, 121)
    _fused(A, B, OutType.BF16, Act.SILU, ws=False)
    err = capfd.readouterr().err
    assert what in err and "gemm_fused_workspace_size()" in err
    _fused(A, B, OutType.BF16, Act.SILU)
    assert "skipped" not in capfd.readouterr().err
