"""Refusals and queries of the fused calls and the typed quantiser: no GPU is touched."""
from __future__ import annotations

import pytest

P = 0x1000  # an aligned address that no accepted call reaches


@pytest.fixture
def call(lib):
    def run(ot=1, M=5, N=40, Kp=256, A=P, B=P, sA=P, sB=P, D=P, Ar=192, Br=192, ep=None, ldd=None):
        return lib.gemm_fused(ot, M, N, Kp, A, B, sA, sB, D, Ar, Br, ep, ldd=ldd)
    return run


def _ep(lib, **kw):
    kw.setdefault("ld_aux", 40)
    return lib.Epilogue(**kw)


@pytest.mark.parametrize("args,code", [
    (dict(ot=3), "ERR_INVALID_OUT_TYPE"), (dict(M=-1), "ERR_INVALID_SHAPE"), (dict(N=0), "ERR_INVALID_SHAPE"),
    (dict(Kp=0), "ERR_INVALID_SHAPE"), (dict(Kp=200), "ERR_INVALID_SHAPE"), (dict(Ar=90), "ERR_INVALID_STRIDE"),
    (dict(Br=200), "ERR_INVALID_STRIDE"), (dict(Br=160), "ERR_INVALID_STRIDE"), (dict(A=0), "ERR_NULL_POINTER"),
    (dict(sB=0), "ERR_NULL_POINTER"), (dict(D=0), "ERR_NULL_POINTER"), (dict(A=P + 2), "ERR_MISALIGNED"),
    (dict(B=P + 16), "ERR_MISALIGNED"), (dict(sA=P + 8), "ERR_MISALIGNED"), (dict(D=P + 1), "ERR_MISALIGNED"),
    (dict(ldd=39), "ERR_INVALID_STRIDE")])
def test_operands_refused(lib, call, capfd, args, code):
    n0 = lib.launch_count()
    assert call(**args) == getattr(lib, code) == lib.last_error()
    assert "[mxfp6]" in capfd.readouterr().err
    assert lib.launch_count() == n0


@pytest.mark.parametrize("kw,code", [
    (dict(act=5), "ERR_UNSUPPORTED"), (dict(act=-1), "ERR_UNSUPPORTED"), (dict(aux=P, aux_op=3), "ERR_UNSUPPORTED"),
    (dict(bias=P, bias_type=3), "ERR_INVALID_OUT_TYPE"), (dict(bias=P + 2, bias_type=0), "ERR_MISALIGNED"),
    (dict(aux_op=1), "ERR_NULL_POINTER"), (dict(aux=P, aux_op=1, aux_type=7), "ERR_INVALID_OUT_TYPE"),
    (dict(aux=P + 1, aux_op=2, aux_type=1), "ERR_MISALIGNED"), (dict(aux=P, aux_op=1, ld_aux=39), "ERR_INVALID_STRIDE")])
def test_epilogue_refused(lib, call, capfd, kw, code):
    assert call(ep=_ep(lib, **kw)) == getattr(lib, code)
    capfd.readouterr()


@pytest.mark.parametrize("kw,code", [
    (dict(N=160), "ERR_INVALID_SHAPE"), (dict(scales=0), "ERR_NULL_POINTER"), (dict(packed=0), "ERR_NULL_POINTER"),
    (dict(rb=64), "ERR_INVALID_STRIDE"), (dict(rb=100), "ERR_INVALID_STRIDE"), (dict(packed=P + 16), "ERR_MISALIGNED"),
    (dict(scales=P + 4), "ERR_MISALIGNED"), (dict(M=-2), "ERR_INVALID_SHAPE")])
def test_quantised_output_refused(lib, capfd, kw, code):
    a = dict(M=5, N=128, packed=P, scales=P, rb=96) | kw
    rc = lib.gemm_fused_quant(a["M"], a["N"], 256, P, P, P, P, a["packed"], a["scales"], 192, 192,
                              packed_row_bytes=a["rb"])
    assert rc == getattr(lib, code)
    capfd.readouterr()


@pytest.mark.parametrize("kw,code", [
    (dict(t=3), "ERR_INVALID_OUT_TYPE"), (dict(rows=-1), "ERR_INVALID_SHAPE"), (dict(cols=33), "ERR_INVALID_SHAPE"),
    (dict(cols=0), "ERR_INVALID_SHAPE"), (dict(padded=32), "ERR_INVALID_SHAPE"),
    (dict(padded=96, tiled=True), "ERR_INVALID_SHAPE"), (dict(ld=63), "ERR_INVALID_STRIDE"),
    (dict(x=0), "ERR_NULL_POINTER"), (dict(x=P + 1), "ERR_MISALIGNED"), (dict(packed=P + 2), "ERR_MISALIGNED")])
def test_typed_quantiser_refused(lib, capfd, kw, code):
    a = dict(x=P, t=2, rows=4, cols=64, ld=64, padded=64, packed=P, tiled=False) | kw
    assert lib.quantize_device_typed(a["x"], a["t"], a["rows"], a["cols"], a["ld"], a["padded"], a["packed"], P,
                                     tiled=a["tiled"]) == getattr(lib, code)
    assert "[mxfp6]" in capfd.readouterr().err


def test_workspace_query(lib):
    assert lib.gemm_fused_workspace_size(0, 128, 256) == 0
    # split K: partials of whole 32-column chunks for every row
    r = lib.route(lib.OutType.BF16, 1, 4001, 8192)
    assert r["splits"] > 1
    assert lib.gemm_fused_workspace_size(1, 4001, 8192) >= r["splits"] * 4032 * 4
    # a compact A adds its padded copy
    assert lib.gemm_fused_workspace_size(300, 4001, 8192, 6120) >= 300 * 6144


def test_aux_given_as_an_address_needs_its_pitch(lib):
    with pytest.raises(ValueError):
        lib.Epilogue(aux=P, aux_op=lib.AuxOp.ADD)


@pytest.fixture
def torch():
    return pytest.importorskip("torch")


@pytest.fixture
def seen(lib, monkeypatch):
    """The arguments of the C calls, which are not made."""
    got = []
    for name in ("_gemm_fused", "_quantize_dev_t"):
        monkeypatch.setattr(lib, name, lambda *a: got.append(a) or 0)
    return got


@pytest.mark.parametrize("dtype,kind", [("float32", "F32"), ("float16", "F16"), ("bfloat16", "BF16")])
def test_epilogue_takes_a_tensors_type_and_stride(lib, torch, dtype, kind):
    t = getattr(torch, dtype)
    bias, aux = torch.zeros(40, dtype=t), torch.zeros(5, 56, dtype=t)[:, 8:48]
    want = int(lib.OutType[kind])
    for e in (lib.Epilogue(bias, aux=aux, aux_op=lib.AuxOp.ADD),
              lib.Epilogue(bias, want, aux=aux, aux_type=want, aux_op=lib.AuxOp.ADD)):
        s = e.struct
        assert (s.bias, s.bias_type, s.aux, s.aux_type, s.ld_aux) == (bias.data_ptr(), want, aux.data_ptr(), want, 56)
    assert lib.Epilogue(aux=aux[:1]).struct.ld_aux >= 40 and lib.Epilogue(aux=aux[0]).struct.ld_aux == 40
    assert lib.Epilogue(bias=P, aux=P, ld_aux=40).struct.bias_type == lib.OutType.F32
    for other in set(lib.OutType) - {want}:
        for kw in (dict(bias=bias, bias_type=other), dict(aux=aux, aux_type=other)):
            with pytest.raises(ValueError, match="elements"):
                lib.Epilogue(**kw)


def test_epilogue_refuses_what_it_would_read_wrongly(lib, torch):
    for kw in (dict(bias=torch.zeros(40, dtype=torch.float64)), dict(aux=torch.zeros(5, 40, dtype=torch.float64)),
               dict(bias=torch.zeros(80)[::2]), dict(aux=torch.zeros(40, 5).T), dict(aux=torch.zeros(5, 80)[:, ::2], ld_aux=80)):
        with pytest.raises(ValueError):
            lib.Epilogue(**kw)


def test_fused_output_tensor(lib, torch, call, seen):
    D = torch.zeros(5, 64, dtype=torch.float16)[:, :40]
    for kw, ldd in ((dict(D=D), 64), (dict(D=D, ldd=70), 70), (dict(D=D[:1].contiguous(), M=1), 40), (dict(D=P), 40),
                    (dict(D=torch.zeros(200, dtype=torch.uint8)), 40)):
        assert call(**kw) == 0 and seen[-1][9] == ldd
    n = len(seen)
    for kw in (dict(D=D, ot=lib.OutType.F32), dict(D=D.double()), dict(D=torch.zeros(40, 5, dtype=torch.float16).T),
               dict(D=torch.zeros(4, 5, 40, dtype=torch.float16)[::2])):
        with pytest.raises(ValueError):
            call(**kw)
    assert len(seen) == n


def test_typed_quantiser_input_tensor(lib, torch, seen):
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    assert lib.quantize_device_typed(x, lib.OutType.BF16, 4, 64, 64, 64, P, P) == 0
    for bad, t in ((x, lib.OutType.F32), (x.T, lib.OutType.BF16), (x.double(), lib.OutType.F32)):
        with pytest.raises(ValueError):
            lib.quantize_device_typed(bad, t, 4, 64, 64, 64, P, P)
    assert len(seen) == 1


def test_epilogue_aux_of_more_dimensions(lib, torch):
    aux = torch.zeros(3, 4, 40)
    assert lib.Epilogue(aux=aux).struct.ld_aux == 40  # [batch][token] rows
    with pytest.raises(ValueError, match="ld_aux"):
        lib.Epilogue(aux=aux[:, ::2])
    assert lib.Epilogue(aux=aux[:, ::2], ld_aux=80).struct.ld_aux == 80
