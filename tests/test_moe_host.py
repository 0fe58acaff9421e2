"""Refusals and queries of the mixture-of-experts layer: no GPU is touched."""
from __future__ import annotations

import pytest

P = 0x1000  # an aligned address that no accepted call reaches


def _layer(lib, **kw):
    a = dict(experts=8, hidden=256, inter=128, w1=P, s1=P, w2=P, s2=P, gated=True, act=lib.Act.SILU) | kw
    return lib.MoELayer(**a)


def _call(lib, layer, **kw):
    a = dict(ot=1, tokens=4, top_k=2, x=P, x_type=2, out=P, ws=P, ws_bytes=1 << 30, logits=P) | kw
    return lib.moe(layer, **a)


@pytest.mark.parametrize("layer,call,code", [
    (dict(experts=0), {}, "ERR_INVALID_SHAPE"), (dict(experts=513), {}, "ERR_INVALID_SHAPE"),
    (dict(hidden=200), {}, "ERR_INVALID_SHAPE"), (dict(inter=0), {}, "ERR_INVALID_SHAPE"),
    (dict(experts=512, hidden=1 << 23), {}, "ERR_INVALID_SHAPE"), (dict(act=9), {}, "ERR_UNSUPPORTED"),
    ({}, dict(tokens=-1), "ERR_INVALID_SHAPE"), ({}, dict(tokens=129), "ERR_INVALID_SHAPE"),
    ({}, dict(top_k=0), "ERR_INVALID_SHAPE"), ({}, dict(top_k=17), "ERR_INVALID_SHAPE"),
    ({}, dict(top_k=9), "ERR_INVALID_SHAPE"), ({}, dict(ot=3), "ERR_INVALID_OUT_TYPE"),
    ({}, dict(x_type=-1), "ERR_INVALID_OUT_TYPE"), (dict(w1=0), {}, "ERR_NULL_POINTER"),
    (dict(s2=0), {}, "ERR_NULL_POINTER"), ({}, dict(x=0), "ERR_NULL_POINTER"), ({}, dict(out=0), "ERR_NULL_POINTER"),
    ({}, dict(logits=None), "ERR_NULL_POINTER"), ({}, dict(logits=None, ids=P), "ERR_NULL_POINTER"),
    ({}, dict(ldx=255), "ERR_INVALID_STRIDE"), ({}, dict(ldo=128), "ERR_INVALID_STRIDE"),
    ({}, dict(residual=P, ld_residual=8), "ERR_INVALID_STRIDE"), (dict(w2=P + 16), {}, "ERR_MISALIGNED"),
    (dict(s1=P + 8), {}, "ERR_MISALIGNED"), ({}, dict(x=P + 1), "ERR_MISALIGNED"),
    ({}, dict(logits=P + 2), "ERR_MISALIGNED"), ({}, dict(ws=0), "ERR_WORKSPACE"), ({}, dict(ws=P + 128), "ERR_WORKSPACE"),
    ({}, dict(ws_bytes=100), "ERR_WORKSPACE")])
def test_refused(lib, capfd, layer, call, code):
    n0 = lib.launch_count()
    assert _call(lib, _layer(lib, **layer), **call) == getattr(lib, code) == lib.last_error()
    assert "[mxfp6] moe" in capfd.readouterr().err
    assert lib.launch_count() == n0


def test_workspace_query(lib):
    layer = _layer(lib)
    for tokens, k in ((0, 2), (129, 2), (4, 0), (4, 17)):
        assert lib.moe_workspace_size(layer, tokens, k) == 0
    assert lib.moe_workspace_size(_layer(lib, hidden=100), 4, 2) == 0
    sizes = [lib.moe_workspace_size(layer, t, 2) for t in range(1, 129)]
    # quantised rows, hidden rows and FP32 rows for every choice
    assert all(n >= 2 * t * (256 + 128 + 4 * 256) for t, n in enumerate(sizes, 1))


def test_tensors_types_and_strides(lib, monkeypatch):
    torch = pytest.importorskip("torch")
    seen = []
    monkeypatch.setattr(lib, "_moe", lambda *a: seen.append(a) or 0)
    layer, F16, BF16 = _layer(lib), lib.OutType.F16, lib.OutType.BF16
    x = torch.zeros(4, 300, dtype=torch.bfloat16)[:, 1:257]
    out, res = torch.zeros(4, 261, dtype=torch.float16)[:, :256], torch.zeros(4, 260, dtype=torch.float16)[:, :256]
    good = dict(ot=F16, x=x, x_type=BF16, out=out, residual=res, logits=torch.zeros(4, 8),
                ids=torch.zeros(4, 2, dtype=torch.int32), weights=torch.zeros(4, 2))
    pitches = lambda a: (a[6], a[12], a[14])  # noqa: E731
    assert _call(lib, layer, **good) == 0 and pitches(seen[-1]) == (300, 260, 261)
    assert _call(lib, layer, **good | dict(ldx=301, ldo=302, ld_residual=303)) == 0 and pitches(seen[-1]) == (301, 303, 302)
    dense = dict(x=x.reshape(2, 512), out=torch.zeros(1024, dtype=torch.float16), residual=None)
    assert _call(lib, layer, **good | dense) == 0 and pitches(seen[-1]) == (256, 256, 256)
    assert _call(lib, layer, **good | dict(tokens=1, x=x[:1], out=P, residual=P)) == 0 and pitches(seen[-1]) == (256, 256, 256)
    n = len(seen)
    for bad in (dict(x_type=F16), dict(ot=BF16), dict(residual=res.float()), dict(out=out.double()),
                dict(x=torch.zeros(256, 4, dtype=torch.bfloat16).T), dict(out=torch.zeros(8, 261, dtype=torch.float16)[:, :200]),
                dict(logits=torch.zeros(4, 8, dtype=torch.bfloat16)), dict(logits=torch.zeros(4, 16)[:, :8]),
                dict(ids=torch.zeros(4, 2, dtype=torch.int64)), dict(ids=torch.zeros(2, 4, dtype=torch.int32).T),
                dict(weights=torch.zeros(4, 2, dtype=torch.float16))):
        with pytest.raises(ValueError):
            _call(lib, layer, **good | bad)
    assert len(seen) == n
