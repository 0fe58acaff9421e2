"""Mixture-of-experts layer for a few tokens (mxfp6_moe) against an FP64 restatement of its formulas."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import mxfp6_b200 as lib
from fused_ref import DTYPE, SLOPE, Operand, act64, check_rounded, values
from mxfp6_b200 import Act, OutType

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _q64(h):
    """(MXFP6 values of FP64 rows, step between neighbouring values around each) by the quantiser's rule."""
    b = h.view(h.shape[0], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    s = torch.exp2(torch.ceil(torch.log2(torch.where(top > 0, top, torch.full_like(top, 7.5)) / 7.5)))
    m = (b / s).abs()
    step = torch.where(m < 2, 0.125, torch.where(m < 4, 0.25, 0.5))
    return (torch.round(b / s / step) * step * s).view(h.shape), (step * s).expand_as(b).reshape(h.shape)


class Layer:
    def __init__(self, E, H, I, gated=True, act=Act.SILU, seed=0):
        R1 = 2 * I if gated else I
        self.E, self.H, self.I, self.gated, self.act = E, H, I, gated, act
        self.W1, self.W2 = Operand(E * R1, H, H ** -0.5, seed + 1), Operand(E * H, I, I ** -0.5, seed + 2)
        self.w1, self.w2 = self.W1.values.view(E, R1, H), self.W2.values.view(E, H, I)
        self.layer = lib.MoELayer(E, H, I, self.W1.packed, self.W1.scales, self.W2.packed, self.W2.scales, gated, act)

    def reference(self, x, ids, weights, residual=None):
        """(out in FP64, a bound on the kernel's error before rounding). Each accumulator is within 1e-5 of its
        largest magnitude. A hidden value within that of a rounding border may take the neighbouring code (its
        step), and a block whose scale could change may move every value by a step of the larger scale."""
        q = lib.quantize_to_mxfp6(x.float().cpu().numpy())
        xv = values(q.packed_data, q.scales, *x.shape)
        T, I = x.shape[0], self.I
        out = torch.zeros(T, self.H, dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(out)
        ids, weights = ids.cpu(), weights.double()
        for e in sorted(set(ids.flatten().tolist())):
            if not 0 <= e < self.E:
                continue
            t, j = (ids == e).nonzero(as_tuple=True)
            t, j = t.cuda(), j.cuda()
            v = xv[t] @ self.w1[e].T
            da = 1e-5 * v.abs().max()
            g = act64(self.act, v[:, :I])
            dg = SLOPE[self.act] * da + 2.0 ** -20 * v[:, :I].abs()
            h, dh = (g * v[:, I:], dg * v[:, I:].abs() + (g.abs() + dg) * da) if self.gated else (g, dg)
            hq, step = _q64(h)
            lo, hi = _q64(h - dh)[0], _q64(h + dh)[0]
            moved = torch.maximum((lo - hq).abs(), (hi - hq).abs())
            top, slack = (z.abs().view(len(t), -1, 32).amax(-1) for z in (h, dh))
            edge = torch.ceil(torch.log2((top - slack).clamp(min=1e-300) / 7.5)) != \
                torch.ceil(torch.log2((top + slack).clamp(min=1e-300) / 7.5))
            moved = torch.where(edge.repeat_interleave(32, 1), torch.maximum(moved, 2 * step), moved)
            y = hq @ self.w2[e].T
            dy = moved @ self.w2[e].abs().T + 1e-5 * y.abs().max()
            w = weights[t, j].unsqueeze(1)
            out.index_add_(0, t, w * y)
            tol.index_add_(0, t, w.abs() * (dy + 2.0 ** -21 * y.abs()))
        if residual is not None:
            out, tol = out + residual.double(), tol + 2.0 ** -23 * residual.double().abs()
        return out, tol


def _randn(*shape, seed, std=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def _space(layer, T, k):
    n = lib.moe_workspace_size(layer.layer, T, k)
    return torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda"), n  # 0xFF: NaN scales and values


def _moe(layer, ot, x, xt, k, **kw):
    T = x.shape[0]
    buf = torch.full((T + 1, layer.H), 99.0, dtype=DTYPE[ot], device="cuda")
    ws, n = _space(layer, T, k)
    rc = lib.moe(layer.layer, ot, T, k, x, xt, buf, ws, n, ldx=x.stride(0), **kw)
    assert rc == lib.OK, rc
    torch.cuda.synchronize()
    assert lib.device_status() == 0
    assert (buf[T] == 99.0).all()
    return buf[:T]


def _routed(layer, T, k, seed=0, ot=OutType.BF16, xt=None, renormalize=True, residual=None):
    xt = ot if xt is None else xt
    x = _randn(T, layer.H, seed=seed + 10, dtype=DTYPE[xt])
    logits = _randn(T, layer.E, seed=seed + 11, std=1.5)
    ids = torch.full((T, k), -7, dtype=torch.int32, device="cuda")
    w = torch.full((T, k), -7.0, device="cuda")
    out = _moe(layer, ot, x, xt, k, logits=logits, ids=ids, weights=w, renormalize=renormalize, residual=residual)
    s = torch.sort(logits.double(), dim=1, descending=True, stable=True)
    assert torch.equal(ids.long(), s.indices[:, :k])
    p = torch.softmax(logits.double(), 1).gather(1, s.indices[:, :k])
    if renormalize:
        p = p / p.sum(1, keepdim=True)
    assert ((w.double() - p).abs() <= 2.0 ** -20 * p).all()  # two exponentials, a sum and a quotient in FP32
    check_rounded(out, *layer.reference(x, ids, w, residual), ot, f"T={T}")
    return out


# Tile widths 16, 32, 64, 128; one to many slabs and tiles; more items than CTAs; an expert in several tiles.
@pytest.mark.parametrize("T,E,k,H,I", [(1, 1, 1, 128, 128), (1, 8, 2, 256, 384), (3, 64, 8, 512, 128), (7, 8, 2, 1024, 512),
                                       (16, 16, 4, 384, 256), (17, 4, 1, 256, 256), (40, 8, 2, 256, 640),
                                       (61, 60, 6, 512, 384), (128, 16, 8, 256, 256), (128, 2, 2, 384, 128),
                                       (128, 64, 8, 128, 128), (2, 40, 16, 2048, 1408), (5, 512, 3, 128, 128),
                                       (20, 100, 5, 128, 128), (30, 200, 4, 128, 128), (128, 300, 16, 128, 128),
                                       (17, 33, 16, 256, 128), (32, 7, 1, 640, 128), (4, 256, 8, 128, 256)])
@pytest.mark.parametrize("gated", [True, False])
def test_sizes(T, E, k, H, I, gated):
    _routed(Layer(E, H, I, gated), T, k, ot=OutType.F16)


@pytest.mark.parametrize("act", list(Act))
@pytest.mark.parametrize("renormalize", [True, False])
def test_activations_and_types(act, renormalize):
    layer = Layer(6, 256, 256, act != Act.RELU, act)
    for ot, xt in ((OutType.F32, OutType.BF16), (OutType.BF16, OutType.F16), (OutType.F16, OutType.F32)):
        _routed(layer, 9, 2, ot=ot, xt=xt, renormalize=renormalize, residual=_randn(9, 256, seed=4, dtype=DTYPE[ot]))


@pytest.mark.parametrize("T,E,k", [(1, 64, 8), (16, 64, 2), (40, 24, 6), (128, 130, 3)])
def test_shares_of_the_whole_softmax(T, E, k):
    _routed(Layer(E, 128, 128), T, k, seed=3, ot=OutType.F32, renormalize=False)


def test_every_token_on_one_expert():
    """128 tokens of one expert where the tile holds 32: four passes over its weights."""
    layer = Layer(64, 256, 256)
    x = _randn(128, 256, seed=5, dtype=torch.bfloat16)
    ids = torch.full((128, 1), 37, dtype=torch.int32, device="cuda")
    w = _randn(128, 1, seed=6)
    check_rounded(_moe(layer, OutType.F32, x, OutType.BF16, 1, ids=ids, weights=w), *layer.reference(x, ids, w), OutType.F32)


def test_given_ids_skipped_and_repeated():
    layer = Layer(5, 256, 128)
    T, k = 12, 4
    ids = torch.randint(-2, 8, (T, k), generator=torch.Generator().manual_seed(7)).int()
    ids[3], ids[4], ids[5] = -1, 2, torch.tensor([5, 2 ** 31 - 1, -2 ** 31, 70000 - 65536])
    w = _randn(T, k, seed=8)
    x, res = _randn(T, 256, seed=9), _randn(T, 256, seed=10)
    given, w0 = ids.cuda(), w.clone()
    out = _moe(layer, OutType.F32, x, OutType.F32, k, ids=given, weights=w, residual=res)
    assert torch.equal(given.cpu(), ids) and torch.equal(w, w0)
    check_rounded(out, *layer.reference(x, ids, w, res), OutType.F32)
    assert torch.equal(out[3], res[3])  # nothing chosen: the residual
    out = _moe(layer, OutType.F32, x, OutType.F32, k, ids=given, weights=w)
    assert (out[3] == 0).all()
    none = torch.full((T, k), -1, dtype=torch.int32, device="cuda")
    assert (_moe(layer, OutType.F32, x, OutType.F32, k, ids=none, weights=w) == 0).all()


def test_routing_edges():
    E, k, H = 40, 6, 128
    layer = Layer(E, H, 128)
    inf, nan = float("inf"), float("nan")
    L = torch.zeros(9, E)
    L[1] = -inf                                   # nothing to choose
    L[2] = nan
    L[3, :] = -inf
    L[3, [5, 33]] = torch.tensor([1.0, 2.0])      # fewer than k
    L[4, [3, 38]] = inf                           # counts as the largest finite value
    L[5, ::2], L[5, 1::2] = 7.0, nan              # ties among the even ones
    L[6] = -3e38
    L[7, 20] = 3.4e38
    L[8] = -0.0
    L[8, 1::2] = 0.0                              # equal: ties
    x = _randn(9, H, seed=11)
    for renorm in (True, False):
        ids = torch.empty(9, k, dtype=torch.int32, device="cuda")
        w = torch.empty(9, k, device="cuda")
        out = _moe(layer, OutType.F32, x, OutType.F32, k, logits=L.cuda(), ids=ids, weights=w, renormalize=renorm)
        got, gw = ids.tolist(), w.cpu()
        assert got[0] == list(range(k)) and got[1] == got[2] == [-1] * k
        assert got[3] == [33, 5] + [-1] * (k - 2) and got[4] == [3, 38, 0, 1, 2, 4]
        assert got[5] == [0, 2, 4, 6, 8, 10] and got[6] == list(range(k)) and got[7] == [20, 0, 1, 2, 3, 4]
        assert got[8] == list(range(k))
        assert (gw[1] == 0).all() and (gw[2] == 0).all() and (gw[3, 2:] == 0).all()
        want = 1 / k if renorm else 1 / E
        assert torch.allclose(gw[0], torch.full((k,), want), rtol=1e-6) and torch.allclose(gw[4, :2], torch.tensor([0.5, 0.5]))
        assert torch.allclose(gw[3, :2].double(), torch.softmax(torch.tensor([2.0, 1.0]).double(), 0), rtol=1e-6)
        assert gw[7, 0] == 1 and (gw[7, 1:] == 0).all()
        check_rounded(out, *layer.reference(x, ids, w), OutType.F32)
        assert (out[1] == 0).all() and (out[2] == 0).all()


# Row strides and bases that rule out wide loads or stores, and the residual in place.
@pytest.mark.parametrize("xt,ot", [(OutType.BF16, OutType.BF16), (OutType.F32, OutType.F16)])
def test_strides_and_in_place(xt, ot):
    layer = Layer(4, 256, 128)
    T, k = 5, 2
    x = _randn(T, 300, seed=12, dtype=DTYPE[xt])[:, 1:257]
    ids = torch.tensor([[0, 1], [1, 2], [2, 3], [3, 0], [1, 3]], dtype=torch.int32, device="cuda")
    w = _randn(T, k, seed=13)
    flat = _randn(T * 261 + 3, seed=14, dtype=DTYPE[ot])
    out = flat[3:].view(T, 261)
    before = flat.clone()
    ws, n = _space(layer, T, k)
    rc = lib.moe(layer.layer, ot, T, k, x, xt, out, ws, n, ids=ids, weights=w, residual=out, ldx=300, ldo=261, ld_residual=261)
    assert rc == lib.OK
    torch.cuda.synchronize()
    check_rounded(out[:, :256], *layer.reference(x, ids, w, before[3:].view(T, 261)[:, :256]), ot)
    assert torch.equal(out[:, 256:], before[3:].view(T, 261)[:, 256:]) and torch.equal(flat[:3], before[:3])


def test_repeatable_and_empty():
    layer = Layer(16, 256, 256)
    a, b = _routed(layer, 50, 4, ot=OutType.F32), _routed(layer, 50, 4, ot=OutType.F32)
    assert torch.equal(a, b)
    n0 = lib.launch_count()
    assert lib.moe(layer.layer, OutType.F16, 0, 2, 0, OutType.F16, 0, 0, 0) == lib.OK
    assert lib.launch_count() == n0


def test_two_layers_in_a_graph():
    """A decoding step of two layers that share one workspace, captured and replayed on new inputs; then
    eager calls on the same stream between replays."""
    l1, l2 = Layer(8, 256, 384, seed=20), Layer(8, 256, 384, False, Act.GELU, seed=30)
    T, k, ot = 6, 2, OutType.F32
    x, mid, out = _randn(T, 256, seed=40), torch.empty(T, 256, device="cuda"), torch.empty(T, 256, device="cuda")
    g1, g2 = _randn(T, 8, seed=41), _randn(T, 8, seed=42)
    ids = [torch.empty(T, k, dtype=torch.int32, device="cuda") for _ in range(2)]
    w = [torch.empty(T, k, device="cuda") for _ in range(2)]
    ws, n = _space(l1, T, k)
    s = torch.cuda.Stream()

    def step():
        assert lib.moe(l1.layer, ot, T, k, x, ot, mid, ws, n, logits=g1, ids=ids[0], weights=w[0], residual=x, stream=s) == lib.OK
        assert lib.moe(l2.layer, ot, T, k, mid, ot, out, ws, n, logits=g2, ids=ids[1], weights=w[1], residual=mid,
                       stream=s) == lib.OK

    def check():
        torch.cuda.synchronize()
        assert lib.device_status() == 0
        check_rounded(mid, *l1.reference(x, ids[0], w[0], x), ot)
        check_rounded(out, *l2.reference(mid, ids[1], w[1], mid), ot)

    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step()
    for seed in (50, 60):
        x.copy_(_randn(T, 256, seed=seed))
        g1.copy_(_randn(T, 8, seed=seed + 1))
        g2.copy_(_randn(T, 8, seed=seed + 2))
        g.replay()
        check()
        with torch.cuda.stream(s):
            step()
        check()


def test_two_streams_at_once():
    """Two layers on two streams, each with its own workspace, beside few-row GEMMs on both: the results of the same
    calls one after another."""
    ot, T, k = OutType.F32, 24, 3
    layers = [Layer(16, 256, 384, seed=80), Layer(16, 256, 256, False, Act.GELU, seed=90)]
    A, B = Operand(20, 1024, 1.0, 91), Operand(640, 1024, 0.03, 92)
    streams = [torch.cuda.Stream() for _ in layers]
    xs = [_randn(T, 256, seed=100 + i) for i in range(2)]
    gs = [_randn(T, 16, seed=110 + i) for i in range(2)]
    spaces = [_space(layer, T, k) for layer in layers]
    outs = [[torch.empty(T, 256, device="cuda") for _ in range(8)] for _ in layers]
    ds = [[torch.empty(20, 640, device="cuda") for _ in range(8)] for _ in layers]

    def call(i, r):
        ws, n = spaces[i]
        assert lib.moe(layers[i].layer, ot, T, k, xs[i], ot, outs[i][r], ws, n, logits=gs[i], stream=streams[i]) == lib.OK
        assert lib.gemm_fused(ot, 20, 640, 1024, A.packed, B.packed, A.scales, B.scales, ds[i][r], 768, 768,
                              stream=streams[i]) == lib.OK

    torch.cuda.synchronize()
    for i in range(2):
        call(i, 0)
        torch.cuda.synchronize()
    for r in range(1, 8):
        for i in range(2):
            call(i, r)
    torch.cuda.synchronize()
    assert lib.device_status() == 0
    for i in range(2):
        for r in range(1, 8):
            assert torch.equal(outs[i][r], outs[i][0]) and torch.equal(ds[i][r], ds[0][0])


def test_prompt_and_decode_share_weights():
    """The layer's weights are GEMM operands as they are: one expert's up product through gemm_fused equals
    the layer's, for an expert without a gate and an identity-free comparison of the whole layer."""
    layer = Layer(3, 256, 256, False, Act.RELU)
    T = 20
    x = _randn(T, 256, seed=70, dtype=torch.bfloat16)
    e, rb = 1, 192
    xq = torch.zeros(T * rb, dtype=torch.uint8, device="cuda")
    sx = torch.zeros(lib.tiled_scale_bytes(T, 256), dtype=torch.uint8, device="cuda")
    hq, sh = torch.zeros_like(xq), torch.zeros_like(sx)
    y = torch.empty(T, 256, device="cuda")
    w1, w2 = layer.W1.packed[e * 256:(e + 1) * 256], layer.W2.packed[e * 256:(e + 1) * 256]
    atoms = 2 * 2 * 512
    s1, s2 = layer.W1.scales[e * atoms:(e + 1) * atoms], layer.W2.scales[e * atoms:(e + 1) * atoms]
    assert lib.quantize_device_typed(x, OutType.BF16, T, 256, 256, 256, xq, sx, tiled=True) == lib.OK
    assert lib.gemm_fused_quant(T, 256, 256, xq, w1, sx, s1, hq, sh, rb, rb, lib.Epilogue(act=Act.RELU)) == lib.OK
    assert lib.gemm_fused(OutType.F32, T, 256, 256, hq, w2, sh, s2, y, rb, rb) == lib.OK
    ids = torch.full((T, 1), e, dtype=torch.int32, device="cuda")
    out = _moe(layer, OutType.F32, x, OutType.BF16, 1, ids=ids, weights=torch.ones(T, 1, device="cuda"))
    ref, tol = layer.reference(x, ids, torch.ones(T, 1, device="cuda"))
    check_rounded(y, ref, tol, OutType.F32)
    check_rounded(out, ref, tol, OutType.F32)


@pytest.mark.parametrize("T,k,E", [(1, 8, 64), (40, 2, 8), (61, 6, 64)])
def test_weight_scales_of_every_slab(T, k, E):
    """Weight scales that differ by up to 2^40 from one 128-column slab to the next, over many more slabs than stages: a
    product with a scale of the stage's previous slab would be far off. Every call gives the same bits."""
    H, I = 4096, 128
    layer = Layer(E, H, I, act=Act.NONE, seed=120)
    rng = np.random.default_rng(121)
    R1 = E * 2 * I
    # one slab of every eight counts, at a place of its own for each row; the others are 2^-40 of it
    live = rng.integers(0, 8, (R1, 1)) == np.arange(H // 128)[None] % 8
    raw = np.where(np.repeat(live, 4, 1), 124, 84).astype(np.uint8)
    layer.W1.scales = torch.from_numpy(lib.preprocess_scale(raw, R1, H)).cuda()
    layer.W1.values = values(layer.W1.packed.cpu().numpy(), raw, R1, H)
    layer.w1 = layer.W1.values.view(E, 2 * I, H)
    layer.layer = lib.MoELayer(E, H, I, layer.W1.packed, layer.W1.scales, layer.W2.packed, layer.W2.scales, True, Act.NONE)
    x = _randn(T, H, seed=122)
    ids = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(t))[:k] for t in range(T)]).int().cuda()
    w = _randn(T, k, seed=123)
    first = _moe(layer, OutType.F32, x, OutType.F32, k, ids=ids, weights=w)
    check_rounded(first, *layer.reference(x, ids, w), OutType.F32)
    ws, n = _space(layer, T, k)
    outs = [torch.empty_like(first) for _ in range(20)]
    for _ in range(10):
        for out in outs:
            assert lib.moe(layer.layer, OutType.F32, T, k, x, OutType.F32, out, ws, n, ids=ids, weights=w) == lib.OK
        torch.cuda.synchronize()
        assert all(torch.equal(out, first) for out in outs)
    assert lib.device_status() == 0


def test_strides_of_tensors():
    """x, out and residual as views of wider rows, their strides taken from the tensors."""
    layer, T, k, ot = Layer(4, 256, 128), 5, 2, OutType.BF16
    x = _randn(T, 272, seed=130, dtype=torch.bfloat16)[:, 8:264]
    res = _randn(T, 300, seed=131, dtype=torch.bfloat16)[:, :256]
    buf = torch.full((T, 261), 9.0, dtype=torch.bfloat16, device="cuda")
    ids = torch.tensor([[0, 1], [1, 2], [2, 3], [3, 0], [1, 3]], dtype=torch.int32, device="cuda")
    w = _randn(T, k, seed=132)
    ws, n = _space(layer, T, k)
    assert lib.moe(layer.layer, ot, T, k, x, ot, buf[:, :256], ws, n, ids=ids, weights=w, residual=res) == lib.OK
    torch.cuda.synchronize()
    assert lib.device_status() == 0 and (buf[:, 256:] == 9.0).all()
    check_rounded(buf[:, :256], *layer.reference(x, ids, w, res), ot)


@pytest.mark.parametrize("inter", [12288, 14336, 28672, 57344])
@pytest.mark.parametrize("T", [3, 40])
def test_long_inter_in_fp32(inter, T):
    """FP32 output of a long down product stays within the library's 1e-5. The up rows pick one value of x each, so the
    hidden values are exact and nothing but the down product's sum is off."""
    H = 128
    W1 = np.zeros((inter, H), np.float32)
    W1[np.arange(inter), np.arange(inter) % H] = 1.0
    q = lib.quantize_to_mxfp6(W1)
    W2 = Operand(H, inter, 1.0, 140)
    raw = np.random.default_rng(142).integers(115, 135, (H, inter // 32)).astype(np.uint8)  # products of many magnitudes
    W2.scales = torch.from_numpy(lib.preprocess_scale(raw, H, inter)).cuda()
    W2.values = values(W2.packed.cpu().numpy(), raw, H, inter)
    s1 = torch.from_numpy(lib.preprocess_scale(q.scales, inter, H)).cuda()
    w1 = torch.from_numpy(q.packed_data).cuda()
    layer = type("L", (), {"H": H, "layer": lib.MoELayer(1, H, inter, w1, s1, W2.packed, W2.scales, False, Act.NONE)})
    x = _randn(T, H, seed=141)
    ids, w = torch.zeros(T, 1, dtype=torch.int32, device="cuda"), torch.ones(T, 1, device="cuda")
    qx = lib.quantize_to_mxfp6(x.cpu().numpy())
    xv = values(qx.packed_data, qx.scales, T, H)
    ref = xv.repeat(1, inter // H) @ W2.values.T
    got = _moe(layer, OutType.F32, x, OutType.F32, 1, ids=ids, weights=w)
    off = float((got.double() - ref).abs().max() / ref.abs().max())
    assert off <= 1e-5, off
    assert torch.equal(got, _moe(layer, OutType.F32, x, OutType.F32, 1, ids=ids, weights=w))
    half = _moe(layer, OutType.BF16, x, OutType.F32, 1, ids=ids, weights=w)
    check_rounded(half, ref, 1e-4 * ref.abs().max(), OutType.BF16)
