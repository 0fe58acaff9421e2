"""Measured cases of the feed-forward operators: the fused GEMM, the feed-forward pass it makes up,
the typed activation quantiser and the mixture-of-experts layer for a few tokens.

With own = False, run() computes each operator from elementary torch operations in 32 bits; with
own = True it makes the calls a user makes of the library. All operands are MXFP6 (FP6 E2M3 codes,
four per three bytes, one E8M0 scale per 32 along the row) in the library's device layouts."""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
PACKED = 0.75 + 1 / 32  # bytes of one element: its code and its share of the block's scale


# ---- cases -------------------------------------------------------------------------------------------

def listed():
    return [
        # one token through a projection with bias and residual: weight bytes and latency
        dict(name="gemm one token", op="gemm", M=1, N=4096, K=4096, out="bf16", act="none", bias=True, aux="add"),
        # a ragged batch of a few dozen tokens, odd N, FP32 output
        dict(name="gemm 37 tokens odd", op="gemm", M=37, N=5001, K=2080, out="f32", act="gelu", bias=True, aux="none"),
        # a prompt's up projection on the repository's 2048-row shapes
        dict(name="gemm prompt", op="gemm", M=2048, N=6144, K=2048, out="f16", act="gelu_tanh", bias=True, aux="none"),
        # a long batch: the gate of a gated feed-forward times its up half
        dict(name="gemm large gate", op="gemm", M=4096, N=8192, K=8192, out="bf16", act="silu", bias=False, aux="mul"),
        # a whole feed-forward block for a small decoding batch and for a prompt
        dict(name="mlp 16 tokens", op="mlp", T=16, H=2048, I=8192, out="bf16", act="gelu"),
        dict(name="mlp prompt", op="mlp", T=2000, H=4096, I=16384, out="bf16", act="silu"),
        # activations on their way into a GEMM: a small batch, and a prompt's
        dict(name="quantize small", op="quantize", rows=48, cols=4096, type="bf16"),
        dict(name="quantize prompt", op="quantize", rows=8192, cols=8192, type="bf16"),
        # mixture of experts: one token of many small experts (latency), a few tokens of large experts,
        # a decoding batch that reaches every expert, and the largest: 128 tokens over 1.2 GB of weights
        dict(name="moe one token", op="moe", T=1, E=64, k=8, H=2048, I=1024, gated=True, act="silu", out="bf16"),
        dict(name="moe 7 tokens", op="moe", T=7, E=8, k=2, H=4096, I=8192, gated=True, act="silu", out="bf16"),
        dict(name="moe 61 tokens", op="moe", T=61, E=64, k=6, H=2048, I=1408, gated=True, act="silu", out="f16"),
        dict(name="moe 128 tokens", op="moe", T=128, E=64, k=4, H=4096, I=2048, gated=True, act="gelu_tanh", out="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gemm", "gemm", "mlp", "quantize", "moe", "moe"])
    if op == "gemm":
        out = rng.choice(["f32", "f16", "bf16"])
        return dict(op=op, M=_log(rng, 1, 4096), N=_log(rng, 8, 8192), K=32 * _log(rng, 8, 128 if out == "f32" else 256),
                    out=out, act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), bias=rng.random() < 0.7,
                    aux=rng.choice(["none", "add", "mul"]))
    if op == "mlp":
        return dict(op=op, T=_log(rng, 1, 2000), H=128 * _log(rng, 4, 32), I=128 * _log(rng, 8, 128),
                    out=rng.choice(["f16", "bf16"]), act=rng.choice(["relu", "gelu", "gelu_tanh", "silu"]))
    if op == "quantize":
        return dict(op=op, rows=_log(rng, 1, 8192), cols=32 * _log(rng, 4, 256), type=rng.choice(["f32", "f16", "bf16"]))
    while True:
        c = dict(op=op, T=_log(rng, 1, 128), E=rng.choice([8, 16, 32, 60, 64]), k=rng.randint(1, 8),
                 H=128 * _log(rng, 4, 32), I=128 * _log(rng, 2, 64), gated=rng.random() < 0.75,
                 act=rng.choice(["relu", "gelu", "gelu_tanh", "silu"]), out=rng.choice(["f16", "bf16"]))
        if c["E"] * c["H"] * c["I"] <= 64 * 4096 * 2048:
            return c


def work(case):
    op = case["op"]
    if op == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        e = BYTES[case["out"]]
        return {"bytes": PACKED * K * (M + N) + e * M * N * (1 if case["aux"] == "none" else 2) + (4 * N if case["bias"] else 0),
                "flops": 2.0 * M * N * K}
    if op == "mlp":
        T, H, I = case["T"], case["H"], case["I"]
        return {"bytes": PACKED * 2 * H * I + 3 * 2 * T * H + 4 * (H + I), "flops": 4.0 * T * H * I}
    if op == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (BYTES[case["type"]] + PACKED), "flops": 0}
    T, E, k, H, I = (case[n] for n in ("T", "E", "k", "H", "I"))
    chosen = E * (1 - (1 - k / E) ** T)  # experts that T tokens reach, expected
    mats = 3 if case["gated"] else 2
    return {"bytes": chosen * mats * H * I * PACKED + 3 * 2 * T * H + 4 * T * (E + 2 * k), "flops": 2.0 * T * k * mats * H * I}


# ---- MXFP6 in elementary operations -------------------------------------------------------------------

def _kpad(K):
    return (K + 127) // 128 * 128


def _quantize(x):
    """FP32 [rows][cols], cols % 32 == 0 -> codes and E8M0 scale codes: the smallest power of two that is
    at least max|x| / 7.5 per 32 (code 127 for a block of zeros), codes to nearest even, at most 7.5."""
    b = x.view(x.shape[0], -1, 32)
    top = b.abs().amax(-1)
    m, e = torch.frexp(top / 7.5)
    s = torch.where(top == 0, 127, (e - (m == 0.5).int() + 127).clamp(0, 254))
    v = torch.ldexp(b.abs(), (127 - s).unsqueeze(-1)).clamp(max=7.5)
    p = ((v >= 2).int() + (v >= 4).int()).float()             # binade above [0, 2), whose step is 1/8
    n = torch.round(torch.ldexp(v, 3 - p))                    # whole steps of the binade, ties to even
    up = n == 16                                              # rounded into the next binade
    p, n = torch.where(up, p + 1, p), torch.where(up, torch.full_like(n, 8), n)
    code = torch.where(p == 0, n, 8 * (p + 1) + (n - 8)).to(torch.uint8)
    neg = (b < 0).to(torch.uint8) * 32
    return (code + neg).view(x.shape), s.to(torch.uint8)


def _values(codes):
    """E2M3 codes -> their values."""
    c = codes.to(torch.int16)
    e, m = (c >> 3) & 3, c & 7
    mag = torch.where(e == 0, m, (8 + m) << (e - 1).clamp(min=0)).float() * 0.125
    return torch.where(c >= 32, -mag, mag)


def _pack(codes):
    g = codes.view(codes.shape[0], -1, 4).int()
    w = g[..., 0] | (g[..., 1] << 6) | (g[..., 2] << 12) | (g[..., 3] << 18)
    return torch.stack([w & 255, (w >> 8) & 255, w >> 16], -1).to(torch.uint8).view(codes.shape[0], -1)


def _unpack(packed):
    g = packed.view(packed.shape[0], -1, 3).int()
    w = g[..., 0] | (g[..., 1] << 8) | (g[..., 2] << 16)
    return torch.stack([w & 63, (w >> 6) & 63, (w >> 12) & 63, w >> 18], -1).to(torch.uint8).view(packed.shape[0], -1)


def _tile(scales):
    """Raw scales [rows][K/32] -> atoms of 128 rows x 4 blocks; rows past the last hold 127."""
    rows, nb = scales.shape
    full = torch.full(((rows + 127) // 128 * 128, nb), 127, dtype=torch.uint8, device=scales.device)
    full[:rows] = scales
    return full.view(-1, 4, 32, nb // 4, 4).permute(0, 3, 2, 1, 4).reshape(-1).contiguous()


def _untile(tiled, rows, nb):
    return tiled.view(-1, nb // 4, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, nb)[:rows]


def _matrix(packed, tiled, rows, Kp):
    """A device operand as the FP32 values it stands for."""
    s = _untile(tiled, rows, Kp // 32).int() - 127
    return torch.ldexp(_values(_unpack(packed)).view(rows, -1, 32), s.unsqueeze(-1)).view(rows, Kp)


def _through_fp6(x):
    codes, s = _quantize(x)
    return torch.ldexp(_values(codes).view(x.shape[0], -1, 32), (s.int() - 127).unsqueeze(-1)).view(x.shape)


def _act(name, v):
    if name == "relu":
        return torch.relu(v)
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    if name == "silu":
        return v / (1 + torch.exp(-v))
    return v


# ---- inputs ----------------------------------------------------------------------------------------------

def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def _operand(g, rows, K, std):
    """A quantised [rows][K] matrix of normal values in the device layout: packed rows of kpad(K) codes
    with a zero tail, tiled scales."""
    Kp = _kpad(K)
    x = torch.zeros(rows, Kp, device="cuda")
    x[:, :K] = _normal(g, rows, K, std=std)
    codes, s = _quantize(x)
    return _pack(codes), _tile(s)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, st = case["op"], {"case": case, "keep": {}}  # keep: a user's own workspaces and output buffers
    if op == "gemm":
        M, N, K, t = case["M"], case["N"], case["K"], TYPES[case["out"]]
        st["A"], st["sA"] = _operand(g, M, K, 1.0)
        st["B"], st["sB"] = _operand(g, N, K, 1 / math.sqrt(K))
        st["bias"] = _normal(g, N, std=0.2) if case["bias"] else None
        st["aux"] = _normal(g, M, N).to(t) if case["aux"] != "none" else None
    elif op == "mlp":
        T, H, I, t = case["T"], case["H"], case["I"], TYPES[case["out"]]
        st["x"], st["residual"] = _normal(g, T, H).to(t), _normal(g, T, H).to(t)
        st["B1"], st["sB1"] = _operand(g, I, H, 1 / math.sqrt(H))
        st["B2"], st["sB2"] = _operand(g, H, I, 1 / math.sqrt(I))
        st["b1"], st["b2"] = _normal(g, I, std=0.2), _normal(g, H, std=0.2)
    elif op == "quantize":
        st["x"] = (_normal(g, case["rows"], case["cols"]) * torch.exp(_normal(g, case["rows"], 1))).to(TYPES[case["type"]])
    else:
        T, E, H, I, t = case["T"], case["E"], case["H"], case["I"], TYPES[case["out"]]
        R1 = 2 * I if case["gated"] else I  # gated: the gate's rows, then the up half's
        st["x"], st["logits"] = _normal(g, T, H).to(t), _normal(g, T, E, std=1.5)
        st["w1"], st["s1"] = _operand(g, E * R1, H, 1 / math.sqrt(H))
        st["w2"], st["s2"] = _operand(g, E * H, I, 1 / math.sqrt(I))
    return st


# ---- one pass -------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if op == "gemm":
        return _gemm(state)
    if op == "mlp":
        return _mlp(state)
    if op == "quantize":
        return _quant(state)
    return _moe(state)


def _gemm(st):
    if own:
        return _own_gemm(st)
    c = st["case"]
    Kp = _kpad(c["K"])
    v = _matrix(st["A"], st["sA"], c["M"], Kp) @ _matrix(st["B"], st["sB"], c["N"], Kp).T
    if c["bias"]:
        v = v + st["bias"]
    v = _act(c["act"], v)
    if c["aux"] == "add":
        v = v + st["aux"].float()
    if c["aux"] == "mul":
        v = v * st["aux"].float()
    return v.to(TYPES[c["out"]])


def _mlp(st):
    if own:
        return _own_mlp(st)
    c = st["case"]
    T, H, I = c["T"], c["H"], c["I"]
    h = _act(c["act"], _through_fp6(st["x"].float()) @ _matrix(st["B1"], st["sB1"], I, H).T + st["b1"])
    y = _through_fp6(h) @ _matrix(st["B2"], st["sB2"], H, I).T + st["b2"]
    return (y + st["residual"].float()).to(TYPES[c["out"]])


def _quant(st):
    if own:
        return _own_quant(st)
    codes, s = _quantize(st["x"].float())
    return _pack(codes), s


def _moe(st):
    if own:
        return _own_moe(st)
    c = st["case"]
    T, E, k, H, I = (c[n] for n in ("T", "E", "k", "H", "I"))
    R1 = 2 * I if c["gated"] else I
    order = torch.sort(st["logits"], dim=1, descending=True, stable=True)  # equal logits: lowest index first
    ids, w = order.indices[:, :k], torch.softmax(order.values[:, :k], 1)
    # every token through every expert, then only the chosen ones' share
    x = _through_fp6(st["x"].float())
    w1 = _matrix(st["w1"], st["s1"], E * R1, H)
    h = torch.matmul(x, w1.T).view(T, E, R1)
    del w1
    h = _act(c["act"], h[..., :I]) * h[..., I:] if c["gated"] else _act(c["act"], h)
    h = _through_fp6(h.reshape(T * E, I)).view(T, E, I)
    y = torch.bmm(h.transpose(0, 1), _matrix(st["w2"], st["s2"], E * H, I).view(E, H, I).transpose(1, 2))
    dense = torch.zeros(T, E, device="cuda").scatter_(1, ids, w)
    out = (y * dense.T.unsqueeze(-1)).sum(0)
    return out.to(TYPES[c["out"]]), ids.int(), w


# ---- the library's calls -----------------------------------------------------------------------------------

def _lib():
    if "mxfp6_b200" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "mxfp6-gemm_b200"))
    import mxfp6_b200
    return mxfp6_b200


def _kind(lib, name):
    return {"f32": lib.OutType.F32, "f16": lib.OutType.F16, "bf16": lib.OutType.BF16}[name]


def _activation(lib, name):
    return {"none": lib.Act.NONE, "relu": lib.Act.RELU, "gelu": lib.Act.GELU, "gelu_tanh": lib.Act.GELU_TANH,
            "silu": lib.Act.SILU}[name]


def _space(n):
    return torch.empty(n, dtype=torch.uint8, device="cuda") if n else None


def _checked(rc):
    if rc:
        raise RuntimeError("mxfp6 status %d" % rc)


def _own_gemm(st):
    c, keep = st["case"], st["keep"]
    M, N, Kp = c["M"], c["N"], _kpad(c["K"])
    lib = _lib()
    if not keep:
        keep["ot"] = _kind(lib, c["out"])
        keep["n"] = lib.gemm_fused_workspace_size(M, N, Kp, Kp * 3 // 4)
        keep["ws"] = _space(keep["n"])
        keep["ep"] = lib.Epilogue(bias=st["bias"], bias_type=lib.OutType.F32, act=_activation(lib, c["act"]),
                                  aux=st["aux"], aux_type=keep["ot"],
                                  aux_op={"none": lib.AuxOp.NONE, "add": lib.AuxOp.ADD, "mul": lib.AuxOp.MUL}[c["aux"]])
    D = torch.empty(M, N, dtype=TYPES[c["out"]], device="cuda")
    _checked(lib.gemm_fused(keep["ot"], M, N, Kp, st["A"], st["B"], st["sA"], st["sB"], D, Kp * 3 // 4, Kp * 3 // 4,
                            keep["ep"], keep["ws"], keep["n"]))
    return D


def _own_mlp(st):
    c, keep = st["case"], st["keep"]
    T, H, I = c["T"], c["H"], c["I"]
    lib = _lib()
    if not keep:
        keep["ot"] = _kind(lib, c["out"])
        keep["n"] = max(lib.gemm_fused_workspace_size(T, I, H, H * 3 // 4), lib.gemm_fused_workspace_size(T, H, I, I * 3 // 4))
        keep["ws"] = _space(keep["n"])
        keep["xq"], keep["sx"] = _space(T * H * 3 // 4), _space(lib.tiled_scale_bytes(T, H))
        keep["hq"], keep["sh"] = _space(T * I * 3 // 4), _space(lib.tiled_scale_bytes(T, I))
        keep["up"] = lib.Epilogue(bias=st["b1"], bias_type=lib.OutType.F32, act=_activation(lib, c["act"]))
        keep["down"] = lib.Epilogue(bias=st["b2"], bias_type=lib.OutType.F32, aux=st["residual"], aux_type=keep["ot"],
                                    aux_op=lib.AuxOp.ADD)
    y = torch.empty(T, H, dtype=TYPES[c["out"]], device="cuda")
    _checked(lib.quantize_device_typed(st["x"], keep["ot"], T, H, H, H, keep["xq"], keep["sx"], tiled=True))
    _checked(lib.gemm_fused_quant(T, I, H, keep["xq"], st["B1"], keep["sx"], st["sB1"], keep["hq"], keep["sh"],
                                  H * 3 // 4, H * 3 // 4, keep["up"], keep["ws"], keep["n"]))
    _checked(lib.gemm_fused(keep["ot"], T, H, I, keep["hq"], st["B2"], keep["sh"], st["sB2"], y, I * 3 // 4, I * 3 // 4,
                            keep["down"], keep["ws"], keep["n"]))
    return y


def _own_quant(st):
    c = st["case"]
    lib = _lib()
    rows, cols = c["rows"], c["cols"]
    packed = torch.empty(rows, cols * 3 // 4, dtype=torch.uint8, device="cuda")
    scales = torch.empty(rows, cols // 32, dtype=torch.uint8, device="cuda")
    _checked(lib.quantize_device_typed(st["x"], _kind(lib, c["type"]), rows, cols, cols, cols, packed, scales))
    return packed, scales


def _own_moe(st):
    c, keep = st["case"], st["keep"]
    lib = _lib()
    T, k, H = c["T"], c["k"], c["H"]
    if not keep:
        keep["ot"] = _kind(lib, c["out"])
        keep["layer"] = lib.MoELayer(c["E"], H, c["I"], st["w1"], st["s1"], st["w2"], st["s2"], gated=c["gated"],
                                     act=_activation(lib, c["act"]))
        keep["n"] = lib.moe_workspace_size(keep["layer"], T, k)
        keep["ws"] = _space(keep["n"])
    out = torch.empty(T, H, dtype=TYPES[c["out"]], device="cuda")
    ids = torch.empty(T, k, dtype=torch.int32, device="cuda")
    w = torch.empty(T, k, device="cuda")
    _checked(lib.moe(keep["layer"], keep["ot"], T, k, st["x"], keep["ot"], out, keep["ws"], keep["n"],
                     logits=st["logits"], ids=ids, weights=w))
    return out, ids, w


# ---- the definition in 64 bits ---------------------------------------------------------------------------------

def _table():
    mags = [j / 8 for j in range(8)] + [(1 + j / 8) * 2.0 ** (e - 1) for e in (1, 2, 3) for j in range(8)]
    return torch.tensor(mags + [-m for m in mags], dtype=torch.float64, device="cuda")


def _exact_matrix(packed, tiled, row0, rows, Kp):
    """Rows [row0, row0 + rows) of a device operand in FP64, from its bytes' bits."""
    shift = torch.arange(8, device="cuda", dtype=torch.uint8)
    bits = (packed[row0:row0 + rows].unsqueeze(-1) >> shift) & 1
    codes = (bits.view(rows, Kp, 6).int() << torch.arange(6, device="cuda")).sum(-1)
    r, j = torch.arange(row0, row0 + rows, device="cuda").view(-1, 1), torch.arange(Kp // 32, device="cuda")
    at = ((r // 128) * (Kp // 128) + j // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + j % 4
    return _table()[codes] * torch.exp2(tiled[at].double() - 127).repeat_interleave(32, 1)


def _exact_fp6(x):
    b = x.view(x.shape[0], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    s = torch.exp2(torch.ceil(torch.log2(torch.where(top > 0, top, 7.5) / 7.5)).clamp(-127, 127))
    v = b / s
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(1, 7.5))) - 3)
    return ((v / step).round() * step).clamp(-7.5, 7.5).mul(s).view(x.shape)


def _exact_act(name, v):
    if name == "relu":
        return v.clamp(min=0)
    if name == "gelu":
        return v * torch.special.ndtr(v)
    if name == "gelu_tanh":
        return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
    if name == "silu":
        return v * torch.sigmoid(v)
    return v


def _exact_product(x, packed, tiled, row0, rows, Kp):
    parts = [x @ _exact_matrix(packed, tiled, row0 + r, min(1024, rows - r), Kp).T for r in range(0, rows, 1024)]
    return torch.cat(parts, 1)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "gemm":
        M, N, Kp = case["M"], case["N"], _kpad(case["K"])
        a = torch.cat([_exact_matrix(st["A"], st["sA"], r, min(1024, M - r), Kp) for r in range(0, M, 1024)])
        v = _exact_product(a, st["B"], st["sB"], 0, N, Kp)
        v = _exact_act(case["act"], v + st["bias"].double() if case["bias"] else v)
        return v if case["aux"] == "none" else v + st["aux"].double() if case["aux"] == "add" else v * st["aux"].double()
    if op == "mlp":
        h = _exact_product(_exact_fp6(st["x"].double()), st["B1"], st["sB1"], 0, case["I"], case["H"]) + st["b1"].double()
        h = _exact_fp6(_exact_act(case["act"], h))
        return _exact_product(h, st["B2"], st["sB2"], 0, case["H"], case["I"]) + st["b2"].double() + st["residual"].double()
    if op == "quantize":
        return None
    T, E, k, H, I = (case[n] for n in ("T", "E", "k", "H", "I"))
    R1 = 2 * I if case["gated"] else I
    p, ids = torch.sort(torch.softmax(st["logits"].double(), 1), dim=1, descending=True, stable=True)
    ids, w = ids[:, :k], p[:, :k] / p[:, :k].sum(1, keepdim=True)
    x, out = _exact_fp6(st["x"].double()), torch.zeros(T, H, dtype=torch.float64, device="cuda")
    for e in range(E):
        t, slot = (ids == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        h = _exact_product(x[t], st["w1"], st["s1"], e * R1, R1, H)
        h = _exact_act(case["act"], h[:, :I]) * h[:, I:] if case["gated"] else _exact_act(case["act"], h)
        y = _exact_product(_exact_fp6(h), st["w2"], st["s2"], e * H, H, I)
        out.index_add_(0, t, y * w[t, slot].unsqueeze(1))
    return out, None, w
