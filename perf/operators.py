"""Cases of the 4-bit (MX) linear layers and of the gated block norm, with their plain forms.

Four operators of a transformer block served with 4-bit Linear layers:

* quantize: rows of x in blocks of 32 columns, each block one power-of-two scale 2^(floor(log2 max|x|) - 2) and
  32 values of the 4-bit type e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives; round to nearest, ties to even,
  saturating), and the values they stand for read back;
* product: Y = T(epilogue(A W^T + bias)) of two such matrices, the epilogue nothing, GELU or + residual;
* norm: x' = T(res_scale x + gate * post(h)), y = T(pre(x') (1 + scale) + shift), post / pre a LayerNorm, an
  RMSNorm or nothing, gate / scale / shift per group of rows;
* block: norm with its y in 4 bits, product with GELU and its output in 4 bits, product + residual.

Scales are stored one byte each (exponent + 127) in tiles of 128 rows x 4 blocks: byte
(row % 32) * 16 + (row % 128) // 32 * 4 + block % 4 of the 512-byte tile (row // 128, block // 4).
"""
import math
import sys

import torch

own = False

TYPES = {"fp16": torch.float16, "fp32": torch.float32}
#: the values of the 16 codes
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EPS = 1e-5
#: the largest listed products and norms bound what a drawn case costs
MOST_MNK, MOST_ROWS_C = 189809 * 4096 * 1024, 189809 * 1024


def listed():
    return [
        # one row of the hidden stream (C = 1024): a single node's activations, all latency
        {"name": "quantize_row", "op": "quantize", "rows": 1, "K": 1024, "type": "fp16"},
        # fp32 rows whose last block is cut (K = 1000) and whose stride is not their length
        {"name": "quantize_ragged", "op": "quantize", "rows": 4099, "K": 1000, "type": "fp32"},
        # the whole hidden stream of the full model before a Linear
        {"name": "quantize_hidden", "op": "quantize", "rows": 189809, "K": 1024, "type": "fp16"},
        # q|k|v|self of one node: the weights are all that is read
        {"name": "product_row", "op": "product", "M": 1, "N": 4096, "K": 1024, "type": "fp16", "epi": "bias"},
        # the output head on a coarse grid: 80 variables, fp32 out, rows not a multiple of a tile
        {"name": "product_head", "op": "product", "M": 40321, "N": 80, "K": 1024, "type": "fp32", "epi": "bias"},
        # a middle-sized hidden mesh at width 512, q|k|v|self
        {"name": "product_mesh", "op": "product", "M": 10242, "N": 2048, "K": 512, "type": "fp16", "epi": "bias"},
        # mlp1 of the full model's processor: GELU, the output is most of the traffic
        {"name": "product_gelu", "op": "product", "M": 189809, "N": 4096, "K": 1024, "type": "fp16", "epi": "gelu"},
        # mlp2 of the full model's processor: the long sum, + residual
        {"name": "product_residual", "op": "product", "M": 189809, "N": 1024, "K": 4096, "type": "fp16", "epi": "residual"},
        # one node between two blocks, pre-norm with modulation
        {"name": "norm_row", "op": "norm", "rows": 1, "C": 1024, "type": "fp16", "post": "none", "pre": "layer", "gate": True, "mod": True, "group": 0},
        # fp32, odd width, RMS norms, each row with its own modulation
        {"name": "norm_ragged", "op": "norm", "rows": 2562, "C": 1000, "type": "fp32", "post": "rms", "pre": "rms", "gate": True, "mod": True, "group": 1},
        # the full model's hidden stream between two blocks, one modulation for all rows
        {"name": "norm_hidden", "op": "norm", "rows": 189809, "C": 1024, "type": "fp16", "post": "layer", "pre": "layer", "gate": True, "mod": True, "group": 0},
        # norm, mlp1, mlp2 of one block at width 512 on a middle-sized mesh, four members with a modulation each
        {"name": "block_mesh", "op": "block", "rows": 40968, "C": 512, "F": 2048, "type": "fp16", "post": "none", "pre": "layer", "gate": True, "mod": True, "group": 10242},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["quantize", "product", "product", "norm", "norm", "block"])
    t = rng.choice(["fp16", "fp16", "fp32"])
    if op == "quantize":
        k = _log(rng, 8, 4096)
        return {"op": op, "rows": _log(rng, 1, min(189809, MOST_ROWS_C // k)), "K": k, "type": t}
    if op == "product":
        n, k = _log(rng, 8, 4096), _log(rng, 32, 4096)
        return {"op": op, "M": _log(rng, 1, min(189809, MOST_MNK // (n * k))), "N": n, "K": k, "type": t,
                "epi": rng.choice(["bias", "gelu", "residual"])}
    c = 32 * _log(rng, 4, 32) if op == "block" else _log(rng, 16, 4096)
    rows = _log(rng, 1, 40968 if op == "block" else min(189809, MOST_ROWS_C // c))
    case = {"op": op, "rows": rows, "C": c, "type": "fp16" if op == "block" else t, "post": rng.choice(["none", "layer", "rms"]),
            "pre": rng.choice(["layer", "rms"]), "gate": rng.random() < 0.7, "mod": rng.random() < 0.7,
            "group": rng.choice([0, 1, max(1, rows // 4)])}
    if op == "block":
        case["F"] = 4 * c
    return case


# ------------------------------------------------------------------ 4-bit blocks in elementary operations

def _round_e2m1(u):
    """u to the nearest e2m1 value, ties to the even code, |u| > 6 to 6."""
    a = u.abs().clamp(max=6.0)
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
    return torch.copysign(torch.round(a / step) * step, u)


def _blocks(x):
    """x [rows, K] fp32 -> (values [rows, nb, 32] of e2m1, exponents [rows, nb]); a cut last block ends in zeros."""
    rows, k = x.shape
    nb = -(-k // 32)
    b = torch.nn.functional.pad(x, (0, 32 * nb - k)).view(rows, nb, 32)
    top = b.abs().amax(-1)
    e = torch.where(top > 0, torch.frexp(top).exponent - 3, -127).clamp(min=-127)
    return _round_e2m1(b * torch.exp2(-e.float()).unsqueeze(-1)), e


def _values(x):
    q, e = _blocks(x)
    return (q * torch.exp2(e.float()).unsqueeze(-1)).view(x.shape[0], -1)[:, :x.shape[1]]


def _pack(x):
    """The codes [rows, 16 nb] (two a byte, the even column low) and the tiled scale bytes of x."""
    q, e = _blocks(x)
    a = q.abs()
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8) | (torch.signbit(q).to(torch.uint8) << 3)
    code = code.view(x.shape[0], -1, 2)
    s = (e + 127).to(torch.uint8)
    rows, nb = s.shape
    rt, kt = -(-rows // 128), -(-nb // 4)
    s = torch.nn.functional.pad(s, (0, 4 * kt - nb, 0, 128 * rt - rows))
    return (code[..., 0] | (code[..., 1] << 4)).contiguous(), s.view(rt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)


def _unpack(codes, scales, k):
    """The fp32 values [rows, k] that codes and tiled scales stand for."""
    rows, nb = codes.shape[0], codes.shape[1] // 16
    rt, kt = -(-rows // 128), -(-nb // 4)
    one = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    pair = torch.stack((one.repeat(16), one.repeat_interleave(16)), -1)
    e = scales.view(rt, kt, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(128 * rt, 4 * kt)[:rows, :nb].float() - 127
    return (pair[codes.int()].view(rows, nb, 32) * torch.exp2(e).unsqueeze(-1)).view(rows, -1)[:, :k]


def _norm(v, kind, w, b):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * w
    return v if b is None else v + b


def _gelu(v):
    return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))


def _group_rows(case, device):
    """The modulation row of each row."""
    r = torch.arange(case["rows"], device=device)
    return r // case["group"] if case["group"] else torch.zeros_like(r)


def _norm_plain(s):
    """(x' rounded to T, y in fp32)."""
    c = s["case"]
    g = _group_rows(c, s["x"].device)
    h = _norm(s["h"].float(), c["post"], s["post_w"], s["post_b"])
    if c["gate"]:
        h = s["gate"].float()[g] * h
    x = (s["res_scale"] * s["x"].float() + h).to(s["x"].dtype)
    y = _norm(x.float(), c["pre"], s["pre_w"], s["pre_b"])
    if c["mod"]:
        y = y * (1.0 + s["scale"].float()[g]) + s["shift"].float()[g]
    return x, y


# ------------------------------------------------------------------ inputs

def _rows(g, rows, k, t, spread=1.0):
    """Rows as a residual stream has them: a normal part whose width differs by column and by row, the rows in a
    buffer whose stride is a multiple of 16 bytes."""
    col = torch.exp(0.5 * torch.randn(k, device="cuda", generator=g))
    row = torch.exp(0.25 * torch.randn(rows, 1, device="cuda", generator=g))
    x = torch.empty(rows, -(-k // 8) * 8, device="cuda", dtype=t)
    x.zero_()
    x[:, :k] = torch.randn(rows, k, device="cuda", generator=g).mul_(spread * row).mul_(col)
    return x[:, :k]


def _space(rows, k, t):
    return torch.empty(rows, -(-k // 8) * 8, device="cuda", dtype=t)[:, :k]


def _mx4_space(rows, k):
    nb = -(-k // 32)
    return (torch.empty(rows, 16 * nb, device="cuda", dtype=torch.uint8),
            torch.empty(-(-rows // 128) * -(-nb // 4) * 512, device="cuda", dtype=torch.uint8))


def _weights(g, n, k):
    return _pack(torch.randn(n, k, device="cuda", generator=g) / math.sqrt(k))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]
    s = {"case": case}
    if case["op"] == "quantize":
        s["x"] = _rows(g, case["rows"], case["K"], t)
        s["codes"], s["scales"] = _mx4_space(case["rows"], case["K"])
        s["y"] = _space(case["rows"], case["K"], t)
        return s
    if case["op"] == "product":
        m, n, k = case["M"], case["N"], case["K"]
        s["A"], s["sA"] = _pack(_rows(g, m, k, t).float())
        s["W"], s["sW"] = _weights(g, n, k)
        s["bias"] = torch.randn(n, device="cuda", generator=g).to(t)
        s["R"] = _rows(g, m, n, t) if case["epi"] == "residual" else None
        s["y"] = _space(m, n, t)
        return s
    rows, c = case["rows"], case["C"]
    groups = -(-rows // case["group"]) if case["group"] else 1
    s["x"], s["h"] = _rows(g, rows, c, t), _rows(g, rows, c, t, 0.5)
    for k in ("gate", "scale", "shift"):
        s[k] = _rows(g, groups, c, t, 0.2) if case["gate" if k == "gate" else "mod"] else None
    for k in ("post", "pre"):
        s[k + "_w"] = 1.0 + 0.1 * torch.randn(c, device="cuda", generator=g)
        s[k + "_b"] = 0.1 * torch.randn(c, device="cuda", generator=g) if case[k] == "layer" else None
    s["res_scale"] = 0.75
    s["out"], s["y"] = _space(rows, c, t), _space(rows, c, t)
    if case["op"] == "block":
        f = case["F"]
        s["W1"], s["sW1"] = _weights(g, f, c)
        s["W2"], s["sW2"] = _weights(g, c, f)
        s["b1"], s["b2"] = (torch.randn(n, device="cuda", generator=g).to(t) for n in (f, c))
        s["a4"], s["f4"] = _mx4_space(rows, c), _mx4_space(rows, f)
    return s


# ------------------------------------------------------------------ one pass

def _vb():
    if "varda.cpp_b200" not in sys.path:
        sys.path.insert(0, "varda.cpp_b200")
    import varda_b200
    return varda_b200


def _run_own(s):
    vb, case = _vb(), s["case"]
    dt = vb.FP16 if case["type"] == "fp16" else vb.FP32
    st = torch.cuda.current_stream().cuda_stream
    ld = lambda a: 0 if a is None else a.stride(0)  # noqa: E731
    if case["op"] == "quantize":
        rows, k, x, y = case["rows"], case["K"], s["x"], s["y"]
        vb.mx4_quantize(dt, x, ld(x), rows, k, s["codes"], ld(s["codes"]), s["scales"], stream=st)
        vb.mx4_dequantize(dt, s["codes"], ld(s["codes"]), s["scales"], rows, k, y, ld(y), stream=st)
        return {"y": y}
    if case["op"] == "product":
        y, r = s["y"], s["R"]
        vb.gemm_mx4(dt, s["A"], ld(s["A"]), s["sA"], s["W"], ld(s["W"]), s["sW"], s["bias"], y, ld(y), r, ld(r), case["M"],
                    case["N"], case["K"], epilogue={"bias": 0, "gelu": 1, "residual": 2}[case["epi"]], stream=st)
        return {"y": y}
    kind = {"none": vb.NORM_NONE, "layer": vb.NORM_LAYER, "rms": vb.NORM_RMS}
    rows, c, x, out, y = case["rows"], case["C"], s["x"], s["out"], s["y"]
    norm = dict(h=s["h"], ldh=ld(s["h"]), post=kind[case["post"]], post_w=s["post_w"], post_b=s["post_b"], gate=s["gate"],
                ldgate=ld(s["gate"]), res_scale=s["res_scale"], out=out, ldo=ld(out), pre=kind[case["pre"]], pre_w=s["pre_w"],
                pre_b=s["pre_b"], scale=s["scale"], shift=s["shift"], ldmod=ld(s["scale"]), rows_per_group=case["group"],
                eps=EPS, stream=st)
    if case["op"] == "norm":
        vb.block_norm(dt, rows, c, x, ld(x), y=y, ldy=ld(y), **norm)
        return {"x": out, "y": y}
    f, (a, sa), (u, su) = case["F"], s["a4"], s["f4"]
    vb.block_norm(dt, rows, c, x, ld(x), y_codes=a, ldc=ld(a), y_scales=sa, **norm)
    vb.gemm_mx4_quant(dt, a, ld(a), sa, s["W1"], ld(s["W1"]), s["sW1"], s["b1"], u, ld(u), su, rows, f, c, epilogue=1, stream=st)
    vb.gemm_mx4(dt, u, ld(u), su, s["W2"], ld(s["W2"]), s["sW2"], s["b2"], y, ld(y), out, ld(out), rows, c, f, epilogue=2, stream=st)
    return {"x": out, "z": y}


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    if case["op"] == "quantize":
        return {"y": _values(s["x"].float()).to(s["x"].dtype)}
    if case["op"] == "product":
        k = case["K"]
        y = _unpack(s["A"], s["sA"], k) @ _unpack(s["W"], s["sW"], k).t() + s["bias"].float()
        if case["epi"] == "gelu":
            y = _gelu(y)
        if case["epi"] == "residual":
            y = y + s["R"].float()
        return {"y": y.to(s["y"].dtype)}
    x, y = _norm_plain(s)
    if case["op"] == "norm":
        return {"x": x, "y": y.to(x.dtype)}
    u = _gelu(_values(y) @ _unpack(s["W1"], s["sW1"], case["C"]).t() + s["b1"].float())
    z = _values(u) @ _unpack(s["W2"], s["sW2"], case["F"]).t() + s["b2"].float() + x.float()
    return {"x": x, "z": z.to(x.dtype)}


# ------------------------------------------------------------------ floors and 64-bit values

def _mx4_bytes(rows, k):
    nb = -(-k // 32)
    return rows * nb * 17


def work(case):
    t = 2 if case["type"] == "fp16" else 4
    if case["op"] == "quantize":
        rows, k = case["rows"], case["K"]
        return {"bytes": 2 * t * rows * k + _mx4_bytes(rows, k), "flops": 2 * rows * k}
    if case["op"] == "product":
        m, n, k = case["M"], case["N"], case["K"]
        outs = 2 if case["epi"] == "residual" else 1
        return {"bytes": _mx4_bytes(m, k) + _mx4_bytes(n, k) + t * n + outs * t * m * n, "flops": 2 * m * n * k}
    rows, c = case["rows"], case["C"]
    groups = -(-rows // case["group"]) if case["group"] else 1
    b = 4 * t * rows * c + t * groups * c * (case["gate"] + 2 * case["mod"])
    if case["op"] == "norm":
        return {"bytes": b, "flops": 12 * rows * c}
    f = case["F"]
    return {"bytes": b + _mx4_bytes(f, c) + _mx4_bytes(c, f) + t * (f + c), "flops": 4 * rows * c * f + 12 * rows * c}


def _codes_to_double(codes, scales, k):
    """[rows, k] in 64 bits, each value from its code's bits: sign, two exponent bits, one mantissa bit."""
    rows, width = codes.shape
    col = torch.arange(k, device=codes.device)
    code = (codes[:, col // 2].to(torch.int16) >> (4 * (col % 2)).to(torch.int16)) & 15
    ex, man = (code >> 1) & 3, (code & 1).double()
    mag = torch.where(ex == 0, 0.5 * man, (1.0 + 0.5 * man) * torch.exp2(ex.double() - 1.0))
    row = torch.arange(rows, device=codes.device).unsqueeze(1)
    blk = (col // 32).unsqueeze(0)
    tiles = -(-(width // 16) // 4)
    at = ((row // 128) * tiles + blk // 4) * 512 + (row % 32) * 16 + (row % 128) // 32 * 4 + blk % 4
    return torch.where(code >= 8, -mag, mag) * torch.exp2(scales[at].double() - 127.0)


def _quantized_double(x):
    """The values of the 4-bit blocks of x in 64 bits, by the distances to the eight magnitudes."""
    rows, k = x.shape
    out = torch.empty_like(x)
    for b in range(0, k, 32):
        v = x[:, b:b + 32]
        top = v.abs().amax(1, keepdim=True)
        e = torch.floor(torch.log2(top.clamp(min=2.0 ** -149)))  # the logarithm of a power of two may round below it
        e = e + (torch.exp2(e + 1.0) <= top).double() - (torch.exp2(e) > top).double()
        unit = torch.exp2((e - 2.0).clamp(min=-127.0))
        a = (v / unit).abs()
        code = torch.zeros_like(a)
        for i in range(7):
            mid = (E2M1[i] + E2M1[i + 1]) / 2.0
            code += ((a >= mid) if i % 2 else (a > mid)).double()
        out[:, b:b + 32] = torch.sign(v) * torch.tensor(E2M1, device=x.device, dtype=torch.float64)[code.long()] * unit
    return out


def _norm_double(v, kind, w, b):
    if kind == "none":
        return v
    m = v.mean(1, keepdim=True) if kind == "layer" else 0.0
    var = ((v - m) ** 2).mean(1, keepdim=True)
    return (v - m) / (var + EPS) ** 0.5 * w.double() + (0.0 if b is None else b.double())


def _linear_double(a, w, b):
    return a @ w.t() + b.double()


def exact(case, seed):
    s = prepare(case, seed)
    rows = case.get("rows") or case["M"]
    parts = []
    if case["op"] == "product":
        w = _codes_to_double(s["W"], s["sW"], case["K"])
    if case["op"] == "block":
        w1, w2 = _codes_to_double(s["W1"], s["sW1"], case["C"]), _codes_to_double(s["W2"], s["sW2"], case["F"])
    for lo in range(0, rows, 16384):  # whole scale tiles of 128 rows
        r = slice(lo, min(rows, lo + 16384))
        if case["op"] == "quantize":
            parts.append({"y": _quantized_double(s["x"][r].double())})
            continue
        if case["op"] == "product":
            tile = -(-(s["A"].shape[1] // 16) // 4) * 512
            y = _linear_double(_codes_to_double(s["A"][r], s["sA"][lo // 128 * tile:], case["K"]), w, s["bias"])
            if case["epi"] == "gelu":
                y = y * 0.5 * torch.special.erfc(-y / math.sqrt(2.0))
            if case["epi"] == "residual":
                y = y + s["R"][r].double()
            parts.append({"y": y})
            continue
        at = torch.arange(lo, r.stop, device="cuda") // max(1, case["group"]) * (case["group"] > 0)
        h = _norm_double(s["h"][r].double(), case["post"], s["post_w"], s["post_b"])
        x = s["res_scale"] * s["x"][r].double() + (h * s["gate"].double()[at] if case["gate"] else h)
        held = x.to(s["x"].dtype).double()  # the stream is held in T, and y is the norm of what is held
        y = _norm_double(held, case["pre"], s["pre_w"], s["pre_b"])
        if case["mod"]:
            y = y + y * s["scale"].double()[at] + s["shift"].double()[at]
        if case["op"] == "norm":
            parts.append({"x": x, "y": y})
            continue
        u = _linear_double(_quantized_double(y), w1, s["b1"])
        u = u * 0.5 * torch.special.erfc(-u / math.sqrt(2.0))
        parts.append({"x": x, "z": _linear_double(_quantized_double(u), w2, s["b2"]) + held})
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
