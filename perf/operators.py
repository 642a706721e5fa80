"""The MXFP4 operators' calls, with their sizes: quantisation to microscaled 4-bit floating point, the
product of two such operands with its epilogues, and the chains in which a quantised DiT block runs them
(adaLN norm -> QKV or output projection, the whole feed-forward network).

MXFP4: elements of E2M1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two to a byte with the even
element in the low four bits; one E8M0 scale 2^(code - 127) for 32 elements along K,
code - 127 = floor(log2(max |x|)) - 2, at least -127; a block that holds an infinity or a NaN has code 255
and stands for NaN. The scales of [rows, K] are [ceil(K / 256), rows, 8]: block b of row r at
[b // 8, r, b % 8], the last slab's unused bytes 0.

Two model geometries are in use, as in cases.py: ``stream`` (hidden 4096, FFN 16384; frames of 1560
tokens, chunks of 3120, 7020 at 720 x 1248, a prompt of 347) and ``wide`` (hidden 5120, FFN 13824, chunks
of 10800 tokens, 512 condition tokens). Activations are N(0, 1) with 0.5 % of their channels scaled by 20,
weights N(0, 0.02), biases N(0, 0.01).
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MAX_FLOPS = 2 * 10800 * 5120 * 15360


def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "joyai-video-edit_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import joyomni_ops
    return joyomni_ops


def listed():
    return [
        # the shortest prompt of the condition stream: a launch and little else
        {"name": "quant_64x4096", "kind": "quant", "rows": 64, "K": 4096, "dtype": "bf16"},
        # a small picture's tokens in the other 16-bit type, odd row count, odd number of blocks
        {"name": "quant_1371x5152_fp16", "kind": "quant", "rows": 1371, "K": 5152, "dtype": "fp16"},
        # the input of a benchmark chunk's FFN-down: the largest activation of the block
        {"name": "quant_10800x13824", "kind": "quant", "rows": 10800, "K": 13824, "dtype": "bf16"},
        # one token: the modulation vector through a projection, W from HBM
        {"name": "product_1x4096x12288", "kind": "product", "rows": 1, "K": 4096, "N": 12288, "epilogue": "plain",
         "dtype": "bf16"},
        # the condition stream's QKV layer for the usual prompt: odd rows, weight-bound
        {"name": "product_347x5120x15360", "kind": "product", "rows": 347, "K": 5120, "N": 15360, "epilogue": "plain",
         "dtype": "bf16"},
        # FFN-up with GELU of one 480 x 832 frame, fp16
        {"name": "product_gelu_1560_fp16", "kind": "product", "rows": 1560, "K": 4096, "N": 16384, "epilogue": "gelu",
         "dtype": "fp16"},
        # FFN-down with the gated residual of a 720 x 1248 chunk
        {"name": "product_residual_7020", "kind": "product", "rows": 7020, "K": 16384, "N": 4096, "epilogue": "residual",
         "dtype": "bf16"},
        # the QKV projection of a benchmark chunk: the largest product
        {"name": "product_10800x5120x15360", "kind": "product", "rows": 10800, "K": 5120, "N": 15360,
         "epilogue": "plain", "dtype": "bf16"},
        # adaLN norm into the QKV layer, the usual prompt
        {"name": "norm_project_347", "kind": "project", "rows": 347, "K": 4096, "N": 12288, "dtype": "bf16"},
        # adaLN norm into a square projection, one 480 x 832 chunk in the wide geometry
        {"name": "norm_project_3120", "kind": "project", "rows": 3120, "K": 5120, "N": 5120, "dtype": "bf16"},
        # the feed-forward network of the shortest prompt: three launches on 64 rows
        {"name": "ffn_64", "kind": "ffn", "rows": 64, "K": 5120, "N": 13824, "dtype": "bf16"},
        # the feed-forward network of one 480 x 832 chunk
        {"name": "ffn_3120", "kind": "ffn", "rows": 3120, "K": 4096, "N": 16384, "dtype": "bf16"},
    ]


def _spread(rng, low, high, unit):
    """A multiple of ``unit`` in [low, high], even over the logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(unit, min(high, int(round(v / unit)) * unit))


def draw(rng):
    kind = rng.choice(["quant", "product", "product", "project", "ffn"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    rows = _spread(rng, 1, 10800, 1)
    K = _spread(rng, 1024, 16384, 32)
    if kind == "quant":
        return {"kind": kind, "rows": rows, "K": K, "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    K = _spread(rng, 1024, 8192, 32) if kind != "product" else K
    N = _spread(rng, 1024, 16384, 32 if kind == "ffn" else 8)
    most = MAX_FLOPS // (2 * K * N * (2 if kind == "ffn" else 1))
    case = {"kind": kind, "rows": min(rows, most), "K": K, "N": N, "dtype": dtype}
    if kind == "product":
        case["epilogue"] = rng.choice(["plain", "gelu", "residual"])
    return case


# ------------------------------------------------------------------------------------------- plain form
def _scale_exponents(x):
    """x [R, K] fp32 -> the blocks' exponents [R, K / 32] (int32; 128 where a block is not finite)."""
    amax = x.reshape(x.shape[0], -1, 32).abs().amax(-1)  # NaN where a block holds one
    e = torch.frexp(amax)[1] - 3  # amax = m 2^e with m in [0.5, 1): floor(log2(amax)) = e - 1
    e = torch.where(amax == 0, torch.full_like(e, -127), e.clamp(min=-127))
    return torch.where(torch.isfinite(amax), e, torch.full_like(e, 128))


def _elements(x, e):
    """The E2M1 elements (fp32 values) of x [R, K] fp32 for block exponents e."""
    a = torch.ldexp(torch.ldexp(x.abs().reshape(x.shape[0], -1, 32), (-(e // 2))[..., None]), (-(e - e // 2))[..., None])
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = (torch.round(a / step) * step).clamp(max=6)  # ties to even: also to the even code
    return torch.copysign(q, x.reshape(q.shape))


def _quant_values(x):
    """What the MXFP4 quantisation of x [R, K] fp32 stands for, fp32."""
    e = _scale_exponents(x)
    v = torch.ldexp(torch.ldexp(_elements(x, e), (e // 2)[..., None]), (e - e // 2)[..., None])
    return torch.where((e == 128)[..., None], torch.full_like(v, math.nan), v).reshape(x.shape)


_CODE_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _decode(q, s, dtype=torch.float32):
    """Codes [R, K / 2] (uint8) and scales [slabs, R, 8] (uint8) -> the values they stand for."""
    table = torch.tensor(_CODE_VALUES, dtype=dtype, device=q.device)
    v = torch.stack([table[(q & 15).long()], table[(q >> 4).long()]], -1).reshape(q.shape[0], -1, 32)
    e = s.permute(1, 0, 2).reshape(q.shape[0], -1)[:, : v.shape[1]].to(torch.int32) - 127
    v = torch.ldexp(torch.ldexp(v, (e // 2)[..., None]), (e - e // 2)[..., None])
    return torch.where((e == 128)[..., None], torch.full_like(v, math.nan), v).reshape(q.shape[0], -1)


def _norm(x, scale, shift):
    d = x - x.mean(-1, keepdim=True)
    return d * torch.rsqrt((d * d).mean(-1, keepdim=True) + EPS) * (1 + scale) + shift


def _gelu(x):
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))


def _product(a, w, s, bias):
    return a @ _decode(w, s).t() + bias.float()


# ------------------------------------------------------------------------------------------------ inputs
def _codes(x):
    """x [R, K] fp32 -> its MXFP4 codes [R, K / 2] and scales [slabs, R, 8], both uint8."""
    R, K = x.shape
    e = _scale_exponents(x)
    v = _elements(x, e)
    a = v.abs()
    c = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    c = (c | torch.signbit(v).to(torch.uint8) * 8).reshape(R, K // 2, 2)
    s = torch.zeros(R, -(-K // 256) * 8, dtype=torch.uint8, device=x.device)
    s[:, : K // 32] = (e + 127).to(torch.uint8)
    return (c[..., 0] | c[..., 1] << 4).contiguous(), s.view(R, -1, 8).permute(1, 0, 2).contiguous()


def _activations(rows, K, dtype, g):
    x = torch.randn(rows, K, generator=g, device="cuda")
    cols = torch.randperm(K, generator=g, device="cuda")[: max(1, K // 200)]
    x[:, cols] *= 20
    return x.to(DTYPES[dtype])


def _weights(N, K, g):
    return _codes((0.02 * torch.randn(N, K, generator=g, device="cuda")).to(torch.bfloat16).float())


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, K, kind, dt = case["rows"], case["K"], case["kind"], DTYPES[case["dtype"]]
    s = {"case": case}
    if kind == "quant":
        s["x"] = _activations(rows, K, case["dtype"], g)
        return s
    N = case["N"]
    vec = lambda n, std: (std * torch.randn(n, generator=g, device="cuda")).to(dt)  # noqa: E731
    if kind == "product":
        s["a"], s["sa"] = _codes(_activations(rows, K, case["dtype"], g).float())
    else:
        s["x"] = _activations(rows, K, case["dtype"], g)
        s["scale"], s["shift"] = vec((1, K), 0.2), vec((1, K), 0.2)
    s["w"], s["sw"] = _weights(N, K, g)
    s["bias"] = vec(N, 0.01)
    if kind == "ffn":
        s["w2"], s["sw2"] = _weights(K, N, g)
        s["bias2"], s["gate"] = vec(K, 0.01), vec(K, 0.5)
    elif case.get("epilogue") == "residual":
        s["residual"], s["gate"] = _activations(rows, N, case["dtype"], g), vec(N, 0.5)
    return s


# --------------------------------------------------------------------------------------------------- run
def _run_plain(st):
    c, kind = st["case"], st["case"]["kind"]
    dt = DTYPES[c["dtype"]]
    if kind == "quant":
        return _quant_values(st["x"].float()).to(torch.bfloat16)
    if kind == "product":
        y = _product(_decode(st["a"], st["sa"]), st["w"], st["sw"], st["bias"])
        if c["epilogue"] == "gelu":
            y = _gelu(y)
        if c["epilogue"] == "residual":
            y = st["residual"].float() + y * st["gate"].float()
        return y.to(dt)
    x = st["x"].float()
    a = _quant_values(_norm(x, st["scale"].float(), st["shift"].float()))
    y = _product(a, st["w"], st["sw"], st["bias"])
    if kind == "project":
        return y.to(dt)
    h = _quant_values(_gelu(y))
    return (x + _product(h, st["w2"], st["sw2"], st["bias2"]) * st["gate"].float()).to(dt)


def _run_own(st):
    jo = _package()
    c, kind = st["case"], st["case"]["kind"]
    dt, rows, K = DTYPES[c["dtype"]], c["rows"], c["K"]
    fp4 = lambda t: t.view(torch.float4_e2m1fn_x2)  # noqa: E731
    e8 = lambda t: t.view(torch.float8_e8m0fnu)  # noqa: E731

    def room(k):
        return (torch.empty(rows, k // 2, dtype=torch.float4_e2m1fn_x2, device="cuda"),
                torch.empty(-(-k // 256), rows, 8, dtype=torch.float8_e8m0fnu, device="cuda"))

    if kind == "quant":
        q, s = room(K)
        jo.per_block_quant_mxfp4(st["x"], q, s)
        return jo.mxfp4_dequantize(q, s, torch.bfloat16)
    w, sw = fp4(st["w"]).t(), e8(st["sw"])
    if kind == "product":
        a, sa = fp4(st["a"]), e8(st["sa"])
        if c["epilogue"] == "residual":
            return jo.mxfp4_scaled_mm_gated_residual(a, w, sa, sw, st["residual"], st["gate"], st["bias"])
        mm = jo.mxfp4_scaled_mm_gelu_tanh if c["epilogue"] == "gelu" else jo.mxfp4_scaled_mm
        return mm(a, w, sa, sw, dt, st["bias"])
    q, s = room(K)
    jo.fused_norm_scale_shift_mxfp4(st["x"], None, None, st["scale"], st["shift"], "layer", EPS, q, s)
    if kind == "project":
        return jo.mxfp4_scaled_mm(q, w, s, sw, dt, st["bias"])
    h, sh = room(c["N"])
    jo.mxfp4_scaled_mm_gelu_tanh_quant(q, w, s, sw, st["bias"], h, sh)
    return jo.mxfp4_scaled_mm_gated_residual(h, fp4(st["w2"]).t(), sh, e8(st["sw2"]), st["x"], st["gate"], st["bias2"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# -------------------------------------------------------------------------------------------------- work
def work(case):
    rows, K, kind = case["rows"], case["K"], case["kind"]
    size = 4 if case["dtype"] == "fp32" else 2
    mx = 0.5 + 1 / 32  # bytes of an MXFP4 element with its share of the scale
    if kind == "quant":  # the input, the codes and the values that they stand for
        return {"bytes": rows * K * (size + mx + 2), "flops": 0}
    N = case["N"]
    if kind == "product":
        more = rows * N * size + N * size if case["epilogue"] == "residual" else 0
        return {"bytes": (rows + N) * K * mx + rows * N * size + N * size + more, "flops": 2 * rows * N * K}
    if kind == "project":
        return {"bytes": rows * K * size + N * K * mx + rows * N * size + (2 * K + N) * size, "flops": 2 * rows * N * K}
    return {"bytes": 2 * rows * K * size + 2 * N * K * mx + (4 * K + N) * size, "flops": 4 * rows * N * K}


# ----------------------------------------------------------------------------- the definition, in 64 bits
def _nearest(x):
    """x [R, K] float64 -> the values of its MXFP4 quantisation: each block's scale from the definition,
    each element the nearest of the eight magnitudes, the one with the even code where two are as near."""
    out = torch.empty_like(x)
    mags = torch.tensor(_CODE_VALUES[:8], dtype=torch.float64, device=x.device)
    for r in range(0, x.shape[0], 256):  # 256 rows at a time: memory
        b = x[r:r + 256].reshape(-1, 32)
        amax = b.abs().max(-1, keepdim=True).values
        fine = torch.isfinite(amax)
        safe = torch.where(fine & (amax > 0), amax, torch.ones_like(amax))
        e = torch.floor(torch.log2(safe))
        e = torch.where(torch.exp2(e) > safe, e - 1, torch.where(torch.exp2(e + 1) <= safe, e + 1, e)) - 2
        scale = torch.exp2(torch.where(amax == 0, torch.full_like(e, -127.0), e.clamp(min=-127.0)))
        a = b.abs() / scale
        best, dist = torch.zeros_like(a), a.clone()  # magnitude 0, code 0
        for code in range(1, 8):
            d = (a - mags[code]).abs()
            nearer = d < dist if code % 2 else d <= dist  # codes ascend: a tie is between neighbours
            best, dist = torch.where(nearer, mags[code], best), torch.where(nearer, d, dist)
        v = torch.where(b < 0, -best, best) * scale
        out[r:r + 256] = torch.where(fine, v, torch.full_like(v, math.nan)).reshape(-1, x.shape[1])
    return out


def _value64(q, s):
    low, high = (q & 15).long(), (q >> 4).long()
    codes = torch.stack([low, high], 2).reshape(q.shape[0], -1)
    mag = codes & 7
    expo, man = mag >> 1, (mag & 1).double()
    v = torch.where(expo == 0, man / 2, (1 + man / 2) * torch.exp2((expo - 1).double()))
    v = torch.where(codes > 7, -v, v)
    block = torch.arange(v.shape[1], device=q.device) // 32
    scale = s.double()[block // 8, :, block % 8].t()
    return torch.where(scale == 255, math.nan, v * torch.exp2(scale - 127))


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    f = {k: v.double() for k, v in st.items() if k in ("x", "bias", "bias2", "gate", "scale", "shift", "residual")}
    if kind == "quant":
        return _nearest(f["x"])

    def gelu(v):
        return v * torch.sigmoid(2 * (2 / math.pi) ** 0.5 * (v + 0.044715 * v ** 3))

    if kind == "product":
        y = torch.matmul(_value64(st["a"], st["sa"]), _value64(st["w"], st["sw"]).t().contiguous()) + f["bias"]
        if case["epilogue"] == "gelu":
            return gelu(y)
        return f["residual"] + y * f["gate"] if case["epilogue"] == "residual" else y
    var, mean = torch.var_mean(f["x"], dim=1, keepdim=True, unbiased=False)
    n = (f["x"] - mean) / torch.sqrt(var + EPS) * (1 + f["scale"]) + f["shift"]
    y = torch.matmul(_nearest(n), _value64(st["w"], st["sw"]).t().contiguous()) + f["bias"]
    if kind == "project":
        return y
    z = torch.matmul(_nearest(gelu(y)), _value64(st["w2"], st["sw2"]).t().contiguous()) + f["bias2"]
    return f["x"] + z * f["gate"]
