"""Layers in microscaled floating point, as cases that can be timed: rows and weights to blocks of 32 values that share a power of
two (e4m3 or e2m1 elements), the norm that leaves its rows so, products of 8-bit rows with 4-bit weights, and sparse experts of such
products.  Sizes are those of ``vllm_distributed_amd/models/configs`` (whole, or one rank's shard) and ragged ones between.

kinds
  quantize  rows to 8 bits (an attention's output in front of its projection), or a weight to 4 bits and back to 16
  norm      residual + branch, RMS norm, 8-bit rows
  linear    a projection of 16-bit rows: to 8 bits, product with 4-bit weights, bias
  normed    the norm and the projection behind it, as a decoder layer runs them
  gate_up   both halves of a gated feed-forward, its activation, 8-bit rows for the projection that follows
  experts   a sparse block behind its router: gate and up, clamped or SiLU, down, weighted sum
"""
import math

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LARGEST = {8: 448.0, 4: 6.0}
EPS = 1e-5


def listed():
    return [
        # 1031 rows of attention output on a 70B model, in front of its output projection
        {"name": "quantize_rows", "kind": "quantize", "bits": 8, "rows": 1031, "width": 8192, "dtype": "bf16"},
        # an 8B model's gate and up matrix, quantised when it is loaded, and widened again
        {"name": "quantize_weight", "kind": "quantize", "bits": 4, "rows": 28672, "width": 4096, "dtype": "bf16"},
        # one stream's token on an 8B model: latency
        {"name": "norm_1", "kind": "norm", "rows": 1, "width": 4096, "dtype": "fp16"},
        # a prompt step on a 70B model
        {"name": "norm_prompt", "kind": "norm", "rows": 8131, "width": 8192, "dtype": "bf16"},
        # one stream's output projection of gpt-oss (64 heads of 64 into 2880 columns, with a bias): latency
        {"name": "linear_1", "kind": "linear", "rows": 1, "n": 2880, "k": 4096, "bias": True, "dtype": "bf16"},
        # 48 streams through a 70B model's down projection: the weights' bytes
        {"name": "linear_48", "kind": "linear", "rows": 48, "n": 8192, "k": 28672, "bias": False, "dtype": "bf16"},
        # prompts through a 70B model's down projection: the matrix cores
        {"name": "linear_prompt", "kind": "linear", "rows": 4096, "n": 8192, "k": 28672, "bias": False, "dtype": "bf16"},
        # a scheduler step of 411 rows into an 8B model's query, key and value projection
        {"name": "normed_qkv_411", "kind": "normed", "rows": 411, "n": 6144, "k": 4096, "bias": False, "dtype": "bf16"},
        # 13 streams through a 70B model's gate and up projection
        {"name": "gate_up_13", "kind": "gate_up", "rows": 13, "inter": 28672, "k": 8192, "dtype": "bf16"},
        # prompts through an 8B model's gate and up projection
        {"name": "gate_up_prompt", "kind": "gate_up", "rows": 6007, "inter": 14336, "k": 4096, "dtype": "bf16"},
        # 16 streams through the 128 experts of gpt-oss-120b: a few rows an expert
        {"name": "experts_decode", "kind": "experts", "tokens": 16, "experts": 128, "chosen": 4, "hidden": 2880, "inter": 2880,
         "limit": 7.0, "dtype": "bf16"},
        # prompts through the 32 experts of gpt-oss-20b: 250 rows an expert
        {"name": "experts_prompt", "kind": "experts", "tokens": 2003, "experts": 32, "chosen": 4, "hidden": 2880, "inter": 2880,
         "limit": 7.0, "dtype": "bf16"},
    ]


# (rows, columns) of a projection's weight: query / key / value, output and down projections of 8B and 70B models, whole and in
# eighths, gpt-oss' attention, and generic ones whose tiles come out ragged
PROJECTIONS = [(6144, 4096), (4096, 4096), (4096, 14336), (10240, 8192), (8192, 8192), (8192, 28672), (1280, 8192), (8192, 1024),
               (8192, 3584), (5120, 2880), (2880, 4096), (1000, 1056), (264, 4640), (4104, 2208)]
# (inner width, hidden) of gated feed-forwards
GATED = [(14336, 4096), (28672, 8192), (3584, 8192), (1792, 4096), (1408, 2048), (2560, 6144), (640, 1120)]
# experts, chosen, hidden, inner width, limit of the clamped activation (0: SiLU), most tokens
SPARSE = [(128, 4, 2880, 2880, 7.0, 256), (32, 4, 2880, 2880, 7.0, 2000), (8, 2, 4096, 14336, 0.0, 1500), (64, 6, 2048, 1408, 0.0, 2000)]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize", "norm", "linear", "linear", "normed", "gate_up", "experts"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "quantize":
        bits, width = rng.choice([8, 4]), 32 * _log_int(rng, 1, 896)
        return {"kind": kind, "bits": bits, "rows": _log_int(rng, 1, min(30000, (1 << 27) // width)), "width": width,
                "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    if kind == "norm":
        width = rng.choice([2048, 2880, 4096, 5120, 8192, 32 * rng.randint(4, 256)])
        return {"kind": kind, "rows": _log_int(rng, 1, 8000), "width": width, "dtype": dtype}
    if kind in ("linear", "normed"):
        n, k = rng.choice(PROJECTIONS)
        return {"kind": kind, "rows": _log_int(rng, 1, min(8000, 4096 * 8192 * 28672 // (n * k))), "n": n, "k": k,
                "bias": rng.random() < 0.3, "dtype": dtype}
    if kind == "gate_up":
        inter, k = rng.choice(GATED)
        return {"kind": kind, "rows": _log_int(rng, 1, min(6000, 6007 * 14336 * 4096 // (inter * k))), "inter": inter, "k": k,
                "dtype": dtype}
    experts, chosen, hidden, inter, limit, most = rng.choice(SPARSE)
    return {"kind": kind, "tokens": _log_int(rng, 1, most), "experts": experts, "chosen": chosen, "hidden": hidden, "inter": inter,
            "limit": limit, "dtype": dtype}


# ------------------------------------------------------------------ the formats, in elementary operations
def _exponent(a, bits):
    """The smallest e with a <= largest * 2^e, of a >= 0 (448 = 0.875 * 2^9, 6 = 0.75 * 2^3)."""
    m, x = torch.frexp(a)
    e = x - (9 if bits == 8 else 3) + (m > (0.875 if bits == 8 else 0.75)).to(x.dtype)
    return torch.where(a > 0, e, torch.full_like(e, -127)).clamp(-127, 127)


def _round4(u):
    """u, |u| <= 6, to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with its sign, ties to the even code."""
    a = u.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).to(u.dtype)
    return torch.copysign(torch.round(a / step) * step, u)


def _blocks(v, bits):
    """v [..., K] -> (elements [..., K/32, 32], exponents [..., K/32, 1]): v ~ element * 2^exponent."""
    b = v.reshape(*v.shape[:-1], v.shape[-1] // 32, 32)
    e = _exponent(b.abs().amax(-1, keepdim=True), bits)
    u = torch.ldexp(b, -e)
    return (_round4(u) if bits == 4 else u.to(torch.float8_e4m3fn).to(v.dtype)), e


def _rounded(v, bits):
    """v as its blocks stand for it."""
    u, e = _blocks(v, bits)
    return torch.ldexp(u, e).reshape(v.shape)


def _scale_bytes(e):
    return (e.squeeze(-1) + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _rows8(v):
    """v in the form that 8-bit rows have: elements [..., K] and scales [..., K/32]."""
    u, e = _blocks(v, 8)
    return u.to(torch.float8_e4m3fn).reshape(v.shape), _scale_bytes(e)


def _pack4(u, e):
    """Blocks of 4-bit values -> ([..., K/2] codes, the even element in the low half, [..., K/32] scale bytes)."""
    mag = (u.abs() * 2).to(torch.int64)
    code = torch.tensor([0, 1, 2, 3, 4, 0, 5, 0, 6, 0, 0, 0, 7], dtype=torch.uint8, device=u.device)[mag]
    code = (code | (torch.signbit(u).to(torch.uint8) << 3)).reshape(*u.shape[:-2], -1, 2)
    return code[..., 0] | (code[..., 1] << 4), (e.squeeze(-1) + 127).to(torch.uint8)


def _widen4(packed, scales):
    """What _pack4 left, in 32 bits."""
    lut = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=packed.device)
    v = torch.stack([lut[(packed & 15).to(torch.int32)], lut[(packed >> 4).to(torch.int32)]], dim=-1)
    v = v.reshape(*scales.shape, 32)
    return torch.ldexp(v, (scales.to(torch.int32) - 127).unsqueeze(-1)).reshape(*packed.shape[:-1], -1)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(DEV).manual_seed(int(seed) * 11 + 5)


def _normal(g, *shape, std=1.0, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, std, generator=g)


def _activations(g, rows, width, dtype):
    """Rows as they come between layers: normal values, some columns many times the others' size."""
    cols = torch.exp(_normal(g, width, std=0.6))
    return (_normal(g, rows, width) * cols).to(dtype)


def _weights(g, *shape):
    """A 4-bit matrix (or several) of normal weights, a slice at a time: its codes and scale bytes."""
    flat = math.prod(shape[:-1])
    packed = torch.empty(flat, shape[-1] // 2, dtype=torch.uint8, device=DEV)
    scales = torch.empty(flat, shape[-1] // 32, dtype=torch.uint8, device=DEV)
    for lo in range(0, flat, 32768):
        hi = min(flat, lo + 32768)
        packed[lo:hi], scales[lo:hi] = _pack4(*_blocks(_normal(g, hi - lo, shape[-1], std=shape[-1] ** -0.5), 4))
    return packed.view(*shape[:-1], -1), scales.view(*shape[:-1], -1)


def prepare(case, seed):
    g, kind, dtype = _gen(seed), case["kind"], TYPES[case["dtype"]]
    s = dict(case, type=dtype)
    if kind == "quantize":
        s["x"] = _activations(g, case["rows"], case["width"], dtype) if case["bits"] == 8 else _normal(
            g, case["rows"], case["width"], std=case["width"] ** -0.5).to(dtype)
    if kind in ("norm", "normed"):
        width = case["width"] if kind == "norm" else case["k"]
        s["x"] = _activations(g, case["rows"], width, dtype)
        s["residual"] = (4 * _normal(g, case["rows"], width)).to(dtype)
        s["gain"] = (1 + 0.2 * _normal(g, width)).to(dtype)
    if kind in ("linear", "gate_up"):
        s["x"] = _activations(g, case["rows"], case["k"], dtype)
    if kind in ("linear", "normed"):
        s["w"] = _weights(g, case["n"], case["k"])
        s["bias"] = _normal(g, case["n"]).to(dtype) if case["bias"] else None
    if kind == "gate_up":
        s["w"] = _weights(g, 2 * case["inter"], case["k"])
    if kind == "experts":
        experts, hidden, inter = case["experts"], case["hidden"], case["inter"]
        s["x"] = (0.5 * _normal(g, case["tokens"], hidden)).to(dtype)
        s["w13"], s["w2"] = _weights(g, experts, 2 * inter, hidden), _weights(g, experts, hidden, inter)
        s["b13"] = s["b2"] = None
        if case["limit"]:
            s["b13"], s["b2"] = _normal(g, experts, 2 * inter, std=0.5).to(dtype), _normal(g, experts, hidden, std=0.5).to(dtype)
        top = torch.topk(_normal(g, case["tokens"], experts), case["chosen"], dim=-1)
        s["topw"], s["topi"] = torch.softmax(top.values, -1), top.indices.to(torch.int32)
    if own:     # weights in the kernels' layout, which a program makes once when it loads them
        from vllm_distributed_amd.ops import quant
        if "w" in s:
            s["weight"] = quant.pack_mx(*s["w"], halves=2 if kind == "gate_up" else 1)
        if kind == "experts":
            s["weight13"], s["weight2"] = quant.pack_mx(*s["w13"], halves=2), quant.pack_mx(*s["w2"])
            s["bias13"] = None if s["b13"] is None else quant.pad_mx_bias(s["b13"], halves=2)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    kind = s["kind"]
    if own:
        from vllm_distributed_amd import ops
        if kind == "quantize":
            rows = ops.mx_quantize(s["x"], s["bits"])
            return [rows.q, rows.s] if s["bits"] == 8 else [ops.mx_dequantize(rows, s["type"]), rows.s]
        if kind == "norm":
            rows, residual = ops.fused_add_rms_norm_mx(s["x"], s["residual"], s["gain"], EPS)
            return [rows.q, rows.s, residual]
        if kind == "linear":
            return [ops.mx_linear(s["x"], s["weight"], s["bias"])]
        if kind == "normed":
            rows, residual = ops.fused_add_rms_norm_mx(s["x"], s["residual"], s["gain"], EPS)
            return [ops.mx_linear(rows, s["weight"], s["bias"]), residual]
        if kind == "gate_up":
            rows = ops.mx_gate_up(s["x"], s["weight"])
            return [rows.q, rows.s]
        return [ops.mx_experts(s["x"], s["topw"], s["topi"], s["weight13"], s["weight2"], s["bias13"], s["b2"], limit=s["limit"])]
    x = s["x"].float()
    if kind == "quantize":
        if s["bits"] == 8:
            return list(_rows8(x))
        u, e = _blocks(x, 4)
        return [torch.ldexp(u, e).reshape(x.shape).to(s["type"]), _scale_bytes(e)]
    if kind in ("norm", "normed"):
        x = x + s["residual"].float()
        residual = x.to(s["type"])
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s["gain"].float()
        if kind == "norm":
            return [*_rows8(x), residual]
    if kind in ("linear", "normed"):
        y = _rounded(x, 8) @ _widen4(*s["w"]).t()
        y = (y if s["bias"] is None else y + s["bias"].float()).to(s["type"])
        return [y] if kind == "linear" else [y, residual]
    if kind == "gate_up":
        h = _rounded(x, 8) @ _widen4(*s["w"]).t()
        gate, up = h[:, :s["inter"]], h[:, s["inter"]:]
        return list(_rows8(gate * torch.sigmoid(gate) * up))
    # every expert over every row, of which each row keeps those that it chose
    at = (s["topi"].long(), torch.arange(x.shape[0], device=x.device).unsqueeze(1))
    h = torch.matmul(_rounded(x, 8).unsqueeze(0), _widen4(*s["w13"]).transpose(1, 2))
    if s["b13"] is not None:
        h = h + s["b13"].float().unsqueeze(1)
    gate, up = h[..., :s["inter"]], h[..., s["inter"]:]
    if s["limit"]:
        gate, up = gate.clamp(max=s["limit"]), up.clamp(-s["limit"], s["limit"])
        a = (up + 1) * gate * torch.sigmoid(1.702 * gate)
    else:
        a = gate * torch.sigmoid(gate) * up
    y = torch.matmul(_rounded(a, 8), _widen4(*s["w2"]).transpose(1, 2))
    if s["b2"] is not None:
        y = y + s["b2"].float().unsqueeze(1)
    return [(y[at] * s["topw"].unsqueeze(-1)).sum(1).to(s["type"])]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind, size = case["kind"], TYPES[case["dtype"]].itemsize
    if kind == "quantize":
        n = case["rows"] * case["width"]      # 8 bits: read, write; 4 bits: to 4.25 bits, and from them
        out = n * 33 / 32 if case["bits"] == 8 else n * (2 * 17 / 32 + size)
        return {"bytes": n * size + out, "flops": 3 * n}
    if kind == "norm":
        n = case["rows"] * case["width"]
        return {"bytes": n * (3 * size + 33 / 32) + case["width"] * size, "flops": 8 * n}
    if kind in ("linear", "normed"):
        m, n, k = case["rows"], case["n"], case["k"]
        rows = m * k * (3 if kind == "normed" else 1) * size
        return {"bytes": rows + n * k * 17 / 32 + (m * n + n * case["bias"]) * size, "flops": 2 * m * n * k}
    if kind == "gate_up":
        m, i, k = case["rows"], case["inter"], case["k"]
        return {"bytes": m * k * size + 2 * i * k * 17 / 32 + m * i * 33 / 32, "flops": 4 * m * i * k}
    t, c, e, h, i = case["tokens"], case["chosen"], case["experts"], case["hidden"], case["inter"]
    used = e * (1 - (1 - c / e) ** t)         # experts that rows chose
    return {"bytes": used * 3 * i * h * 17 / 32 + 2 * t * h * size, "flops": 6 * t * c * i * h}


# ------------------------------------------------------------------ the same in 64 bits
def _values(packed, scales):
    """The numbers that 4-bit codes and scale bytes stand for, from the bits: sign, two of exponent, one of mantissa."""
    c = torch.stack([packed & 15, packed >> 4], -1).reshape(*packed.shape[:-1], -1).int()
    ex, ma, sign = (c >> 1) & 3, (c & 1).double(), 1.0 - 2.0 * (c >> 3).double()
    mag = torch.where(ex == 0, ma * 0.5, (1 + 0.5 * ma) * torch.exp2((ex - 1).double()))
    return sign * mag * torch.exp2(scales.double() - 127).repeat_interleave(32, dim=-1)


def _nearest(v, bits):
    """v in 64 bits -> (elements, what a block's elements are multiplied by): the grid of the format, by its step at each size."""
    b = v.unflatten(-1, (-1, 32))
    top = LARGEST[bits]
    a = b.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2((a / top).clamp_min(2.0 ** -150)))
    e = torch.where(a > top * torch.exp2(e), e + 1, torch.where(a <= top * torch.exp2(e - 1), e - 1, e))     # (a rounded logarithm)
    scale = torch.exp2(e.clamp(-127, 127))
    u = b / scale
    low, mantissa = (-6, 3) if bits == 8 else (0, 1)
    step = torch.exp2(torch.floor(torch.log2(u.abs().clamp_min(2.0 ** low))).clamp_min(low) - mantissa)
    return torch.round(u / step) * step, scale, u


def _as_rows(v, bits=8):
    u, scale, _ = _nearest(v, bits)
    return (u * scale).flatten(-2)


def exact(case, seed):
    """Elements of 8-bit rows that follow computed numbers are given before their rounding, which is within the format's half step of either
    neighbour; scales of such rows have no such value (a number beside a power of two may fall to either side)."""
    s, kind = prepare(case, seed), case["kind"]
    x = s["x"].double()
    if kind == "quantize":
        u, scale, _ = _nearest(x, case["bits"])
        if case["bits"] == 8:
            return [u.flatten(-2), scale.squeeze(-1)]
        return [(u * scale).flatten(-2), scale.squeeze(-1)]
    residual = None
    if kind in ("norm", "normed"):
        residual = x + s["residual"].double()
        x = residual / torch.sqrt((residual ** 2).sum(-1, keepdim=True) / residual.shape[-1] + EPS) * s["gain"].double()
        if kind == "norm":
            return [_nearest(x, 8)[2].flatten(-2), None, residual]
    if kind in ("linear", "normed"):
        y = _as_rows(x) @ _values(*s["w"]).T
        y = y if s["bias"] is None else y + s["bias"].double()
        return [y] if residual is None else [y, residual]
    if kind == "gate_up":
        h = _as_rows(x) @ _values(*s["w"]).T
        g, u = h.chunk(2, -1)
        return [_nearest(g / (1 + torch.exp(-g)) * u, 8)[2].flatten(-2), None]
    rows, out = _as_rows(x), torch.zeros_like(x)
    for e in range(case["experts"]):
        t, j = (s["topi"] == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        h = rows[t] @ _values(s["w13"][0][e], s["w13"][1][e]).T
        h = h if s["b13"] is None else h + s["b13"][e].double()
        g, u = h.chunk(2, -1)
        if case["limit"]:
            g, u = g.clamp(max=case["limit"]), u.clamp(-case["limit"], case["limit"])
            a = (u + 1) * g / (1 + torch.exp(-1.702 * g))
        else:
            a = g / (1 + torch.exp(-g)) * u
        y = _as_rows(a) @ _values(s["w2"][0][e], s["w2"][1][e]).T
        y = y if s["b2"] is None else y + s["b2"][e].double()
        out.index_add_(0, t, y * s["topw"][t, j].double().unsqueeze(1))
    return [out]
