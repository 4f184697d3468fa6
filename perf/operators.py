"""Block-scaled operands: making them from activations and weights, reading them back, and the MXFP4 product.

Every case is one pass of one operator, or of two that are used together, on the current stream.  ``listed()`` holds
representatives of each, ``draw()`` spreads over the ranges they stand for.  ``run`` computes the definition with elementary
torch operations in f32, or (``own``) makes the framework's calls.
"""
import math

import torch

own = False

EPS = 1e-6
BLOCK = {"mxfp8": 32, "mxfp4": 32, "nvfp4": 16}
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
MOST_VALUES = 16384 * 8192                  # no drawn pass over rows holds more than the largest listed one
MOST_FLOPS = 2.0 * 8192 ** 3                # nor costs a drawn product more


def listed():
    return [
        # one token's activations in front of a linear layer: the smallest call, where the launch is the cost
        {"name": "quantize_mxfp8_1x4096", "op": "quantize", "fmt": "mxfp8", "dtype": "bf16", "rows": 1, "n": 4096},
        # a large prompt batch in front of a linear layer
        {"name": "quantize_mxfp8_16384x8192", "op": "quantize", "fmt": "mxfp8", "dtype": "f16", "rows": 16384, "n": 8192},
        # rows of odd length to two-level 4 bits and back: calibration of a layer whose width fits no block
        {"name": "round_trip_nvfp4_4000x5001", "op": "round_trip", "fmt": "nvfp4", "dtype": "bf16", "rows": 4000, "n": 5001},
        # a gated MLP's weight kept as [K, N] for the dense product, to 4 bits along K and back, as a model is loaded and checked
        {"name": "round_trip_mxfp4_weight", "op": "round_trip", "fmt": "mxfp4", "dtype": "bf16", "rows": 14336, "n": 4096, "transposed": True},
        # the norm in front of a layer's first product, one token
        {"name": "add_norm_mxfp8_1x4096", "op": "add_norm", "fmt": "mxfp8", "dtype": "bf16", "rows": 1, "n": 4096},
        # the same for a prompt of ordinary, not round, length
        {"name": "add_norm_mxfp8_1500x5120", "op": "add_norm", "fmt": "mxfp8", "dtype": "bf16", "rows": 1500, "n": 5120},
        # and for a large prompt batch
        {"name": "add_norm_mxfp8_16384x8192", "op": "add_norm", "fmt": "mxfp8", "dtype": "f16", "rows": 16384, "n": 8192},
        # the gated activation in front of the MLP's second product: halves of one tensor, a decode batch and a prompt
        {"name": "silu_mul_mxfp8_16x14336", "op": "silu_mul", "fmt": "mxfp8", "dtype": "bf16", "rows": 16, "n": 14336},
        {"name": "silu_mul_mxfp8_1500x14336", "op": "silu_mul", "fmt": "mxfp8", "dtype": "bf16", "rows": 1500, "n": 14336},
        # linear layers on one token, on a serving batch whose activations are quantised on the way, and the large square product
        {"name": "linear_mxfp4_1x14336x4096", "op": "linear", "m": 1, "n": 14336, "k": 4096, "dynamic": False},
        {"name": "linear_mxfp4_200x14336x4096", "op": "linear", "m": 200, "n": 14336, "k": 4096, "dynamic": True},
        {"name": "linear_mxfp4_8192", "op": "linear", "m": 8192, "n": 8192, "k": 8192, "dynamic": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _log_multiple(rng, lo, hi, unit):
    return max(unit, _log(rng, lo, hi) // unit * unit)


def draw(rng):
    op = rng.choice(["quantize", "round_trip", "add_norm", "add_norm", "silu_mul", "linear", "linear", "linear"])
    if op == "linear":
        n, k = _log_multiple(rng, 512, 16384, 4), _log_multiple(rng, 512, 16384, 128)
        m = max(1, min(_log(rng, 1, 8192), int(MOST_FLOPS / (2.0 * n * k))))
        return {"op": op, "m": m, "n": n, "k": k, "dynamic": rng.random() < 0.4}
    n = _log(rng, 100, 28672)
    n = n if rng.random() < 0.3 else max(64, n // 64 * 64)
    c = {"op": op, "fmt": "mxfp8", "dtype": rng.choice(["f16", "bf16"]), "rows": min(_log(rng, 1, 16384), MOST_VALUES // n), "n": n}
    if op == "round_trip":
        c.update(fmt=rng.choice(["mxfp8", "mxfp4", "nvfp4"]), transposed=rng.random() < 0.3)
    return c


# ---- inputs ------------------------------------------------------------------------------------------------------------
class _Make:
    """seeded inputs on the GPU"""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def activations(self, rows, n, dtype, std=1.0):
        """normal values, one channel in 128 twenty times as large"""
        x = torch.empty((rows, n), dtype=torch.float32, device="cuda").normal_(0.0, std, generator=self.g)
        loud = torch.randint(n, (max(1, n // 128),), device="cuda", generator=self.g)
        x[:, loud] *= 20.0
        return x.to(dtype)

    def normal(self, rows, n, dtype, std):
        return torch.empty((rows, n), dtype=dtype, device="cuda").normal_(0.0, std, generator=self.g)

    def gain(self, n, dtype):
        return torch.empty(n, dtype=dtype, device="cuda").uniform_(0.5, 1.5, generator=self.g)

    def codes(self, rows, cols, lo, hi):
        return torch.randint(lo, hi, (rows, cols), dtype=torch.uint8, device="cuda", generator=self.g)


def _padded(case):
    """columns of the quantised rows: the row rounded up to whole blocks"""
    b = BLOCK[case["fmt"]]
    return -(-case["n"] // b) * b


def _buffers(rows, cols, fmt):
    """the quantised rows and their scales, in torch's types where it has them (4 bits: two values a byte)"""
    data = torch.zeros((rows, cols), dtype=torch.float8_e4m3fn, device="cuda") if fmt == "mxfp8" else torch.zeros((rows, cols // 2), dtype=torch.uint8, device="cuda")
    scales = torch.zeros((rows, cols // BLOCK[fmt]), dtype=torch.uint8, device="cuda")
    return data, scales.view(torch.float8_e4m3fn if fmt == "nvfp4" else torch.float8_e8m0fnu)


def prepare(case, seed):
    mk, op = _Make(seed), case["op"]
    s = {"case": case}
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        s.update(y=mk.codes(n, k // 2, 0, 256), ys=mk.codes(n, k // 32, 117, 122).view(torch.float8_e8m0fnu),
                 z=torch.zeros((m, n), dtype=torch.bfloat16, device="cuda"))
        if case["dynamic"]:
            s.update(a=mk.activations(m, k, torch.bfloat16), x=torch.zeros((m, k // 2), dtype=torch.uint8, device="cuda"),
                     xs=torch.zeros((m, k // 32), dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu))
        else:
            s.update(x=mk.codes(m, k // 2, 0, 256), xs=mk.codes(m, k // 32, 124, 129).view(torch.float8_e8m0fnu))
        return s
    rows, n, dt = case["rows"], case["n"], DTYPES[case["dtype"]]
    s["out"], s["scales"] = _buffers(rows, _padded(case), case["fmt"])
    if op == "round_trip":
        s["x"] = mk.normal(n, rows, dt, n ** -0.5).t() if case.get("transposed") else mk.activations(rows, n, dt)
        s["back"] = torch.zeros((rows, n), dtype=dt, device="cuda")
        # a calibrated scale of the whole tensor: its largest value reaches the largest element times the largest scale
        s["tensor_scale"] = float(s["x"].abs().max().float()) / (6.0 * 448.0) if case["fmt"] == "nvfp4" else 1.0
    elif op == "quantize":
        s["x"] = mk.activations(rows, n, dt)
    elif op == "add_norm":
        s.update(x=mk.activations(rows, n, dt, 0.3), residual=mk.activations(rows, n, dt), w=mk.gain(n, dt),
                 residual_out=torch.zeros((rows, n), dtype=dt, device="cuda"))
    else:
        both = mk.activations(rows, 2 * n, dt)              # one product gives gate and up side by side
        s.update(gate=both[:, :n], up=both[:, n:])
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------
def _to_e2m1(v):
    """the code of the nearest e2m1 value, ties to the even code: halfway points between neighbours, who wins each in turn"""
    a = v.abs()
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    return code.to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)


def _quantize(v, cols, fmt, g=1.0):
    """f32 rows -> (data, scales), padded with zeros to `cols` columns"""
    rows, n = v.shape
    if cols > n:
        v = torch.nn.functional.pad(v, (0, cols - n))
    v = v.reshape(rows, -1, BLOCK[fmt])
    most = v.abs().amax(-1, keepdim=True)
    lost = ~torch.isfinite(most)
    if fmt == "nvfp4":
        g = torch.tensor(g, dtype=torch.float32, device=v.device)
        scale = (most * (1.0 / (6.0 * g))).clamp(max=448.0).to(torch.float8_e4m3fn)
        unit = scale.float()
        v = torch.where(unit > 0, v * (1.0 / (unit * g)), torch.zeros_like(v))
        scale = torch.where(lost, torch.full_like(unit, float("nan")), unit).to(torch.float8_e4m3fn)
    else:
        byte = (torch.frexp(most).exponent - 1 - (8 if fmt == "mxfp8" else 2) + 127).clamp(0, 254)
        byte = torch.where(most == 0, torch.zeros_like(byte), byte)
        v = torch.ldexp(v, 127 - byte)
        scale = torch.where(lost, torch.full_like(byte, 255), byte).to(torch.uint8).view(torch.float8_e8m0fnu)
    v = torch.where(lost, torch.zeros_like(v), v)
    if fmt == "mxfp8":
        data = v.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).reshape(rows, cols)
    else:
        code = _to_e2m1(v).reshape(rows, cols // 2, 2)
        data = code[..., 0] | (code[..., 1] << 4)
    return data, scale.reshape(rows, -1)


def _values(data, scales, fmt, g=1.0, dtype=torch.float32):
    """the values that quantised rows stand for"""
    if fmt == "mxfp8":
        v = data.to(dtype)
    else:
        table = torch.tensor(E2M1 + [-e for e in E2M1], dtype=dtype, device=data.device)
        v = torch.stack((table[(data & 15).long()], table[(data >> 4).long()]), -1).reshape(data.shape[0], -1)
    return (v.reshape(v.shape[0], -1, BLOCK[fmt]) * scales.to(dtype).unsqueeze(-1)).reshape(v.shape) * g


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "linear":
        x, xs = _quantize(s["a"].float(), case["k"], "mxfp4") if case["dynamic"] else (s["x"], s["xs"])
        return (_values(x, xs, "mxfp4") @ _values(s["y"], s["ys"], "mxfp4").t()).to(torch.bfloat16)
    cols, fmt = _padded(case), case["fmt"]
    if op == "quantize":
        return _quantize(s["x"].float(), cols, fmt)
    if op == "round_trip":
        data, scales = _quantize(s["x"].float(), cols, fmt, s["tensor_scale"])
        return _values(data, scales, fmt, s["tensor_scale"])[:, :case["n"]].to(s["x"].dtype)
    if op == "add_norm":
        c = s["residual"].float() + s["x"].float()
        v = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS) * s["w"].float()
        return _quantize(v, cols, fmt) + (c.to(s["x"].dtype),)
    g = s["gate"].float()
    return _quantize(g / (1.0 + torch.exp(-g)) * s["up"].float(), cols, fmt)


# ---- the framework's calls ---------------------------------------------------------------------------------------------
_package = None


def _ct():
    global _package
    if _package is None:
        from __graft_entry__ import load_package
        _package = load_package()
    return _package


def _tile(m, n):
    """256 x 256 tiles where they fill the chip's 256 compute units, smaller ones otherwise"""
    return [256, 256] if -(-m // 256) * -(-n // 256) >= 256 else [128, 128]


def _rows_of(ct, t):
    return ct.partition(t, [1, t.shape[1]])


def _own(s):
    ct, case = _ct(), s["case"]
    op = case["op"]
    if op == "linear":
        if case["dynamic"]:
            ct.block_quantize(s["a"], _rows_of(ct, s["x"]), _rows_of(ct, s["xs"]), "mxfp4")
        ct.linear_tile_mxfp4(ct.partition(s["z"], _tile(case["m"], case["n"])), s["x"], s["y"], s["xs"], s["ys"])
        return s["z"]
    fmt, out, scales = case["fmt"], _rows_of(ct, s["out"]), _rows_of(ct, s["scales"])
    if op == "quantize":
        ct.block_quantize(s["x"], out, scales, fmt)
    elif op == "round_trip":
        ct.block_quantize(s["x"], out, scales, fmt, s["tensor_scale"])
        ct.block_dequantize(s["out"], s["scales"], _rows_of(ct, s["back"]), fmt, s["tensor_scale"])
        return s["back"]
    elif op == "add_norm":
        ct.add_rms_norm_quantize(s["residual"], s["x"], s["w"], out, scales, _rows_of(ct, s["residual_out"]), EPS, fmt)
        return s["out"], s["scales"], s["residual_out"]
    else:
        ct.silu_mul_quantize(s["gate"], s["up"], out, scales, fmt)
    return s["out"], s["scales"]


def run(s):
    return _own(s) if own else _plain(s)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        # (activations that are quantised on the way are read; their 4-bit form is read and written inside the pass)
        return {"bytes": (n + (0 if case["dynamic"] else m)) * k * (0.5 + 1 / 32) + (2.0 * m * k if case["dynamic"] else 0.0) + 2.0 * m * n, "flops": 2.0 * m * n * k}
    values, size = float(case["rows"]) * case["n"], 4 if case["dtype"] == "f32" else 2
    quantised = case["rows"] * _padded(case) * ((1.0 if case["fmt"] == "mxfp8" else 0.5) + 1 / BLOCK[case["fmt"]])
    if op == "quantize":
        return {"bytes": size * values + quantised, "flops": 3.0 * values}
    if op == "round_trip":                                  # two passes: the quantised rows are one's output and the other's input
        return {"bytes": 2 * size * values + 2 * quantised, "flops": 4.0 * values}
    if op == "add_norm":
        return {"bytes": 3 * size * values + size * case["n"] + quantised, "flops": 8.0 * values}
    return {"bytes": 2 * size * values + quantised, "flops": 8.0 * values}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------
def _on_grid(v, mantissa, lowest, most):
    """v rounded to nearest even on a grid of `mantissa` bits behind the leading one, exponents from `lowest` on, saturated"""
    e = torch.where(v == 0, lowest, (torch.frexp(v)[1] - 1).clamp(min=lowest)) - mantissa
    step = torch.exp2(e.double())
    return (torch.round(v / step) * step).clamp(-most, most)


def _exact_quantized(v, cols, fmt, g):
    """(elements, scales) as values in 64 bits"""
    rows, b = v.shape[0], BLOCK[fmt]
    full = torch.zeros((rows, cols), dtype=torch.float64, device=v.device)
    full[:, :v.shape[1]] = v
    full = full.view(rows, cols // b, b)
    top = torch.maximum(full.amax(-1), -full.amin(-1))
    if fmt == "nvfp4":
        scale = _on_grid((top / (6.0 * g)).clamp(max=448.0), 3, -6, 448.0)
        unit = torch.where(scale > 0, scale * g, torch.full_like(scale, math.inf))
    else:
        at = torch.where(top > 0, torch.floor(torch.log2(top)), torch.full_like(top, -1000.0))
        at = at + (torch.exp2(at + 1) <= top).double() - (torch.exp2(at) > top).double() * (top > 0)    # (the logarithm may round across a power of two)
        scale = torch.exp2((at - (8 if fmt == "mxfp8" else 2)).clamp(-127, 127))
        unit = scale
    scaled = full / unit.unsqueeze(-1)
    q = _on_grid(scaled, 3, -6, 448.0) if fmt == "mxfp8" else _on_grid(scaled, 1, 0, 6.0)
    return q, scale


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        x = _values(s["x"], s["xs"], "mxfp4", dtype=torch.float64)
        if case["dynamic"]:
            q, scale = _exact_quantized(s["a"].double(), case["k"], "mxfp4", 1.0)
            x = (q * scale.unsqueeze(-1)).view(case["m"], case["k"])
        return x @ _values(s["y"], s["ys"], "mxfp4", dtype=torch.float64).t()
    cols, fmt = _padded(case), case["fmt"]
    if op in ("quantize", "round_trip"):
        g = s.get("tensor_scale", 1.0)
        q, scale = _exact_quantized(s["x"].double(), cols, fmt, g)
        if op == "round_trip":
            return (q * (scale * g).unsqueeze(-1)).view(case["rows"], cols)[:, :case["n"]]
        return q.view(case["rows"], cols), scale
    if op == "add_norm":
        c = s["residual"].double() + s["x"].double()
        v = c / torch.sqrt(c.square().sum(-1, keepdim=True) / case["n"] + EPS) * s["w"].double()
        q, scale = _exact_quantized(v, cols, fmt, 1.0)
        return q.view(case["rows"], cols), scale, c
    g = s["gate"].double()
    q, scale = _exact_quantized(g * torch.sigmoid(g) * s["up"].double(), cols, fmt, 1.0)
    return q.view(case["rows"], cols), scale
