"""Timed cases of the microscaled operators (``ancha_b200/microscaled.py``), beside their plain form.

Three operators, each with the number formats "mxf8" (E4M3 elements, one power of two for each 32 of
a row), "mxf4" (E2M1 elements, one power of two for each 32) and "nvf4" (E2M1 elements, one E4M3 scale
for each 16 and an f32 scale of the whole array):

* ``norm``: stream = stream + x, y = stream / sqrt(mean(stream^2) + eps) * gain, y quantised;
* ``quantize``: rows quantised, and with the 4-bit formats expanded again (8-bit elements and scales
  are returned as torch's float8 types);
* ``linear``: act(x . weight^T + bias) + residual of two quantised operands, the output in 16 or 32
  bits or quantised again;

and ``ffn``, the three together as a pre-norm feed-forward block calls them: norm, a product with
GELU whose output is quantised, a product onto the residual stream.

``own`` false runs elementary torch operations in f32; true runs the library.
"""
import math

import torch

own = False

BLOCK = {"mxf8": 32, "mxf4": 32, "nvf4": 16}
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


# ---------------------------------------------------------------------------------------- cases

def _norm(name, rows, dim, fmt, x, stream):
    return {"name": name, "op": "norm", "rows": rows, "dim": dim, "format": fmt, "x": x, "stream": stream}


def _quantize(name, rows, dim, fmt, x):
    return {"name": name, "op": "quantize", "rows": rows, "dim": dim, "format": fmt, "x": x}


def _linear(name, m, n, k, fmt, out, act="none", bias=True, residual=False):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "format": fmt, "out": out, "act": act,
            "bias": bias, "residual": residual}


def _ffn(name, rows, dim, hidden, fmt, x, stream):
    return {"name": name, "op": "ffn", "rows": rows, "dim": dim, "hidden": hidden, "format": fmt, "x": x, "stream": stream}


def listed():
    return [
        # One token before its projection: nothing but latency.
        _norm("norm 1x512 mxf8", 1, 512, "mxf8", "bf16", "bf16"),
        # The residual stream of one 8 s chunk (60 bands x 801 frames, width 384) between two blocks.
        _norm("norm 48060x384 mxf8", 48060, 384, "mxf8", "f32", "f32"),
        # Rows that are neither whole blocks nor whole vectors.
        _norm("norm 1201x1001 mxf4", 1201, 1001, "mxf4", "f16", "f32"),
        # A long batch of wide rows in 16 bits.
        _norm("norm 16384x4096 nvf4", 16384, 4096, "nvf4", "bf16", "bf16"),
        # The feed-forward's hidden rows of one chunk, quantised for the second product.
        _quantize("quantize 48060x1536 mxf8", 48060, 1536, "mxf8", "f16"),
        # The rows of one band, their width no whole number of blocks.
        _quantize("quantize 801x516 nvf4", 801, 516, "nvf4", "bf16"),
        # A wide layer's f32 weight at load time.
        _quantize("quantize 4096x4096 mxf4", 4096, 4096, "mxf4", "f32"),
        # Feed-forward in, its GELU output quantised for the next product: one chunk.
        _linear("linear 48060x1536x384 mxf8 gelu", 48060, 1536, 384, "mxf8", "mxf8", "gelu"),
        # A feed-forward block over the tokens of one chunk.
        _ffn("ffn 48060x384x1536 mxf4", 48060, 384, 1536, "mxf4", "f16", "f32"),
        # One token through a wide layer: the weight's bytes.
        _linear("linear 1x4096x4096 mxf4", 1, 4096, 4096, "mxf4", "bf16"),
        # A few rows, nothing a whole tile: k ends inside a block, n inside a tile.
        _linear("linear 133x1544x1000 mxf8", 133, 1544, 1000, "mxf8", "f32", "tanh", True, True),
        # A large product: the tensor cores' rate.
        _linear("linear 8192x8192x8192 nvf4", 8192, 8192, 8192, "nvf4", "bf16", "none", False),
    ]


def _size(rng, lo, hi):
    """A size between lo and hi, even in its logarithm; half of them rounded to a multiple of 8."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if v >= 16 and rng.random() < 0.5:
        v = v // 8 * 8
    return min(hi, max(lo, v))


def draw(rng):
    op = rng.choice(["norm", "quantize", "linear", "linear", "ffn"])
    fmt = rng.choice(["mxf8", "mxf4", "nvf4"])
    if op == "norm":
        dim = _size(rng, 16, 8192)
        rows = _size(rng, 1, min(48060, (1 << 26) // dim))
        return {"op": op, "rows": rows, "dim": dim, "format": fmt, "x": rng.choice(["f32", "bf16", "f16"]),
                "stream": rng.choice(["f32", "same"])}
    if op == "quantize":
        dim = _size(rng, 16, 8192)
        rows = _size(rng, 1, min(48060, (1 << 26) // dim))
        return {"op": op, "rows": rows, "dim": dim, "format": fmt, "x": rng.choice(["f32", "bf16", "f16"])}
    if op == "ffn":
        dim = _size(rng, 16, 2048)
        hidden = _size(rng, 16, 8192)
        rows = _size(rng, 1, min(48060, (1 << 26) // max(dim, hidden)))
        return {"op": op, "rows": rows, "dim": dim, "hidden": hidden, "format": fmt,
                "x": rng.choice(["bf16", "f16"]), "stream": rng.choice(["f32", "same"])}
    k = _size(rng, 16, 8192)
    n = _size(rng, 16, 8192)
    m = _size(rng, 1, min(48060, (1 << 26) // max(n, k)))
    return {"op": op, "m": m, "n": n, "k": k, "format": fmt,
            "out": rng.choice(["f32", "bf16", "f16", "mxf8"]),
            "act": rng.choice(["none", "gelu", "tanh"]), "bias": rng.random() < 0.7, "residual": rng.random() < 0.4}


def _element_bytes(fmt, rows, cols):
    nb = -(-cols // BLOCK[fmt])
    return rows * (cols if fmt == "mxf8" else (cols + 1) // 2) + rows * nb


def _bytes(name):
    return 4 if name == "f32" else 2


def work(case):
    fmt = case["format"]
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        out = case["out"]
        b = _element_bytes(fmt, m, k) + _element_bytes(fmt, n, k)
        b += m * n * _bytes(out) if out in DTYPE else _element_bytes(out, m, n)
        b += 4 * n * case["bias"] + 4 * m * n * case["residual"]
        return {"bytes": b, "flops": 2 * m * n * k}
    rows, dim = case["rows"], case["dim"]
    if case["op"] == "ffn":
        h = case["hidden"]
        b = rows * dim * (2 * _bytes(case["x"]) + 2 * _bytes(_stream(case)))
        b += _element_bytes(fmt, h, dim) + _element_bytes(fmt, dim, h) + 4 * (h + 2 * dim)
        return {"bytes": b, "flops": 4 * rows * dim * h + 10 * rows * dim}
    b = rows * dim * _bytes(case["x"]) + _element_bytes(fmt, rows, dim)
    if fmt != "mxf8":
        b += 2 * rows * dim  # expanded again
    if case["op"] == "norm":
        b += 2 * rows * dim * _bytes(_stream(case)) + 4 * dim
    return {"bytes": b, "flops": (10 if case["op"] == "norm" else 4) * rows * dim}


def _stream(case):
    return case["x"] if case["stream"] == "same" else case["stream"]


# --------------------------------------------------------------------------- plain quantisation

def _blocks(v, fmt):
    """Rows of v cut into blocks, the last one filled with zeros: [rows, blocks, block]."""
    b = BLOCK[fmt]
    pad = -v.shape[1] % b
    if pad:
        v = torch.nn.functional.pad(v, (0, pad))
    return v.reshape(v.shape[0], -1, b)


def _round_e2m1(t):
    """The nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with the sign of t, ties to the even code."""
    a = t.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).to(t.dtype)
    return torch.copysign(torch.clamp(torch.round(a / step) * step, max=6.0), t)


def _plain_quantize(v, fmt, g):
    """f32 rows -> (elements as f32 [rows, blocks, block], scale codes as uint8 [rows, blocks]).
    A block with an infinity or a NaN gets the scale NaN and elements 0."""
    v = _blocks(v, fmt)
    a = v.abs().amax(-1)
    bad = ~torch.isfinite(v).all(-1)
    if fmt == "nvf4":
        s = torch.clamp(torch.where(bad, torch.zeros_like(a), a) / (6.0 * g), max=448.0).to(torch.float8_e4m3fn)
        code = s.view(torch.uint8)
        d = s.float() * g
        t = torch.where((d > 0).unsqueeze(-1), v / d.unsqueeze(-1), torch.zeros_like(v))
        e = _round_e2m1(torch.clamp(t, -6.0, 6.0))
        nan = 127
    else:
        # The least power of two at which the largest magnitude still rounds into the range.
        bits = a.view(torch.int32)
        mantissa = bits & 0x7FFFFF
        top = (mantissa > 0x680000) if fmt == "mxf8" else (mantissa >= 0x600000)
        code = torch.clamp((bits >> 23) - (8 if fmt == "mxf8" else 2) + top.int(), min=0)
        t = v * ((254 - code) << 23).view(torch.float32).unsqueeze(-1)  # 2^(127 - code), from its bits
        t = torch.where(bad.unsqueeze(-1), torch.zeros_like(t), t)
        e = t.to(torch.float8_e4m3fn).float() if fmt == "mxf8" else _round_e2m1(t)
        nan = 255
    e = torch.where(bad.unsqueeze(-1), torch.zeros_like(e), e)
    return e, torch.where(bad, torch.full_like(code, nan), code).to(torch.uint8)


def _scale_values(code, fmt, g):
    if fmt == "nvf4":
        return code.view(torch.float8_e4m3fn).float() * g
    c = code.int()  # 2^(code - 127) from its bits; code 0 is f32's subnormal 2^-127, code 255 is NaN
    bits = torch.where(c == 255, 0x7FC00000, torch.where(c == 0, 0x00400000, c << 23))
    return bits.to(torch.int32).view(torch.float32)


def _tiled(code):
    """Scale codes [rows, blocks] in the library's order [rows / 128][blocks / 4][32][4][4], zeros behind the ends."""
    rows, nb = code.shape
    c = torch.nn.functional.pad(code, (0, -nb % 4, 0, -rows % 128))
    return c.view(-1, 4, 32, c.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous()


def _untiled(tiles, rows, nb):
    c = tiles.permute(0, 3, 2, 1, 4).reshape(tiles.shape[0] * 128, -1)
    return c[:rows, :nb]


def _packed(e, fmt, cols):
    """Elements as stored bytes: rows padded with zeros to a multiple of 16 bytes."""
    e = e.reshape(e.shape[0], -1)[:, :cols]
    if fmt == "mxf8":
        return torch.nn.functional.pad(e, (0, -cols % 16)).to(torch.float8_e4m3fn).view(torch.uint8)
    a = torch.nn.functional.pad(e, (0, -cols % 32))
    grid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=e.device)
    code = torch.bucketize(a.abs(), grid).to(torch.uint8) | (torch.signbit(a).to(torch.uint8) << 3)
    return code[:, 0::2] | (code[:, 1::2] << 4)


def _unpacked(data, fmt, cols):
    if fmt == "mxf8":
        return data.view(torch.float8_e4m3fn)[:, :cols].float()
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0.0, -.5, -1, -1.5, -2, -3, -4, -6], device=data.device)
    code = torch.stack((data & 15, data >> 4), -1).reshape(data.shape[0], -1)[:, :cols]
    return table[code.int()]


def _expanded(data, tiles, fmt, rows, cols, g):
    """Stored bytes and tiled scales -> f32 values."""
    b = BLOCK[fmt]
    s = _scale_values(_untiled(tiles, rows, -(-cols // b)), fmt, g)
    return _unpacked(data, fmt, cols) * s.repeat_interleave(b, 1)[:, :cols]


def _result(v, fmt, g):
    """What run() returns for rows v quantised to fmt: E4M3 elements and tiled scales, or the values in bf16
    (which holds every product of a 4-bit element and its scale; nvf4's array scale rounds there)."""
    e, code = _plain_quantize(v, fmt, g)
    rows, cols = v.shape
    if fmt == "mxf8":
        e = torch.nn.functional.pad(e.reshape(rows, -1)[:, :cols], (0, -cols % 16))
        return {"elements": e.to(torch.float8_e4m3fn), "scales": _tiled(code).view(torch.float8_e8m0fnu)}
    s = _scale_values(code, fmt, g)
    return {"values": (e * s.unsqueeze(-1)).reshape(rows, -1)[:, :cols].to(torch.bfloat16)}


def _requantized(v, fmt, g):
    """f32 rows -> the f32 values that they have once quantised."""
    e, code = _plain_quantize(v, fmt, g)
    return (e * _scale_values(code, fmt, g).unsqueeze(-1)).reshape(v.shape[0], -1)[:, :v.shape[1]]


# ------------------------------------------------------------------------------------- prepare

def _rows(g, rows, dim, dtype):
    """Activations as a trained network has them: channels of unlike size, a few of them large."""
    scale = torch.exp(0.5 * torch.randn(dim, device="cuda", generator=g))
    scale = torch.where(torch.rand(dim, device="cuda", generator=g) < 0.01, 8 * scale, scale)
    return (torch.randn(rows, dim, device="cuda", generator=g) * scale).to(dtype)


def _operand(g, rows, cols, fmt, spread):
    """A quantised array as a user's program holds it: stored bytes, tiled scales, array scale."""
    v = _rows(g, rows, cols, torch.float32) * spread
    a = (v.abs().amax() / (448.0 * 6.0)).reshape(1) if fmt == "nvf4" else None
    e, code = _plain_quantize(v, fmt, a)
    return {"data": _packed(e, fmt, cols).contiguous(), "scales": _tiled(code), "global": a, "rows": rows, "cols": cols,
            "format": fmt}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case)
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        s["xq"] = _operand(g, m, k, case["format"], 1.0)
        s["wq"] = _operand(g, n, k, case["format"], 0.5 / math.sqrt(k))
        s["b"] = torch.randn(n, device="cuda", generator=g) * 0.1 if case["bias"] else None
        s["r"] = torch.randn(m, n, device="cuda", generator=g) if case["residual"] else None
        s["g"] = None
        return s
    x = _rows(g, case["rows"], case["dim"], torch.float32)
    s["g"] = None
    if case["op"] != "quantize":
        s["res"] = _rows(g, case["rows"], case["dim"], DTYPE[_stream(case)])
        s["gain"] = 1 + 0.1 * torch.randn(case["dim"], device="cuda", generator=g)
        s["g"] = torch.full((1,), 0.01, device="cuda") if case["format"] == "nvf4" else None
    elif case["format"] == "nvf4":
        s["g"] = (x.abs().amax() / (448.0 * 6.0)).reshape(1)
    if case["op"] == "ffn":
        h, dim = case["hidden"], case["dim"]
        s["w1"] = _operand(g, h, dim, case["format"], 0.5 / math.sqrt(dim))
        s["w2"] = _operand(g, dim, h, case["format"], 0.5 / math.sqrt(h))
        s["b1"] = torch.randn(h, device="cuda", generator=g) * 0.1
        s["b2"] = torch.randn(dim, device="cuda", generator=g) * 0.1
        s["g2"] = torch.full((1,), 0.004, device="cuda") if case["format"] == "nvf4" else None
    s["in"] = x.to(DTYPE[case["x"]])
    return s


# ----------------------------------------------------------------------------------------- run

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _plain_norm(s):
    """(the new stream, the normed rows in f32). The norm's mean and root are taken in 64 bits and rounded
    once: the quantisers that follow have borders, next to which the last bit decides."""
    stream = (s["res"].float() + s["in"].float()).to(s["res"].dtype)
    v = stream.float()
    r = torch.rsqrt(v.double().square().mean(-1, keepdim=True) + EPS).float()
    return stream, v * r * s["gain"]


def _gelu(y):
    return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))


def _plain_values(q):
    return _expanded(q["data"], q["scales"], q["format"], q["rows"], q["cols"], q["global"])


def _run_plain(s):
    fmt = s["format"]
    if s["op"] == "quantize":
        return _result(s["in"].float(), fmt, s["g"])
    if s["op"] == "norm":
        stream, y = _plain_norm(s)
        return {"stream": stream, **_result(y, fmt, s["g"])}
    if s["op"] == "ffn":
        stream, y = _plain_norm(s)
        hidden = _gelu(_requantized(y, fmt, s["g"]) @ _plain_values(s["w1"]).t() + s["b1"])
        out = _requantized(hidden, fmt, s["g2"]) @ _plain_values(s["w2"]).t() + s["b2"] + stream.float()
        return {"stream": stream, "y": out.to(s["in"].dtype)}
    y = _plain_values(s["xq"]) @ _plain_values(s["wq"]).t()
    if s["b"] is not None:
        y = y + s["b"]
    if s["act"] == "gelu":
        y = _gelu(y)
    elif s["act"] == "tanh":
        y = torch.tanh(y)
    if s["r"] is not None:
        y = y + s["r"]
    return {"y": y.to(DTYPE[s["out"]])} if s["out"] in DTYPE else _result(y, s["out"], s["g"])


def _run_own(s):
    from ancha_b200 import microscaled as mx

    def operand(q):
        return mx.Microscaled(q["format"], q["rows"], q["cols"], q["data"], q["scales"], q["global"])

    def result(q):
        if q.format == "mxf8":
            return {"elements": q.data.view(torch.float8_e4m3fn), "scales": q.scales.view(torch.float8_e8m0fnu)}
        return {"values": mx.dequantize(q, torch.bfloat16)}

    if s["op"] == "quantize":
        return result(mx.quantize(s["in"], s["format"], s["g"]))
    if s["op"] == "norm":
        q, stream = mx.add_rms_norm(s["in"], s["res"], s["gain"], EPS, s["format"], s["g"])
        return {"stream": stream, **result(q)}
    if s["op"] == "ffn":
        q, stream = mx.add_rms_norm(s["in"], s["res"], s["gain"], EPS, s["format"], s["g"])
        hidden = mx.linear(q, operand(s["w1"]), s["b1"], "gelu", format=s["format"], global_scale=s["g2"])
        return {"stream": stream, "y": mx.linear(hidden, operand(s["w2"]), s["b2"], "none", stream, dtype=s["in"].dtype)}
    a, w = operand(s["xq"]), operand(s["wq"])
    if s["out"] in DTYPE:
        return {"y": mx.linear(a, w, s["b"], s["act"], s["r"], dtype=DTYPE[s["out"]])}
    return result(mx.linear(a, w, s["b"], s["act"], s["r"], format=s["out"], global_scale=s["g"]))


# --------------------------------------------------------------------------------------- exact

def _grid(fmt):
    """The non-negative values of the element type, in order of their codes."""
    if fmt == "mxf8":
        v = [m / 8 * 2.0 ** -6 for m in range(8)]
        return v + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:-1]
    return [0, .5, 1, 1.5, 2, 3, 4, 6]


def _power(e):
    """2^e in 64 bits of whole numbers e in [-300, 300]."""
    table = torch.tensor([2.0 ** i for i in range(-300, 301)], dtype=torch.float64, device=e.device)
    return table[e.long() + 300]


def _nearest(t, grid):
    """The grid value nearest to each of t >= 0 in 64 bits, ties to the even code, saturating."""
    grid = torch.tensor(grid, dtype=torch.float64, device=t.device)
    hi = torch.clamp(torch.searchsorted(grid, t), max=len(grid) - 1)
    lo = torch.clamp(hi - 1, min=0)
    up, down = grid[hi] - t, t - grid[lo]
    take = (up < down) | ((up == down) & (hi % 2 == 0))
    return torch.where(take, grid[hi], grid[lo])


def _exact_quantize(y, fmt, g):
    """64-bit rows -> (elements [rows, cols], scales [rows, blocks]) by the formats' definition."""
    rows, cols = y.shape
    b = BLOCK[fmt]
    z = torch.zeros(rows, -(-cols // b) * b, dtype=torch.float64, device=y.device)
    z[:, :cols] = y
    z = z.view(rows, -1, b)
    a = z.abs().max(2).values
    if fmt == "nvf4":
        s = _nearest(a / (6.0 * g.double()), _grid("mxf8")) * g.double()
    else:
        most, power = ((464.0, 8) if fmt == "mxf8" else (7.0, 2))
        m, e = torch.frexp(a)  # a = m 2^e with m in [0.5, 1)
        e = torch.where(a > 0, e.long() - 1 - power, -127)
        r = a / _power(e)
        e = torch.where((r > most) | ((r == most) & (fmt != "mxf8")), e + 1, e)
        s = _power(e.clamp(min=-127))
    t = torch.where(s.unsqueeze(2) > 0, z.abs() / s.unsqueeze(2), torch.zeros_like(z))
    q = _nearest(t, _grid(fmt)) * torch.sign(z)
    return q.view(rows, -1)[:, :cols], s


def _exact_result(y, fmt, g):
    q, s = _exact_quantize(y, fmt, g)
    rows, cols = y.shape
    if fmt != "mxf8":
        return {"values": q * s.repeat_interleave(BLOCK[fmt], 1)[:, :cols]}
    wide = torch.zeros(rows, -(-cols // 16) * 16, dtype=torch.float64, device=y.device)
    wide[:, :cols] = q
    mt, kt = -(-rows // 128), -(-s.shape[1] // 4)
    full = torch.full((mt * 128, kt * 4), 2.0 ** -127, dtype=torch.float64, device=y.device)
    full[:rows, :s.shape[1]] = s
    return {"elements": wide, "scales": full.reshape(mt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4)}


def _exact_values(q):
    """The values a quantised operand stands for, in 64 bits."""
    rows, cols, b = q["rows"], q["cols"], BLOCK[q["format"]]
    nb = -(-cols // b)
    r = torch.arange(rows, device="cuda").unsqueeze(1)
    c = torch.arange(nb, device="cuda").unsqueeze(0)
    code = q["scales"][r // 128, c // 4, r % 32, (r % 128) // 32, c % 4].long()
    g8 = torch.tensor(_grid("mxf8") + [math.nan], dtype=torch.float64, device="cuda")
    g8 = torch.cat((g8, -g8))
    if q["format"] == "nvf4":
        s = g8[code] * q["global"].double()
    else:
        s = _power(code - 127)
    if q["format"] == "mxf8":
        e = g8[q["data"].long()][:, :cols]
    else:
        g4 = torch.tensor(_grid("mxf4"), dtype=torch.float64, device="cuda")
        g4 = torch.cat((g4, -g4))
        col = torch.arange(cols, device="cuda")
        e = g4[((q["data"][:, col // 2].long() >> (4 * (col % 2))) & 15)]
    return e * s.repeat_interleave(b, 1)[:, :cols]


def _exact_requantized(y, fmt, g):
    q, s = _exact_quantize(y, fmt, g)
    return q * s.repeat_interleave(BLOCK[fmt], 1)[:, :y.shape[1]]


def exact(case, seed):
    s = prepare(case, seed)
    fmt = case["format"]
    if case["op"] == "quantize":
        return _exact_result(s["in"].double(), fmt, s["g"])
    if case["op"] in ("norm", "ffn"):
        total = s["res"].double() + s["in"].double()
        v = total.to(s["res"].dtype).double()  # the stream as it is held
        y = v / torch.sqrt(v.square().sum(1, keepdim=True) / case["dim"] + EPS) * s["gain"].double()
        if case["op"] == "norm":
            return {"stream": total, **_exact_result(y, fmt, s["g"])}
        h = _exact_requantized(y, fmt, s["g"]) @ _exact_values(s["w1"]).t() + s["b1"].double()
        h = h * 0.5 * torch.erfc(-h / math.sqrt(2.0))
        y = _exact_requantized(h, fmt, s["g2"]) @ _exact_values(s["w2"]).t() + s["b2"].double()
        return {"stream": total, "y": y + v}
    y = _exact_values(s["xq"]) @ _exact_values(s["wq"]).t()
    if case["bias"]:
        y += s["b"].double()
    if case["act"] == "gelu":
        y = y * 0.5 * torch.erfc(-y / math.sqrt(2.0))
    elif case["act"] == "tanh":
        y = 1 - 2 / (torch.exp(2 * y) + 1)
    if case["residual"]:
        y += s["r"].double()
    return {"y": y} if case["out"] in DTYPE else _exact_result(y, case["out"], s["g"])
