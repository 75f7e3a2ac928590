"""The operators of a layer's linear path in 8-bit floating point, as measurable cases.

An encoder layer in e4m3 is a run of four kinds of call: the norm of the residual stream, with the
last product's addition, writes the next product's 8-bit operand; a product takes it against
8-bit weights; the gated product writes the operand of the product behind it; and what attention
returns is coded by itself, as the weights are when a model is loaded.  Every block of 128 values
along the summed axis has one scale.  Activations have blocks of one row, scaled by a power of two
that a byte holds ("e8m0"); weights have blocks of 128 rows, whose scale is such a byte or a float
("f32"), as a checkpoint has it.

`own` chooses between the framework's calls and the same operators in elementary torch operations.
Inputs come from the seed alone.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
BLOCK = 128
TOP = 448.0                    # the largest e4m3 value
LEAST = 2.0 ** -126            # the smallest scale
EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": 0, "f16": 1, "bf16": 2}
SCALES = {"e8m0": 0, "f32": 1}


# ---- the cases -----------------------------------------------------------------------------

def _codes(rows, cols, source):
    return {"op": "codes", "rows": rows, "cols": cols, "source": source}


def _weight_codes(rows, cols, scale):
    return {"op": "weight_codes", "rows": rows, "cols": cols, "source": "f32", "scale": scale}


def _norm(rows, cols, stream, delta):
    return {"op": "norm", "rows": rows, "cols": cols, "stream": stream, "delta": delta}


def _product(rows, cols, depth, out, scale):
    return {"op": "product", "rows": rows, "cols": cols, "depth": depth, "out": out, "scale": scale}


def _gated(rows, cols, depth, scale):
    return {"op": "gated", "rows": rows, "cols": cols, "depth": depth, "scale": scale}


def listed():
    return [
        # What attention returns for an odd number of tokens, ahead of the output product.
        {"name": "context_codes", **_codes(9001, 768, "f16")},
        # A large model's weight matrix, coded once when it is loaded.
        {"name": "weight_codes", **_weight_codes(8192, 4096, "f32")},
        # One token's wide row, with no batch to hide latency behind.
        {"name": "norm_token", **_norm(1, 8192, "bf16", "bf16")},
        # The tokens of a batch of 32 passages of 32 to 256 tokens.
        {"name": "norm_batch", **_norm(4616, 768, "f32", "f16")},
        # Bulk indexing: 256 passages of 64 to 512 tokens.
        {"name": "norm_bulk", **_norm(74640, 768, "f32", "f16")},
        # One token against a large matrix: the weights' bytes are the time.
        {"name": "product_token", **_product(1, 8192, 4096, "bf16", "e8m0")},
        # A search box's query of 32 tokens through q, k and v.
        {"name": "product_query", **_product(32, 2304, 768, "f16", "e8m0")},
        # The feed-forward's second product for a batch of passages, into a 32-bit stream.
        {"name": "product_batch", **_product(4616, 768, 2048, "f32", "f32")},
        # A large model's product over a long batch of odd length.
        {"name": "product_large", **_product(16391, 8192, 4096, "bf16", "e8m0")},
        # The feed-forward's gate and up products of a query.
        {"name": "gated_query", **_gated(32, 2048, 768, "e8m0")},
        # The same for a batch of passages, on weights with float scales.
        {"name": "gated_batch", **_gated(4616, 2048, 768, "f32")},
        # And for bulk indexing.
        {"name": "gated_bulk", **_gated(74640, 2048, 768, "e8m0")},
    ]


def _log_int(rng, lo, hi, step=1):
    return max(step, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step)


def draw(rng):
    op = rng.choice(["codes", "weight_codes", "norm", "norm", "product", "product", "product", "gated", "gated"])
    scale = rng.choice(["e8m0", "f32"])
    if op == "codes":
        cols = _log_int(rng, 256, 8192, 16)
        return _codes(_log_int(rng, 1, 30000000 // cols), cols, rng.choice(["f32", "f16", "bf16"]))
    if op == "weight_codes":
        return _weight_codes(_log_int(rng, 128, 8192), _log_int(rng, 256, 4096, 16), scale)
    if op == "norm":
        cols = _log_int(rng, 256, 8192, 16)
        stream = rng.choice(["f32", "bf16", "f16"])
        return _norm(_log_int(rng, 1, 40000000 // cols), cols, stream, rng.choice([stream, "f16", "bf16", "none"]))
    if op == "product":
        cols, depth = _log_int(rng, 64, 8192), _log_int(rng, 256, 4096, 16)
        most = min(70000, 450000000000 // (cols * depth))
        return _product(_log_int(rng, 1, most), cols, depth, rng.choice(["bf16", "f16", "f32"]), scale)
    cols, depth = _log_int(rng, 256, 8192, 16), _log_int(rng, 256, 4096, 16)
    most = min(70000, 200000000000 // (cols * depth))
    return _gated(_log_int(rng, 1, most), cols, depth, scale)


# ---- shared sizes --------------------------------------------------------------------------

def _blocks(cols):
    return (cols + BLOCK - 1) // BLOCK


def _rows16(rows):
    return (rows + 15) // 16 * 16


# ---- the plain form ------------------------------------------------------------------------

def _block_scales(top, scale):
    """The blocks' scales and their inverses, in 32 bits, from the largest magnitudes."""
    if scale == "f32":
        top = top.clamp(min=TOP * LEAST)
        return top / TOP, TOP / top
    # the smallest power of two whose 448-fold is not below `top`: a mantissa over 1.75 carries
    byte = ((top.view(torch.int32) + 0x1FFFFF) >> 23) - 8
    byte = byte.clamp(min=1)
    return (byte << 23).view(torch.float32), ((254 - byte) << 23).view(torch.float32)


def _stored(scales, scale):
    """Scales as they are stored: floats, or the exponent's byte."""
    return scales if scale == "f32" else (scales.view(torch.int32) >> 23).to(torch.uint8)


def _to_codes(y):
    """e4m3 codes of 32-bit rows in blocks of one row, and the scales [block][row]."""
    rows, cols = y.shape
    n = _blocks(cols)
    y = torch.nn.functional.pad(y, (0, n * BLOCK - cols)).view(rows, n, BLOCK)
    size = y.abs()
    top = torch.where(torch.isfinite(y), size, torch.zeros_like(size)).amax(2)
    s, inv = _block_scales(top, "e8m0")
    q = y * inv[:, :, None]
    q = torch.where(torch.isfinite(y), q, torch.full_like(q, math.nan)).to(torch.float8_e4m3fn)
    return q.view(torch.uint8).view(rows, n * BLOCK)[:, :cols].contiguous(), _stored(s.t().contiguous(), "e8m0")


def _to_weight_codes(w, scale):
    """e4m3 codes of a 32-bit matrix in blocks of 128 x 128, and the scales [row block][block]."""
    rows, cols = w.shape
    m, n = _blocks(rows), _blocks(cols)
    y = torch.nn.functional.pad(w, (0, n * BLOCK - cols, 0, m * BLOCK - rows)).view(m, BLOCK, n, BLOCK)
    size = y.abs()
    top = torch.where(torch.isfinite(y), size, torch.zeros_like(size)).amax((1, 3))
    s, inv = _block_scales(top, scale)
    q = y * inv[:, None, :, None]
    q = torch.where(torch.isfinite(y), q, torch.full_like(q, math.nan)).to(torch.float8_e4m3fn).view(torch.uint8)
    return q.view(m * BLOCK, n * BLOCK)[:rows, :cols].contiguous(), _stored(s, scale)


def _floats(scales, scale):
    return scales if scale == "f32" else (scales.to(torch.int32) << 23).view(torch.float32)


def _values(codes, scales):
    """What activations' codes and scales stand for, in 32 bits."""
    rows, cols = codes.shape
    s = _floats(scales[:, :rows], "e8m0").t().repeat_interleave(BLOCK, 1)[:, :cols]
    return codes.view(torch.float8_e4m3fn).to(torch.float32) * s


def _weight_values(codes, scales, scale):
    rows, cols = codes.shape
    s = _floats(scales, scale).repeat_interleave(BLOCK, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]
    return codes.view(torch.float8_e4m3fn).to(torch.float32) * s


def _gelu(x):
    return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x * x * x)))


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "codes":
        return _coded(*_to_codes(s["x"].float()))
    if op == "weight_codes":
        return _coded(*_to_weight_codes(s["x"].float(), case["scale"]))
    if op == "norm":
        h = s["x"].float()
        if s["delta"] is not None:
            h = (h + s["delta"].float()).to(s["x"].dtype)
        y = h.float()
        y = y * torch.rsqrt((y * y).mean(1, keepdim=True) + EPS) * s["gamma"]
        out = _coded(*_to_codes(y))
        if s["delta"] is not None:
            out["sum"] = h
        return out
    a = _values(s["a"], s["a_scales"])
    c = a @ _weight_values(s["w"], s["w_scales"], case["scale"]).t()
    if op == "product":
        return {"out": c.to(TYPES[case["out"]])}
    up = a @ _weight_values(s["w1"], s["w1_scales"], case["scale"]).t()
    return _coded(*_to_codes(_gelu(c) * up))


def _coded(codes, scales):
    """Codes and scales as what they stand for: e4m3 values, and floats or powers of two."""
    if scales.dtype == torch.uint8:
        scales = scales.view(torch.float8_e8m0fnu)
    return {"codes": codes.view(torch.float8_e4m3fn), "scales": scales}


# ---- inputs --------------------------------------------------------------------------------

def _hidden(g, rows, cols):
    """Hidden states: a few channels much larger than the others, tokens of different sizes."""
    x = torch.randn(rows, cols, generator=g, device=DEV)
    x *= torch.exp(0.5 * torch.randn(cols, generator=g, device=DEV))
    x[:, torch.randint(cols, (max(1, cols // 200),), generator=g, device=DEV)] *= 12.0
    return x * torch.exp(0.3 * torch.randn(rows, 1, generator=g, device=DEV))


def _weights(g, rows, cols):
    return torch.randn(rows, cols, generator=g, device=DEV) * (1.5 / math.sqrt(cols))


def _padded(scales, rows):
    """Activations' scales with the row stride that the calls take: rows rounded up to 16."""
    out = torch.zeros(scales.shape[0], _rows16(rows), dtype=scales.dtype, device=DEV)
    out[:, :rows] = scales
    return out


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op, rows, cols = case["op"], case["rows"], case["cols"]
    s = {"case": case}
    if op in ("codes", "weight_codes"):
        s["x"] = (_hidden if op == "codes" else _weights)(g, rows, cols).to(TYPES[case["source"]])
    elif op == "norm":
        s["x"] = _hidden(g, rows, cols).to(TYPES[case["stream"]])
        s["delta"] = None
        if case["delta"] != "none":
            s["delta"] = (0.3 * _hidden(g, rows, cols)).to(TYPES[case["delta"]])
            s["sum"] = torch.empty_like(s["x"])
        s["gamma"] = 1.0 + 0.2 * torch.randn(cols, generator=g, device=DEV)
    else:
        depth = case["depth"]
        x = _hidden(g, rows, depth)
        x *= torch.rsqrt((x * x).mean(1, keepdim=True))
        s["a"], a_scales = _to_codes(x)
        s["a_scales"] = _padded(a_scales, rows)
        s["w"], s["w_scales"] = _to_weight_codes(_weights(g, cols, depth), case["scale"])
        if op == "product":
            s["out"] = torch.empty(rows, cols, dtype=TYPES[case["out"]], device=DEV)
            return s
        s["w1"], s["w1_scales"] = _to_weight_codes(_weights(g, cols, depth), case["scale"])
    s["codes"] = torch.empty(rows, cols, dtype=torch.uint8, device=DEV)
    if op == "weight_codes":
        s["scales"] = torch.empty(_blocks(rows), _blocks(cols), device=DEV,
                                  dtype=torch.uint8 if case["scale"] == "e8m0" else torch.float32)
    else:
        s["scales"] = torch.empty(_blocks(cols), _rows16(rows), dtype=torch.uint8, device=DEV)
    return s


# ---- one pass ------------------------------------------------------------------------------

def _own(s):
    from witchcraft_amd import fp8

    case = s["case"]
    op, rows, cols = case["op"], case["rows"], case["cols"]
    stream = torch.cuda.current_stream().cuda_stream
    if op == "product":
        fp8.matmul_device(s["a"].data_ptr(), s["a_scales"].data_ptr(), rows, s["w"].data_ptr(), s["w_scales"].data_ptr(),
                          cols, case["depth"], SCALES[case["scale"]], s["out"].data_ptr(), CODE[case["out"]], stream)
        return {"out": s["out"]}
    codes, scales = s["codes"], s["scales"]
    if op == "weight_codes":
        fp8.quantize_weights_device(s["x"].data_ptr(), CODE[case["source"]], rows, cols, SCALES[case["scale"]],
                                    codes.data_ptr(), scales.data_ptr(), stream)
        return _coded(codes, scales)
    if op == "codes":
        fp8.quantize_device(s["x"].data_ptr(), CODE[case["source"]], rows, cols, codes.data_ptr(), scales.data_ptr(),
                            stream)
    elif op == "norm":
        delta = s["delta"]
        fp8.rmsnorm_device(s["x"].data_ptr(), CODE[case["stream"]], 0 if delta is None else delta.data_ptr(),
                           CODE.get(case["delta"], 0), rows, cols, s["gamma"].data_ptr(), EPS,
                           0 if delta is None else s["sum"].data_ptr(), codes.data_ptr(), scales.data_ptr(), stream)
    else:
        fp8.gated_gelu_device(s["a"].data_ptr(), s["a_scales"].data_ptr(), rows, s["w"].data_ptr(),
                              s["w_scales"].data_ptr(), s["w1"].data_ptr(), s["w1_scales"].data_ptr(), cols,
                              case["depth"], SCALES[case["scale"]], codes.data_ptr(), scales.data_ptr(), stream)
    out = _coded(codes, scales[:, :rows])
    if op == "norm" and s["delta"] is not None:
        out["sum"] = s["sum"]
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ---------------------------------------------------------

def work(case):
    op, rows, cols = case["op"], case["rows"], case["cols"]
    size = {"f32": 4, "f16": 2, "bf16": 2, "none": 0}
    scale = 4 if case.get("scale") == "f32" else 1
    if op == "codes":
        return {"bytes": rows * cols * (size[case["source"]] + 1) + rows * _blocks(cols), "flops": 2 * rows * cols}
    if op == "weight_codes":
        return {"bytes": rows * cols * 5 + _blocks(rows) * _blocks(cols) * scale, "flops": 2 * rows * cols}
    if op == "norm":
        stream, delta = size[case["stream"]], size[case["delta"]]
        per = stream + delta + (stream if delta else 0) + 1
        return {"bytes": rows * cols * per + 4 * cols + rows * _blocks(cols), "flops": 6 * rows * cols}
    depth = case["depth"]
    a = rows * (depth + _blocks(depth))
    w = cols * depth + _blocks(cols) * _blocks(depth) * scale
    if op == "product":
        return {"bytes": a + w + rows * cols * size[case["out"]], "flops": 2 * rows * cols * depth}
    return {"bytes": a + 2 * w + rows * (cols + _blocks(cols)), "flops": 4 * rows * cols * depth}


# ---- the definition in 64 bits -------------------------------------------------------------

def _table():
    """The value of every e4m3 code: sign, four bits of exponent (bias 7), three of fraction."""
    t = []
    for code in range(256):
        sign, e, f = -1.0 if code & 128 else 1.0, (code >> 3) & 15, code & 7
        if e == 15 and f == 7:
            t.append(math.nan)
        else:
            t.append(sign * (math.ldexp(f, -9) if e == 0 else math.ldexp(8 + f, e - 10)))
    return torch.tensor(t, dtype=torch.float64, device=DEV)


def _exact_scales(scales, scale):
    return scales.double() if scale == "f32" else torch.exp2(scales.double() - 127.0)


def _exact_operand(codes, scales, scale, table):
    """Values of codes; each 128 columns are multiplied by their column of scales [rows][blocks]."""
    v = table[codes.long()]
    s = _exact_scales(scales, scale)
    for b in range(s.shape[1]):
        v[:, b * BLOCK:(b + 1) * BLOCK] *= s[:, b:b + 1]
    return v


def _exact_codes(y, rows_per_block, scale):
    """What the codes stand for before they are rounded to e4m3, and the scales."""
    rows, cols = y.shape
    m, n = -(-rows // rows_per_block), _blocks(cols)
    scales = torch.empty(m, n, dtype=torch.float64, device=DEV)
    for b in range(n):
        part = y[:, b * BLOCK:(b + 1) * BLOCK].abs().amax(1)
        if rows_per_block > 1:
            part = torch.stack([p.max() for p in part.split(rows_per_block)])
        scales[:, b] = part
    scales /= TOP
    scales = scales.clamp(min=LEAST)
    if scale == "e8m0":
        scales = torch.exp2(torch.ceil(torch.log2(scales)))
    v = y.clone()
    for b in range(n):
        s = scales[:, b:b + 1]
        v[:, b * BLOCK:(b + 1) * BLOCK] /= s.repeat_interleave(rows_per_block, 0)[:rows]
    return v, scales


def exact(case, seed):
    """`run` in 64 bits.  Codes are given as the values they are the nearest e4m3 to; a power-of-two scale
    that steps where a computed maximum crosses a border has no value between the steps: None."""
    s = prepare(case, seed)
    op = case["op"]
    if op == "codes":
        v, scales = _exact_codes(s["x"].double(), 1, "e8m0")
        return {"codes": v, "scales": scales.t()}
    if op == "weight_codes":
        v, scales = _exact_codes(s["x"].double(), BLOCK, case["scale"])
        return {"codes": v, "scales": scales}
    if op == "norm":
        out = {}
        h = s["x"].double()
        if s["delta"] is not None:
            h = h + s["delta"].double()
            out["sum"] = h
            h = h.to(s["x"].dtype).double()  # the norm is the stored sum's
        y = h / torch.sqrt(h.square().mean(1, keepdim=True) + EPS) * s["gamma"].double()
        return {"codes": _exact_codes(y, 1, "e8m0")[0], "scales": None, **out}
    table = _table()
    rows, cols = case["rows"], case["cols"]

    def weights(codes, scales):
        return _exact_operand(codes, scales.repeat_interleave(BLOCK, 0)[:cols], case["scale"], table).t()

    a = _exact_operand(s["a"], s["a_scales"][:, :rows].t(), "e8m0", table)
    c = a @ weights(s["w"], s["w_scales"])
    if op == "product":
        return {"out": c}
    up = a @ weights(s["w1"], s["w1_scales"])
    y = c * (0.5 + 0.5 * torch.tanh(math.sqrt(2.0 / math.pi) * (c + 0.044715 * c ** 3))) * up
    return {"codes": _exact_codes(y, 1, "e8m0")[0], "scales": None}
