"""The operators between a layer's shared projection and its attention, as measurable cases.

Many requests in one packed batch, each with a low-rank adapter of its own or none, go through one
shared product (in 8 bits or 16); the adapters' products are added to its rows ("adapter").  Queries
and keys then take a norm for each head and the rotation by their positions, which have one axis for
text and several for images and video ("rotate").

`own` chooses between the framework's calls and the same operators in elementary torch operations.
Inputs come from the seed alone.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
BLOCK = 128
EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
CODE = {"f32": 0, "f16": 1, "bf16": 2, "e4m3": 3}


# ---- the cases -----------------------------------------------------------------------------

def _adapter(tokens, requests, adapters, rank, depth, cols, slices, x, w, y):
    """Rows of `tokens` tokens and `depth` values against `adapters` adapters of up to `rank`, beside a
    product of `slices` projections of `cols` columns each.  x, w, y: the types of the rows, of the
    adapters and of the product's results."""
    return {"op": "adapter", "tokens": tokens, "requests": requests, "adapters": adapters, "rank": rank,
            "depth": depth, "cols": cols, "slices": slices, "x": x, "w": w, "y": y}


def _rotate(tokens, requests, heads, key_heads, dim, rot, pairing, axes, norms, kind, far=0):
    """`heads` + `key_heads` heads of `dim` values, of which the first `rot` are turned, "halves" or
    "neighbours" together, by positions of `axes` axes that start at `far`."""
    return {"op": "rotate", "tokens": tokens, "requests": requests, "heads": heads, "key_heads": key_heads, "dim": dim,
            "rot": rot, "pairing": pairing, "axes": axes, "norms": norms, "type": kind, "far": far}


def listed():
    return [
        # One token of one request beside a large projection: latency.
        {"name": "adapter_token", **_adapter(1, 1, 8, 16, 4096, 4096, 1, "bf16", "bf16", "bf16")},
        # One token of each of 64 requests, no two with the same adapter: the adapters' bytes.
        {"name": "adapter_requests", **_adapter(64, 64, 64, 16, 4096, 4096, 1, "bf16", "bf16", "bf16")},
        # A search box's query of 32 tokens through q, k and v.
        {"name": "adapter_query", **_adapter(32, 1, 4, 16, 768, 768, 3, "e4m3", "f16", "f16")},
        # A batch of 32 passages of several tenants through q, k and v in 8 bits.
        {"name": "adapter_batch", **_adapter(4616, 32, 8, 16, 768, 768, 3, "e4m3", "f16", "f16")},
        # The same batch through the feed-forward's second product, into a 32-bit stream.
        {"name": "adapter_stream", **_adapter(4616, 32, 4, 64, 2048, 768, 1, "f16", "f16", "f32")},
        # Bulk indexing of 256 passages through q, k and v.
        {"name": "adapter_bulk", **_adapter(74640, 256, 16, 16, 768, 768, 3, "e4m3", "f16", "f16")},
        # A large model's product over long passages, with wide adapters.
        {"name": "adapter_large", **_adapter(16391, 9, 3, 64, 4096, 8192, 1, "bf16", "bf16", "bf16")},
        # One token far into a long text.
        {"name": "rotate_token", **_rotate(1, 1, 32, 8, 128, 128, "halves", 1, True, "bf16", 130000)},
        # A batch of 32 passages, rotated without norms.
        {"name": "rotate_batch", **_rotate(4616, 32, 12, 12, 64, 64, "halves", 1, False, "f16")},
        # Patches of page images in a vision encoder, with a row and a column each; an odd head size.
        {"name": "rotate_patches", **_rotate(10007, 8, 16, 16, 80, 80, "halves", 2, False, "bf16")},
        # Page images among text, positions in time, height and width, norms, shared keys.
        {"name": "rotate_pages", **_rotate(16391, 9, 32, 8, 128, 128, "halves", 3, True, "bf16", 1000)},
        # Bulk indexing of 256 passages, norms, neighbouring values turned together.
        {"name": "rotate_bulk", **_rotate(74640, 256, 12, 12, 64, 64, "neighbours", 1, True, "f16")},
    ]


def _log_int(rng, lo, hi, step=1):
    return max(step, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi)))) / step)) * step)


def draw(rng):
    if rng.random() < 0.55:
        depth, cols, slices = _log_int(rng, 256, 8192, 16), _log_int(rng, 64, 8192, 16), rng.choice([1, 1, 2, 3])
        cols = min(cols, 8192 // slices // 16 * 16)
        rank = rng.choice([8, 16, 16, 24, 32, 64, 128])
        w = rng.choice(["bf16", "f16"])
        x, y = rng.choice([w, w, "e4m3"]), rng.choice(["bf16", "f16", "f32"])
        per_row = depth * SIZE[x] + 2 * cols * slices * SIZE[y]
        most = min(75000, 600000000 // per_row, 12000000000 // (slices * rank * (depth + cols)))
        tokens = _log_int(rng, 1, most)
        requests = tokens if rng.random() < 0.2 and tokens <= 512 else _log_int(rng, 1, min(tokens, 300))
        weights = 2 * slices * rank * (depth + cols)
        adapters = _log_int(rng, 1, min(128, max(1, 500000000 // weights)))
        return _adapter(tokens, requests, adapters, rank, depth, cols, slices, x, w, y)
    dim = rng.choice([32, 64, 72, 80, 96, 128, 128, 160, 256])
    rot = rng.choice([dim, dim, dim, dim // 2 // 8 * 8])
    key_heads = rng.choice([1, 2, 4, 8, 12, 16])
    heads = key_heads * rng.choice([1, 1, 2, 4, 7])
    kind = rng.choice(["bf16", "f16", "f32"])
    most = min(75000, 600000000 // (2 * (heads + key_heads) * dim * SIZE[kind]))
    tokens = _log_int(rng, 1, most)
    return _rotate(tokens, _log_int(rng, 1, min(tokens, 300)), heads, key_heads, dim, rot,
                   rng.choice(["halves", "neighbours"]), rng.choice([1, 1, 2, 3]), rng.random() < 0.6, kind,
                   rng.choice([0, 0, _log_int(rng, 100, 1000000)]))


# ---- shared by both forms: who has which adapter, how fast a pair turns --------------------

def _adapted(case):
    """How many requests have an adapter: of eight or more, every eighth has none."""
    return case["requests"] - case["requests"] // 8


def _frequencies(case):
    """Radians per step of each pair, falling by powers of 10,000, and the axis that it follows."""
    pairs = case["rot"] // 2
    freqs = [10000.0 ** (-i / pairs) for i in range(pairs)]
    return freqs, [i * case["axes"] // pairs for i in range(pairs)]


# ---- inputs --------------------------------------------------------------------------------

def _hidden(g, rows, cols):
    """Hidden states: a few channels much larger than the others, tokens of different sizes."""
    x = torch.randn(rows, cols, generator=g, device=DEV)
    x *= torch.exp(0.5 * torch.randn(cols, generator=g, device=DEV))
    x[:, torch.randint(cols, (max(1, cols // 200),), generator=g, device=DEV)] *= 12.0
    return x * torch.exp(0.3 * torch.randn(rows, 1, generator=g, device=DEV))


def _lengths(h, tokens, requests):
    """Lengths of one or more that add up to `tokens`."""
    cuts = (torch.randperm(tokens - 1, generator=h)[:requests - 1] + 1).sort().values
    return torch.diff(torch.cat([torch.tensor([0]), cuts, torch.tensor([tokens])]))


def _coded(x):
    """Rows as e4m3 codes with a power-of-two scale for each block of 128, stored [block][row], rows
    rounded up to 16."""
    rows, cols = x.shape
    n = -(-cols // BLOCK)
    v = torch.nn.functional.pad(x, (0, n * BLOCK - cols)).view(rows, n, BLOCK)
    byte = (((v.abs().amax(2).view(torch.int32) + 0x1FFFFF) >> 23) - 8).clamp(min=1)
    inv = ((254 - byte) << 23).view(torch.float32)
    codes = (v * inv[:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8).view(rows, n * BLOCK)[:, :cols].contiguous()
    scales = torch.zeros(n, (rows + 15) // 16 * 16, dtype=torch.uint8, device=DEV)
    scales[:, :rows] = byte.t().to(torch.uint8)
    return codes, scales


def _prepare_adapter(case, g, h):
    t, k, n, s, r = case["tokens"], case["depth"], case["cols"], case["slices"], case["rank"]
    adapters, wt = case["adapters"], TYPES[case["w"]]
    x = _hidden(g, t, k)
    x *= torch.rsqrt((x * x).mean(1, keepdim=True))
    state = {"x_scales": None}
    if case["x"] == "e4m3":
        state["x"], state["x_scales"] = _coded(x)
    else:
        state["x"] = x.to(TYPES[case["x"]])
    del x
    # a third of the adapters have half the rank (in whole eights): the rest of their rows and columns is zero
    ranks = torch.full((adapters,), r, dtype=torch.int32)
    ranks[1::3] = max(8, r // 2 // 8 * 8)
    kept = torch.arange(r)[None] < ranks[:, None]
    a = torch.randn(adapters, s, r, k, generator=g, device=DEV) / math.sqrt(k)
    b = torch.randn(adapters, s * n, r, generator=g, device=DEV) * (0.5 / math.sqrt(r))
    state["a"] = (a * kept.to(DEV)[:, None, :, None]).to(wt)
    state["b"] = (b * kept.to(DEV)[:, None, :]).to(wt)
    state["ranks"] = ranks.to(DEV)
    state["scales"] = (2.0 ** torch.randint(-1, 3, (adapters,), generator=h)).to(torch.float32).to(DEV)
    which = torch.randperm(adapters, generator=h)
    with_one = _adapted(case)
    ids = torch.full((case["requests"],), -1, dtype=torch.int64)
    place = torch.randperm(case["requests"], generator=h)[:with_one]
    ids[place] = which[torch.arange(with_one) % adapters]
    state["ids"] = ids.repeat_interleave(_lengths(h, t, case["requests"])).to(torch.int32).to(DEV)
    state["y"] = torch.randn(t, s * n, generator=g, device=DEV).to(TYPES[case["y"]])
    state["out"] = torch.empty_like(state["y"])
    if own:
        from witchcraft_amd import adapters as module

        size = module.workspace_bytes(t, k, s, r)
        state["work"] = torch.empty(max(size, 1), dtype=torch.uint8, device=DEV)
    return state


def _positions(case, h):
    """Positions [axes][tokens].  One axis: each request counts from `far`.  More: each request is a run of
    images, of 16 to 64 columns; the last axis is the column, the one before it the row, the first the image."""
    out = []
    for n in _lengths(h, case["tokens"], case["requests"]).tolist():
        i = torch.arange(n)
        if case["axes"] == 1:
            out.append(case["far"] + i[None])
            continue
        width = int(torch.randint(16, 65, (), generator=h))
        grid = [i // (width * width), i // width % width, i % width]
        out.append(case["far"] + torch.stack(grid[3 - case["axes"]:]))
    return torch.cat(out, 1).to(torch.int32).contiguous()


def _prepare_rotate(case, g, h):
    t, d, kind = case["tokens"], case["dim"], TYPES[case["type"]]
    heads, key_heads = case["heads"], case["key_heads"]
    # the fused projection's rows: queries, keys and values
    state = {"qkv": torch.randn(t, (heads + 2 * key_heads) * d, generator=g, device=DEV).mul_(2.0).to(kind)}
    state["positions"] = _positions(case, h).to(DEV)
    state["q_gamma"] = state["k_gamma"] = None
    if case["norms"]:
        state["q_gamma"] = 1.0 + 0.2 * torch.randn(d, generator=g, device=DEV)
        state["k_gamma"] = 1.0 + 0.2 * torch.randn(d, generator=g, device=DEV)
    state["q"] = torch.empty(t, heads, d, dtype=kind, device=DEV)
    state["k"] = torch.empty(t, key_heads, d, dtype=kind, device=DEV)
    if own:
        from witchcraft_amd import rotary

        state["table"] = torch.from_numpy(rotary.table(*_frequencies(case)).view("int64")).to(DEV)
    return state


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    h = torch.Generator().manual_seed(seed)
    state = (_prepare_adapter if case["op"] == "adapter" else _prepare_rotate)(case, g, h)
    state["case"] = case
    return state


# ---- the plain form ------------------------------------------------------------------------

def _rows(state, kind):
    """The rows' values: as they are, or what codes and scales stand for."""
    x = state["x"]
    if state["x_scales"] is None:
        return x.to(kind)
    t, k = x.shape
    scale = torch.exp2(state["x_scales"][:, :t].t().to(kind) - 127.0).repeat_interleave(BLOCK, 1)[:, :k]
    return x.view(torch.float8_e4m3fn).to(kind) * scale


def _plain_adapter(s):
    case = s["case"]
    n, slices = case["cols"], case["slices"]
    x, out = _rows(s, torch.float32), s["y"].float()
    for g in range(case["adapters"]):
        rows = (s["ids"] == g).nonzero()[:, 0]
        if rows.numel() == 0:
            continue
        part = x[rows]
        for i in range(slices):
            down = part @ s["a"][g, i].float().t()
            up = down @ s["b"][g, i * n:(i + 1) * n].float().t()
            out[rows, i * n:(i + 1) * n] += s["scales"][g] * up
    return {"out": out.to(s["y"].dtype)}


def _plain_rotate(s):
    case = s["case"]
    t, d, rot, heads, key_heads = case["tokens"], case["dim"], case["rot"], case["heads"], case["key_heads"]
    freqs, axis = _frequencies(case)
    # angles of far positions need 64 bits
    turn = s["positions"][torch.tensor(axis, device=DEV)].double() * torch.tensor(freqs, dtype=torch.float64, device=DEV)[:, None]
    cos, sin = torch.cos(turn).t().float()[:, None], torch.sin(turn).t().float()[:, None]
    q, k = s["qkv"][:, :heads * d], s["qkv"][:, heads * d:(heads + key_heads) * d]
    out = {}
    for name, x, gamma in (("q", q, s["q_gamma"]), ("k", k, s["k_gamma"])):
        x = x.reshape(t, -1, d).float()
        if gamma is not None:
            x = x * torch.rsqrt((x * x).mean(2, keepdim=True) + EPS) * gamma
        if case["pairing"] == "halves":
            a, b = x[:, :, :rot // 2], x[:, :, rot // 2:rot]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], 2)
        else:
            a, b = x[:, :, 0:rot:2], x[:, :, 1:rot:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], 3).flatten(2)
        out[name] = torch.cat([turned, x[:, :, rot:]], 2).to(s["qkv"].dtype)
    return out


# ---- one pass ------------------------------------------------------------------------------

def _own_adapter(s):
    from witchcraft_amd import adapters

    case = s["case"]
    n = case["cols"] * case["slices"]
    # a 32-bit stream takes the sums in place, here as in the plain form
    out = s["y"] if case["y"] == "f32" else s["out"]
    adapters.add_device(s["x"].data_ptr(), CODE[case["x"]], 0 if s["x_scales"] is None else s["x_scales"].data_ptr(),
                        case["depth"], case["tokens"], case["depth"], s["ids"].data_ptr(), case["adapters"],
                        s["a"].data_ptr(), s["b"].data_ptr(), CODE[case["w"]], s["ranks"].data_ptr(),
                        s["scales"].data_ptr(), case["rank"], (case["cols"],) * case["slices"], s["y"].data_ptr(), n,
                        out.data_ptr(), n, CODE[case["y"]], s["work"].data_ptr(), s["work"].numel(),
                        torch.cuda.current_stream().cuda_stream)
    return {"out": out}


def _own_rotate(s):
    from witchcraft_amd import rotary

    case = s["case"]
    d, heads, key_heads = case["dim"], case["heads"], case["key_heads"]
    row, at = (heads + 2 * key_heads) * d, s["qkv"].data_ptr()
    norms = case["norms"]
    rotary.rotate_device(at, row, heads, at + heads * d * SIZE[case["type"]], row, key_heads, CODE[case["type"]],
                         case["tokens"], d, s["q_gamma"].data_ptr() if norms else 0, s["k_gamma"].data_ptr() if norms else 0,
                         EPS, s["table"].data_ptr(), case["rot"],
                         rotary.HALVES if case["pairing"] == "halves" else rotary.NEIGHBOURS, s["positions"].data_ptr(),
                         case["axes"], s["q"].data_ptr(), heads * d, s["k"].data_ptr(), key_heads * d,
                         torch.cuda.current_stream().cuda_stream)
    return {"q": s["q"], "k": s["k"]}


def run(state):
    if state["case"]["op"] == "adapter":
        return _own_adapter(state) if own else _plain_adapter(state)
    return _own_rotate(state) if own else _plain_rotate(state)


# ---- what a pass cannot do without ---------------------------------------------------------

def work(case):
    t = case["tokens"]
    if case["op"] == "rotate":
        values = t * (case["heads"] + case["key_heads"]) * case["dim"]
        return {"bytes": 2 * values * SIZE[case["type"]] + 4 * t * case["axes"],
                "flops": values * ((4 if case["norms"] else 0) + 3 * case["rot"] / case["dim"])}
    k, n, inner = case["depth"], case["cols"] * case["slices"], case["slices"] * case["rank"]
    share = _adapted(case) / case["requests"]  # of the rows, about
    used = min(case["adapters"], _adapted(case))
    x = share * t * (k * SIZE[case["x"]] + (-(-k // BLOCK) if case["x"] == "e4m3" else 0))
    return {"bytes": x + 2 * t * n * SIZE[case["y"]] + 4 * t + used * 2 * (inner * k + n * case["rank"]),
            "flops": 2 * share * t * (inner * k + n * case["rank"])}


# ---- the definition in 64 bits -------------------------------------------------------------

def _exact_adapter(s):
    """y[t] + scale (B A x[t]) for each row with an adapter, one slice of columns after the other."""
    case = s["case"]
    n = case["cols"]
    x, out = _rows(s, torch.float64), s["y"].double()
    for g in sorted(set(s["ids"].tolist()) - {-1}):
        mine = s["ids"] == g
        inner = torch.einsum("tk,srk->tsr", x[mine], s["a"][g].double()) * s["scales"][g].double()
        b = s["b"][g].double().view(case["slices"], n, case["rank"])
        out[mine] += torch.cat([inner[:, i] @ b[i].t() for i in range(case["slices"])], 1)
    return {"out": out}


def _exact_rotate(s):
    """Each pair as a complex number times e^(i angle)."""
    case = s["case"]
    t, d, rot, heads = case["tokens"], case["dim"], case["rot"], case["heads"]
    freqs, axis = _frequencies(case)
    angle = torch.stack([s["positions"][a].double() * f for f, a in zip(freqs, axis)], 1)
    turn = torch.polar(torch.ones_like(angle), angle)
    rows = s["qkv"].view(t, -1, d)
    out = {}
    for name, x, gamma in (("q", rows[:, :heads], s["q_gamma"]), ("k", rows[:, heads:heads + case["key_heads"]], s["k_gamma"])):
        y = x.double()
        if gamma is not None:
            y = y / torch.sqrt(y.square().sum(2, keepdim=True) / d + EPS) * gamma.double()
        at = torch.arange(rot, device=DEV)
        first, second = (at[:rot // 2], at[rot // 2:]) if case["pairing"] == "halves" else (at[0::2], at[1::2])
        z = torch.complex(y[:, :, first], y[:, :, second]) * turn[:, None]
        y[:, :, first], y[:, :, second] = z.real, z.imag
        out[name] = y
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return (_exact_adapter if case["op"] == "adapter" else _exact_rotate)(s)
