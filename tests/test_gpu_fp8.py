"""The 8-bit operators against their definition in 64 bits.

Codes.  e4m3 rounds to the nearest, ties to even, so a code's value is at most half a step off what
it stands for: 2^-4 of the value, or 2^-10 scales in the subnormal range.  Where the coded value is
the input itself (the quantizers), codes and scales are compared bit for bit.  Where it is computed
in f32 first (norm, gated product), the value may lie either side of a border: codes are held to the
half step plus the computation's bound, and a power-of-two scale may take its neighbour only if the
block's maximum lies within that bound of the border.

Products.  Codes of few bits and small integers have exact products and sums, so any kernel must give
the correctly rounded result (`exact` tests, over all shapes).  On ordinary data an f32 result is
within f32 summation rounding, (K + 16) 2^-23 sum |a w|; an f16 or bf16 result within its own half step
(2^-11, 2^-8 of the value) plus the fp8 matrix instructions' alignment: each product is kept to 2^-12
of the largest of its group at worst (2^-13 as measured), so a K block is off by at most 128 * 2^-12 of its largest
product, and, errors of either sign, by far less in the 2-norm.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DEV = "cuda:0"
U = 2.0 ** -24
TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (2, torch.bfloat16)}
EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step, relative
E8M0, F32S = 0, 1

# value of every code, and the non-negative finite ones in order
TABLE = np.array([(-1.0 if c & 128 else 1.0) * (np.ldexp(c & 7, -9) if not c & 0x78 else
                  np.ldexp(8 + (c & 7), ((c >> 3) & 15) - 10)) for c in range(256)])
TABLE[[0x7f, 0xff]] = np.nan
GRID = TABLE[:0x7f]


@pytest.fixture(scope="module")
def fp8():
    from witchcraft_amd import fp8 as f
    return f


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _blocks(n):
    return (n + 127) // 128


def _rows16(m):
    return (m + 15) // 16 * 16


def _round_e4m3(v):
    """Codes of |v| <= 448 in 64 bits, nearest, ties to even; NaN elsewhere."""
    a = np.abs(v)
    hi = np.clip(np.searchsorted(GRID, a), 1, len(GRID) - 1)
    lo = hi - 1
    up = a - GRID[lo] > GRID[hi] - a
    tie = a - GRID[lo] == GRID[hi] - a
    code = np.where(up | (tie & (hi % 2 == 0)), hi, lo).astype(np.uint8)
    return np.where(np.isfinite(v), code | (np.signbit(v) << 7).astype(np.uint8), 0x7f).astype(np.uint8)


def _same_codes(got, want):
    """Equal, any NaN code for a NaN code."""
    nan = (want & 0x7f) == 0x7f
    return np.array_equal(np.where(nan, 0x7f, want), np.where((got & 0x7f) == 0x7f, 0x7f, got))


def _byte_of(top):
    """The E8M0 byte of a block whose largest magnitude is `top` (64 bits): least e with top <= 448 2^e."""
    f, e = np.frexp(np.asarray(top, np.float64) / 448.0)
    e = np.where(f == 0.5, e - 1, e)
    return np.where(top > 0, np.maximum(e, -126), -126) + 127


def _guarded(n, dtype=torch.uint8, fill=0x5a, before=64):
    """A device buffer of n elements with guard bytes on both sides."""
    b = torch.empty(0, dtype=dtype).element_size()
    raw = torch.full((before * b + n * b + 256,), fill, dtype=torch.uint8, device=DEV)
    return raw, raw[before * b:before * b + n * b].view(dtype) if n else raw[:0].view(dtype)


def _untouched(raw, view, fill=0x5a):
    n = view.numel() * view.element_size()
    off = 64 * view.element_size()
    return bool((raw[:off] == fill).all()) and bool((raw[off + n:] == fill).all())


# ---- activations -----------------------------------------------------------------------------

def _special_rows(m, k, seed):
    r = np.random.default_rng(seed)
    x = r.standard_normal((m, k)) * np.exp(r.normal(0, 3, (m, 1)))
    x[0, :] = 0.0
    if m > 1:
        x[1, ::3] = np.nan
        x[1, 1] = np.inf
    if m > 2:
        x[2, :] = -np.inf
    if m > 3:
        x[3, :] = r.choice([448.0, 449.0, 224.0, -448.0, 1.0, 1.0625, 1.1875, 2.0 ** -9, -0.0, 2.0 ** -10], k)
    if m > 4:
        x[4, :] = r.choice([6e-8, -6e-8, 0.0, 1.2e-7], k)  # f16 subnormals
    return x


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,K", [(1, 16), (1, 128), (3, 144), (17, 768), (5, 4112), (1000, 272), (37, 8192), (4097, 16)])
def test_quantize_bitexact(fp8, kind, M, K):
    code, t = TYPES[kind]
    x = torch.from_numpy(_special_rows(M, K, M + K)).to(t).to(DEV)
    if kind != "f16" and M > 5:
        x[5] = 3e38  # near the type's top, and (below) subnormal in f32
    if kind == "f32" and M > 6:
        x[6] = 1e-41
    v = x.double().cpu().numpy()
    raw, codes = _guarded(M * K)
    sraw, scales = _guarded(_blocks(K) * _rows16(M))
    fp8.quantize_device(x.data_ptr(), code, M, K, codes.data_ptr(), scales.data_ptr(), _stream())
    torch.cuda.synchronize()
    got, s = codes.cpu().numpy().reshape(M, K), scales.cpu().numpy().reshape(_blocks(K), _rows16(M))
    assert _untouched(raw, codes) and _untouched(sraw, scales)
    assert (s[:, M:] == 0x5a).all()
    size = np.where(np.isfinite(v), np.abs(v), 0.0)
    for b in range(_blocks(K)):
        part = slice(128 * b, min(K, 128 * b + 128))
        byte = _byte_of(size[:, part].max(1))
        assert np.array_equal(s[b, :M], byte), b
        assert _same_codes(got[:, part], _round_e4m3(v[:, part] * 2.0 ** (127.0 - byte[:, None]))), b


def test_quantize_large_offsets(fp8):
    """Codes past 2^32: rows at the end of a matrix of more than 4 GiB."""
    M, K = 270000, 16000
    x = torch.zeros(M, K, dtype=torch.bfloat16, device=DEV)
    x[-3:] = torch.randn(3, K, device=DEV).to(torch.bfloat16)
    codes = torch.empty(M, K, dtype=torch.uint8, device=DEV)
    scales = torch.empty(_blocks(K), _rows16(M), dtype=torch.uint8, device=DEV)
    fp8.quantize_device(x.data_ptr(), 2, M, K, codes.data_ptr(), scales.data_ptr(), _stream())
    v = x[-3:].double().cpu().numpy()
    s = scales[:, M - 3:M].cpu().numpy()
    byte = np.stack([_byte_of(np.abs(v[:, 128 * b:128 * b + 128]).max(1)) for b in range(_blocks(K))])
    assert np.array_equal(s, byte)
    e = np.repeat(byte.T, 128, 1)[:, :K]
    assert _same_codes(codes[-3:].cpu().numpy(), _round_e4m3(v * 2.0 ** (127.0 - e)))
    assert int(codes[:-3].max()) == 0 and bool((scales[:, :M - 3] == 1).all())


# ---- weights ---------------------------------------------------------------------------------

@pytest.mark.parametrize("scale", [E8M0, F32S])
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("N,K", [(1, 16), (128, 128), (129, 144), (300, 768), (257, 1040), (7, 2048)])
def test_quantize_weights_bitexact(fp8, kind, N, K, scale):
    code, t = TYPES[kind]
    r = np.random.default_rng(N + K)
    x = r.standard_normal((N, K)) * np.exp(r.normal(0, 2, (N, 1)))
    if N > 128:
        x[128:] = 0.0
    x[0, 3] = np.nan
    x[N // 2, 9] = np.inf
    w = torch.from_numpy(x).to(t).to(DEV)
    v = w.double().cpu().numpy()
    nb, kb = _blocks(N), _blocks(K)
    raw, codes = _guarded(N * K)
    sraw, scales = _guarded(nb * kb, torch.float32 if scale else torch.uint8)
    fp8.quantize_weights_device(w.data_ptr(), code, N, K, scale, codes.data_ptr(), scales.data_ptr(), _stream())
    torch.cuda.synchronize()
    got, s = codes.cpu().numpy().reshape(N, K), scales.cpu().numpy().reshape(nb, kb)
    assert _untouched(raw, codes) and _untouched(sraw, scales)
    for i in range(nb):
        for b in range(kb):
            part = v[128 * i:128 * i + 128, 128 * b:128 * b + 128]
            top = np.where(np.isfinite(part), np.abs(part), 0.0).max()
            if scale == F32S:
                top = np.maximum(np.float32(top), np.float32(448 * 2.0 ** -126))
                assert s[i, b] == top / np.float32(448)
                with np.errstate(over="ignore", invalid="ignore"):
                    q = (part.astype(np.float32) * (np.float32(448) / top)).astype(np.float64)
                q = np.clip(q, -448, 448) if np.isfinite(part).all() else np.where(np.isfinite(part), np.clip(q, -448, 448), np.nan)
            else:
                byte = int(_byte_of(top))
                assert s[i, b] == byte
                q = part * 2.0 ** (127 - byte)
            assert _same_codes(got[128 * i:128 * i + 128, 128 * b:128 * b + 128], _round_e4m3(q)), (i, b)


# ---- norm ------------------------------------------------------------------------------------

def _check_codes(codes, scales, y, rel, floor=0.0):
    """Codes [M, K] and bytes [blocks, M] against values y in 64 bits, known to `rel` of their size (and
    `floor`, per value).  Returns the bytes that are a neighbour's."""
    M, K = y.shape
    other = 0
    floor = np.broadcast_to(floor, y.shape)
    for b in range(_blocks(K)):
        part = slice(128 * b, min(K, 128 * b + 128))
        v, f = y[:, part], floor[:, part]
        size = np.where(np.isfinite(v), np.abs(v), 0.0)
        lo = _byte_of(np.max(np.maximum(size * (1 - rel) - f, 0.0), 1))
        hi = _byte_of(np.max(size * (1 + rel) + f, 1))
        byte = scales[b].astype(int)
        assert ((byte >= lo) & (byte <= hi)).all(), (b, byte, lo, hi)
        other += int((byte != _byte_of(size.max(1))).sum())
        s = 2.0 ** (byte[:, None] - 127.0)
        got = TABLE[codes[:, part]] * s
        assert np.array_equal(np.isnan(got), ~np.isfinite(v)), b
        ok = np.isfinite(v)
        tol = np.maximum(np.abs(v) * 2.0 ** -4, 2.0 ** -10 * s) * (1 + rel) + np.abs(v) * rel + f * 1.0625
        assert (np.abs(got - v)[ok] <= tol[ok]).all(), (b, float((np.abs(got - v) / tol)[ok].max()))
    return other


def _norm_case(fp8, xk, dk, M, D, place="apart", seed=0, gamma=None, fix=None):
    (xc, xt), r = TYPES[xk], np.random.default_rng(seed + M + D)
    x = torch.from_numpy(r.standard_normal((M, D)) * np.exp(r.normal(0, 1, (M, 1)))).to(xt).to(DEV)
    if fix is not None:
        fix(x)
    g = torch.from_numpy(1 + 0.3 * r.standard_normal(D) if gamma is None else gamma).float().to(DEV)
    delta, dc, total = None, 0, None
    h = x.float()
    if dk:
        dc, dt = TYPES[dk]
        delta = torch.from_numpy(0.5 * r.standard_normal((M, D))).to(dt).to(DEV)
        h = (h + delta.float()).to(xt)
        total = {"apart": torch.empty_like(x), "x": x, "delta": delta, "none": None}[place]
    raw, codes = _guarded(M * D)
    sraw, scales = _guarded(_blocks(D) * _rows16(M))
    fp8.rmsnorm_device(x.data_ptr(), xc, delta.data_ptr() if dk else 0, dc, M, D, g.data_ptr(), 1e-6,
                       total.data_ptr() if total is not None else 0, codes.data_ptr(), scales.data_ptr(), _stream())
    torch.cuda.synchronize()
    assert _untouched(raw, codes) and _untouched(sraw, scales)
    if total is not None:
        assert torch.equal(total.view(torch.uint8), h.to(xt).contiguous().view(torch.uint8))
    s = scales.cpu().numpy().reshape(_blocks(D), _rows16(M))
    assert (s[:, M:] == 0x5a).all()
    h = h.double().cpu().numpy()
    with np.errstate(invalid="ignore", over="ignore"):
        y = h / np.sqrt((h * h).mean(1, keepdims=True) + 1e-6) * g.double().cpu().numpy()
    return codes.cpu().numpy().reshape(M, D), s[:, :M], y


# f32 steps of a value: squares and their sum (a lane's chain, then trees: 4 values of up to 16 chunks,
# 6 and 16 joins), halved by the root; division, addition, root, two products
NORM_REL = (96 / 2 + 8) * U


@pytest.mark.parametrize("D", [16, 128, 144, 768, 1024, 1040, 4096, 4112, 16384, 16400, 40000])
@pytest.mark.parametrize("xk,dk", [("f32", None), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f32")])
def test_rmsnorm(fp8, xk, dk, D):
    for M in (1, 5, 33):
        codes, s, y = _norm_case(fp8, xk, dk, M, D)
        _check_codes(codes, s, y, NORM_REL)


@pytest.mark.parametrize("xk", list(TYPES))
@pytest.mark.parametrize("dk", list(TYPES))
def test_rmsnorm_types_and_places(fp8, xk, dk):
    sizes = {"f32": 4, "f16": 2, "bf16": 2}
    for D in (768, 2048, 16400):
        for place in ("apart", "x", "none") + (("delta",) if sizes[xk] == sizes[dk] else ()):
            if place == "delta" and xk != dk:
                continue  # the sum's type is x's: checked through its bytes where the types agree
            codes, s, y = _norm_case(fp8, xk, dk, 7, D, place)
            _check_codes(codes, s, y, NORM_REL)


def test_rmsnorm_rows_that_are_not_finite(fp8):
    def fix(x):
        x[0] = 0.0
        x[1, 5] = float("nan")
        x[2, 700] = float("inf")
        x[3] = 1e30  # the sum of squares overflows: every value becomes 0
        x[4] = 1e-30
    codes, s, y = _norm_case(fp8, "f32", None, 9, 768, fix=fix)
    y[2] = 0.0  # an infinite sum of squares leaves 0, and 0 * inf is NaN
    y[2, 700] = np.nan
    y[3] = 0.0
    _check_codes(codes, s, y, NORM_REL)
    assert (s[:, 0] == 1).all() and (codes[0] == 0).all()


def test_rmsnorm_many_rows(fp8):
    codes, s, y = _norm_case(fp8, "f32", "f16", 70001, 768)
    other = _check_codes(codes, s, y, NORM_REL)
    assert other <= 70001 * 6 * 1e-4  # borders are met by chance only


def test_longest_rows(fp8):
    """K = 2^21 through the quantizers and the norm (whose lanes sum 2,048 squares one after another)."""
    K = 1 << 21
    x = torch.randn(3, K, generator=torch.Generator(device=DEV).manual_seed(4), device=DEV)
    v = x.double().cpu().numpy()
    codes = torch.empty(3, K, dtype=torch.uint8, device=DEV)
    scales = torch.empty(_blocks(K), 16, dtype=torch.uint8, device=DEV)
    fp8.quantize_device(x.data_ptr(), 0, 3, K, codes.data_ptr(), scales.data_ptr(), _stream())
    byte = _byte_of(np.abs(v).reshape(3, -1, 128).max(2))
    assert np.array_equal(scales[:, :3].cpu().numpy(), byte.T)
    assert _same_codes(codes.cpu().numpy(), _round_e4m3(v * 2.0 ** (127.0 - np.repeat(byte, 128, 1))))
    blocks = torch.empty(1, _blocks(K), dtype=torch.uint8, device=DEV)
    fp8.quantize_weights_device(x.data_ptr(), 0, 3, K, E8M0, codes.data_ptr(), blocks.data_ptr(), _stream())
    byte = byte.max(0)
    assert np.array_equal(blocks.cpu().numpy()[0], byte)
    assert _same_codes(codes.cpu().numpy(), _round_e4m3(v * 2.0 ** (127.0 - np.repeat(byte, 128)[None])))
    got = _norm_case(fp8, "bf16", "f16", 2, K)
    _check_codes(*got, ((2048 + 22) / 2 + 8) * U)


def test_most_workgroups(fp8):
    """More rows and blocks than a launch has workgroups: the last ones are reached."""
    M = (4 << 20) + 5
    x = torch.zeros(M, 16, dtype=torch.bfloat16, device=DEV)
    x[-3:] = torch.randn(3, 16, device=DEV).to(torch.bfloat16)
    g = torch.ones(16, device=DEV)
    codes = torch.full((M, 16), 77, dtype=torch.uint8, device=DEV)
    scales = torch.full((1, _rows16(M)), 77, dtype=torch.uint8, device=DEV)
    fp8.rmsnorm_device(x.data_ptr(), 2, 0, 0, M, 16, g.data_ptr(), 1e-6, 0, codes.data_ptr(), scales.data_ptr(), _stream())
    assert int(codes[:-3].max()) == 0 and bool((scales[:, :M - 3] == 1).all()) and bool((scales[:, M:] == 77).all())
    v = x[-3:].double().cpu().numpy()
    y = v / np.sqrt((v * v).mean(1, keepdims=True) + 1e-6)
    _check_codes(codes[-3:].cpu().numpy(), scales[:, M - 3:M].cpu().numpy(), y, NORM_REL)
    del x, codes
    N = (128 << 20) + 200
    w = torch.zeros(N, 16, dtype=torch.bfloat16, device=DEV)
    w[-1] = torch.randn(16, device=DEV).to(torch.bfloat16)
    codes = torch.full((N, 16), 77, dtype=torch.uint8, device=DEV)
    scales = torch.full((_blocks(N),), 77, dtype=torch.uint8, device=DEV)
    fp8.quantize_weights_device(w.data_ptr(), 2, N, 16, E8M0, codes.data_ptr(), scales.data_ptr(), _stream())
    v = w[-1].double().cpu().numpy()
    byte = _byte_of(np.abs(v).max())
    assert bool((scales[:-1] == 1).all()) and int(scales[-1]) == byte
    assert not bool(codes[:-1].any()) and _same_codes(codes[-1].cpu().numpy(), _round_e4m3(v * 2.0 ** (127.0 - byte)))


# ---- products --------------------------------------------------------------------------------

def _operand(values, scale_bytes, M, K):
    """Device codes and padded scales (rows past M: NaN) from e4m3 values and bytes [blocks, M]."""
    codes = _round_e4m3(values)
    s = np.full((_blocks(K), _rows16(M)), 255, np.uint8)
    s[:, :M] = scale_bytes
    return torch.from_numpy(codes).to(DEV), torch.from_numpy(s).to(DEV)


def _exact_case(M, N, K, scale, seed):
    """Operands of small integers: every partial sum is exact in f32.  Scales: powers of two that differ
    by row and block in a range that keeps the sums exact (2^0 .. 2^3 a side; |a w| <= 4, K <= 8192:
    sums below 2^21 over steps of 2^-2)."""
    r = np.random.default_rng(seed)
    vals = np.array([-2, -1.5, -1, -0.5, 0, 0.5, 1, 1.5, 2])
    a, w = r.choice(vals, (M, K)), r.choice(vals, (N, K))
    ab = r.integers(127, 130, (_blocks(K), M))
    wb = r.integers(126, 129, (_blocks(N), _blocks(K)))
    acodes, ascales = _operand(a, ab, M, K)
    wcodes = torch.from_numpy(_round_e4m3(w)).to(DEV)
    ws = 2.0 ** (wb - 127.0)
    wscales = torch.from_numpy(ws.astype(np.float32) if scale else wb.astype(np.uint8)).to(DEV)
    av = a * np.repeat(2.0 ** (ab.T - 127.0), 128, 1)[:, :K]
    wv = w * np.repeat(np.repeat(ws, 128, 0)[:N], 128, 1)[:, :K]
    return acodes, ascales, wcodes, wscales, av, wv


def _matmul(fp8, a, sa, w, sw, N, kind, scale):
    (M, K), (code, t) = a.shape, TYPES[kind]
    raw, c = _guarded(M * N, t)
    fp8.matmul_device(a.data_ptr(), sa.data_ptr(), M, w.data_ptr(), sw.data_ptr(), N, K, scale, c.data_ptr(), code,
                      _stream())
    torch.cuda.synchronize()
    assert _untouched(raw, c)
    return c.view(M, N)


SHAPES = [
    (1, 1, 16), (1, 16, 128), (1, 2304, 768), (2, 77, 144), (15, 64, 2048), (16, 130, 400), (17, 128, 768),
    (31, 768, 2048), (32, 2304, 768), (33, 257, 1040), (64, 512, 128), (65, 513, 256), (100, 1000, 272),
    (127, 384, 2064), (128, 128, 4096), (129, 768, 768), (200, 40, 112), (255, 2048, 768), (256, 256, 256),
    (257, 259, 384), (300, 2304, 768), (511, 128, 2048), (513, 770, 528), (1000, 640, 768), (2049, 1100, 304),
    (4616, 768, 2048), (5000, 1, 768), (5000, 515, 128), (1, 8192, 4096), (7, 5000, 8192), (48, 9000, 512),
]


@pytest.mark.parametrize("scale", [E8M0, F32S])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_matmul_exact(fp8, M, N, K, scale):
    a, sa, w, sw, av, wv = _exact_case(M, N, K, scale, M + N + K)
    want = torch.from_numpy(av).to(DEV) @ torch.from_numpy(wv).to(DEV).t()
    for kind, (_, t) in TYPES.items():
        got = _matmul(fp8, a, sa, w, sw, N, kind, scale)
        ref = want.float() if kind == "f32" else want.float().to(t)
        assert torch.equal(got, ref), (kind, int((got != ref).sum()))


# One shape at least on each side of every border of the kernels' choice, tiles that end inside on both
# axes, workgroups that walk several tiles, and more than 64 K blocks.
VARIANTS = [
    (16, 4096, 144), (16, 4100, 144), (15, 8192, 256), (16, 8200, 128), (13, 16384, 128), (16, 16400, 272),
    (17, 4096, 400), (32, 8192, 144), (31, 8200, 272), (32, 16384, 144), (33, 16390, 128), (64, 8192, 400),
    (64, 16390, 144), (65, 4100, 1040), (70, 5001, 8336), (512, 2048, 400), (513, 2041, 272), (512, 2000, 8336),
    (1024, 2048, 144), (1024, 2041, 8336), (1025, 2048, 272), (1100, 1600, 8336), (2048, 2048, 144), (2030, 2041, 8336),
    (2049, 2048, 400), (3000, 2041, 8336), (4096, 2041, 144), (4097, 2048, 272), (6144, 2041, 272), (6145, 2048, 144),
    (6150, 2041, 8336), (16413, 1027, 272), (16413, 1032, 16), (33000, 515, 384), (1500, 770, 16400),
]


@pytest.mark.parametrize("scale", [E8M0, F32S])
@pytest.mark.parametrize("M,N,K", VARIANTS)
def test_matmul_variants(fp8, M, N, K, scale):
    """As test_matmul_exact: at K = 16,400 sums stay below 2^20 over steps of 2^-3."""
    test_matmul_exact(fp8, M, N, K, scale)


def _signs(shape, seed):
    """Codes of -1, 0 and 1 on the device, and a function that gives a stretch of columns in 64 bits."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    v = torch.randint(0, 3, shape, generator=g, device=DEV, dtype=torch.uint8)
    codes = torch.tensor([0, 0x38, 0xb8], dtype=torch.uint8, device=DEV)[v.int()]
    table = torch.from_numpy(TABLE).to(DEV)
    return codes, lambda a, b: table[codes[:, a:b].int()]


def _unit_scales(n, k, rows):
    return torch.full((_blocks(k), _rows16(n)) if rows else (_blocks(n), _blocks(k)), 127, dtype=torch.uint8, device=DEV)


def _long_product(a, w, K):
    return sum(a(k, min(K, k + 131072)) @ w(k, min(K, k + 131072)).t() for k in range(0, K, 131072))


@pytest.mark.parametrize("M,N", [(3, 70), (65, 4100)])
def test_matmul_longest_rows(fp8, M, N):
    """K = 2^21; sums of signs are exact."""
    K = 1 << 21
    (a, av), (w, wv) = _signs((M, K), 1), _signs((N, K), 2)
    want = _long_product(av, wv, K).float()
    for kind in ("f32", "bf16"):
        got = _matmul(fp8, a, _unit_scales(M, K, True), w, _unit_scales(N, K, False), N, kind, E8M0)
        assert torch.equal(got, want.to(TYPES[kind][1])), kind


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_matmul_large_offsets(fp8, kind):
    """More than 2^31 results."""
    M, N, K = 300001, 8200, 16
    (a, av), (w, wv) = _signs((M, K), 3), _signs((N, K), 4)
    got = _matmul(fp8, a, _unit_scales(M, K, True), w, _unit_scales(N, K, False), N, kind, E8M0)
    want = av(0, K).to(TYPES[kind][1]).float(), wv(0, K).float()
    for m in range(0, M, 20000):
        assert torch.equal(got[m:m + 20000].float(), want[0][m:m + 20000] @ want[1].t()), m


def _ordinary(fp8, M, N, K, scale, seed):
    """Quantized normal data with outlying channels, through the quantizers, and the values it stands for."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(M, K, generator=g, device=DEV) * torch.exp(0.5 * torch.randn(K, generator=g, device=DEV))
    x[:, K // 3] *= 20
    a, sa = torch.empty(M, K, dtype=torch.uint8, device=DEV), torch.zeros(_blocks(K), _rows16(M), dtype=torch.uint8, device=DEV)
    fp8.quantize_device(x.data_ptr(), 0, M, K, a.data_ptr(), sa.data_ptr(), _stream())
    w, sw, wv = _ordinary_weights(fp8, N, K, scale, g)
    table = torch.from_numpy(TABLE).to(DEV)
    av = table[a.long()] * torch.exp2(sa[:, :M].double() - 127).t().repeat_interleave(128, 1)[:, :K]
    return a, sa, w, sw, av, wv


def _ordinary_weights(fp8, N, K, scale, g):
    x = torch.randn(N, K, generator=g, device=DEV) / K ** 0.5
    w = torch.empty(N, K, dtype=torch.uint8, device=DEV)
    sw = torch.empty(_blocks(N), _blocks(K), dtype=torch.float32 if scale else torch.uint8, device=DEV)
    fp8.quantize_weights_device(x.data_ptr(), 0, N, K, scale, w.data_ptr(), sw.data_ptr(), _stream())
    s = sw.double() if scale else torch.exp2(sw.double() - 127)
    wv = torch.from_numpy(TABLE).to(DEV)[w.long()] * s.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    return w, sw, wv


def _alignment_bound(av, wv):
    """Per result: 128 * 2^-12 of the largest |a w| of every K block, from row maxima (an upper bound)."""
    M, K = av.shape
    out = torch.zeros(M, wv.shape[0], dtype=torch.float64, device=DEV)
    for b in range(_blocks(K)):
        part = slice(128 * b, 128 * b + 128)
        out += av[:, part].abs().amax(1)[:, None] * wv[:, part].abs().amax(1)[None, :]
    return out * 128 * 2.0 ** -12


@pytest.mark.parametrize("scale", [E8M0, F32S])
@pytest.mark.parametrize("M,N,K", [(1, 768, 2048), (9, 300, 784), (32, 2304, 768), (130, 770, 2048), (1500, 768, 768),
                                   (777, 1030, 4096), (3000, 2304, 768)])
def test_matmul_ordinary(fp8, M, N, K, scale):
    a, sa, w, sw, av, wv = _ordinary(fp8, M, N, K, scale, M + N)
    want = av @ wv.t()
    total = av.abs() @ wv.abs().t()
    align = _alignment_bound(av, wv)
    for kind in TYPES:
        got = _matmul(fp8, a, sa, w, sw, N, kind, scale).double()
        err = (got - want).abs()
        bound = (K + 16) * 2.0 ** -23 * total
        if kind != "f32":
            bound = (bound + align) * (1 + EPS[kind]) + EPS[kind] * want.abs() + 2.0 ** -25  # f16 subnormals' half step
        assert bool((err <= bound).all()), (kind, float((err / bound).max()))
        # in the 2-norm: rounding at most its half step, alignment errors of either sign, at most
        # 2^-12 / sqrt(3) of a product that is at most 9 times the typical one
        norm = float(err.norm() / want.norm())
        assert norm <= (1e-6 if kind == "f32" else EPS[kind] + 9 * 2.0 ** -12 / 3 ** 0.5), (kind, norm)


def test_matmul_repeats_its_bits(fp8):
    for M, N, K in ((1, 2304, 768), (32, 768, 2048), (700, 1030, 784), (2100, 2304, 768)):
        a, sa, w, sw, _, _ = _ordinary(fp8, M, N, K, F32S, 3)
        for kind in TYPES:
            first = _matmul(fp8, a, sa, w, sw, N, kind, F32S)
            assert torch.equal(first, _matmul(fp8, a, sa, w, sw, N, kind, F32S))


@pytest.mark.parametrize("M,N", [(5, 40), (40, 300), (600, 777), (2500, 1024)])
def test_matmul_rows_stand_alone(fp8, M, N):
    """A NaN code, a NaN scale or an infinite-looking row changes its own row only; a row's bits do not
    depend on what is behind the last row."""
    K = 400
    a, sa, w, sw, av, wv = _exact_case(M, N, K, E8M0, 5)
    want = (av @ wv.T)
    a[1, 399] = 0x7f
    sa[3, 3] = 255
    for kind in ("f32", "bf16"):
        got = _matmul(fp8, a, sa, w, sw, N, kind, E8M0).double().cpu().numpy()
        ref = torch.from_numpy(want).float().to(TYPES[kind][1]).double().numpy()
        assert np.isnan(got[[1, 3]]).all()
        keep = [i for i in range(M) if i not in (1, 3)]
        assert np.array_equal(got[keep], ref[keep])


def test_matmul_scale_bytes(fp8):
    """Every scale byte, on both sides, as far as the result's exponent is a float's."""
    M, N, K = 256, 40, 128
    one = np.full((M, K), 1.0)
    sa = np.arange(256)[None, :].repeat(1, 0)
    a, sad = _operand(one, sa, M, K)
    w = torch.from_numpy(_round_e4m3(np.full((N, K), 0.5))).to(DEV)
    for wb in (100, 127, 140):
        sw = torch.full((1, 1), wb, dtype=torch.uint8, device=DEV)
        e = np.arange(256) + wb - 254 + 6.0  # 128 * 0.5
        for kind in ("f32", "bf16"):
            got = _matmul(fp8, a, sad, w, sw, N, kind, E8M0).double().cpu().numpy()
            assert np.isnan(got[255]).all()
            rows = (e >= -126) & (e <= 127) & (np.arange(256) < 255)
            assert np.array_equal(got[rows], np.broadcast_to(2.0 ** e[rows, None], (rows.sum(), N))), (wb, kind)


def test_matmul_every_code(fp8):
    """Each of the 256 codes times one, in both operands' places and both kinds of instruction."""
    M, K = 256, 16
    codes = torch.arange(256, dtype=torch.uint8, device=DEV)
    a = torch.zeros(M, K, dtype=torch.uint8, device=DEV)
    a[:, 7] = codes
    one = torch.zeros(3, K, dtype=torch.uint8, device=DEV)
    one[:, 7] = 0x38
    sa = torch.full((1, 256), 127, dtype=torch.uint8, device=DEV)
    sw = torch.full((2, 1), 127, dtype=torch.uint8, device=DEV)
    for kind in TYPES:
        got = _matmul(fp8, a, sa, one, sw, 3, kind, E8M0).double().cpu().numpy()
        assert np.array_equal(got, np.repeat(TABLE[:, None], 3, 1), equal_nan=True), kind
        got = _matmul(fp8, one, sa[:, :16].contiguous(), a, sw, 256, kind, E8M0).double().cpu().numpy()
        assert np.array_equal(got, np.repeat(TABLE[None], 3, 0), equal_nan=True), kind


# ---- gated product ---------------------------------------------------------------------------

GATED_SHAPES = [
    (1, 16, 16), (1, 2048, 768), (2, 144, 144), (16, 256, 400), (17, 128, 768), (31, 400, 2048), (32, 2048, 768),
    (33, 272, 1040), (64, 512, 128), (65, 528, 256), (100, 1008, 272), (128, 128, 4096), (129, 768, 768),
    (255, 2048, 768), (257, 272, 384), (513, 784, 528), (1000, 640, 768), (2049, 1104, 304), (4616, 2048, 768),
    (5000, 16, 768),
]


def _gelu(x):
    return x * (0.5 + 0.5 * torch.tanh((2 / np.pi) ** 0.5 * (x + 0.044715 * x ** 3)))


def _gated(fp8, a, sa, w0, s0, w1, s1, scale):
    (M, K), N = a.shape, w0.shape[0]
    raw, codes = _guarded(M * N)
    sraw, scales = _guarded(_blocks(N) * _rows16(M))
    fp8.gated_gelu_device(a.data_ptr(), sa.data_ptr(), M, w0.data_ptr(), s0.data_ptr(), w1.data_ptr(), s1.data_ptr(), N,
                          K, scale, codes.data_ptr(), scales.data_ptr(), _stream())
    torch.cuda.synchronize()
    assert _untouched(raw, codes) and _untouched(sraw, scales)
    s = scales.cpu().numpy().reshape(_blocks(N), _rows16(M))
    assert (s[:, M:] == 0x5a).all()
    return codes.cpu().numpy().reshape(M, N), s[:, :M]


# gelu in f32: the exponent's argument is a few 2^-24 off, relative; times its size, at most
# 8 (2.31 + 0.103 * 64) log2(e)^0 = 72 for |gate| <= 8, three roundings deep: 72 * 3 * 2^-24, and the
# exp2, reciprocal and three products at 4 * 2^-23
GELU_REL = 72 * 3 * U + 10 * 2 * U


@pytest.mark.parametrize("scale", [E8M0, F32S])
@pytest.mark.parametrize("M,N,K", GATED_SHAPES)
def test_gated_exact_products(fp8, M, N, K, scale):
    """Gate and up are exact, small (|gate| <= 8: few non-zero values a row); what is left is the gelu."""
    r = np.random.default_rng(M + N + K)
    a, sa, w0, s0, av, _ = _exact_case(M, N, K, scale, M * 3 + N + K)
    keep = np.zeros((M, K), bool)  # 4 values a row, one scale: |gate| <= 4 * 2 * 2 / 2
    for i in range(M):
        keep[i, r.integers(0, K, 4)] = True
    v = np.where(keep, r.choice([-1.0, -0.5, 0.5, 1.0, 1.5], (M, K)), 0.0)
    a, sa = _operand(v, np.full((_blocks(K), M), 127), M, K)
    b = r.integers(126, 128, (2, _blocks(N), _blocks(K)))
    wv = r.choice([-1.0, -0.5, 0.0, 0.5, 1.0], (2, N, K))
    dev = [torch.from_numpy(_round_e4m3(x)).to(DEV) for x in wv]
    sw = [torch.from_numpy((2.0 ** (x - 127.0)).astype(np.float32) if scale else x.astype(np.uint8)).to(DEV) for x in b]
    full = [torch.from_numpy(wv[i] * np.repeat(np.repeat(2.0 ** (b[i] - 127.0), 128, 0)[:N], 128, 1)[:, :K]).to(DEV)
            for i in (0, 1)]
    x = torch.from_numpy(v).to(DEV)
    y = (_gelu(x @ full[0].t()) * (x @ full[1].t())).cpu().numpy()
    codes, s = _gated(fp8, a, sa, dev[0], sw[0], dev[1], sw[1], scale)
    _check_codes(codes, s, y, GELU_REL)


@pytest.mark.parametrize("scale", [E8M0, F32S])
@pytest.mark.parametrize("M,N,K", [(1, 2048, 768), (32, 2048, 768), (70, 400, 1040), (777, 2048, 768), (3000, 1040, 784)])
def test_gated_ordinary(fp8, M, N, K, scale):
    a, sa, w0, s0, av, wv0 = _ordinary(fp8, M, N, K, scale, M + N)
    w1, s1, wv1 = _ordinary_weights(fp8, N, K, scale, torch.Generator(device=DEV).manual_seed(M))
    g, u = av @ wv0.t(), av @ wv1.t()
    dg = (K + 16) * 2.0 ** -23 * (av.abs() @ wv0.abs().t()) + _alignment_bound(av, wv0)
    du = (K + 16) * 2.0 ** -23 * (av.abs() @ wv1.abs().t()) + _alignment_bound(av, wv1)
    y = _gelu(g) * u
    # |gelu'| <= 1.13; the gelu's own error for gates up to 100: 100 (2.31 + 0.103 * 1e4) would be all
    # of its value, but there gelu is x or 0 to 2^-24 (|gate| >= 8), so GELU_REL holds of max(|gelu|, 1e-9)
    floor = 1.13 * dg * (u.abs() + du) + _gelu(g).abs() * du + 1e-9 * u.abs()
    codes, s = _gated(fp8, a, sa, w0, s0, w1, s1, scale)
    _check_codes(codes, s, y.cpu().numpy(), GELU_REL, floor.cpu().numpy())
    again = _gated(fp8, a, sa, w0, s0, w1, s1, scale)
    assert np.array_equal(codes, again[0]) and np.array_equal(s, again[1])
    # in the 2-norm: e4m3's half step of values spread over a step, 2^-4 / sqrt(3)
    got = TABLE[codes] * np.repeat(2.0 ** (s.T - 127.0), 128, 1)[:, :N]
    y = y.cpu().numpy()
    assert np.linalg.norm(got - y) <= 2.0 ** -4 / 3 ** 0.5 * np.linalg.norm(y)


@pytest.mark.parametrize("scale", [E8M0, F32S])
@pytest.mark.parametrize("M,N,K", [(70, 400, 8336), (700, 1424, 400), (700, 1440, 8336), (1100, 1040, 400), (2100, 1040, 8336), (2100, 1936, 400),
                                   (2100, 2064, 272), (4200, 1040, 8336), (8201, 1040, 144), (33000, 272, 16)])
def test_gated_variants(fp8, M, N, K, scale):
    """Both sides of the borders at one strip of 32, 64 and of 128 rows per compute unit, several tiles per
    workgroup, more than 64 K blocks."""
    test_gated_exact_products(fp8, M, N, K, scale)


@pytest.mark.parametrize("M,N", [(70, 272), (1100, 1040), (2100, 1040), (4200, 1040)])
def test_gated_infinite_products(fp8, M, N):
    """A product past f32's range has a NaN code and does not count towards its block's scale; huge finite
    ones do, and a gate of -2^64 closes to -0."""
    K = 272
    a, w0, w1 = np.zeros((M, K)), np.zeros((N, K)), np.zeros((N, K))
    a[1::2, 0], a[:, 200] = 1, 1
    n = np.arange(N)
    w0[n % 4 == 0, 0] = w1[n % 4 == 0, 0] = 1       # 2^64 * 2^64
    w0[n % 4 == 1, 200], w1[n % 4 == 1, 200] = 2, 1.5
    w0[n % 4 == 2, 200], w1[n % 4 == 2, 0] = 1, 1   # gelu(1) 2^64
    w0[n % 4 == 3, 0], w1[n % 4 == 3, 0] = -1, 1
    w0[128:256], w1[128:256] = 0, 0                 # a block with one finite value
    w0[130, 200] = w1[130, 200] = w0[140, 0] = w1[140, 0] = 1
    bytes_ = np.full((_blocks(K), M), 127)
    bytes_[0] += 64
    ac, asc = _operand(a, bytes_, M, K)
    w = [torch.from_numpy(_round_e4m3(v)).to(DEV) for v in (w0, w1)]
    unit = _unit_scales(N, K, False)
    x = a.copy()
    x[:, 0] *= 2.0 ** 64
    gate, up = torch.from_numpy(x @ w0.T), x @ w1.T
    with np.errstate(over="ignore"):
        y = (_gelu(gate).numpy() * up).astype(np.float32).astype(np.float64)
    assert np.isinf(y[1, 0]) and np.isfinite(y[0]).all()
    codes, s = _gated(fp8, ac, asc, w[0], unit, w[1], unit, E8M0)
    _check_codes(codes, s, y, GELU_REL)


@pytest.mark.parametrize("M", [5, 40, 600])
def test_gated_rows_stand_alone(fp8, M):
    N, K = 272, 400
    a, sa, w0, s0, av, wv0 = _exact_case(M, N, K, E8M0, 5)
    _, _, w1, s1, _, wv1 = _exact_case(M, N, K, E8M0, 6)
    sa[:, :M] -= 8  # small gates
    base, bs = _gated(fp8, a, sa, w0, s0, w1, s1, E8M0)
    a[1, 399] = 0x7f
    sa[3, 3] = 255
    codes, s = _gated(fp8, a, sa, w0, s0, w1, s1, E8M0)
    assert ((codes[[1, 3]] & 0x7f) == 0x7f).all() and (s[:, [1, 3]] == 1).all()
    keep = [i for i in range(M) if i not in (1, 3)]
    assert np.array_equal(codes[keep], base[keep]) and np.array_equal(s[:, keep], bs[:, keep])


# ---- together --------------------------------------------------------------------------------

class _FeedForward:
    """x += wo(gelu(norm(x) wi0^T) * (norm(x) wi1^T)), as three calls and the next norm's addition."""

    def __init__(self, fp8, T, D=768, F=2048, seed=0, scale=E8M0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.f, self.T, self.D, self.F, self.scale = fp8, T, D, F, scale
        self.x = torch.randn(T, D, generator=g, device=DEV)
        self.gamma = [1 + 0.2 * torch.randn(D, generator=g, device=DEV) for _ in range(2)]
        self.raw = [torch.randn(n, k, generator=g, device=DEV) / k ** 0.5 for n, k in ((F, D), (F, D), (D, F))]
        self.w = []
        for w in self.raw:
            n, k = w.shape
            c = torch.empty(n, k, dtype=torch.uint8, device=DEV)
            s = torch.empty(_blocks(n), _blocks(k), dtype=torch.float32 if scale else torch.uint8, device=DEV)
            fp8.quantize_weights_device(w.data_ptr(), 0, n, k, scale, c.data_ptr(), s.data_ptr(), _stream())
            self.w.append((c, s))
        e = lambda *shape, t=torch.uint8: torch.empty(*shape, dtype=t, device=DEV)  # noqa: E731
        r = _rows16(T)
        self.c, self.cs, self.h, self.hs = e(T, D), e(_blocks(D), r), e(T, F), e(_blocks(F), r)
        self.d, self.y = e(T, D, t=torch.float16), e(T, D, t=torch.float32)

    def run(self, stream):
        p, f = (lambda t: t.data_ptr()), self.f
        (w0, s0), (w1, s1), (wo, so) = self.w
        f.rmsnorm_device(p(self.x), 0, 0, 0, self.T, self.D, p(self.gamma[0]), 1e-6, 0, p(self.c), p(self.cs), stream)
        f.gated_gelu_device(p(self.c), p(self.cs), self.T, p(w0), p(s0), p(w1), p(s1), self.F, self.D, self.scale,
                            p(self.h), p(self.hs), stream)
        f.matmul_device(p(self.h), p(self.hs), self.T, p(wo), p(so), self.D, self.F, self.scale, p(self.d), 1, stream)
        f.rmsnorm_device(p(self.x), 0, p(self.d), 1, self.T, self.D, p(self.gamma[1]), 1e-6, p(self.y), p(self.c),
                         p(self.cs), stream)

    def outputs(self):
        return [t.clone() for t in (self.c, self.cs[:, :self.T], self.d, self.y)]


@pytest.mark.parametrize("scale", [E8M0, F32S])
@pytest.mark.parametrize("T", [1, 33, 700, 2300])
def test_feed_forward_run(fp8, T, scale):
    """Three operand roundings of at most 2^-4 / sqrt(3) = 0.036 rms a factor: gate and up 0.051 each,
    their product 0.072, its codes 0.036, wo 0.036: 0.089 of the block's output in the 2-norm."""
    ff = _FeedForward(fp8, T, seed=T, scale=scale)
    ff.run(_stream())
    x = ff.x.double()
    n = x / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-6) * ff.gamma[0].double()
    w = [t.double() for t in ff.raw]
    d = (_gelu(n @ w[0].t()) * (n @ w[1].t())) @ w[2].t()
    assert float((ff.d.double() - d).norm() / d.norm()) <= 0.089
    assert torch.equal(ff.y, ff.x + ff.d.float())
    h = ff.y.double()
    y = (h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6) * ff.gamma[1].double()).cpu().numpy()
    _check_codes(ff.c.cpu().numpy(), ff.cs[:, :T].cpu().numpy(), y, NORM_REL)


def test_graph_replays_equal_eager(fp8):
    for T in (3, 40, 900):
        ff = _FeedForward(fp8, T, seed=T)
        ff.run(_stream())
        torch.cuda.synchronize()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=side):
            ff.run(torch.cuda.current_stream().cuda_stream)
        for i in range(4):
            ff.x.copy_(torch.randn(T, 768, generator=torch.Generator(device=DEV).manual_seed(i), device=DEV))
            ff.run(_stream())
            want = ff.outputs()
            for t in (ff.c, ff.h, ff.d, ff.y):
                t.zero_()
            graph.replay()
            torch.cuda.synchronize()
            for got, ref in zip(ff.outputs(), want):
                assert torch.equal(got.view(torch.uint8), ref.view(torch.uint8)), (T, i)


def test_two_streams_at_once(fp8):
    runs = [_FeedForward(fp8, T, seed=T) for T in (50, 1100)]
    want = []
    for ff in runs:
        ff.run(_stream())
        torch.cuda.synchronize()
        want.append(ff.outputs())
    streams = [torch.cuda.Stream() for _ in runs]
    for _ in range(5):
        for ff, s in zip(runs, streams):
            ff.run(s.cuda_stream)
    torch.cuda.synchronize()
    for ff, ref in zip(runs, want):
        for got, r in zip(ff.outputs(), ref):
            assert torch.equal(got.view(torch.uint8), r.view(torch.uint8))


def test_host_forms(fp8):
    """The numpy entry points give the device forms' results."""
    r = np.random.default_rng(8)
    x, g = r.standard_normal((37, 400)).astype(np.float32), (1 + 0.1 * r.standard_normal(400)).astype(np.float32)
    delta = r.standard_normal((37, 400)).astype(np.float16)
    codes, scales, total = fp8.rmsnorm(x, g, 1e-6, delta)
    assert np.array_equal(total, x + delta.astype(np.float32)) and not scales[:, 37:].any()
    h = total.astype(np.float64)
    _check_codes(codes, scales[:, :37], h / np.sqrt((h * h).mean(1, keepdims=True) + 1e-6) * g, NORM_REL)
    alone = fp8.rmsnorm(x.astype(np.float16), g)
    assert len(alone) == 2 and alone[0].shape == (37, 400)
    q, s = fp8.quantize(x)
    w = [r.standard_normal((272, 400)).astype(np.float32) / 20 for _ in range(2)]
    for st in (E8M0, F32S):
        w0, w1 = (fp8.quantize_weights(v, st) for v in w)
        wv = [TABLE[c] * np.repeat(np.repeat(sc if st else 2.0 ** (sc - 127.0), 128, 0)[:272], 128, 1)[:, :400]
              for c, sc in (w0, w1)]
        av = TABLE[q] * np.repeat(2.0 ** (s[:, :37].T - 127.0), 128, 1)[:, :400]
        want, size = av @ wv[0].T, np.abs(av) @ np.abs(wv[0]).T
        assert (np.abs(fp8.matmul((q, s), w0) - want) <= 416 * 2.0 ** -23 * size).all()
        half = fp8.matmul((q, s), w0, dtype=np.float16)
        assert half.dtype == np.float16 and np.linalg.norm(half - want) <= 2.0 ** -9 * np.linalg.norm(want)
        gc, gs = fp8.gated_gelu((q, s), w0, w1)
        y = _gelu(torch.from_numpy(want)).numpy() * (av @ wv[1].T)
        got = TABLE[gc] * np.repeat(2.0 ** (gs[:, :37].T - 127.0), 128, 1)[:, :272]
        assert np.linalg.norm(got - y) <= 2.0 ** -4 / 3 ** 0.5 * np.linalg.norm(y)
