"""What the fp8 matrix instructions keep of a sum, for 16-bit results and the gated product.

They align the products of eight consecutive K to the largest of the eight and keep 2^-13 of it; sums of
groups are f32.  The kept bit itself is tested, in a sum whose large part another block cancels, and the
size of the errors on ordinary data, for every kernel that forms them.

Errors behind a rounding.  Let R round to a grid and s be a sum whose place between two grid points is
uniform.  Then E|R(s + e) - R(s)| = |e|: with a step h, the chance of another grid point is |e| / h, and it
is h away.  So the sum of |result - R(definition)| over many results is that of the errors before the
rounding, which no single result shows.

Those errors.  In a group whose largest product lies in [2^x, 2^(x+1)) a product loses at most what is below
q = 2^(x-13): |a w| mod q, nothing for most of them, as a product of two codes has eight bits.  Products have
either sign, so E|e| is at most the root of the losses' squares (and some 0.8 of it for many of one size).
One bit less kept doubles q and brings further products under it.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_fp8 import (DEV, E8M0, F32S, TABLE, TYPES, _blocks, _gated, _gelu, _matmul, _operand, _ordinary,  # noqa: E402
                          _ordinary_weights, _round_e4m3, _unit_scales, fp8)  # noqa: F401

# One size at least for every kernel of 16-bit results, and of the gated product.
PRODUCTS = [(16, 2304), (32, 2304), (300, 2304), (1000, 1152), (1000, 2304), (3000, 2304), (4616, 2048), (6500, 2304)]
GATED = [(32, 2048), (700, 1440), (1900, 2048), (2100, 2048)]
PLACES = [(0, 7), (7, 0), (13, 8), (69, 66), (120, 127)]  # of a large and a small product, in one group of eight


def _group_case(M, N, large, small):
    """Rows of 256 * 256 + a * 4 in one group, and a block of -256 * 256: sums a * 4, a multiple of 2^-13 2^16."""
    K = 256
    a, w = np.zeros((M, K)), np.zeros((N, K))
    a[:, large], w[:, large] = 256, 256
    a[:, small], w[:, small] = np.resize([2.0, -2.0, 4.0, 0.0, 8.0], M), np.where(np.arange(N) % 2, 4.0, -4.0)
    a[:, 128 + small], w[:, 128 + small] = 256, -256
    return _operand(a, np.full((2, M), 127), M, K), torch.from_numpy(_round_e4m3(w)).to(DEV), np.outer(a[:, small], w[:, small])


@pytest.mark.parametrize("M,N", PRODUCTS)
def test_products_keep_2_13th_of_a_group(fp8, M, N):
    for large, small in PLACES:
        (a, sa), w, want = _group_case(M, N, large, small)
        for scale in (E8M0, F32S):
            sw = _unit_scales(N, 256, False) if scale == E8M0 else torch.ones(_blocks(N), 2, device=DEV)
            for kind in TYPES:
                got = _matmul(fp8, a, sa, w, sw, N, kind, scale)
                assert torch.equal(got.cpu().double(), torch.from_numpy(want)), (large, small, kind, scale)


@pytest.mark.parametrize("M,N", GATED)
def test_gated_product_keeps_2_13th_of_a_group(fp8, M, N):
    """gelu(x) = x to 2^-24 for x = 8 and above, and 0 for -8 and below: codes of x^2 or of (next to) 0."""
    for large, small in PLACES:
        (a, sa), w, want = _group_case(M, N, large, small)
        for scale in (E8M0, F32S):
            sw = _unit_scales(N, 256, False) if scale == E8M0 else torch.ones(_blocks(N), 2, device=DEV)
            codes, s = _gated(fp8, a, sa, w, sw, w, sw, scale)
            got = TABLE[codes] * np.repeat(2.0 ** (s.T - 127.0), 128, 1)[:, :N]
            assert np.array_equal(got, np.where(want > 0, want * want, 0.0)), (large, small, scale)


def _mean_square(a, sa, w, sw):
    """Per result, the bound on the errors' mean square, from codes and scales [row][block]: what groups of eight lose,
    and f32 sums of groups and blocks, whose parts are of the whole's size (values of either sign)."""
    table = torch.from_numpy(TABLE).float().to(DEV)
    a, w = table[a.long()], table[w.long()].t().contiguous()
    (M, K), N = a.shape, w.shape[1]
    out = torch.zeros(M, N, dtype=torch.float64, device=DEV)
    for m in range(M):
        p = (a[m][:, None] * w).abs().view(K // 8, 8, N)
        q = torch.exp2(torch.floor(torch.log2(p.amax(1, keepdim=True).clamp(min=2.0 ** -30))) - 13)
        lost, size = torch.fmod(p, q).square().sum(1).double(), p.square().sum(1).double()
        lost += size * (K / 8 + K / 128 + 16) * 2.0 ** -48
        for b in range(_blocks(K)):
            out[m] += lost[16 * b:16 * b + 16].sum(0) * (sa[m, b] * sw[:, b]).square()
    return out


def _floats(scales, rows):
    """Weights' scales by row, [N][block]."""
    s = scales.double() if scales.dtype == torch.float32 else torch.exp2(scales.double() - 127)
    return s.repeat_interleave(128, 0)[:rows]


def _some_rows(M):
    return torch.arange(0, M, max(1, M // 60), device=DEV)


@pytest.mark.parametrize("scale", [E8M0, F32S])
@pytest.mark.parametrize("M,N", PRODUCTS)
def test_product_errors(fp8, M, N, scale):
    K = 784
    a, sa, w, sw, av, wv = _ordinary(fp8, M, N, K, scale, M + N)
    rows = _some_rows(M)
    want = av[rows] @ wv.t()
    bound = _mean_square(a[rows], torch.exp2(sa.t()[rows].double() - 127), w, _floats(sw, N)).sqrt()
    for kind in ("f16", "bf16"):
        got = _matmul(fp8, a, sa, w, sw, N, kind, scale)[rows].double()
        err = (got - want.to(TYPES[kind][1]).double()).abs().sum()
        assert float(err) <= float(bound.sum()), (kind, float(err / bound.sum()))


@pytest.mark.parametrize("scale", [E8M0, F32S])
@pytest.mark.parametrize("M,N", GATED)
def test_gated_product_errors(fp8, M, N, scale):
    """Codes are the grid here, with the definition's own scales; the gelu adds at most 2^-20 of |gelu u| (its
    exponent's rounding, times an argument of a few units).  A block's scale is a neighbour's where its maximum lies
    within the error of a border: for maxima spread evenly over a binade's logarithm, |e| / (maximum ln 2)."""
    K = 784
    a, sa, w0, s0, av, wv0 = _ordinary(fp8, M, N, K, scale, M + N)
    w1, s1, wv1 = _ordinary_weights(fp8, N, K, scale, torch.Generator(device=DEV).manual_seed(M))
    rows = torch.arange(0, M, max(1, M // 500), device=DEV)
    g, u = av[rows] @ wv0.t(), av[rows] @ wv1.t()
    y = _gelu(g) * u
    slope = 1.13 * u.abs()
    act = a[rows], torch.exp2(sa.t()[rows].double() - 127)
    eg, eu = _mean_square(*act, w0, _floats(s0, N)), _mean_square(*act, w1, _floats(s1, N))
    sd = (eg * slope.square() + eu * _gelu(g).square()).sqrt() + y.abs() * 2.0 ** -20
    codes, s = _gated(fp8, a, sa, w0, s0, w1, s1, scale)
    keep = rows.cpu().numpy()
    codes, s = torch.from_numpy(codes[keep]).to(DEV), torch.from_numpy(s[:, keep].copy()).to(DEV)
    table = torch.from_numpy(TABLE).to(DEV)
    error = allowed = neighbours = expected = 0.0
    for b in range(_blocks(N)):
        part = slice(128 * b, min(N, 128 * b + 128))
        top, at = y[:, part].abs().max(1)
        step = torch.exp2(torch.ceil(torch.log2(top / 448)))
        neighbours += int((torch.exp2(s[b].double() - 127) != step).sum())
        expected += float((sd[:, part].gather(1, at[:, None])[:, 0] / (top * np.log(2))).sum())
        same = torch.exp2(s[b].double() - 127) == step
        ref = table[torch.from_numpy(_round_e4m3((y[:, part] / step[:, None]).cpu().numpy())).to(DEV).long()] * step[:, None]
        got = table[codes[:, part].long()] * step[:, None]
        error += float((got - ref).abs()[same].sum())
        allowed += float(sd[:, part][same].sum())
    assert error <= allowed, error / allowed
    assert neighbours <= 4 + 3 * expected, (neighbours, expected)
