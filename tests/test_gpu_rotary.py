"""Head norms and rotation on the GPU against the definition in 64 bits.

Tolerances.  Sums of squares: at most 16 terms in a lane and 6 additions across lanes, each off by half a step
of f32 (2^-24), half of which reaches the inverse root; the root and the products with it and gamma are off by at
most 5 more half steps.  Sines and cosines are within 2^-23: their argument's rounding, the series' end (3e-8) and
the last rounding.  So a turned value a c - b s is within (|a| + |b|) 20 2^-24 of the definition's, plus half a
step of the output's type.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DEV = "cuda:0"
TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (2, torch.bfloat16)}
LEAST = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half the smallest subnormal
HALVES, NEIGHBOURS = 0, 1


@pytest.fixture(scope="module")
def rotary():
    from witchcraft_amd import rotary
    return rotary


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _turns(freqs, axis, pos):
    """Cosines and sines [rows][pairs] of position * frequency, f64 (positions of axes that are not there: 0)."""
    pos = torch.cat([pos, torch.zeros(8 - pos.shape[0], pos.shape[1], dtype=pos.dtype, device=pos.device)])
    t = pos[torch.tensor(list(axis), device=pos.device, dtype=torch.long)].double().t() * torch.tensor(list(freqs), dtype=torch.float64, device=pos.device)
    return torch.cos(t)[:, None], torch.sin(t)[:, None]


def _want(x, gamma, eps, freqs, axis, pos, pairing):
    """The definition, and |a| + |b| of what each value was made from."""
    y = x.double()
    if gamma is not None:
        y = y / torch.sqrt((y * y).mean(2, keepdim=True) + eps) * gamma.double()
    size = y.abs()
    r = 2 * len(freqs)
    if r:
        c, s = _turns(freqs, axis, pos)
        first = torch.arange(r // 2, device=x.device) * (1 if pairing == HALVES else 2)
        second = first + (r // 2 if pairing == HALVES else 1)
        a, b = y[:, :, first], y[:, :, second]
        y, size = y.clone(), size.clone()
        y[:, :, first], y[:, :, second] = a * c - b * s, b * c + a * s
        size[:, :, first] = size[:, :, second] = a.abs() + b.abs()
    return y, size


def _check(got, want, size, kind):
    tol = size * 20 * 2.0 ** -24 + want.abs() * (torch.finfo(got.dtype).eps / 2) * 1.001 + LEAST[kind]
    off = (got.double() - want).abs() - tol
    assert bool((off <= 0).all()), (kind, float(off.max()), int((off > 0).sum()))


class Rows:
    """q and k as columns of one projection's rows, with values behind them and rows behind the last."""

    def __init__(self, T, qh, kh, D, dtype, seed, gap=16, scale=2.0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.T, self.qh, self.kh, self.D = T, qh, kh, D
        self.ld = (qh + kh) * D + gap
        self.all = (scale * torch.randn(T + 2, self.ld, generator=g, device=DEV)).to(dtype)
        self.at = self.all.data_ptr()
        self.at_k = self.at + qh * D * self.all.element_size()

    def parts(self):
        x = self.all[:self.T]
        return (x[:, :self.qh * self.D].reshape(self.T, self.qh, self.D),
                x[:, self.qh * self.D:(self.qh + self.kh) * self.D].reshape(self.T, self.kh, self.D))


def _run(rotary, r, code, qg, kg, eps, tab, rot, pairing, pos, out=None):
    """In place, or into `out`."""
    o = out or r
    rotary.rotate_device(r.at, r.ld, r.qh, r.at_k, r.ld, r.kh, code, r.T, r.D, 0 if qg is None else qg.data_ptr(),
                         0 if kg is None else kg.data_ptr(), eps, tab.data_ptr(), rot, pairing, pos.data_ptr(), pos.shape[0],
                         o.at, o.ld, o.at_k, o.ld, _stream())


def _case(rotary, kind, T, qh, kh, D, rot, pairing, axes, norm, in_place, seed=0, far=100):
    code, dt = TYPES[kind]
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    freqs = list(10000.0 ** (-np.arange(rot // 2) / max(1, rot // 2)))
    axis = [i * axes // max(1, rot // 2) for i in range(rot // 2)]
    tab = torch.from_numpy(rotary.table(freqs, axis).view(np.int64)).to(DEV)
    pos = torch.randint(-far, far, (axes, T), generator=g, device=DEV, dtype=torch.int32)
    qg = 1 + 0.3 * torch.randn(D, generator=g, device=DEV) if norm in ("both", "q") else None
    kg = 1 + 0.3 * torch.randn(D, generator=g, device=DEV) if norm in ("both", "k") else None
    r = Rows(T, qh, kh, D, dt, seed)
    out = None if in_place else Rows(T, qh, kh, D, dt, seed + 7, gap=32)
    before, o = r.all.clone(), out or r
    was = o.all.clone()
    q, k = (x.clone() for x in r.parts())
    print(f"[rotary] {kind} T={T} heads={qh}+{kh} D={D} rot={rot} pairing={pairing} axes={axes} norm={norm}", flush=True)
    _run(rotary, r, code, qg, kg, 1e-6, tab, rot, pairing, pos, out)
    torch.cuda.synchronize()
    for got, x, gamma in zip(o.parts(), (q, k), (qg, kg)):
        if x.shape[1]:
            _check(got, *_want(x, gamma, 1e-6, freqs, axis, pos, pairing), kind)
    # columns behind q and k, rows behind the last, and inputs that are no outputs: as they were
    w = (qh + kh) * D
    bits = lambda x: x.contiguous().view(torch.uint8)  # noqa: E731
    assert torch.equal(bits(o.all[:, w:]), bits(was[:, w:])) and torch.equal(bits(o.all[T:]), bits(was[T:]))
    assert in_place or torch.equal(bits(r.all), bits(before))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pairing", [HALVES, NEIGHBOURS])
@pytest.mark.parametrize("D,rot", [(8, 8), (8, 0), (16, 8), (24, 16), (32, 32), (40, 24), (64, 64), (64, 32), (72, 72), (80, 80),
                                   (96, 48), (104, 104), (128, 128), (128, 64), (136, 16), (160, 160), (256, 256), (264, 256), (512, 512),
                                   (512, 8)])
def test_head_sizes(rotary, kind, pairing, D, rot):
    _case(rotary, kind, 5, 3, 2, D, rot, pairing, 1, "both", False, seed=D + rot)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("norm", ["none", "q", "k", "both"])
@pytest.mark.parametrize("axes", [1, 2, 3, 8])
@pytest.mark.parametrize("in_place", [False, True])
def test_norms_and_axes(rotary, kind, norm, axes, in_place):
    _case(rotary, kind, 19, 4, 2, 64, 64, HALVES, axes, norm, in_place, seed=axes)


@pytest.mark.parametrize("T,qh,kh,D", [(1, 1, 0, 64), (1, 0, 1, 64), (1, 32, 8, 128), (1, 300, 7, 64), (2, 1, 1, 8), (3, 65, 64, 512),
                                       (17, 12, 12, 64), (33, 7, 1, 80), (255, 1, 1, 256), (700, 12, 12, 64), (1025, 5, 3, 128),
                                       (4616, 12, 12, 64), (9001, 1, 1, 32), (2500, 64, 8, 128), (20000, 3, 0, 16)])
@pytest.mark.parametrize("kind,pairing", [("f32", NEIGHBOURS), ("f16", HALVES), ("bf16", NEIGHBOURS)])
def test_rows_and_heads(rotary, kind, pairing, T, qh, kh, D):
    """From one token to more rows than a round of workgroups takes; more heads than a workgroup's."""
    _case(rotary, kind, T, qh, kh, D, D, pairing, 2, "both", T % 2 == 0, seed=T)


def test_most_heads(rotary):
    _case(rotary, "bf16", 2, 65535, 65535, 8, 8, HALVES, 1, "both", True)


@pytest.mark.parametrize("at", [0, 1, 4095, 1 << 20, (1 << 24) + 1, 2 ** 31 - 1, -2 ** 31, -1])
def test_far_positions(rotary, at):
    """Angles in 64 bits lose at most half a step of theirs, 2^-22 at 2^31 radians: compared with the table's own
    turns, in whole numbers, which lose nothing."""
    D, freqs = 128, [1.0, 0.7071, 3.1, 1e-3] + list(1e6 ** (-np.arange(60) / 60))
    table = rotary.table(freqs)
    tab = torch.from_numpy(table.view(np.int64)).to(DEV)
    r = Rows(3, 2, 1, D, torch.float32, 5)
    q, k = (x.clone() for x in r.parts())
    pos = torch.full((1, 3), at, dtype=torch.int32, device=DEV)
    _run(rotary, r, 0, None, None, 1e-6, tab, D, HALVES, pos)
    # the turn's fraction as an exact integer, then as an angle in one turn
    angle = [((int(e) >> 3) * at % (1 << 61)) / 2.0 ** 61 * 2 * np.pi for e in table.tolist()]
    one = torch.ones((1, 3), dtype=torch.int32, device=DEV)
    for got, x in zip(r.parts(), (q, k)):
        _check(got, *_want(x, None, 0, angle, [0] * 64, one, HALVES), "f32")
    if abs(at) <= 1 << 24:
        for got, x in zip(r.parts(), (q, k)):
            _check(got, *_want(x, None, 0, freqs, [0] * 64, pos, HALVES), "f32")


def test_every_quarter(rotary):
    """Angles all around the circle, on and beside the borders between the series."""
    n = 4096
    freqs = [2 * np.pi / 1024] * 4
    pos = torch.arange(n, dtype=torch.int32, device=DEV)[None] - n // 2
    tab = torch.from_numpy(rotary.table(freqs).view(np.int64)).to(DEV)
    r = Rows(n, 1, 1, 8, torch.float32, 3)
    q, k = (x.clone() for x in r.parts())
    _run(rotary, r, 0, None, None, 0.0, tab, 8, NEIGHBOURS, pos)
    for got, x in zip(r.parts(), (q, k)):
        _check(got, *_want(x, None, 0, freqs, [0] * 4, pos, NEIGHBOURS), "f32")


def test_axes_that_are_not_there(rotary):
    """Pairs of an axis past the positions' are not turned."""
    freqs, axis = [0.5] * 32, [0, 1, 2, 7] * 8
    tab = torch.from_numpy(rotary.table(freqs, axis).view(np.int64)).to(DEV)
    r = Rows(9, 2, 2, 64, torch.float16, 3)
    q, k = (x.clone() for x in r.parts())
    pos = torch.arange(18, dtype=torch.int32, device=DEV).view(2, 9)
    _run(rotary, r, 1, None, None, 0.0, tab, 64, HALVES, pos)
    for got, x in zip(r.parts(), (q, k)):
        _check(got, *_want(x, None, 0, freqs, axis, pos, HALVES), "f16")
        still = [i + h for i in range(32) if axis[i] > 1 for h in (0, 32)]
        assert torch.equal(got[:, :, still], x[:, :, still])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_special_values(rotary, kind):
    """Heads of zeros, tiny, large, infinite and NaN values: only their own head is touched by them."""
    code, dt = TYPES[kind]
    D, freqs = 64, list(10000.0 ** (-np.arange(32) / 32))
    tab = torch.from_numpy(rotary.table(freqs).view(np.int64)).to(DEV)
    r = Rows(6, 2, 1, D, dt, 11)
    q, k = r.parts()
    r.all[0, :D] = 0
    r.all[1, :D] *= 2.0 ** -12
    r.all[2, :D] *= 2.0 ** 12
    r.all[3, 5] = float("nan")
    r.all[4, 7] = float("inf")
    q, k = (x.clone() for x in r.parts())
    g = torch.ones(D, device=DEV)
    pos = torch.arange(6, dtype=torch.int32, device=DEV)[None]
    _run(rotary, r, code, g, g, 1e-6, tab, D, HALVES, pos)
    got_q, got_k = r.parts()
    want, size = _want(q, g, 1e-6, freqs, [0] * 32, pos, HALVES)
    ok = torch.ones(6, 2, dtype=torch.bool, device=DEV)
    ok[3, 0] = ok[4, 0] = False
    _check(got_q[ok], want[ok], size[ok], kind)
    assert bool((got_q[0, 0] == 0).all())
    assert bool(got_q[3, 0].isnan().all())               # NaN in the sum of squares
    assert bool((got_q[4, 0].isnan() | (got_q[4, 0] == 0)).all()) and bool(got_q[4, 0, [7, 39]].isnan().all())  # 1 / inf
    _check(got_k, *_want(k, g, 1e-6, freqs, [0] * 32, pos, HALVES), kind)
    # without a norm an infinity reaches its own pair only
    r = Rows(2, 1, 1, D, dt, 12)
    r.all[0, 7] = float("inf")
    q, _ = (x.clone() for x in r.parts())
    _run(rotary, r, code, None, None, 0.0, tab, D, HALVES, pos[:, :2])
    got, _ = r.parts()
    bad = ~got[0, 0].isfinite()
    assert bad.nonzero().flatten().tolist() in ([7, 39], [7])  # inf sin(0) is NaN, cos(0) inf is inf


def test_gammas_and_eps(rotary):
    """Gammas on 4-byte boundaries, negative and zero ones; an eps of zero; a head of zeros with it is NaN, as 0 / 0."""
    D, freqs = 32, [0.3] * 16
    tab = torch.from_numpy(rotary.table(freqs).view(np.int64)).to(DEV)
    g = torch.linspace(-2, 2, D + 3, device=DEV)
    g[9] = 0
    pos = torch.arange(7, dtype=torch.int32, device=DEV)[None]
    for eps in (0.0, 0.5):
        r = Rows(7, 3, 1, D, torch.bfloat16, 2)
        r.all[3, :D] = 0
        q, k = (x.clone() for x in r.parts())
        _run(rotary, r, 2, g[1:D + 1], g[3:], eps, tab, D, HALVES, pos)
        got_q, got_k = r.parts()
        want, size = _want(q, g[1:D + 1], eps, freqs, [0] * 16, pos, HALVES)
        if eps == 0:
            assert bool(got_q[3, 0].isnan().all())
            got_q, want, size = (torch.cat([x[:3], x[4:]]) for x in (got_q, want, size))
        _check(got_q, want, size, "bf16")
        _check(got_k, *_want(k, g[3:], eps, freqs, [0] * 16, pos, HALVES), "bf16")


def test_rows_past_32_bits(rotary):
    """Rows whose bytes and values lie past 2^32."""
    D, T, ld = 64, 5, 1 << 30
    freqs = [0.3] * 32
    tab = torch.from_numpy(rotary.table(freqs).view(np.int64)).to(DEV)
    x = torch.empty((T - 1) * ld + 2 * D, dtype=torch.float16, device=DEV)
    q = torch.randn(T, 1, D, device=DEV).half()
    k = torch.randn(T, 1, D, device=DEV).half()
    for t in range(T):
        x[t * ld:t * ld + D], x[t * ld + D:t * ld + 2 * D] = q[t, 0], k[t, 0]
    pos = torch.arange(T, dtype=torch.int32, device=DEV)[None]
    rotary.rotate_device(x.data_ptr(), ld, 1, x.data_ptr() + 2 * D, ld, 1, 1, T, D, 0, 0, 0.0, tab.data_ptr(), D, HALVES,
                         pos.data_ptr(), 1, x.data_ptr(), ld, x.data_ptr() + 2 * D, ld, _stream())
    for at, was in ((0, q), (D, k)):
        got = torch.stack([x[t * ld + at:t * ld + at + D] for t in range(T)])[:, None]
        _check(got, *_want(was, None, 0, freqs, [0] * 32, pos, HALVES), "f16")


def test_host_form(rotary):
    rng = np.random.default_rng(4)
    freqs, axis = rotary.frequencies(48, 1e5), [0] * 8 + [1] * 16
    for dt, kind in ((np.float32, "f32"), (np.float16, "f16")):
        q, k = rng.standard_normal((11, 4, 64)).astype(dt), rng.standard_normal((11, 2, 64)).astype(dt)
        pos, g = rng.integers(-50, 5000, (2, 11)), rng.standard_normal(64).astype(np.float32)
        got = rotary.rotate(q, k, pos, rotary.table(freqs, axis), q_gamma=g, pairing=NEIGHBOURS)
        for o, x, gamma in zip(got, (q, k), (torch.from_numpy(g), None)):
            _check(torch.from_numpy(o), *_want(torch.from_numpy(x), gamma, 1e-6, freqs, axis, torch.from_numpy(pos), NEIGHBOURS), kind)
    q = rng.standard_normal((3, 2, 16)).astype(np.float32)
    none = rotary.table([])
    a, b = rotary.rotate(q, q[:, :0], np.zeros(3, np.int32), none)
    assert np.array_equal(a, q) and b.shape == (3, 0, 16)


def test_graph_replays_equal_eager(rotary):
    r, out = Rows(300, 12, 4, 64, torch.bfloat16, 1), Rows(300, 12, 4, 64, torch.bfloat16, 2)
    g = torch.ones(64, device=DEV)
    tab = torch.from_numpy(rotary.table(rotary.frequencies(64)).view(np.int64)).to(DEV)
    pos = torch.arange(300, dtype=torch.int32, device=DEV)[None].contiguous()
    args = (2, g, g, 1e-6, tab, 64, HALVES, pos, out)
    _run(rotary, r, *args)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        _run(rotary, r, *args)
    for i in range(4):
        r.all.copy_(torch.randn(r.all.shape, device=DEV))
        pos.add_(i)
        _run(rotary, r, *args)
        want = out.all.clone()
        out.all.zero_()
        graph.replay()
        torch.cuda.synchronize()
        w = 16 * 64
        assert torch.equal(out.all[:300, :w], want[:300, :w])


def test_streams_at_once(rotary):
    streams = [torch.cuda.Stream() for _ in range(3)]
    tab = torch.from_numpy(rotary.table(rotary.frequencies(128)).view(np.int64)).to(DEV)
    pos = torch.arange(900, dtype=torch.int32, device=DEV)[None].contiguous()
    g = torch.ones(128, device=DEV)
    sets = [(Rows(900, 8, 2, 128, torch.float16, s), Rows(900, 8, 2, 128, torch.float16, 9)) for s in range(3)]
    want = []
    for r, o in sets:
        _run(rotary, r, 1, g, g, 1e-6, tab, 128, HALVES, pos, o)
        want.append(o.all.clone())
        o.all.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for s, (r, o) in zip(streams, sets):
            with torch.cuda.stream(s):
                _run(rotary, r, 1, g, g, 1e-6, tab, 128, HALVES, pos, o)
    torch.cuda.synchronize()
    for (r, o), w in zip(sets, want):
        assert torch.equal(o.all[:900, :1280], w[:900, :1280])
