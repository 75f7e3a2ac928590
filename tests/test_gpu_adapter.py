"""Low-rank adapters on the GPU against the definition in 64 bits.

Whole numbers: small ones in x, A and B make every sum a whole number below 2^24, and the inner products have at
most 16 bits, so results are exact before their one rounding and are compared bit for bit; that holds every part
of every kernel.  Other values: sums of n terms in f32 are within n 2^-23 of the sum of their magnitudes (a step
of f32 an addition, as matrix units may cut), the parts that the inner product is taken in within 2^-16 of it (two
parts, 16-bit results; three hold all of it), and the results' rounding within half a step of their type.

Two parts: h in 2^e .. 2^(e + 1).  The first keeps bf16's 8 bits and leaves less than 2^(e - 7), exactly; the second
rounds that to 8 bits, whose step there is at most 2^(e - 8 - 7): off by at most half of it, 2^(e - 16).
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DEV = "cuda:0"
CODE = {"f32": 0, "f16": 1, "bf16": 2, "e4m3": 3}
TYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def adapters():
    from witchcraft_amd import adapters
    return adapters


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _bits(x):
    return x.contiguous().view(torch.uint8)


class Case:
    """Inputs with gaps between rows, and values around the outputs that have to stay."""

    def __init__(self, T, K, cols, R, G, x="f16", w="f16", y="f16", seed=0, whole=True, ids=None, ranks=None, scales=True, gap=16):
        self.T, self.K, self.cols, self.R, self.G, self.S, self.N = T, K, tuple(cols), R, G, len(cols), sum(cols)
        self.kx, self.kw, self.ky = x, w, y
        g = torch.Generator(device=DEV).manual_seed(seed)
        h = torch.Generator().manual_seed(seed)

        def values(*shape, top):
            if whole:
                return torch.randint(-top, top + 1, shape, generator=g, device=DEV).float()
            return torch.randn(*shape, generator=g, device=DEV)
        v = values(T, K, top=2)
        self.xs = None
        if x == "e4m3":
            blocks, m16 = (K + 127) // 128, (T + 15) // 16 * 16
            byte = torch.randint(126, 129, (blocks, m16), generator=g, device=DEV) if whole else torch.randint(120, 131, (blocks, m16), generator=g, device=DEV)
            if whole:
                v = v * 2  # times 1/2, 1 or 2
            self.x = torch.zeros(T, K + gap, dtype=torch.uint8, device=DEV)
            self.x[:, :K] = v.to(torch.float8_e4m3fn).view(torch.uint8)
            self.xs = byte.to(torch.uint8)
            scale = torch.exp2(byte[:, :T].t().double() - 127).repeat_interleave(128, 1)[:, :K]
            self.xv = self.x[:, :K].contiguous().view(torch.float8_e4m3fn).double() * scale
        else:
            self.x = torch.zeros(T, K + gap, dtype=TYPE[x], device=DEV)
            self.x[:, :K] = v.to(TYPE[x])
            self.xv = self.x[:, :K].double()
        self.a, self.b = values(G, self.S, R, K, top=1).to(TYPE[w]), values(G, self.N, R, top=3).to(TYPE[w])
        if not whole:
            self.a, self.b = self.a / K ** 0.5, self.b / R ** 0.5
        self.ranks = None
        if ranks is not None:
            self.ranks = torch.tensor(ranks, dtype=torch.int32, device=DEV)
            for i, n in enumerate(ranks):
                n = min(max(n, 0), R)
                self.a[i, :, n:], self.b[i, :, n:] = 0, 0
                up = (n + 7) // 8 * 8  # behind it anything may lie
                self.a[i, :, up:], self.b[i, :, up:] = float("nan"), float("nan")
        self.scales = torch.exp2(torch.randint(-1, 3, (G,), generator=h).float()).to(DEV) if scales else None
        self.ids = torch.randint(-1, G, (T,), generator=h, dtype=torch.int32) if ids is None else torch.as_tensor(ids, dtype=torch.int32)
        self.ids = self.ids.to(DEV)
        self.y = torch.zeros(T + 1, self.N + gap, dtype=TYPE[y], device=DEV)
        self.y.copy_(values(T + 1, self.N + gap, top=100))

    def run(self, adapters, out=None, work=None):
        """Into a buffer of its own, or in place with out = self.y."""
        from_ = self.y
        out = torch.full((self.T + 2, self.N + 32), 7.0, dtype=self.y.dtype, device=DEV) if out is None else out
        size = adapters.workspace_bytes(self.T, self.K, self.S, self.R)
        if work is None:  # of exactly the size, with NaN in it and a guard behind
            self.work = torch.full((size + 256,), 255, dtype=torch.uint8, device=DEV)
            work = self.work
        adapters.add_device(self.x.data_ptr(), CODE[self.kx], 0 if self.xs is None else self.xs.data_ptr(), self.x.stride(0), self.T,
                            self.K, self.ids.data_ptr(), self.G, self.a.data_ptr(), self.b.data_ptr(), CODE[self.kw],
                            0 if self.ranks is None else self.ranks.data_ptr(), 0 if self.scales is None else self.scales.data_ptr(),
                            self.R, self.cols, from_.data_ptr(), from_.stride(0), out.data_ptr(), out.stride(0), CODE[self.ky],
                            work.data_ptr(), size, _stream())
        return out

    def want(self):
        """The definition, and the tolerance of sums, ahead of the rounding."""
        out, tol = self.y[:self.T, :self.N].double(), torch.zeros(self.T, self.N, dtype=torch.float64, device=DEV)
        part = 2.0 ** -16 if self.ky != "f32" else 2.0 ** -22
        a, b = self.a.double().nan_to_num(0.0), self.b.double().nan_to_num(0.0)
        for g in sorted(set(self.ids.tolist())):
            if not 0 <= g < self.G:
                continue
            rows = (self.ids == g).nonzero()[:, 0]
            f = 1.0 if self.scales is None else float(self.scales[g])
            n0 = 0
            for s, n in enumerate(self.cols):
                x, aa, bb = self.xv[rows], a[g, s], b[g, n0:n0 + n]
                h = x @ aa.t()
                add = f * (h @ bb.t())
                out[rows, n0:n0 + n] += add
                far = (x.abs() @ aa.abs().t()) @ bb.abs().t()
                tol[rows, n0:n0 + n] = abs(f) * (far * (self.K + 3 * self.R + 16) * 2.0 ** -23 + (h.abs() @ bb.abs().t()) * part)
                n0 += n
        return out, tol

    def check(self, out, whole=True):
        got = out[:self.T, :self.N]
        want, tol = self.want()
        if whole:
            assert float(want.abs().max()) < 2 ** 24
            bad = got != want.to(got.dtype)
            assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist())
        else:
            # f32 sums of y and the addition, then the type's rounding
            tol = tol + want.abs() * (torch.finfo(got.dtype).eps / 2 + 2.0 ** -23) * 1.01
            off = (got.double() - want).abs() - tol
            assert bool((off <= 0).all()), (float(off.max()), int((off > 0).sum()))

    def around(self, out, was=7.0):
        """Columns and rows behind the output stay as they were, and so does what lies behind the workspace."""
        assert bool((out[self.T:] == was).all()) and bool((out[:self.T, self.N:] == was).all())
        assert bool((self.work[-256:] == 255).all())


def _go(adapters, *args, whole=True, **kw):
    print(f"[adapter] {args} {kw}", flush=True)
    c = Case(*args, whole=whole, **kw)
    out = c.run(adapters)
    torch.cuda.synchronize()
    c.check(out, whole)
    c.around(out)
    return c, out


ROWS = [1, 2, 15, 16, 17, 64, 100, 257, 300]


@pytest.mark.parametrize("T", ROWS)
@pytest.mark.parametrize("x,w,y", [("f16", "f16", "f16"), ("bf16", "bf16", "bf16"), ("e4m3", "f16", "f32"), ("e4m3", "bf16", "f32"),
                                   ("f16", "f16", "f32"), ("bf16", "bf16", "f16"), ("e4m3", "bf16", "bf16")])
def test_rows_and_types(adapters, T, x, w, y):
    _go(adapters, T, 272, (96,), 16, 5, x=x, w=w, y=y, seed=T)


@pytest.mark.parametrize("R", [8, 16, 24, 32, 40, 64, 104, 128])
@pytest.mark.parametrize("S", [1, 2, 3, 4])
@pytest.mark.parametrize("w,y", [("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f32")])
def test_ranks_and_slices(adapters, R, S, w, y):
    _go(adapters, 37, 144, (64, 16, 272, 48)[:S], R, 3, x="e4m3" if R % 16 else w, w=w, y=y, seed=R + S)


@pytest.mark.parametrize("K", [16, 32, 112, 128, 144, 768, 1040, 4096, 8208])
@pytest.mark.parametrize("x", ["f16", "e4m3"])
@pytest.mark.parametrize("T", [1, 40])
def test_depths(adapters, K, x, T):
    _go(adapters, T, K, (32,), 8, 2, x=x, y="f32", seed=K)


@pytest.mark.parametrize("cols", [(16,), (240,), (256,), (272,), (1040,), (16, 16, 16, 16), (768, 768, 768), (512, 128, 128), (2048, 16)])
@pytest.mark.parametrize("y", ["f16", "f32"])
def test_columns(adapters, cols, y):
    _go(adapters, 50, 64, cols, 16, 3, y=y, seed=len(cols))


@pytest.mark.parametrize("T", [3000, 5000, 16400, 66001, 70000])
@pytest.mark.parametrize("x,w,y", [("e4m3", "f16", "f16"), ("bf16", "bf16", "bf16"), ("f16", "f16", "f32"), ("e4m3", "bf16", "f32")])
@pytest.mark.parametrize("S,R", [(1, 16), (3, 16), (1, 32), (1, 64), (2, 40)])
def test_many_rows(adapters, T, x, w, y, S, R):
    """Every tile height and split, with requests of odd lengths and some without an adapter."""
    lengths = torch.randint(1, 400, (T,), generator=torch.Generator().manual_seed(T))
    ids = torch.randint(-1, 4, (T,), generator=torch.Generator().manual_seed(R)).repeat_interleave(lengths)[:T]
    _go(adapters, T, 144, (48,) * S, R, 4, x=x, w=w, y=y, ids=ids, seed=T)


@pytest.mark.parametrize("T", [64, 257, 4616, 70000])
def test_every_row_another_adapter(adapters, T):
    """Rows of one tile that all have adapters of their own, in no order; and only a few of many adapters used."""
    G = 300
    ids = torch.arange(T) * 7 % G
    _go(adapters, T, 48, (32,), 8, G, ids=ids, y="f32", seed=T)
    ids = torch.where(torch.arange(T) % 5 == 0, 299, -1)
    _go(adapters, T, 48, (32,), 8, G, ids=ids, y="bf16", x="bf16", w="bf16", seed=T)


def test_ids_that_are_no_adapters(adapters):
    """Rows whose id is out of range are y, bit for bit (NaN payloads and zeros' signs too), and in place not written."""
    T = 70
    ids = torch.tensor([-1, 3, 2 ** 31 - 1, -2 ** 31, 5, 0, 99] * 10, dtype=torch.int32)
    for y in ("f32", "f16", "bf16"):
        c = Case(T, 64, (32, 32), 8, 3, y=y, ids=ids)
        none = ((ids < 0) | (ids >= 3)).to(DEV)
        raw = c.y.view(torch.int32 if y == "f32" else torch.int16)
        raw[:T][none] = torch.randint(-2 ** 15, 2 ** 15, raw[:T][none].shape, device=DEV, dtype=raw.dtype)
        if y == "f32":
            raw[:T][none] <<= 16
        out = c.run(adapters)
        assert torch.equal(_bits(out[:T, :64][none]), _bits(c.y[:T, :64][none]))
        before = c.y.clone()
        c.run(adapters, out=c.y)
        assert torch.equal(_bits(c.y[:T][none]), _bits(before[:T][none]))
        assert torch.equal(_bits(c.y[:T, :64][~none]), _bits(out[:T, :64][~none]))
        assert torch.equal(_bits(c.y[:T, 64:]), _bits(before[:T, 64:])) and torch.equal(_bits(c.y[T:]), _bits(before[T:]))


def test_no_adapters_at_all(adapters):
    c = Case(40, 64, (32,), 8, 1, ids=[0] * 40)
    out = torch.zeros_like(c.y)
    work = torch.empty(adapters.workspace_bytes(40, 64, 1, 8), dtype=torch.uint8, device=DEV)
    adapters.add_device(c.x.data_ptr(), 1, 0, c.x.stride(0), 40, 64, c.ids.data_ptr(), 0, 0, 0, 1, 0, 0, 8, (32,), c.y.data_ptr(), c.y.stride(0),
                        out.data_ptr(), out.stride(0), 1, work.data_ptr(), work.numel(), _stream())
    assert torch.equal(out[:40, :32], c.y[:40, :32])


@pytest.mark.parametrize("R,ranks", [(16, [16, 8, 0, 3, 99, -5]), (64, [64, 8, 16, 33, 0, 40]), (24, [1, 9, 17, 24, 16, 8])])
@pytest.mark.parametrize("w", ["f16", "bf16"])
@pytest.mark.parametrize("T", [30, 700])
def test_ranks_of_their_own(adapters, R, ranks, w, T):
    """Adapters of lower rank, with NaN behind theirs."""
    _go(adapters, T, 80, (48, 80), R, 6, x=w, w=w, y="f32", ranks=ranks, seed=R)


def test_scales(adapters):
    _go(adapters, 40, 64, (32,), 8, 3, scales=False)
    c = Case(40, 64, (32,), 8, 3, y="f32")
    c.scales = torch.tensor([0.0, -1.5, 0.25], device=DEV)
    c.check(c.run(adapters))


@pytest.mark.parametrize("T,K,cols,R", [(1, 4096, (512,), 16), (33, 768, (256, 256, 256), 16), (200, 2048, (768,), 64), (4616, 768, (256,), 16),
                                        (20000, 256, (128,), 128)])
@pytest.mark.parametrize("x,w,y", [("f16", "f16", "f16"), ("bf16", "bf16", "bf16"), ("e4m3", "f16", "f32"), ("bf16", "bf16", "f32"),
                                   ("e4m3", "bf16", "f16"), ("f16", "f16", "f32")])
def test_values(adapters, T, K, cols, R, x, w, y):
    _go(adapters, T, K, cols, R, 7, x=x, w=w, y=y, whole=False, seed=T + R)


@pytest.mark.parametrize("w", ["f16", "bf16"])
@pytest.mark.parametrize("e", [-36, -24, -12, 10, 24])
def test_small_and_large_inner_products(adapters, w, e):
    """Inner products far outside f16's range, and of very different sizes in one row.  f16 rows take their size from
    scales of codes."""
    c = Case(50, 256, (64,), 16, 2, x="e4m3", w=w, y="f32", whole=False, seed=3)
    c.y.zero_()
    c.xs += e if e >= 0 else 0
    if e < 0:
        c.xs -= -e
    c.xv = c.xv * 2.0 ** e
    c.a[:, :, ::3] *= 2.0 ** -9
    out = c.run(adapters)
    want, tol = c.want()
    # a value's parts may be held to 2^-22 of it, and to 2^-39 of the row's largest
    far = torch.zeros_like(tol)
    for g in range(2):
        rows = c.ids == g
        h = (c.xv[rows] @ c.a[g, 0].double().t()).abs().amax(1, keepdim=True)
        far[rows] = 4 * 2.0 ** -39 * h * c.b[g].double().abs().sum(1)[None]
    off = (out[:50, :64].double() - want).abs() - tol - far - want.abs() * 2.0 ** -23
    assert bool((off <= 0).all()), float(off.max())


@pytest.mark.parametrize("w", ["f16", "bf16"])
def test_infinities_and_nan_stay_in_their_row(adapters, w):
    for T in (40, 5000):
        c = Case(T, 64, (64,), 8, 3, x=w, w=w, y="f32", ids=[0, 1, 2, 1] * (T // 4))
        c.b[c.b == 0] = 1  # an infinity times a zero would be NaN
        good = c.run(adapters).clone()
        c.x[5, 3], c.x[6, 3], c.x[7, 3] = float("inf"), float("nan"), float("-inf")
        out = c.run(adapters)
        rest = [i for i in range(T) if i not in (5, 6, 7)]
        assert torch.equal(out[rest], good[rest])
        assert bool(out[6, :64].isnan().all())
        a = c.a[1, 0, :, 3].double()
        for row, v in ((5, float("inf")), (7, float("-inf"))):
            h = torch.where(a == 0, float("nan"), a * v)
            want = c.y[row, :64].double() + (h * c.b[1].double()).sum(1)
            got = out[row, :64].double()
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0, 1, -1), want.nan_to_num(0, 1, -1))


@pytest.mark.parametrize("y", ["f16", "f32"])
@pytest.mark.parametrize("T", [150, 400])
def test_rows_past_32_bits(adapters, T, y):
    """Rows as far apart as may be, whose bytes (and with 400 of them values) lie past 2^32, of x, y and out."""
    K, n, ld = 64, 32, 1 << 24
    if y == "f32" and T > 200:
        ld = 1 << 23
    c = Case(T, K, (n,), 8, 2, y=y, ids=[0, 1, -1, 1, 0] * (T // 5))
    x = torch.empty((T - 1) * ld + K, dtype=torch.float16, device=DEV)
    big = torch.empty((T - 1) * ld + n, dtype=c.y.dtype, device=DEV)
    for t in range(T):
        x[t * ld:t * ld + K], big[t * ld:t * ld + n] = c.x[t, :K], c.y[t, :n]
    work = torch.empty(adapters.workspace_bytes(T, K, 1, 8), dtype=torch.uint8, device=DEV)
    adapters.add_device(x.data_ptr(), 1, 0, ld, T, K, c.ids.data_ptr(), 2, c.a.data_ptr(), c.b.data_ptr(), 1, 0, c.scales.data_ptr(), 8, (n,),
                        big.data_ptr(), ld, big.data_ptr(), ld, CODE[y], work.data_ptr(), work.numel(), _stream())
    c.check(torch.stack([big[t * ld:t * ld + n] for t in range(T)]))


def test_adapters_past_32_bits(adapters):
    """The last of many adapters, whose weights lie past 2^32 bytes."""
    T, K, R, G = 40, 8192, 128, 2300
    a = torch.zeros(G, 1, R, K, dtype=torch.bfloat16, device=DEV)  # 4.8 GB
    b = torch.zeros(G, 64, R, dtype=torch.bfloat16, device=DEV)
    c = Case(T, K, (64,), R, 1, x="bf16", w="bf16", y="f32", scales=False, ids=[0] * T)
    a[-1], b[-1] = c.a[0], c.b[0]
    want, _ = c.want()
    c.a, c.b, c.G = a, b, G
    c.ids = torch.full((T,), G - 1, dtype=torch.int32, device=DEV)
    assert torch.equal(c.run(adapters)[:T, :64], want.float())


def test_host_form(adapters):
    rng = np.random.default_rng(1)
    from witchcraft_amd import fp8
    t, k, g, r = 21, 160, 3, 16
    x = rng.integers(-2, 3, (t, k)).astype(np.float16)
    a, b = rng.integers(-1, 2, (g, 2, r, k)).astype(np.float16), rng.integers(-3, 4, (g, 112, r)).astype(np.float16)
    y, ids, cols = rng.integers(-9, 10, (t, 112)).astype(np.float32), rng.integers(-1, g + 2, t), (80, 32)
    scales = np.array([0.5, 2, 1], np.float32)
    want = y.astype(np.float64)
    for i, e in enumerate(ids):
        if 0 <= e < g:
            h = x[i].astype(np.float64) @ a[e].astype(np.float64).transpose(0, 2, 1)
            want[i] += scales[e] * np.concatenate([b[e, :80].astype(np.float64) @ h[0], b[e, 80:].astype(np.float64) @ h[1]])
    assert np.array_equal(adapters.add(x, ids, a, b, y, scales=scales, cols=cols), want.astype(np.float32))
    assert np.array_equal(adapters.add(fp8.quantize(x), ids, a, b, y.astype(np.float16), scales=scales, cols=cols), want.astype(np.float16))
    assert np.array_equal(adapters.add(x, np.full(t, -1), a, b, y, cols=cols), y)
    assert np.array_equal(adapters.add(x, ids, a, b, y, scales=scales, ranks=[16, 16, 99], cols=cols), want.astype(np.float32))


@pytest.mark.parametrize("T", [20, 3000])
def test_same_bits_every_time(adapters, T):
    c = Case(T, 768, (768,), 16, 5, whole=False, seed=4, y="f32")
    first = c.run(adapters)
    for _ in range(5):
        assert torch.equal(c.run(adapters), first)


@pytest.mark.parametrize("T", [1, 64, 3000])
def test_graph_replays_equal_eager(adapters, T):
    c = Case(T, 256, (256, 256), 16, 4, x="bf16", w="bf16", y="bf16", whole=False, seed=2)
    out = torch.empty(T + 2, 512 + 32, dtype=torch.bfloat16, device=DEV)
    work = torch.empty(adapters.workspace_bytes(T, 256, 2, 16), dtype=torch.uint8, device=DEV)
    c.run(adapters, out, work)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        c.run(adapters, out, work)
    for i in range(4):
        c.x.copy_(torch.randn(c.x.shape, device=DEV))
        c.ids.copy_(torch.randint(-1, 4, (T,)))
        want = c.run(adapters)[:T, :512].clone()
        out.zero_()
        work.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[:T, :512], want)


def test_streams_at_once(adapters):
    cases = [Case(500, 256, (256,), 16, 4, whole=False, seed=s) for s in range(3)]
    streams = [torch.cuda.Stream() for _ in cases]
    want = [c.run(adapters) for c in cases]
    outs = [torch.zeros_like(w) for w in want]
    works = [torch.empty(adapters.workspace_bytes(500, 256, 1, 16), dtype=torch.uint8, device=DEV) for _ in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, c, o, w in zip(streams, cases, outs, works):
            with torch.cuda.stream(s):
                c.run(adapters, o, w)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o[:500, :256], w[:500, :256])


@pytest.mark.parametrize("R,K", [(8, 768), (16, 4096), (64, 4096), (128, 128)])
def test_a_workspace_serves_fewer_rows(adapters, R, K):
    """Sizes of the workspace never fall with the rows, whichever form they are taken in."""
    last = 0
    for T in [1, 16, 100, 191, 192, 193, 383, 385, 511, 512, 513, 700, 1400, 2730, 5000]:
        n = adapters.workspace_bytes(T, K, 1, R)
        assert n >= last, T
        last = n
    for T in (192, 193, 384, 385, 512, 513):
        c = Case(T, K, (64,), R, 2, seed=T)
        work = torch.full((adapters.workspace_bytes(600, K, 1, R) + 256,), 255, dtype=torch.uint8, device=DEV)
        c.work = work
        c.check(c.run(adapters, work=work))
        assert bool((work[-256:] == 255).all())


@pytest.mark.parametrize("K", [16, 32, 112, 128, 144, 496, 768, 2064, 4096])
@pytest.mark.parametrize("x,w", [("f16", "f16"), ("bf16", "bf16"), ("e4m3", "f16"), ("e4m3", "bf16")])
@pytest.mark.parametrize("T,R", [(600, 64), (5003, 16), (2100, 128), (17000, 48)])
def test_depths_of_many_rows(adapters, K, x, w, T, R):
    """Depths that end inside a step of the first product, whose tiles begin at different ones."""
    ids = (torch.arange(T) // 37) % 4 - 1
    _go(adapters, T, K, (48,), R, 3, x=x, w=w, y="f32" if K % 3 else "f16", ids=ids, seed=K + T)


@pytest.mark.parametrize("R", [8, 24, 48, 56, 72, 104, 128])
@pytest.mark.parametrize("S", [1, 2, 4])
@pytest.mark.parametrize("T", [520, 4500, 9000])
@pytest.mark.parametrize("x,y", [("f16", "f32"), ("bf16", "bf16"), ("f16", "f16")])
def test_ranks_of_many_rows(adapters, R, S, T, x, y):
    """Whole and half tiles of the first product and every number of its ranks, every form of the second."""
    ids = (torch.arange(T) // 50) % 5 - 1
    _go(adapters, T, 128, (80, 16, 256, 32)[:S], R, 4, x=x, w=x, y=y, ids=ids, ranks=[R, R // 2, 5, R - 1], seed=R + S + T)


@pytest.mark.parametrize("x", ["f16", "e4m3"])
@pytest.mark.parametrize("R", [8, 64])
def test_tiles_of_far_rows(adapters, x, R):
    """Many rows as far apart as may be: a tile of 64 spans 2^31 bytes of x, a sixteen 2^29 of y."""
    T, K, n, ld = 600, 176, 32, 1 << 24
    c = Case(T, K, (n,), R, 2, x=x, ids=[0, 1, -1, 1, 0] * (T // 5))
    far = torch.empty((T - 1) * ld + K, dtype=c.x.dtype, device=DEV)
    big = torch.empty((T - 1) * ld + n, dtype=c.y.dtype, device=DEV)
    for t in range(T):
        far[t * ld:t * ld + K], big[t * ld:t * ld + n] = c.x[t, :K], c.y[t, :n]
    work = torch.empty(adapters.workspace_bytes(T, K, 1, R), dtype=torch.uint8, device=DEV)
    adapters.add_device(far.data_ptr(), CODE[x], 0 if c.xs is None else c.xs.data_ptr(), ld, T, K, c.ids.data_ptr(), 2, c.a.data_ptr(),
                        c.b.data_ptr(), 1, 0, c.scales.data_ptr(), R, (n,), big.data_ptr(), ld, big.data_ptr(), ld, 1,
                        work.data_ptr(), work.numel(), _stream())
    c.check(torch.stack([big[t * ld:t * ld + n] for t in range(T)]))


@pytest.mark.parametrize("w", ["f16", "bf16"])
@pytest.mark.parametrize("T", [40, 600, 17000])
def test_codes_that_are_no_numbers(adapters, w, T):
    """A NaN code and the scale byte that stands for none make their rows NaN, and no others; every other code and the
    smallest and largest scales count as they are."""
    c = Case(T, 144, (64,), 8, 3, x="e4m3", w=w, y="f32", ids=[0, 1, 2, 1] * (T // 4))
    c.b[c.b == 0] = 1
    good = c.run(adapters).clone()
    c.x[5, 3], c.x[T - 2, 143] = 0x7f, 0xff
    c.xs[0, 6], c.xs[1, T - 5] = 255, 255
    got = c.run(adapters)
    torch.cuda.synchronize()
    bad = [5, 6, T - 5, T - 2]
    assert bool(got[bad, :64].isnan().all())
    keep = torch.ones(T, dtype=torch.bool, device=DEV)
    keep[bad] = False
    assert torch.equal(got[:T, :64][keep], good[:T, :64][keep])


@pytest.mark.parametrize("w", ["f16", "bf16"])
@pytest.mark.parametrize("T", [16, 640])
def test_every_code(adapters, w, T):
    """One code and one weight of one to a row: results are the code's value, bit for bit, times each power of two."""
    codes = torch.tensor([i for i in range(256) if i & 0x7f != 0x7f], dtype=torch.uint8, device=DEV)
    c = Case(T, 128, (16,), 8, 1, x="e4m3", w=w, y="f32", ids=[0] * T, scales=False)
    c.y.zero_(), c.a.zero_(), c.b.zero_()
    c.a[0, 0, 0, 17], c.b[0, :, 0] = 1, 1
    for i in range(0, 254, T):
        part = codes[i:i + T]
        n = len(part)
        c.x.zero_()
        c.x[:n, 17] = part
        for byte in (1, 100, 127, 200, 244):
            c.xs.fill_(byte)
            want = part.view(torch.float8_e4m3fn).double() * 2.0 ** (byte - 127)
            got = c.run(adapters)[:n, :16]
            # a power of two below f32's normal numbers may be taken as zero
            fine = (want.abs() >= 2.0 ** -126) | (want == 0)
            assert torch.equal(got[fine], want.float()[fine, None].expand(-1, 16)), byte


@pytest.mark.parametrize("w", ["f16", "bf16"])
@pytest.mark.parametrize("T", [40, 5000])
def test_infinite_rows(adapters, w, T):
    """An infinite inner product makes its row infinite (or NaN, f16 adapters), never finite, and only that row."""
    c = Case(T, 64, (64,), 8, 1, x=w, w=w, y="f32", ids=[0] * T, scales=False)
    c.a[:, :, :, 3], c.b[:] = 1, c.b.abs() + 1
    good = c.run(adapters).clone()
    c.x[5, 3], c.x[T - 1, 3] = float("inf"), float("-inf")
    got = c.run(adapters)
    assert torch.equal(got[[i for i in range(T) if i not in (5, T - 1)], :64], good[[i for i in range(T) if i not in (5, T - 1)], :64])
    if w == "bf16":
        assert bool((got[5, :64] == float("inf")).all()) and bool((got[T - 1, :64] == float("-inf")).all())
    assert not bool(got[[5, T - 1], :64].isfinite().any())
