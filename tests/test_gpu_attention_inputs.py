"""What stands before attention in one run, on the GPU: residual's norm and codes, the shared q, k and v projection,
the requests' adapters added in place, and q's and k's head norms and rotation in place; against the definition in
64 bits from the codes on (how the norm's codes come about has its own tests).

The bound is carried along: the product's own (sums in f32, alignment to the largest product of a block at 12 bits),
its rounding to f16, what the adapters' sums and parts are off by and their rounding, the norm (a value's error, and the
norm's: the root mean square of a head's errors against its own; 1.1 covers second order at errors of 2^-10), the rotation
of two values' errors, and the last rounding.
"""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DEV = "cuda:0"
HEADS, KEYS, D, HEAD, R, G = 6, 2, 384, 64, 16, 3
COLS = (HEADS * HEAD, KEYS * HEAD, KEYS * HEAD)
N = sum(COLS)
HALF, LEAST = 2.0 ** -11, 2.0 ** -25  # f16: half a step of a value, of the smallest ones
EPS = 1e-6


@pytest.fixture(scope="module")
def fp8():
    from witchcraft_amd import fp8
    return fp8


class Run:
    def __init__(self, fp8, T, seed):
        import numpy as np

        from witchcraft_amd import adapters, rotary
        self.f, self.a, self.r, self.T = fp8, adapters, rotary, T
        g = torch.Generator(device=DEV).manual_seed(seed)
        n = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
        self.x, self.gamma = n(T, D), 1 + 0.2 * n(D)
        self.norms = [(1 + 0.2 * n(HEAD)).contiguous() for _ in range(2)]
        w = n(N, D) / D ** 0.5
        self.w, self.sw = torch.empty(N, D, dtype=torch.uint8, device=DEV), torch.empty((N + 127) // 128, D // 128, dtype=torch.uint8, device=DEV)
        fp8.quantize_weights_device(w.data_ptr(), 0, N, D, 0, self.w.data_ptr(), self.sw.data_ptr(), self.stream())
        self.la, self.lb = (n(G, 3, R, D) / D ** 0.5).half(), (n(G, N, R) / R ** 0.5).half()
        self.scales = torch.tensor([0.5, 1.0, 2.0], device=DEV)
        # requests of 1 .. 100 rows, each with an adapter or none, and their own positions
        lengths = torch.randint(1, 101, (T,), generator=torch.Generator().manual_seed(seed))
        which = torch.repeat_interleave(torch.arange(T), lengths)[:T]
        self.ids = (which % (G + 1) - 1).to(torch.int32).to(DEV)
        self.pos = (torch.arange(T) - torch.searchsorted(which, which)).to(torch.int32).to(DEV)
        self.freqs = rotary.frequencies(HEAD)
        self.table = torch.from_numpy(np.ascontiguousarray(rotary.table(self.freqs)).view(np.uint8)).to(DEV)
        rows = (T + 15) // 16 * 16
        self.c, self.cs = torch.zeros(T, D, dtype=torch.uint8, device=DEV), torch.zeros(D // 128, rows, dtype=torch.uint8, device=DEV)
        self.qkv = torch.full((T + 3, N), 5.0, dtype=torch.float16, device=DEV)
        self.size = adapters.workspace_bytes(T, D, 3, R)
        self.work = torch.full((self.size,), 255, dtype=torch.uint8, device=DEV)

    @staticmethod
    def stream():
        return torch.cuda.current_stream().cuda_stream

    def run(self):
        p, s, T = (lambda t: t.data_ptr()), self.stream(), self.T
        self.f.rmsnorm_device(p(self.x), 0, 0, 0, T, D, p(self.gamma), EPS, 0, p(self.c), p(self.cs), s)
        self.f.matmul_device(p(self.c), p(self.cs), T, p(self.w), p(self.sw), N, D, 0, p(self.qkv), 1, s)
        self.a.add_device(p(self.c), 3, p(self.cs), D, T, D, p(self.ids), G, p(self.la), p(self.lb), 1, 0, p(self.scales), R,
                          COLS, p(self.qkv), N, p(self.qkv), N, 1, p(self.work), self.size, s)
        q, k = p(self.qkv), p(self.qkv) + 2 * HEADS * HEAD
        self.r.rotate_device(q, N, HEADS, k, N, KEYS, 1, T, HEAD, p(self.norms[0]), p(self.norms[1]), EPS, p(self.table), HEAD,
                             self.r.HALVES, p(self.pos), 1, q, N, k, N, s)

    def want(self):
        T = self.T
        codes = lambda c: c.view(torch.float8_e4m3fn).double()  # noqa: E731
        x = codes(self.c) * torch.exp2(self.cs[:, :T].double() - 127).t().repeat_interleave(128, 1)
        w = codes(self.w) * torch.exp2(self.sw.double() - 127).repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)
        out, far = x @ w.t(), (D + 16) * 2.0 ** -23 * (x.abs() @ w.abs().t())
        for b in range(D // 128):
            part = slice(128 * b, 128 * b + 128)
            far += 128 * 2.0 ** -12 * x[:, part].abs().amax(1)[:, None] * w[:, part].abs().amax(1)[None]
        far = far + HALF * (out.abs() + far) + LEAST
        for g in range(G):
            rows, n0, f = (self.ids == g).nonzero()[:, 0], 0, float(self.scales[g])
            for s, n in enumerate(COLS):
                a, b = self.la[g, s].double(), self.lb[g, n0:n0 + n].double()
                h = x[rows] @ a.t()
                e = far[rows, n0:n0 + n] + f * ((D + 3 * R + 16) * 2.0 ** -23 * ((x[rows].abs() @ a.abs().t()) @ b.abs().t())
                                                + 2.0 ** -16 * (h.abs() @ b.abs().t()))
                out[rows, n0:n0 + n] += f * (h @ b.t())
                far[rows, n0:n0 + n] = e + (HALF + 2.0 ** -23) * (out[rows, n0:n0 + n].abs() + e) + LEAST
                n0 += n
        turn = self.pos.double()[:, None] * torch.from_numpy(self.freqs).to(DEV).double()[None]
        cos, sin, half = torch.cos(turn)[:, None], torch.sin(turn)[:, None], HEAD // 2
        n0 = 0
        for heads, gamma in ((HEADS, self.norms[0]), (KEYS, self.norms[1])):
            at = slice(n0, n0 + heads * HEAD)
            y, e, g = out[:, at].reshape(T, heads, HEAD), far[:, at].reshape(T, heads, HEAD), gamma.double()
            r = torch.sqrt((y * y).mean(2, keepdim=True) + EPS)
            e = 1.1 * g.abs() / r * (e + y.abs() / r * (e * e).mean(2, keepdim=True).sqrt())
            y = y / r * g
            a, b, ea, eb = y[..., :half], y[..., half:], e[..., :half], e[..., half:]
            y = torch.cat([a * cos - b * sin, b * cos + a * sin], 2)
            e = torch.cat([ea * cos.abs() + eb * sin.abs(), eb * cos.abs() + ea * sin.abs()], 2)
            e = e + 20 * 2.0 ** -24 * (a.abs() + b.abs()).repeat(1, 1, 2)
            out[:, at], far[:, at] = y.reshape(T, -1), (e + 1.001 * HALF * (y.abs() + e) + LEAST).reshape(T, -1)
            n0 += heads * HEAD
        return out, far


@pytest.mark.parametrize("T", [1, 40, 300, 700, 2300])
def test_run(fp8, T):
    run = Run(fp8, T, T)
    run.run()
    want, far = run.want()
    off = (run.qkv[:T].double() - want).abs() - far
    assert bool((off <= 0).all()), (float(off.max()), int((off > 0).sum()))
    assert bool((run.qkv[T:] == 5).all())
    # the bound is no blanket: errors near the roundings
    assert float((run.qkv[:T].double() - want).norm() / want.norm()) < 2.0 ** -9


@pytest.mark.parametrize("T", [1, 40, 700])
def test_captured_run_equals_eager(fp8, T):
    run = Run(fp8, T, 7 + T)
    run.run()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        run.run()
    for i in range(4):
        run.x.copy_(torch.randn(T, D, generator=torch.Generator(device=DEV).manual_seed(i), device=DEV))
        run.ids.copy_(torch.randint(-1, G, (T,), generator=torch.Generator(device=DEV).manual_seed(i), device=DEV))
        run.run()
        want = run.qkv.clone()
        run.qkv[:T].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(run.qkv.view(torch.int16), want.view(torch.int16)), i


def test_failed_calls_leave_no_error(fp8):
    """Host forms whose buffers no card holds (2 TB, of which nothing is read here), and a device that is not there:
    the next call on the thread succeeds."""
    import ctypes as C

    import numpy as np

    from witchcraft_amd import _lib, adapters, rotary
    buf, lib, cols = np.zeros(4096, np.uint8).ctypes.data, _lib.lib, (C.c_int32 * 1)(64)
    table = rotary.table(rotary.frequencies(8))
    x = np.ones((3, 2, 8), np.float16)
    a, b = np.ones((1, 1, 8, 16), np.float16), np.ones((1, 16, 8), np.float16)

    def good():
        q, _ = rotary.rotate(x, x, np.zeros(3, np.int32), table)
        assert (q == 1).all()
        y = adapters.add(np.ones((3, 16), np.float16), [0, -1, 0], a, b, np.zeros((3, 16), np.float32))
        assert (y == np.array([128, 0, 128])[:, None]).all()
        assert int(torch.ones(5, device=DEV).sum()) == 5

    good()
    for call in (lambda dev: lib.t5h_adapter_add(dev, buf, 1, None, 1 << 20, 1 << 20, buf, 1, buf, buf, 1, None, None, 8, C.addressof(cols), 1,
                                                 buf, buf, 1),
                 lambda dev: lib.t5h_rotary(dev, buf, 64, buf, 64, 0, 1 << 24, 512, None, None, 1e-6, buf, 512, 0, buf, 1, buf, buf)):
        assert call(0) == _lib.T5H_ERR_NOMEM
        good()
        assert call(4096) not in (0, _lib.T5H_ERR_NOMEM)
        good()
