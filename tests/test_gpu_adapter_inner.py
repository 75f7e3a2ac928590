"""How many bits of the inner product reach the results of low-rank adapters, on the GPU.

Rows hold digits and A's rows the digits' places (a few powers of two each, elsewhere zeros), so that an inner product
is a whole number of 23 or 24 bits, whose lowest ones lie below what two bf16 parts hold; every partial sum is a whole
number below 2^24, so f32 sums are exact in any order.  B has one power of two a column, scales are powers of two.
  * f32 results are then the definition's, bit for bit, which takes all three parts of the inner product;
  * 16-bit results may be off by 2^-16 of the inner product's share, and half a step of their type: where y cancels the
    adapter's share this is more than half a step of what is left.
"""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_adapter import DEV, TYPE, Case, adapters  # noqa: E402,F401

# Bits of a digit, places from digit to digit, digits.  Codes: three each in two blocks with scales of their own.
DIGITS = {"f16": (11, 12, 2), "bf16": (8, 8, 3), "e4m3": (4, 4, 6)}


def _two_parts(h):
    """f32 values as the sum of two bf16 parts: the upper 8 bits, and the rest rounded to 8."""
    first = (h.view(torch.int32) & -65536).view(torch.float32)
    return first.double() + (h - first).bfloat16().double()


class Digits(Case):
    def __init__(self, T, cols, R, x, w, y, seed, factor=1.0):
        K, G = 272, 4
        super().__init__(T, K, cols, R, G, x=x, w=w, y=y, seed=seed)
        g = torch.Generator().manual_seed(seed)
        bits, places, count = DIGITS[x]
        v = torch.randint(0, 1 << bits, (T, K), generator=g).float() * (torch.randint(0, 2, (T, 1), generator=g) * 2 - 1)
        if x == "e4m3":
            self.x[:, :K] = v.to(torch.float8_e4m3fn).view(torch.uint8).to(DEV)
            self.xs.fill_(127)
            self.xs[1] += 12  # the upper three digits' block
            self.xv = v.double().to(DEV)
            self.xv[:, 128:256] *= 4096
        else:
            self.x[:, :K] = v.to(TYPE[x]).to(DEV)
            self.xv = self.x[:, :K].double()
        a = torch.zeros(G, self.S, R, K)
        for d in range(count):
            lo, hi = (0, 128) if x == "e4m3" and d < 3 else (128, 256) if x == "e4m3" else (d * K // count, (d + 1) * K // count)
            at = torch.randint(lo, hi, (G, self.S, R, 1), generator=g)
            while d % 3 and x == "e4m3":  # not on another digit of its block
                taken = a.gather(3, at) != 0
                if not bool(taken.any()):
                    break
                at = torch.where(taken, torch.randint(lo, hi, at.shape, generator=g), at)
            a.scatter_(3, at, 2.0 ** (places * (d % 3 if x == "e4m3" else d)))
        self.a = a.to(TYPE[w]).to(DEV)
        b = torch.zeros(G, self.N, R)
        rank = torch.randint(0, R, (G, self.N, 1), generator=g)
        self.rank = rank[:, :, 0].to(DEV)
        b.scatter_(2, rank, 2.0 ** torch.randint(-2, 3, rank.shape, generator=g).float() * (torch.randint(0, 2, rank.shape, generator=g) * 2 - 1))
        self.b = b.to(TYPE[w]).to(DEV)
        self.scales = (factor * 2.0 ** torch.randint(-1, 3, (G,), generator=g).float()).to(DEV)
        self.y.zero_()

    def inner(self):
        """scale h of each column's one rank [T][N], f64 and exact; and that column's weight."""
        h, b = torch.zeros(self.T, self.N, dtype=torch.float64, device=DEV), torch.zeros(self.T, self.N, dtype=torch.float64, device=DEV)
        for g in range(self.G):
            rows, n0 = (self.ids == g).nonzero()[:, 0], 0
            for s, n in enumerate(self.cols):
                of = self.xv[rows] @ self.a[g, s].double().t() * float(self.scales[g])
                h[rows, n0:n0 + n] = of[:, self.rank[g, n0:n0 + n]]
                b[rows, n0:n0 + n] = self.b[g, n0:n0 + n].double().gather(1, self.rank[g, n0:n0 + n, None])[:, 0]
                n0 += n
        return h, b


@pytest.mark.parametrize("x,w", [("f16", "f16"), ("bf16", "bf16"), ("e4m3", "f16"), ("e4m3", "bf16")])
@pytest.mark.parametrize("R", [8, 16, 24, 32, 64, 104, 128])
@pytest.mark.parametrize("T", [1, 40, 700])
def test_f32_results_take_the_whole_inner_product(adapters, T, R, x, w):  # noqa: F811
    print(f"[adapter] T={T} R={R} {x} {w}", flush=True)
    c = Digits(T, (48, 272), R, x, w, "f32", seed=R + T)
    if T == 1:
        c.ids.fill_(2)
    h, b = c.inner()
    assert bool((h * b == (h * b).float()).all())
    mine = c.ids >= 0
    # what is checked needs the third part: two would give other values
    assert float((_two_parts(h[mine].float()) != h[mine]).double().mean()) > 0.5
    out = c.run(adapters)
    torch.cuda.synchronize()
    assert torch.equal(out[:T, :c.N], (h * b).float())
    c.around(out)


@pytest.mark.parametrize("w,y", [("f16", "f16"), ("bf16", "bf16"), ("f16", "bf16"), ("bf16", "f16")])
@pytest.mark.parametrize("R", [8, 16, 32, 64, 128])
@pytest.mark.parametrize("T", [40, 700])
def test_results_that_cancel(adapters, T, R, w, y):  # noqa: F811
    """y is what the adapter adds, rounded and negative: what is left is that rounding.  Scales take the inner products
    to some 2^10, within f16's range."""
    c = Digits(T, (48, 272), R, w, w, y, seed=R + T, factor=2.0 ** -13)
    h, b = c.inner()
    add = h * b
    c.y[:T, :c.N] = (-add).to(c.y.dtype)
    want = c.y[:T, :c.N].double() + add
    out = c.run(adapters)[:T, :c.N].double()
    half = torch.finfo(c.y.dtype).eps / 2
    left = add.abs() * 2.0 ** -16 + (c.y[:T, :c.N].double().abs() + add.abs()) * 2.0 ** -23  # two parts; f32's own sum
    least = 2.0 ** -25 if y == "f16" else 0.0
    tol = left + (want.abs() + left) * half + least
    assert bool(((out - want).abs() <= tol).all()), float(((out - want).abs() - tol).max())
    # and y does cancel: what is left is a step of its type
    mine = c.ids >= 0
    assert float(want[mine].abs().mean()) < 2 * half * float(add[mine].abs().mean())
