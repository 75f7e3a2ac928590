"""Adapters of lower rank than their buffers, whose rows of a and columns of b hold other values behind it: those do not
count, whatever the rank is a multiple of.  Whole numbers, compared bit for bit with the definition over the ranks that
count."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_adapter import DEV, Case, adapters  # noqa: E402,F401


def _cut(c, ranks, value=0.0, whole=1):
    """a and b with `value` from each adapter's rank on, up to whole ones of `whole`."""
    a, b = c.a.clone(), c.b.clone()
    for i, n in enumerate(ranks):
        n = (min(max(n, 0), c.R) + whole - 1) // whole * whole
        a[i, :, n:], b[i, :, n:] = value, value
    return a, b


@pytest.mark.parametrize("R,ranks", [(8, [3, 8, 1, 0]), (16, [3, 9, 16, 12]), (24, [17, 23, 4, 8]), (64, [33, 5, 64, 63]), (128, [100, 1, 127, 66])])
@pytest.mark.parametrize("w,y", [("f16", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("T", [1, 40, 700])
def test_values_behind_the_rank_do_not_count(adapters, T, R, ranks, w, y):  # noqa: F811
    print(f"[adapter] T={T} R={R} ranks={ranks} {w} {y}", flush=True)
    c = Case(T, 144, (48, 80), R, 4, x=w, w=w, y=y, seed=R + T, ids=(torch.arange(T) // 3) % 4)
    given = c.a, c.b
    c.ranks = torch.tensor(ranks, dtype=torch.int32, device=DEV)
    c.a, c.b = _cut(c, ranks)
    want, _ = c.want()
    assert float(want.abs().max()) < 2 ** 24
    c.a, c.b = given
    out = c.run(adapters)
    torch.cuda.synchronize()
    assert torch.equal(out[:T, :c.N], want.to(out.dtype))
    c.around(out)
    # no number at all: in a from the rank on, in b from the next whole eight on
    c.a, _ = _cut(c, ranks, float("nan"))
    _, c.b = _cut(c, ranks, float("nan"), 8)
    out = c.run(adapters)
    torch.cuda.synchronize()
    assert torch.equal(out[:T, :c.N], want.to(out.dtype))


@pytest.mark.parametrize("ranks", [[3, 7, 12], [1, 16, 9]])
def test_host_form(adapters, ranks):  # noqa: F811
    rng = np.random.default_rng(1)
    t, k, g, r = 21, 160, 3, 16
    x = rng.integers(-2, 3, (t, k)).astype(np.float16)
    a, b = rng.integers(-1, 2, (g, 1, r, k)).astype(np.float16), rng.integers(-3, 4, (g, 112, r)).astype(np.float16)
    y, ids = rng.integers(-9, 10, (t, 112)).astype(np.float32), rng.integers(-1, g, t)
    want = y.astype(np.float64)
    for i, e in enumerate(ids):
        if e >= 0:
            n = ranks[e]
            want[i] += b[e, :, :n].astype(np.float64) @ (a[e, 0, :n].astype(np.float64) @ x[i].astype(np.float64))
    assert np.array_equal(adapters.add(x, ids, a, b, y, ranks=ranks), want.astype(np.float32))
