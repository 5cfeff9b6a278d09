"""Adapters with infinite rows, weights, hidden rows and gradients: infinities, their
signs and NaN where the formulas in 64 bits have them, and everything else as it is
without them (bounds: lora_reference)."""
import pytest
import torch

from lora_reference import Adapters, factors

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SEED = [77, 5]
INF = float("inf")


class Plain:
    """The formulas in float64, an adapter's rows at once; dropped elements are zeros."""

    def __init__(self, x, down, up, of, f):
        d = lambda t: t.detach().cpu().double()  # noqa: E731
        self.down, self.up, self.of, self.f = d(down), d(up), of, f
        self.x = torch.where(f > 0, d(x) * f, torch.zeros(()).double())

    def forward(self, base):
        y = base.detach().cpu().double().clone()
        h = torch.zeros(len(self.of), self.down.shape[1], dtype=torch.float64)
        for a in range(len(self.down)):
            on = self.of == a
            h[on] = self.x[on] @ self.down[a].t()
            y[on] += h[on] @ self.up[a].t()
        return y, h

    def backward(self, dy, hidden, base):
        dy, hidden, dx = (t.detach().cpu().double().clone() for t in (dy, hidden, base))
        dd, du = torch.zeros_like(self.down), torch.zeros_like(self.up)
        for a in range(len(self.down)):
            on = self.of == a
            u = dy[on] @ self.up[a]
            z = u @ self.down[a]
            dx[on] += torch.where(self.f[on] > 0, z * self.f[on], torch.zeros(()).double())
            dd[a], du[a] = u.t() @ self.x[on], dy[on].t() @ hidden[on]
        return dx, dd, du


def _same(name, got, want, bound):
    got = got.detach().cpu().double()
    assert torch.equal(got.isnan(), want.isnan()), f"{name}: {int((got.isnan() != want.isnan()).sum())} NaN too many or few"
    for v in (INF, -INF):
        assert torch.equal(got == v, want == v), f"{name}: {int(((got == v) != (want == v)).sum())} of {v}"
    ok = want.isfinite()
    assert bool(((got - want).abs()[ok] <= bound[ok]).all()), name


# (gathered gradients, tiles, tiles of more rows; each count of rank tiles; rows in one
# block's columns and in several)
@pytest.mark.parametrize("n,c,o,r", [(12, 130, 90, 5), (20, 72, 136, 100), (300, 130, 300, 16), (200, 600, 72, 9), (150, 96, 264, 30),
                                     (300, 264, 130, 64), (300, 40, 200, 33), (130, 520, 136, 128), (12_300, 72, 40, 12),
                                     (12_300, 40, 64, 70), (24_600, 40, 33, 50)])
@pytest.mark.parametrize("p", [0.0, 0.25])
@pytest.mark.parametrize("dt", list(DT))
def test_infinities(spc, dev, dt, p, n, c, o, r):
    nat, t, g = spc._native, DT[dt], torch.Generator().manual_seed(n + c + o + r)
    rnd = lambda *s: torch.randn(*s, generator=g).to(t).to(dev)  # noqa: E731
    cut = n // 2 - 1
    kw = dict(offsets=torch.tensor([0, cut, n - 1], device=dev), adapters=torch.tensor([1, 0], dtype=torch.int32, device=dev),
              p=p, seed=torch.tensor(SEED, device=dev) if p else None)
    of = torch.tensor([1] * cut + [0] * (n - 1 - cut) + [-1])
    f = factors(SEED, n, c, p) if p else torch.ones(n, c, dtype=torch.float64)
    x, down, up, base = rnd(n, c), rnd(2, r, c) * 0.1, rnd(2, o, r) * 0.1, rnd(n, o)
    dy, dx_base = rnd(n, o), rnd(n, c)
    x[2:n:3, c - 1] = 0                               # (an infinite weight there: NaN)
    ref = Adapters(x, down, up, offsets=[0, cut, n - 1], adapters=[1, 0], p=p, seed=SEED)
    (_, ey), (h, eh) = ref.forward(base)
    hidden = h.float().to(dev)
    bounds = [b for _, b in ref.backward(dy, hidden, dx_base)]

    def run(x, down, up, dy, hidden):
        w = Plain(x, down, up, of, f)
        y, got_h = nat.lora(x, down, up, base, return_hidden=True, **kw)
        want_y, want_h = w.forward(base)
        _same("hidden", got_h, want_h, eh), _same("y", y, want_y, ey)
        assert torch.equal(nat.lora(x, down, up, base.clone(), return_hidden=False, **kw).isnan(), y.isnan())
        got = nat.lora_backward(dy, x, hidden, down, up, dx_base, **kw)
        for name, a, b, e in zip(("dx", "ddown", "dup"), got, w.backward(dy, hidden, dx_base), bounds):
            _same(name, a, b, e)

    run(x, down, up, dy, hidden)
    for sign in (1, -1):
        v = [t.clone() for t in (x, down, up, dy, hidden)]
        v[0][[1, n - 2], [3, c - 1]] = sign * INF     # a row of each adapter
        run(v[0], *v[1:])
        v = [t.clone() for t in (x, down, up, dy, hidden)]
        v[1][0, r - 1, c - 1] = sign * INF            # a weight
        run(*v)
        v = [t.clone() for t in (x, down, up, dy, hidden)]
        v[2][1, o - 1, r - 1], v[2][0, 2, 0] = sign * INF, INF
        run(*v)
        v = [t.clone() for t in (x, down, up, dy, hidden)]
        v[3][0, o - 1], v[3][n - 3, 1] = sign * INF, INF
        run(*v)
        v = [t.clone() for t in (x, down, up, dy, hidden)]
        v[4][0, r - 1], v[4][n - 3, 0] = sign * INF, INF
        run(*v)
