"""The row layer norm and its gradient where their values end: items without
rows, SiLU far from zero, rows that are not finite, the most items."""
import pytest
import torch

from norm_reference import Reference, check

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf"), 3e38])
@pytest.mark.parametrize("offsets", [[0, 4, 4, 30], [0, 0, 30, 30], [10, 10, 20, 20]])
def test_coefficients_that_no_row_meets(spc, dev, offsets, value):
    """What an empty item's scale and shift hold reaches no gradient, and its
    own are zeros, under an infinite weight too."""
    nat = spc._native
    n, c, nb = 30, 72, 3
    x, dy = _randn(1, n, c).to(dev), _randn(2, n, c).to(dev)
    w, b = (1 + 0.2 * _randn(3, c)).to(dev), (0.2 * _randn(4, c)).to(dev)
    sc, sh = _randn(5, nb, c).to(dev), _randn(6, nb, c).to(dev)
    kw = dict(offsets=torch.tensor(offsets, device=dev), silu=True)
    _, st = nat.layer_norm(x, w, b, scale=sc, shift=sh, return_stats=True, **kw)
    want = nat.layer_norm_backward(dy, x, st, w, b, scale=sc, shift=sh, **kw)
    empty = [i for i in range(nb) if offsets[i] == offsets[i + 1]]
    sc[empty], sh[empty] = value, value
    y, st = nat.layer_norm(x, w, b, scale=sc, shift=sh, return_stats=True, **kw)
    got = nat.layer_norm_backward(dy, x, st, w, b, scale=sc, shift=sh, **kw)
    assert bool(y.isfinite().all()) and all(torch.equal(p, q) for p, q in zip(got, want))
    assert bool((got[3][empty] == 0).all()) and bool((got[4][empty] == 0).all())
    w[:] = float("inf")
    ds = nat.layer_norm_backward(dy, x, st, w, b, scale=sc, shift=sh, **kw)[3]
    assert bool((ds[empty] == 0).all())


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("reach", [5.0, 60.0, 1e4, 1e30])
def test_silu_far_from_zero(spc, dev, dt, reach):
    """z from -4 to 4 times `reach`: values and slopes stay finite and within
    the bounds; the negative tail keeps its relative precision.

    silu = z sg(z) changes by |1 / z + 1 - sg| <= 2 of itself per unit of z where
    z <= -1, and the exponential, the reciprocal and three products are off by
    at most u (2 |z| + 8).  The reciprocal's results below 2^-126 are zeros: sg(z) <
    2^-126 needs z < -87.3, where |z| sg(z) falls with z, so that is at most 87.4 x
    2^-126 of a value."""
    nat = spc._native
    n, c = 60, 200
    x, dy = _randn(1, n, c).to(DT[dt]).to(dev), _randn(2, n, c).to(DT[dt]).to(dev)
    w, b = (reach * (1 + 0.2 * _randn(3, c).abs())).to(dev), (reach * 0.1 * _randn(4, c)).to(dev)
    y, st = nat.layer_norm(x, w, b, silu=True, return_stats=True)
    if dt == "f16" and reach > 1e4:           # past f16: infinite, or the tail's zeros
        assert not bool(y.isnan().any())
        return
    ref = Reference(x, w, b, 1e-6, silu=True)
    value, bound = ref.forward()
    check("y", y, value, bound)
    tail = ref.z <= -1
    u = 2.0 ** -24
    rel = 2 * ref.e_z + u * (2 * ref.z.abs() + 8) + torch.finfo(DT[dt]).eps / 2 * 1.01
    tiny = {"bf16": 88 * 2.0 ** -126, "f32": 88 * 2.0 ** -126, "f16": 2.0 ** -24}[dt]
    # (below the normal range, and where e_z is no small change: nothing to say)
    here = tail & (ref.e_z < 0.1)
    err = (y.cpu().double() - value).abs()
    assert bool((err <= rel * value.abs() * 1.2 + tiny)[here].all())
    outs = ref.backward(dy, 60)
    got = nat.layer_norm_backward(dy, x, st, w, b, silu=True)
    for name, g, (val, bnd), t in zip(("dx", "dweight", "dbias"), got, outs, (x, w, b)):
        if float(val.abs().max()) < torch.finfo(t.dtype).max / 2:
            check(name, g, val, bnd, t.dtype)
        else:
            assert not bool(g.isnan().any())


@pytest.mark.parametrize("c", [24, 200, 1024, 3000])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_gradients_of_rows_that_are_not_finite(spc, dev, dt, c):
    """An infinity or a NaN in a row or its gradient stays in that row's dx and
    that item's sums."""
    nat = spc._native
    n, offsets = 90, [0, 30, 33, 70, 90]
    x, dy = _randn(1, n, c).to(DT[dt]).to(dev), _randn(2, n, c).to(DT[dt]).to(dev)
    sc, sh = (0.3 * _randn(3, 4, c)).to(dev), (0.3 * _randn(4, 4, c)).to(dev)
    kw = dict(scale=sc, shift=sh, offsets=torch.tensor(offsets, device=dev), silu=True)

    def run():
        _, st = nat.layer_norm(x, return_stats=True, **kw)
        return nat.layer_norm_backward(dy, x, st, **kw)

    want = run()
    x[5, c - 1], x[31, 0], dy[40, 3], dy[41, 7] = (float(v) for v in ("inf", "nan", "nan", "-inf"))
    dx, _, _, ds, dh = run()
    bad = [5, 31, 40, 41]
    keep = [i for i in range(n) if i not in bad]
    assert torch.equal(dx[keep], want[0][keep])
    assert not bool(dx[bad].isfinite().all(1).any())
    for g, w in ((ds, want[3]), (dh, want[4])):
        assert torch.equal(g[3], w[3])
        assert not bool(g[:3].isfinite().all(1).any())


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_every_gradient_of_the_most_items(spc, dev, dt):
    """65,535 items, most of them empty: dx, and each item's sums in its place."""
    nat = spc._native
    nb, n, c = 65_535, 3000, 40
    cuts = torch.randint(0, n + 1, (nb - 1,), generator=torch.Generator().manual_seed(1)).sort().values
    off = torch.cat([torch.tensor([3]), cuts.clamp(3, n - 5), torch.tensor([n - 5])])
    x, dy = _randn(2, n, c).to(DT[dt]).to(dev), _randn(3, n, c).to(DT[dt]).to(dev)
    sc, sh = (0.3 * _randn(4, nb, c)).to(dev), (0.3 * _randn(5, nb, c)).to(dev)
    kw = dict(scale=sc, shift=sh, offsets=off.to(dev), silu=True)
    y, st = nat.layer_norm(x, return_stats=True, **kw)
    dx, _, _, ds, dh = nat.layer_norm_backward(dy, x, st, **kw)
    rows = off[1:] - off[:-1]
    some = rows.nonzero()[:, 0]
    assert 1000 < some.numel() < 3000
    item = torch.full((n,), -1)
    item[3:n - 5] = torch.repeat_interleave(torch.arange(some.numel()), rows[some])
    ref = Reference(x, None, None, 1e-6, sc[some], sh[some], item, True)
    check("y", y, *ref.forward())
    outs = ref.backward(dy, 60)
    check("dx", dx, *outs[0], DT[dt])
    check("dscale", ds[some], *outs[3], torch.float32)
    check("dshift", dh[some], *outs[4], torch.float32)
    assert all(bool((g.cpu()[rows == 0] == 0).all()) for g in (ds, dh))


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,c", [(16, 72), (333, 192), (5000, 101), (30_000, 1024)])
def test_sums_of_whole_gradients_are_exact(spc, dev, dt, n, c):
    """dbias and dshift of whole numbers up to 128: sums below 2^24, whatever
    their order, and dweight of rows whose h is +-1 (half the channels each)."""
    nat = spc._native
    dy = torch.randint(-128, 129, (n, c), generator=torch.Generator().manual_seed(n)).to(DT[dt])
    sign = (2.0 * (torch.arange(c) % 2) - 1).expand(n, c)
    x = (sign * 2.0 ** (torch.arange(n)[:, None] % 5)).to(DT[dt])
    w, b = torch.ones(c, device=dev), torch.zeros(c, device=dev)
    _, st = nat.layer_norm(x.to(dev), w, b, 0.0, return_stats=True)
    _, dw, db, _, _ = nat.layer_norm_backward(dy.to(dev), x.to(dev), st, w, b)
    assert torch.equal(db.cpu(), dy.float().sum(0))
    if c % 2 == 0:
        assert torch.equal(dw.cpu(), (dy.float() * sign).sum(0))
    cuts = [0, n // 3, n // 3, n]
    mod = torch.zeros(3, c, device=dev)
    dh = nat.layer_norm_backward(dy.to(dev), x.to(dev), st, scale=mod, shift=mod,
                                 offsets=torch.tensor(cuts, device=dev))[4]
    want = torch.stack([dy[lo:hi].float().sum(0) for lo, hi in zip(cuts, cuts[1:])])
    assert torch.equal(dh.cpu(), want)
