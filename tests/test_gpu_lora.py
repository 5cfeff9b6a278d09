"""spc_lora and spc_lora_backward against their 64-bit form (lora_reference):
ranks, widths, layouts of items, adapters out of order and missing, strides,
dropout, values that are not finite, streams, graphs, refusals."""
import pytest
import torch

from lora_reference import Adapters, adapter_of_rows, factors
from norm_reference import check

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SEED = [0xFEDCBA987654321, 12]


class Case:
    def __init__(self, dev, dt, n, c, o, r, k=1, offsets=None, adapters=None, p=0.0, base=True, scale=True, seed=0):
        g = torch.Generator().manual_seed(seed + n + 3 * c + 5 * o + 7 * r)
        f = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        t = DT[dt]
        self.x = (f(n, c) * (0.5 + f(c).abs())).to(t).to(dev)
        self.down = (f(k, r, c) * c ** -0.5).to(t).to(dev)
        self.up = (f(k, o, r) * 0.2).to(t).to(dev)
        self.dy = f(n, o).to(t).to(dev)
        self.base = f(n, o).to(t).to(dev) if base else None
        self.dx_base = f(n, c).to(t).to(dev) if base else None
        self.kw = dict(scale=(1 + f(k).abs()).to(dev) if scale else None,
                       offsets=None if offsets is None else torch.tensor(offsets, device=dev),
                       adapters=None if adapters is None else torch.tensor(adapters, dtype=torch.int32, device=dev),
                       p=p, seed=torch.tensor(SEED, device=dev) if p else None)
        self.name = f"{dt} {n}x{c}->{o} r{r}"

    def reference(self):
        kw = dict(self.kw)
        kw["seed"] = SEED
        return Adapters(self.x, self.down, self.up, **kw)

    def check(self, nat, backward=True):
        ref = self.reference()
        y, h = nat.lora(self.x, self.down, self.up, self.base, return_hidden=True, **self.kw)
        want_y, want_h = ref.forward(self.base)
        check(f"y {self.name}", y, *want_y)
        check(f"hidden {self.name}", h, *want_h)
        assert torch.equal(nat.lora(self.x, self.down, self.up, self.base, **self.kw), y)
        if not backward:
            return
        grads = nat.lora_backward(self.dy, self.x, h, self.down, self.up, self.dx_base, **self.kw)
        for name, got, want in zip(("dx", "ddown", "dup"), grads, ref.backward(self.dy, h, self.dx_base)):
            check(f"{name} {self.name}", got, *want)
        again = nat.lora_backward(self.dy, self.x, h, self.down, self.up, self.dx_base, **self.kw)
        assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("n,c,o,r", [
    (1, 1, 1, 1), (1, 1024, 2048, 16), (1, 8, 8, 4), (2, 33, 65, 3), (15, 128, 128, 16), (16, 64, 256, 8), (17, 101, 77, 5),
    (33, 512, 96, 32), (64, 257, 1030, 64), (100, 192, 192, 128), (65, 96, 40, 127), (333, 130, 200, 17),
    (1000, 256, 129, 16), (2100, 72, 136, 33), (7, 8200, 40, 16), (9, 40, 16_400, 2)])
@pytest.mark.parametrize("dt", list(DT))
def test_one_adapter(spc, dev, dt, n, c, o, r):
    Case(dev, dt, n, c, o, r).check(spc._native)
    Case(dev, dt, n, c, o, r, base=False, scale=False, p=0.3, seed=1).check(spc._native)


LAYOUTS = {
    "rows": (list(range(41)), [(7 * i) % 5 - 1 for i in range(40)], 40),
    "behind": ([3, 20, 20, 21, 60], [2, 0, 3, 1], 75),
    "none": ([0, 30, 64], [-1, -5], 64),
    "outside": ([0, 30, 64, 70], [4, 1, 2 ** 31 - 1], 70),
    "same": ([0, 10, 33, 50, 90], [1, 1, 1, 1], 90),
    "empty": ([5, 5, 5], [0, 1], 9),
    "uneven": ([0, 1, 300, 301, 1200], [3, 0, 3, 2], 1203),
    "many": (list(range(0, 1001, 5)), [i % 4 for i in range(200)], 1000),
    "beyond": ([0, 50, 900], [0, 2], 70),
    "before": ([-20, 10, 40], [3, 1], 40),
}


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("c,o,r", [(96, 160, 16), (75, 130, 20), (264, 72, 64)])
def test_items(spc, dev, dt, layout, c, o, r):
    off, ids, n = LAYOUTS[layout]
    Case(dev, dt, n, c, o, r, k=4, offsets=off, adapters=ids).check(spc._native)
    Case(dev, dt, n, c, o, r, k=4, offsets=off, adapters=ids, p=0.2, base=False).check(spc._native)


@pytest.mark.parametrize("n,k", [(40, 40), (7, 7), (60, 3), (2000, 4), (1, 1), (128, 64)])
@pytest.mark.parametrize("dt", list(DT))
def test_items_of_equal_rows(spc, dev, dt, n, k):
    """Without offsets, as with them."""
    nat, ids = spc._native, [(3 * i + 1) % 5 - 1 for i in range(k)]
    q = Case(dev, dt, n, 136, 264, 16, k=4, adapters=ids, p=0.1)
    q.check(nat)
    y, h = nat.lora(q.x, q.down, q.up, q.base, return_hidden=True, **q.kw)
    kw = {**q.kw, "offsets": torch.arange(0, n + 1, n // k, device=dev)}
    y1, h1 = nat.lora(q.x, q.down, q.up, q.base, return_hidden=True, **kw)
    assert torch.equal(y, y1) and torch.equal(h, h1)


@pytest.mark.parametrize("dt", list(DT))
def test_strides_and_alignment(spc, dev, dt):
    """Views at any element of wider rows, weights that are slices."""
    nat, t = spc._native, DT[dt]
    g = torch.Generator().manual_seed(3)
    f = lambda *s: torch.randn(*s, generator=g).to(t).to(dev)  # noqa: E731
    n, r, off, ids = 50, 12, [0, 20, 47], [1, 0]
    wide, wide_o = f(n, 400), f(n, 500)
    for c, o, at in ((96, 128, 1), (101, 77, 3), (128, 256, 8), (64, 64, 5)):
        q = Case(dev, dt, n, c, o, r, k=2, offsets=off, adapters=ids, p=0.1)
        q.x, q.dx_base = wide[:, at:at + c], wide[:, at + c:at + 2 * c]
        q.dy, q.base = wide_o[:, at:at + o], wide_o[:, 200 + at:200 + at + o]
        flat = f(2 * r * (c + o) + 9)
        q.down = flat[at:at + 2 * r * c].view(2, r, c) * 0.1
        q.up = flat[at + 2 * r * c:at + 2 * r * (c + o)].view(2, o, r)
        q.check(nat)
    q.x, q.dy = wide[:1, :64].expand(n, 64), wide_o[:1, :64].expand(n, 64)
    q.check(nat)
    q.x, q.dy = f(64, n).t(), f(64, n).t()
    q.check(nat)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dt", list(DT))
def test_values_that_are_not_finite(spc, dev, dt, bad):
    """A row that is not finite changes its own outputs and its adapter's
    gradients; one without an adapter, or an adapter that no row meets, nothing."""
    nat = spc._native
    for n, off, ids in ((90, [0, 31, 60, 80], [1, 2, 1]), (12, [0, 1, 5, 11], [1, 2, 1])):
        q = Case(dev, dt, n, 130, 90, 9, k=4, offsets=off, adapters=ids)
        y0, h0 = nat.lora(q.x, q.down, q.up, q.base, return_hidden=True, **q.kw)
        g0 = nat.lora_backward(q.dy, q.x, h0, q.down, q.up, q.dx_base, **q.kw)
        hit, free = off[1] + 1, n - 1
        q.x[[hit, free]] = bad
        q.dy[[hit, free]] = bad
        q.down[3], q.up[3] = bad, bad
        q.down[0], q.up[0] = bad, bad
        y, h = nat.lora(q.x, q.down, q.up, q.base, return_hidden=True, **q.kw)
        h1 = h.clone()
        h1[free] = bad
        g = nat.lora_backward(q.dy, q.x, h1, q.down, q.up, q.dx_base, **q.kw)
        rest = [i for i in range(n) if i != hit]
        assert torch.equal(y[rest], y0[rest]) and torch.equal(h[rest], h0[rest]) and torch.equal(g[0][rest], g0[0][rest])
        assert not y[hit].isfinite().any() and not h[hit].isfinite().any() and not g[0][hit].isfinite().any()
        for a, b in zip(g[1:], g0[1:]):
            assert torch.equal(a[[0, 1, 3]], b[[0, 1, 3]]) and not a[2].isfinite().any()


@pytest.mark.parametrize("dt", list(DT))
def test_large_values_beside_small(spc, dev, dt):
    """What a value contributes does not depend on the largest one beside it: a
    hidden value that meets zero weights leaves nothing in the others."""
    nat = spc._native
    q = Case(dev, dt, 40, 64, 96, 16, base=False, scale=False)
    big = 32.0 if dt == "f16" else 1e18   # (40 big^2 is finite)
    q.x[:, 0], q.down[0, 3], q.down[0, 3, 0] = big, 0, 1
    q.down[0, :3, 0], q.down[0, 4:, 0] = 0, 0
    q.up[0, :, 3] = 0
    q.dy[:, 5], q.up[0, 5] = big, 0
    q.up[0, 5, 7], q.down[0, 7] = 1, 0
    q.check(nat)


@pytest.mark.parametrize("r", [33, 64])
@pytest.mark.parametrize("dt", list(DT))
def test_large_tiles(spc, dev, dt, r):
    """So many rows of such ranks that a block takes 64 of them; few columns, so that the
    64-bit form is quick."""
    Case(dev, dt, 25_003, 40, 72, r, k=2, offsets=[5, 70, 12_000, 24_990], adapters=[1, -1, 0], p=0.2).check(spc._native)
    Case(dev, dt, 24_576, 33, 8, r, base=False).check(spc._native)


@pytest.mark.parametrize("c,o", [(1, 64), (4, 136), (7, 8), (8, 7), (200, 3), (520, 1), (5, 6), (1, 1)])
@pytest.mark.parametrize("dt", list(DT))
def test_narrow_rows(spc, dev, dt, c, o):
    """Of fewer elements than 16 bytes hold: strides, bases in place, few rows and many,
    nothing beside the results."""
    nat, t = spc._native, DT[dt]
    for n, off, ids in ((70, [0, 9, 40, 60], [2, 0, 1]), (900, [3, 400, 410, 880], [1, 2, -1])):
        for r in (1, 12, 40):
            q = Case(dev, dt, n, c, o, r, k=3, offsets=off, adapters=ids, p=0.25)
            q.x = torch.randn(n, c + 3, device=dev).to(t)[:, 1:1 + c]
            q.dy = torch.randn(n, o + 2, device=dev).to(t)[:, 2:]
            q.check(nat)
            y, h = nat.lora(q.x, q.down, q.up, q.base, return_hidden=True, **q.kw)
            buf = torch.full((n + 2, o), 7.0, dtype=t, device=dev)
            buf[1:-1] = q.base
            nat.lora(q.x, q.down, q.up, buf[1:-1], out=buf[1:-1], **q.kw)
            assert torch.equal(buf[1:-1], y) and (buf[[0, -1]] == 7).all()
            whole = nat.lora_backward(q.dy, q.x, h, q.down, q.up, q.dx_base, **q.kw)
            for i in range(3):
                need = [i == k for k in range(3)]
                part = nat.lora_backward(q.dy, q.x, h, q.down, q.up, q.dx_base, need=need, **q.kw)
                assert torch.equal(part[i], whole[i]) and [p is None for p in part] == [not k for k in need]


@pytest.mark.parametrize("n,rows,k", [(600, 5, 8), (600, 5, 3), (700, 1, 3), (512, 8, 8), (512, 32, 8), (2000, 2, 8)])
@pytest.mark.parametrize("dt", list(DT))
def test_many_short_items(spc, dev, dt, n, rows, k):
    """Few and many adapters, whose rows lie all over."""
    ids = [(i * i + i // 7) % (k + 1) - 1 for i in range(n // rows)]
    off = list(range(0, n // rows * rows + 1, rows))
    Case(dev, dt, n, 136, 72, 16, k=k, offsets=off, adapters=ids).check(spc._native)
    Case(dev, dt, n, 75, 136, 40, k=k, offsets=off, adapters=ids, p=0.2).check(spc._native)


@pytest.mark.parametrize("k", [3, 20])
@pytest.mark.parametrize("dt", list(DT))
def test_many_rows_without_an_adapter(spc, dev, dt, k):
    """Hundreds of them in short items, gathered in several rounds, and behind the
    items."""
    n = 900
    q = Case(dev, dt, n, 70, 200, 12, k=k, offsets=list(range(10, 811, 20)),
             adapters=[i // 13 if i % 13 == 0 and i < 39 else -1 for i in range(40)], p=0.3)
    q.check(spc._native)
    dx = spc._native.lora_backward(q.dy, q.x, None, q.down, q.up, q.dx_base, need=(1, 0, 0), **q.kw)[0]
    rest = (adapter_of_rows(n, k, q.kw["offsets"], q.kw["adapters"]) < 0).to(dev)
    assert int(rest.sum()) == 840 and torch.equal(dx[rest], q.dx_base[rest])


def test_more_elements_than_32_bits_count(spc, dev):
    """Rows past 2^31 elements of x, dy, dx and y are as in calls of their own; the
    gradients are those of the rows that are not zero."""
    nat = spc._native
    g = torch.Generator().manual_seed(1)
    n, c, r = (1 << 21) + 77, 1040, 8
    f = lambda *s: torch.randn(*s, generator=g).bfloat16().to(dev)  # noqa: E731
    down, up = f(2, r, c) * 0.03, f(2, c, r) * 0.3
    ids = torch.tensor([1, -1, 0], dtype=torch.int32, device=dev)
    off = torch.tensor([0, 100, n - 90, n - 3], device=dev)
    x = torch.zeros((n, c), dtype=torch.bfloat16, device=dev)
    x[:100], x[n - 90:] = f(100, c), f(90, c)
    kw = dict(adapters=ids, p=0.25, seed=torch.tensor(SEED, device=dev))
    y, h = nat.lora(x, down, up, x, offsets=off, return_hidden=True, **kw)
    dx, dd, du = nat.lora_backward(x, x, h, down, up, x, offsets=off, **kw)
    for rows, a, first in ((slice(0, 100), 1, 0), (slice(n - 90, n - 3), 0, n - 90)):
        k = rows.stop - rows.start
        q = Adapters(x[rows], down[a:a + 1], up[a:a + 1])
        q.f = factors(SEED, k, c, 0.25, first=first)
        q.x = q.x * q.f
        (wy, ey), (wh, eh) = q.forward(x[rows])
        check("y", y[rows], wy, ey), check("hidden", h[rows], wh, eh)
        (wx, ex), (wd, ed), (wu, eu) = q.backward(x[rows], h[rows], x[rows])
        check("dx", dx[rows], wx, ex), check("ddown", dd[a:a + 1], wd, ed), check("dup", du[a:a + 1], wu, eu)
    for t in (y, dx):
        assert torch.equal(t[n - 3:], x[n - 3:]) and not t[100:n - 90].any()
    assert not h[100:n - 90].any() and not h[n - 3:].any()


def test_in_place_and_partial_gradients(spc, dev):
    nat = spc._native
    for n in (9, 400):
        q = Case(dev, "bf16", n, 96, 80, 8, k=2, offsets=[0, n // 2, n - 2], adapters=[1, 0], p=0.1)
        want = nat.lora(q.x, q.down, q.up, q.base, **q.kw)
        y, h = nat.lora(q.x, q.down, q.up, q.base, return_hidden=True, out=q.base, **q.kw)
        assert torch.equal(y, want) and y.data_ptr() == q.base.data_ptr()
        full = nat.lora_backward(q.dy, q.x, h, q.down, q.up, q.dx_base, **q.kw)
        for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (0, 1, 1), (1, 0, 1), (0, 0, 0)):
            part = nat.lora_backward(q.dy, q.x, h if need[2] else None, q.down, q.up, q.dx_base, need=need, **q.kw)
            for a, b, on in zip(part, full, need):
                assert (a is None) if not on else torch.equal(a, b)


def test_no_rows(spc, dev):
    nat = spc._native
    q = Case(dev, "bf16", 4, 32, 16, 4, k=3, offsets=[0, 0, 0], adapters=[1, 2])
    y, h = nat.lora(q.x[:0], q.down, q.up, q.base[:0], return_hidden=True, **q.kw)
    assert y.shape == (0, 16) and h.shape == (0, 4)
    dx, dd, du = nat.lora_backward(q.dy[:0], q.x[:0], h, q.down, q.up, **q.kw)
    assert dx.shape == (0, 32) and not dd.any() and not du.any()


def test_dropout_is_the_operators_own(spc, dev):
    """lora(x, p) is lora(dropout(x)) in F32, where the factor is rounded alike
    (1 / (1 - p) a power of two, so exactly)."""
    nat = spc._native
    for n in (5, 300):
        q = Case(dev, "f32", n, 200, 60, 8, p=0.5)
        d = nat.dropout(q.x, 0.5, q.kw["seed"])
        kw = {**q.kw, "p": 0.0}
        y, h = nat.lora(q.x, q.down, q.up, q.base, return_hidden=True, **q.kw)
        y1, h1 = nat.lora(d, q.down, q.up, q.base, return_hidden=True, **kw)
        assert torch.equal(y, y1) and torch.equal(h, h1)
        dx, dd, du = nat.lora_backward(q.dy, q.x, h, q.down, q.up, **q.kw)
        dx1, dd1, du1 = nat.lora_backward(q.dy, d, h, q.down, q.up, **kw)
        assert torch.equal(dx, nat.dropout(dx1, 0.5, q.kw["seed"])) and torch.equal(dd, dd1) and torch.equal(du, du1)


def test_gradient_agrees_with_differences(spc, dev):
    """Along a direction, in F32: (y(t) - y(-t)) / 2t . dy, y trilinear, so a
    difference with t = 1/4 is off by t^2 of the triple product alone, which the
    64-bit form gives; both sums are off by what the bounds of y and of the
    gradients add up to."""
    nat = spc._native
    q = Case(dev, "f32", 60, 80, 50, 6, k=2, offsets=[0, 25, 58], adapters=[1, 0], p=0.25, base=False)
    g = torch.Generator().manual_seed(5)
    d = [torch.randn(t.shape, generator=g).to(dev) * s for t, s in ((q.x, 1), (q.down, 0.1), (q.up, 0.1))]
    t = 0.25

    def at(t):
        a = [v + t * w for v, w in zip((q.x, q.down, q.up), d)]
        y = nat.lora(*a, **q.kw)
        r = Adapters(*a, **{**q.kw, "seed": SEED})
        e = float((r.forward()[0][1] * q.dy.cpu().double().abs()).sum())
        return float((y.double() * q.dy.double()).sum()), e

    (up, e1), (dn, e2) = at(t), at(-t)
    h = nat.lora(q.x, q.down, q.up, return_hidden=True, **q.kw)[1]
    grads = nat.lora_backward(q.dy, q.x, h, q.down, q.up, **q.kw)
    slope = sum(float((a.double() * b.double()).sum()) for a, b in zip(grads, d))
    e3 = sum(float((b[1] * w.cpu().double().abs()).sum()) for b, w in zip(q.reference().backward(q.dy, h), d))
    triple = Adapters(*d, **{**q.kw, "seed": SEED}).forward()[0][0]
    cubic = t * t * float((triple * q.dy.cpu().double()).sum())
    assert abs((up - dn) / (2 * t) - slope - cubic) <= (e1 + e2) / (2 * t) + e3


def test_streams_and_graphs(spc, dev):
    """On another stream as on the current one; a captured pass replayed on new
    inputs, another capture beside it, with eager work between."""
    nat = spc._native
    for n, off in ((6, [0, 1, 3, 6]), (500, [0, 100, 250, 480])):
        q = Case(dev, "bf16", n, 136, 72, 16, k=3, offsets=off, adapters=[2, 0, 1], p=0.1)

        def run():
            y, h = nat.lora(q.x, q.down, q.up, q.base, return_hidden=True, **q.kw)
            return (y, h, *nat.lora_backward(q.dy, q.x, h, q.down, q.up, q.dx_base, **q.kw))

        want = run()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = run()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                graphs.append((g, run()))
        for i in range(4):
            q.x.copy_(torch.randn(n, 136))
            q.dy.copy_(torch.randn(n, 72))
            q.kw["adapters"].copy_(torch.tensor([(i + 1) % 4 - 1, 1, i % 3], dtype=torch.int32))
            q.kw["seed"].copy_(torch.tensor([i, 9]))
            for g, _ in graphs:
                g.replay()
            torch.cuda.synchronize()
            want = run()
            for _, got in graphs:
                assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(spc, dev):
    nat = spc._native
    q = Case(dev, "bf16", 6, 32, 24, 4, k=2, offsets=[0, 2, 6], adapters=[0, 1], p=0.1)
    h = nat.lora(q.x, q.down, q.up, return_hidden=True, **q.kw)[1]
    kw = q.kw
    bad = [dict(adapters=None), dict(adapters=kw["adapters"].long()), dict(offsets=None, adapters=torch.zeros(4, dtype=torch.int32, device=dev)), dict(offsets=kw["offsets"][:2]),
           dict(offsets=kw["offsets"].int()), dict(scale=kw["scale"][:1]), dict(scale=kw["scale"].half()),
           dict(seed=None), dict(p=2.0), dict(seed=kw["seed"].cpu())]
    for b in bad:
        with pytest.raises(ValueError):
            nat.lora(q.x, q.down, q.up, **{**kw, **b})
        with pytest.raises(ValueError):
            nat.lora_backward(q.dy, q.x, h, q.down, q.up, **{**kw, **b})
    for args in ((q.x[:, :30], q.down, q.up), (q.x, q.down.float(), q.up), (q.x, q.down[:1], q.up), (q.x, q.down[:, :3], q.up),
                 (q.x, q.down[0], q.up), (q.x, q.down, q.up, q.base[:3]), (q.x, q.down, q.up, q.base.float())):
        with pytest.raises(ValueError):
            nat.lora(*args, **kw)
    for args in ((q.dy[:3], q.x, h, q.down, q.up), (q.dy.float(), q.x, h, q.down, q.up), (q.dy, q.x, h[:, :2], q.down, q.up),
                 (q.dy, q.x, h.half(), q.down, q.up), (q.dy, q.x, None, q.down, q.up),
                 (q.dy, q.x, h, q.down, q.up, q.dx_base[:, :9])):
        with pytest.raises(ValueError):
            nat.lora_backward(*args, **kw)
    flat = torch.zeros(6 * 24 + 8, dtype=torch.bfloat16, device=dev)
    with pytest.raises(ValueError, match="apart"):
        nat.lora(q.x, q.down, q.up, flat[8:].view(6, 24), out=flat[:-8].view(6, 24), **kw)
    big = torch.zeros(1, 129, 32, dtype=torch.bfloat16, device=dev)
    with pytest.raises(nat.SparseConvError):
        nat.lora(q.x, big, torch.zeros(1, 24, 129, dtype=torch.bfloat16, device=dev))
    with pytest.raises(TypeError):
        nat.lora(q.x.double(), q.down.double(), q.up.double(), **kw)


def test_reference_maps_rows():
    assert adapter_of_rows(6, 2, [-3, 1, 9], [1, 0]).tolist() == [1, 0, 0, 0, 0, 0]
