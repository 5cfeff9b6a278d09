"""The general row layer norm and its gradient (nat.layer_norm,
nat.layer_norm_backward, SparseLayerNorm32) against 64 bits.  Bounds:
tests/norm_reference.py."""
import copy

import pytest
import torch

from norm_reference import Reference, check

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# widths on both sides of every team width, odd and even, whole and broken vectors
WIDTHS = [1, 2, 3, 7, 8, 24, 32, 33, 64, 100, 101, 127, 128, 130, 192, 256, 513, 768, 1000, 1024,
          1025, 2048, 2050, 4096, 5003, 8192]


def _inputs(dev, dt, n, c, seed, items=0, affine=True, mdt=None, pdt=torch.float32):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = (r(n, c) * (0.5 + r(c).abs()) + 0.5 * r(c) + 0.3).to(dt)
    w = (1 + 0.2 * r(c)).to(pdt) if affine else None
    b = (0.2 * r(c)).to(pdt) if affine else None
    scale = shift = None
    if items:
        mod = (0.3 * r(items, 2 * c)).to(mdt or dt).to(dev)
        scale, shift = mod[:, :c], mod[:, c:]
    dy = r(n, c).to(dt)
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    return to(x), to(w), to(b), scale, shift, to(dy)


def _items(offsets, n):
    item = torch.full((n,), -1, dtype=torch.int64)
    for i, (lo, hi) in enumerate(zip(offsets, offsets[1:])):
        item[lo:hi] = i
    return item


def _run(nat, dev, name, x, w, b, scale, shift, dy, offsets=None, silu=False, eps=1e-6):
    n, c = x.shape
    off = None if offsets is None else torch.tensor(offsets, dtype=torch.int64, device=dev)
    kw = dict(scale=scale, shift=shift, offsets=off, silu=silu)
    y, stats = nat.layer_norm(x, w, b, eps, return_stats=True, **kw)
    grads = nat.layer_norm_backward(dy, x, stats, w, b, **kw)
    torch.cuda.synchronize()
    ref = Reference(x, w, b, eps, scale, shift, None if offsets is None else _items(offsets, n), silu)
    check(f"{name} y", y, *ref.forward())
    # a row's way into a sum: the rounds of a block's team (512 blocks of at
    # least one row), its lanes and waves (10), its share of 512 chunks (8)
    # and a tree (5)
    outs = ref.backward(dy, -(-n // 512) + 50)
    want = [True, w is not None, b is not None, scale is not None, scale is not None]
    for gname, on, got, (val, bound), t in zip(("dx", "dweight", "dbias", "dscale", "dshift"), want,
                                               grads, outs, (x, w, b, scale, shift)):
        if not on:
            assert got is None
            continue
        assert got.dtype == t.dtype
        check(f"{name} {gname}", got, val, bound, t.dtype)
    return y, stats, grads


@pytest.mark.parametrize("c", WIDTHS)
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_widths(spc, dev, dt, c):
    x, w, b, _, _, dy = _inputs(dev, DT[dt], 37, c, c)
    _run(spc._native, dev, f"affine {dt} c={c}", x, w, b, None, None, dy)
    x, w, b, sc, sh, dy = _inputs(dev, DT[dt], 41, c, c + 1, items=3, affine=False)
    _run(spc._native, dev, f"mod silu {dt} c={c}", x, None, None, sc, sh, dy, [0, 5, 20, 41], True)


@pytest.mark.parametrize("n", [1, 2, 3, 15, 16, 17, 64, 1023, 4097, 30_011])
@pytest.mark.parametrize("dt,c", [("bf16", 128), ("f32", 96), ("f16", 1024)])
def test_rows(spc, dev, dt, c, n):
    x, w, b, _, _, dy = _inputs(dev, DT[dt], n, c, n)
    _run(spc._native, dev, f"{dt} n={n} c={c}", x, w, b, None, None, dy, silu=n % 2 == 0)


@pytest.mark.parametrize("offsets", [
    [0, 700],
    [0, 0, 1, 1, 2, 700],               # empty items between
    [0, 333, 333, 700, 700, 700],       # and at the end
    [13, 40, 41, 600],                  # rows before the first and behind the last
    [0, 0, 0],                          # nothing but empty items
    [700, 700],
    list(range(0, 701, 7)),             # an item in every few rows
])
@pytest.mark.parametrize("c", [40, 512, 2048])
def test_items(spc, dev, offsets, c):
    """Affine and modulated at once: all five gradients."""
    nb = len(offsets) - 1
    x, w, b, sc, sh, dy = _inputs(dev, torch.bfloat16, 700, c, nb, items=nb, mdt=torch.float32)
    y, stats, g = _run(spc._native, dev, f"{nb} items c={c}", x, w, b, sc, sh, dy, offsets, True)
    out = _items(offsets, 700) < 0
    assert bool((y.cpu()[out] == 0).all()) and bool((g[0].cpu()[out] == 0).all())
    assert bool((stats.cpu()[out] == 0).all())


def test_many_items(spc, dev):
    """More items than rows, and the most there can be."""
    nb, n, c = 65_535, 300, 16
    offsets = [min(i // 100, n) for i in range(nb)] + [n]
    x, _, _, sc, sh, dy = _inputs(dev, torch.float32, n, c, 5, items=nb, affine=False)
    off = torch.tensor(offsets, device=dev)
    nat = spc._native
    y, st = nat.layer_norm(x, scale=sc, shift=sh, offsets=off, return_stats=True)
    dx, _, _, ds, dh = nat.layer_norm_backward(dy, x, st, scale=sc, shift=sh, offsets=off)
    item = _items(offsets, n)
    ref = Reference(x, None, None, 1e-6, sc, sh, item)
    check("y", y, *ref.forward())
    want = torch.zeros((nb, c), dtype=torch.float64).index_add_(0, item, dy.cpu().double())
    check("dshift", dh, want, want.abs() * 2.0 ** -20 + 2.0 ** -20, torch.float32)
    assert ds.shape == (nb, c) and bool((ds.cpu()[want.abs().sum(1) == 0] == 0).all())


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("given", ["none", "weight", "bias", "mod f32", "affine bf16"])
def test_parameters(spc, dev, dt, given):
    pdt = torch.bfloat16 if given == "affine bf16" else torch.float32
    x, w, b, sc, sh, dy = _inputs(dev, DT[dt], 130, 72, 3, items=1, mdt=torch.float32, pdt=pdt)
    if given != "mod f32":
        sc = sh = None
    if given in ("none", "bias", "mod f32"):
        w = None
    if given in ("none", "weight", "mod f32"):
        b = None
    _run(spc._native, dev, f"{given} {dt}", x, w, b, sc, sh, dy, silu=True)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_strided_and_offset_rows(spc, dev, dt):
    """Views: column ranges at any element, every other row, broadcast and
    transposed gradients, parameters at odd elements."""
    nat = spc._native
    base, w, b, _, _, dyb = _inputs(dev, DT[dt], 90, 301, 8)
    for c0, c, step in [(0, 128, 1), (8, 128, 1), (1, 128, 1), (2, 100, 2), (3, 77, 3)]:
        x, dy = base[::step, c0:c0 + c], dyb[::step, c0 + 1:c0 + 1 + c]
        _run(nat, dev, f"{dt} cols {c0}+{c} step {step}", x, w[c0:c0 + c], b[c0 + 1:c0 + 1 + c], None,
             None, dy)
    x = base[:, :64].contiguous()
    one = dyb[:1, :64].expand(90, 64)
    _run(nat, dev, f"{dt} broadcast dy", x, w[:64], b[:64], None, None, one)
    _run(nat, dev, f"{dt} transposed", dyb[:64, :90].t(), w[:64], b[:64], None, None,
         base[:64, :90].t())


def test_in_place_and_out(spc, dev):
    nat = spc._native
    x, w, b, _, _, dy = _inputs(dev, torch.bfloat16, 501, 256, 1)
    want, st = nat.layer_norm(x, w, b, return_stats=True)
    out = torch.empty_like(x)
    assert nat.layer_norm(x, w, b, out=out) is out and torch.equal(out, want)
    y = x.clone()
    assert nat.layer_norm(y, w, b, out=y) is y and torch.equal(y, want)


def test_overlapping_out_is_refused(spc, dev):
    nat = spc._native
    buf = torch.randn(40, 64, device=dev)
    for x, out in [(buf[1:], buf[:-1]), (buf[:20, :32], buf.view(-1)[:640].view(20, 32))]:
        with pytest.raises(ValueError, match="apart"):
            nat.layer_norm(x, out=out)
    a, b = buf[:20], buf[20:]
    assert torch.equal(nat.layer_norm(a, out=b), nat.layer_norm(a))


def test_padding_rows_do_not_matter(spc, dev):
    """Rows of no item: whatever they hold (NaN here) reaches neither the
    others nor a sum."""
    nat = spc._native
    n, c = 300, 136
    x, w, b, sc, sh, dy = _inputs(dev, torch.bfloat16, n, c, 2, items=3)
    offsets = [20, 100, 100, 250]
    kw = dict(scale=sc, shift=sh, offsets=torch.tensor(offsets, device=dev), silu=True)
    y, st = nat.layer_norm(x, w, b, return_stats=True, **kw)
    g = nat.layer_norm_backward(dy, x, st, w, b, **kw)
    out = _items(offsets, n) < 0
    x[out.to(dev)] = float("nan")
    dy[out.to(dev)] = float("inf")
    y2, st2 = nat.layer_norm(x, w, b, return_stats=True, **kw)
    g2 = nat.layer_norm_backward(dy, x, st2, w, b, **kw)
    assert all(torch.equal(p, q) for p, q in zip((y, st, *g), (y2, st2, *g2)))


def test_equal_calls_equal_bits(spc, dev):
    nat = spc._native
    x, w, b, sc, sh, dy = _inputs(dev, torch.bfloat16, 5000, 320, 1, items=3)
    off = torch.tensor([0, 1700, 1701, 5000], device=dev)
    kw = dict(scale=sc, shift=sh, offsets=off, silu=True)
    _, st = nat.layer_norm(x, w, b, return_stats=True, **kw)
    first = nat.layer_norm_backward(dy, x, st, w, b, **kw)
    for _ in range(3):
        for p, q in zip(first, nat.layer_norm_backward(dy, x, st, w, b, **kw)):
            assert torch.equal(p, q)


def test_empty(spc, dev):
    nat = spc._native
    x, w, b, sc, sh, dy = _inputs(dev, torch.float32, 0, 64, 1, items=2)
    off = torch.zeros(3, dtype=torch.int64, device=dev)
    y, st = nat.layer_norm(x, w, b, scale=sc, shift=sh, offsets=off, return_stats=True)
    g = nat.layer_norm_backward(dy, x, st, w, b, scale=sc, shift=sh, offsets=off)
    assert y.shape == (0, 64) and st.shape == (0, 2) and g[0].shape == (0, 64)
    assert all(bool((t == 0).all()) for t in g[1:])


def test_need(spc, dev):
    nat = spc._native
    x, w, b, sc, sh, dy = _inputs(dev, torch.bfloat16, 70, 64, 1, items=1)
    kw = dict(scale=sc, shift=sh)
    _, st = nat.layer_norm(x, w, b, return_stats=True, **kw)
    every = nat.layer_norm_backward(dy, x, st, w, b, **kw)
    for bits in range(32):
        need = [bool(bits >> i & 1) for i in range(5)]
        got = nat.layer_norm_backward(dy, x, st, w, b, need=need, **kw)
        for k, p, q in zip(need, got, every):
            assert (p is None) if not k else torch.equal(p, q)


@pytest.mark.parametrize("n", [1, 4, 5, 30])
@pytest.mark.parametrize("c", [8, 72, 600, 1024, 2048, 3000, 8192])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_few_rows(spc, dev, dt, c, n):
    """Calls that one block takes, whose sums are the gradients, and their
    neighbours."""
    nat = spc._native
    x, w, b, _, _, dy = _inputs(dev, DT[dt], n, c, n)
    _run(nat, dev, f"{dt} {n}x{c}", x, w, b, None, None, dy)
    wanted = nat.layer_norm_backward(dy, x, nat.layer_norm(x, w, b, return_stats=True)[1], w, b)
    for need in [(0, 1, 0), (0, 0, 1), (1, 0, 1), (1, 1, 0)]:
        got = nat.layer_norm_backward(dy, x, nat.layer_norm(x, w, b, return_stats=True)[1], w, b,
                                      need=(*need, 1, 1))
        assert got[3:] == (None, None)
        for k, p, q in zip(need, got, wanted):
            assert (p is None) if not k else torch.equal(p, q)
    x, _, _, sc, sh, dy = _inputs(dev, DT[dt], n, c, n + 1, items=1, affine=False)
    _run(nat, dev, f"{dt} mod {n}x{c}", x, None, None, sc, sh, dy, silu=True)
    _run(nat, dev, f"{dt} mod offsets {n}x{c}", x, None, None, sc, sh, dy, [0, n], silu=True)
    _run(nat, dev, f"{dt} empty item {n}x{c}", x, None, None, sc, sh, dy, [0, 0], silu=True)


def test_large_offset_and_special_rows(spc, dev):
    """Rows far from zero; a constant row; rows with an infinity or a NaN stay
    alone with it."""
    nat = spc._native
    x, w, b, _, _, dy = _inputs(dev, torch.float32, 64, 256, 2)
    _run(nat, dev, "far", x + 1000.0, w, b, None, None, dy)
    x[3] = 2.5
    _run(nat, dev, "constant row", x, w, b, None, None, dy)
    clean = nat.layer_norm(x, w, b)
    x[5, 7], x[9, 0] = float("inf"), float("nan")
    y = nat.layer_norm(x, w, b)
    bad = torch.zeros(64, dtype=torch.bool, device=dev)
    bad[5] = bad[9] = True
    assert torch.equal(y[~bad], clean[~bad])
    assert bool(y[bad].isnan().any(1).all())


def test_gradient_against_differences(spc, dev):
    """Central differences of the 64-bit forward pass, element by element
    (h = 1e-5: truncation below 1e-8, rounding below 1e-10 a step), within the
    F32 bounds."""
    nat = spc._native
    n, c, nb = 5, 11, 2
    x, w, b, sc, sh, dy = _inputs(dev, torch.float32, n, c, 4, items=nb)
    offsets = [0, 2, 5]
    off = torch.tensor(offsets, device=dev)
    item = _items(offsets, n)
    kw = dict(scale=sc, shift=sh, offsets=off, silu=True)
    _, st = nat.layer_norm(x, w, b, return_stats=True, **kw)
    got = nat.layer_norm_backward(dy, x, st, w, b, **kw)
    bounds = Reference(x, w, b, 1e-6, sc, sh, item, True).backward(dy, 60)
    args = [t.detach().cpu().double() for t in (x, w, b, sc, sh)]
    dy64 = dy.cpu().double()

    def loss():
        r = Reference(args[0], args[1], args[2], 1e-6, args[3], args[4], item, True)
        return float((r.z * r.sg * dy64).sum())

    for i, (g, (_, bound)) in enumerate(zip(got, bounds)):
        num = torch.empty_like(args[i])
        flat, out = args[i].view(-1), num.view(-1)
        for j in range(flat.numel()):
            v = float(flat[j])
            flat[j] = v + 1e-5
            up = loss()
            flat[j] = v - 1e-5
            out[j] = (up - loss()) / 2e-5
            flat[j] = v
        check(f"differences {i}", g, num, bound + 1e-7, torch.float32)


def _tensor(spc, dev, feats, counts):
    rows = [torch.arange(k) for k in counts]
    coords = torch.cat([torch.stack([torch.full_like(r, i), r % 7, r // 7 % 7, r // 49], 1)
                        for i, r in enumerate(rows)]).to(torch.int32).to(dev)
    return spc.sparse.SparseTensor(feats, coords)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_module_gradients(spc, dev, dt):
    """SparseLayerNorm32 under autograd: the halves of a Linear's output as the
    modulation, gradients through the views and into the parameters."""
    c, counts = 96, [50, 1, 80]
    n = sum(counts)
    x, _, _, _, _, dy = _inputs(dev, DT[dt], n, c, 6)
    g = torch.Generator().manual_seed(9)
    mod = (0.3 * torch.randn(3, 2 * c, generator=g)).to(DT[dt]).to(dev).requires_grad_()
    ln = spc.sparse.SparseLayerNorm32(c).to(dev)
    with torch.no_grad():
        ln.weight += 0.1 * torch.randn(c, generator=g).to(dev)
        ln.bias += 0.1 * torch.randn(c, generator=g).to(dev)
    x.requires_grad_()
    t = _tensor(spc, dev, x, counts)
    scale, shift = mod.chunk(2, 1)
    y = ln(t, scale, shift, silu=True)
    assert y.coords is t.coords and y.feats.dtype == DT[dt]
    y.feats.backward(dy)
    item = torch.repeat_interleave(torch.arange(3), torch.tensor(counts))
    ref = Reference(x, ln.weight, ln.bias, 1e-6, scale, shift, item, True)
    check("y", y.feats, *ref.forward())
    (dx, bx), (dw, bw), (db, bb), (ds, bs), (dh, bh) = ref.backward(dy, 60)
    check("dx", x.grad, dx, bx, DT[dt])
    check("dweight", ln.weight.grad, dw, bw, torch.float32)
    check("dbias", ln.bias.grad, db, bb, torch.float32)
    check("dmod", mod.grad, torch.cat([ds, dh], 1), torch.cat([bs, bh], 1), DT[dt])
    with torch.no_grad():
        assert torch.equal(ln(t, scale, shift, silu=True).feats, y.feats)


def test_module_frozen_and_plain(spc, dev):
    c = 64
    x, _, _, _, _, dy = _inputs(dev, torch.bfloat16, 40, c, 6)
    ln = spc.sparse.SparseLayerNorm32(c, elementwise_affine=False)
    x.requires_grad_()
    t = _tensor(spc, dev, x, [40])
    y = ln(t)
    (dx,) = torch.autograd.grad(y.feats, x, dy)
    ref = Reference(x)
    check("dx", dx, *ref.backward(dy, 60)[0], torch.bfloat16)
    # twice differentiable it is not
    y = ln(_tensor(spc, dev, x, [40])).feats
    (gx,) = torch.autograd.grad(y, x, dy.clone().requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()


def test_other_stream(spc, dev):
    """The call runs on the current stream, behind what it reads."""
    nat = spc._native
    x, w, b, _, _, dy = _inputs(dev, torch.bfloat16, 3000, 512, 3)
    want, st = nat.layer_norm(x, w, b, return_stats=True)
    gw = nat.layer_norm_backward(dy, x, st, w, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        z = torch.zeros_like(x)
        for _ in range(10):
            z = z + x / 10
        z.copy_(x)
        y, st2 = nat.layer_norm(z, w, b, return_stats=True)
        g2 = nat.layer_norm_backward(dy, z, st2, w, b)
    s.synchronize()
    assert torch.equal(y, want) and all(torch.equal(p, q) for p, q in zip(g2[:3], gw[:3]))


def test_graph_capture(spc, dev):
    """Forward and backward captured together and replayed on new values, with
    eager work between the replays; two graphs of one shape do not share a
    workspace."""
    nat = spc._native
    x, w, b, sc, sh, dy = _inputs(dev, torch.bfloat16, 1500, 256, 3, items=2)
    off = torch.tensor([0, 600, 1500], device=dev)
    kw = dict(scale=sc, shift=sh, offsets=off, silu=True)

    def step():
        y, st = nat.layer_norm(x, w, b, return_stats=True, **kw)
        return (y, *nat.layer_norm_backward(dy, x, st, w, b, **kw))

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for i in range(4):
        x.copy_(torch.randn(x.shape, device=dev) + i)
        dy.copy_(torch.randn(x.shape, device=dev))
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = step()
        for _, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_module_capture(spc, dev):
    """The module in a graph: its items' offsets come from a call before."""
    c, counts = 64, [30, 20]
    x, _, _, sc, sh, _ = _inputs(dev, torch.bfloat16, 50, c, 3, items=2)
    ln = spc.sparse.SparseLayerNorm32(c).to(dev)
    t = _tensor(spc, dev, x, counts)
    torch.cuda.synchronize()
    with torch.no_grad():
        with pytest.raises(RuntimeError, match="before capturing"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                ln(t, sc, sh)
        torch.cuda.synchronize()
        ln(t, sc, sh)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ln(t, sc, sh).feats
        for _ in range(3):
            x.copy_(torch.randn(50, c, device=dev))
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, ln(t, sc, sh).feats)


def test_training_pass_capture(spc, dev):
    """Forward and backward of norm and 4-bit Linear in one graph, replayed on
    new values with eager work between; refused while an eager graph of the
    same leaves is alive."""
    c, e, counts = 64, 32, [30, 20]
    sp = spc.sparse
    lin = sp.Q4Linear(e, 2 * c).to(dev)
    lin.quantize_q4_0()
    ln = sp.SparseLayerNorm32(c).to(dev)
    x = torch.randn(50, c, device=dev, requires_grad=True)
    emb = torch.randn(2, e, device=dev, requires_grad=True)
    dy = torch.randn(50, c, device=dev)
    t = _tensor(spc, dev, x.detach(), counts)

    def run(x, emb, ln, lin):
        scale, shift = lin(emb).chunk(2, 1)
        return ln(t.replace(x), scale, shift, silu=True).feats

    leaves = [x, emb, ln.weight, ln.bias, lin.bias]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):          # first calls: operands, offsets
        y = run(x, emb, ln, lin)
        y.backward(dy)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for fn in (lambda: ln(t), lambda: lin(emb)):
        with pytest.raises(RuntimeError, match="eager graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                fn()
        torch.cuda.synchronize()
    del y
    for p in leaves:
        p.grad = None
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = run(x, emb, ln, lin)
        y.backward(dy)
    grads = [p.grad for p in leaves]
    # eager results from other leaves of the same values
    ln2, lin2 = copy.deepcopy(ln), copy.deepcopy(lin)
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(50, c, device=dev) + i)
            emb.copy_(torch.randn(2, e, device=dev))
        dy.copy_(torch.randn(50, c, device=dev))
        g.replay()
        torch.cuda.synchronize()
        x2, emb2 = (v.detach().clone().requires_grad_() for v in (x, emb))
        y2 = run(x2, emb2, ln2, lin2)
        want = torch.autograd.grad(y2, [x2, emb2, ln2.weight, ln2.bias, lin2.bias], dy)
        assert torch.equal(y, y2)
        for p, q in zip(grads, want):
            assert torch.equal(p, q)


def test_offset_past_32_bits(spc, dev):
    """Elements past 2^32: 2^20 + 8 rows of 4,096, 4,100 apart."""
    nat = spc._native
    n, c, ld = (1 << 20) + 8, 4096, 4100
    base = torch.empty((n, ld), dtype=torch.bfloat16, device=dev)
    for i in range(0, n, 1 << 16):
        base[i:i + (1 << 16)].normal_()
    x = base[:, :c]
    y, st = nat.layer_norm(x, return_stats=True)
    rows = [0, 1, (1 << 19) + 3, n - 9, n - 1]
    ref = Reference(x[rows])
    check("y", y[rows], *ref.forward())
    dx = nat.layer_norm_backward(x, x, st)[0]
    check("dx", dx[rows], *ref.backward(x[rows], 60)[0], torch.bfloat16)


def test_refusals_on_device(spc, dev):
    nat = spc._native
    x = torch.zeros((4, 64), device=dev)
    sc = torch.zeros((2, 64), device=dev)
    off = torch.tensor([0, 2, 4], device=dev)
    for kw in [dict(weight=x[0, :63]), dict(scale=sc), dict(scale=sc, shift=sc),
               dict(offsets=off), dict(scale=sc, shift=sc[:1], offsets=off),
               dict(scale=sc, shift=sc, offsets=off.int()),
               dict(scale=sc, shift=sc, offsets=off[:2]), dict(out=x[:, ::2]),
               dict(out=x.half()), dict(weight=torch.zeros(64))]:
        with pytest.raises(ValueError):
            nat.layer_norm(x, **kw)
    with pytest.raises(ValueError):
        nat.layer_norm(x[0])
    with pytest.raises(TypeError):
        nat.layer_norm(x.double())
    with pytest.raises(nat.SparseConvError):
        nat.layer_norm(x, eps=-1.0)
    with pytest.raises(nat.SparseConvError):
        nat.layer_norm(torch.zeros((2, 8193), device=dev))
    st = torch.zeros((4, 2), device=dev)
    for args in [(x[:3], x, st), (x.half(), x, st), (x, x, st[:3]), (x, x, st.double())]:
        with pytest.raises(ValueError):
            nat.layer_norm_backward(*args)
    ln = spc.sparse.SparseLayerNorm32(64).to(dev)
    t = _tensor(spc, dev, x, [2, 2])
    with pytest.raises(ValueError):
        ln(t, sc[:1], sc[:1])
    with pytest.raises(ValueError):
        ln(t.replace(x[:, :32]))
