"""Adapters at the edges of what a call may be: no rows, the largest counts of items
and adapters, adapters that most rows name."""
import ctypes

import pytest
import torch

from test_gpu_lora import DT, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(0, 64), (0, 5, 64), (3, 0, 64)])
@pytest.mark.parametrize("q4", [False, True])
def test_no_rows_train(spc, dev, q4, shape):
    """A batch without rows gives zeros as gradients, as the Linear's own weight has
    them, and a loss of it can be differentiated."""
    lin = spc.sparse.Q4Linear(64, 96).to(dev)
    if q4:
        lin.quantize_q4_0()
    lin.weight.requires_grad_(False)
    lin.add_adapters(2, 8, dropout=0.1)
    ids = torch.zeros(shape[0], dtype=torch.int32, device=dev)
    x = torch.randn(shape, device=dev, requires_grad=True)
    for frozen in (False, True):
        lin.bias.requires_grad_(not frozen)
        y = lin(x.detach() if frozen else x, ids)
        assert y.shape == (*shape[:-1], 96)
        lin.zero_grad(set_to_none=True)
        y.sum().backward()
        for p in (lin.adapter_down, lin.adapter_up, *([] if frozen else [lin.bias])):
            assert p.grad is not None and not p.grad.any()
    assert x.grad.shape == shape
    with torch.no_grad():
        assert lin(x, ids).shape == (*shape[:-1], 96)
    with pytest.raises(ValueError):
        lin(x, ids.long())


@pytest.mark.parametrize("n,rows,k,c,o,r,p", [(8400, 2, 1, 1024, 1024, 32, 0.0), (2200, 2, 1, 1024, 520, 128, 0.1),
                                              (3300, 3, 3, 130, 1024, 100, 0.0), (4200, 2, 2, 1000, 1030, 60, 0.2)])
@pytest.mark.parametrize("dt", list(DT))
def test_sums_in_parts(spc, dev, dt, n, rows, k, c, o, r, p):
    """More items than the slots of the weights' sums hold at a time, of either weight
    or both; each gradient alone has the same bits."""
    ids = [(i * i + i // 7) % (k + 1) - 1 if k > 1 else 0 for i in range(n // rows)]
    q = Case(dev, dt, n, c, o, r, k=k, offsets=list(range(0, n + 1, rows)), adapters=ids, p=p)
    q.check(spc._native)
    h = spc._native.lora(q.x, q.down, q.up, q.base, return_hidden=True, **q.kw)[1]
    whole = spc._native.lora_backward(q.dy, q.x, h, q.down, q.up, q.dx_base, **q.kw)
    for i in range(3):
        part = spc._native.lora_backward(q.dy, q.x, h, q.down, q.up, q.dx_base, need=[i == j for j in range(3)], **q.kw)
        assert torch.equal(part[i], whole[i])


def test_sums_in_parts_captured(spc, dev):
    """Replays on new rows, with eager calls of another size between."""
    nat = spc._native
    q = Case(dev, "bf16", 2200, 1024, 1030, 100, k=2, offsets=list(range(0, 2201, 2)), adapters=[i % 3 - 1 for i in range(1100)], p=0.1)
    h = torch.randn(2200, 100, device=dev)
    run = lambda: nat.lora_backward(q.dy, q.x, h, q.down, q.up, q.dx_base, **q.kw)  # noqa: E731
    run()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run()
    for i in range(3):
        q.x.copy_(torch.randn(2200, 1024))
        q.kw["seed"].copy_(torch.tensor([i, 7]))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, run()))
        nat.lora_backward(q.dy[:9], q.x[:9], h[:9], q.down[:1], q.up[:1])


MOST = 65_535   # of items and of adapters


@pytest.mark.parametrize("k,rows,name", [(MOST, 1, "each its own"), (MOST, 1, "the last"), (MOST, 1, "none"), (1, 2, "the last"),
                                         (3, 3, "in turn")])
@pytest.mark.parametrize("c,o", [(8, 9), (4, 3)])
@pytest.mark.parametrize("dt", list(DT))
def test_largest_counts_of_items_and_adapters(spc, dev, dt, c, o, k, rows, name):
    """Whole numbers, whose sums are exact (131,070 rows of at most 72 in one adapter's),
    so that results are the formulas', rounded once."""
    nat, t, g = spc._native, DT[dt], torch.Generator().manual_seed(k + rows)
    ints = lambda m, *s: torch.randint(-m, m + 1, s, generator=g).double()  # noqa: E731
    n, r = MOST * rows + 5, 1
    i = torch.arange(MOST)
    ids = {"each its own": torch.where(i % 10 == 3, -1, i * 7919 % MOST), "the last": torch.full((MOST,), k - 1),
           "none": torch.full((MOST,), -1), "in turn": i % 4}[name]
    of = torch.cat([ids.repeat_interleave(rows), torch.full((5,), -1)])
    of = torch.where(of >= k, -1, of)
    x, dy, base, dx_base = ints(3, n, c), ints(3, n, o), ints(50, n, o), ints(50, n, c)
    down, up = ints(2, k, r, c), ints(1, k, o, r)
    on = (of >= 0).double()[:, None]
    a = of.clamp(min=0)
    h = (x * down[a, 0]).sum(1, keepdim=True) * on
    u = (dy * up[a, :, 0]).sum(1, keepdim=True) * on
    dd = torch.zeros(k, c, dtype=torch.float64).index_add_(0, a, u * x)
    du = torch.zeros(k, o, dtype=torch.float64).index_add_(0, a, h * dy * on)
    f = lambda v: v.to(t).to(dev)  # noqa: E731
    kw = dict(offsets=torch.arange(0, n, rows, device=dev)[:MOST + 1], adapters=ids.to(torch.int32).to(dev))
    y, hid = nat.lora(f(x), f(down), f(up), f(base), return_hidden=True, **kw)
    dx, ddown, dup = nat.lora_backward(f(dy), f(x), hid, f(down), f(up), f(dx_base), **kw)
    for got, want in ((y, base + h * up[a, :, 0]), (hid, h), (dx, dx_base + u * down[a, 0]), (ddown[:, 0], dd), (dup[:, :, 0], du)):
        assert float(want.abs().max()) < 2 ** 24
        assert torch.equal(got.cpu(), want.to(got.dtype))


@pytest.mark.parametrize("n,rows,k", [(60, 1, 7), (96, 3, 32), (300, 1, 40), (1000, 1, 500)])
@pytest.mark.parametrize("which", ["one", "none", "most"])
@pytest.mark.parametrize("dt", list(DT))
def test_adapters_that_most_rows_name(spc, dev, dt, which, n, rows, k):
    """One adapter of a large bank in all items, in none, in all but a few."""
    items = n // rows
    ids = {"one": [k - 1] * items, "none": [-1] * items,
           "most": [i % k if i % 9 == 4 else -1 if i % 5 == 2 else 1 for i in range(items)]}[which]
    for c, o, r, p in ((130, 72, 12, 0.0), (72, 264, 70, 0.2), (7, 33, 3, 0.1)):
        q = Case(dev, dt, n, c, o, r, k=k, offsets=list(range(0, n + 1, rows)), adapters=ids, p=p)
        q.check(spc._native)
        dx, _, _ = spc._native.lora_backward(q.dy, q.x, None, q.down, q.up, q.dx_base, need=(True, False, False), **q.kw)
        free = [i for i in range(n) if ids[i // rows] < 0]
        assert torch.equal(dx[free], q.dx_base[free])
        # in place, and without a base
        got = _in_place(spc._native, q)
        assert torch.equal(got, dx)
        dx, _, _ = spc._native.lora_backward(q.dy, q.x, None, q.down, q.up, need=(True, False, False), **q.kw)
        assert not dx[free].any()


def _in_place(nat, q):
    """dx written over dx_base, by the entry point that allows it."""
    base = q.dx_base.clone()
    dev = nat._one_device(base)
    prm, keep, (items, c, o, r) = nat._lora_params(q.x, q.x.shape[1], None, q.down, q.up, q.kw["scale"], q.kw["offsets"],
                                                   q.kw["adapters"], q.kw["p"], q.kw["seed"])
    n, dt = q.x.shape[0], nat.dtype_code(q.x.dtype)
    need = nat.lib().spc_lora_workspace_bytes(dt, n, items, prm.n_adapters, c, o, r, 1)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=base.device)
    st = nat._launch(nat.lib().spc_lora_backward, dev, dt, q.dy.data_ptr(), q.dy.stride(0), q.x.data_ptr(), q.x.stride(0), None,
                     n, ctypes.byref(prm), base.data_ptr(), c, base.data_ptr(), None, None, ws.data_ptr(), need)
    assert st == nat.OK
    del keep
    return base
