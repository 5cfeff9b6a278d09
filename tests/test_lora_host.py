"""Dropout and low-rank adapters: the 64-bit reference against published
vectors, torch's own autograd and differences, and what is refused on the host,
before any device work."""
import ctypes

import numpy as np
import pytest
import torch

from lora_reference import Adapters, dropout, factors, philox, threshold


def test_reference_generator_has_the_published_values():
    """Counter and key zero: the known answers that the generator's authors give
    for seven and ten rounds."""
    zero = [np.zeros(1, np.uint64)] * 4
    for rounds, want in ((7, "5f6fb709 0d893f64 4f121f81 4f730a48"), (10, "6627e8d5 e169c58d bc57ac4c 9b00dbd8")):
        assert " ".join("%08x" % int(v[0]) for v in philox(zero, [0, 0], rounds)) == want


def test_reference_mask():
    for p in (0.1, 0.5, 0.9):
        f = factors([1234567890123456789, -5], 2000, 99, p)
        kept = float((f > 0).double().mean())
        q = 1 - threshold(p) / 65536
        assert abs(kept - q) < 5 * (q * (1 - q) / f.numel()) ** 0.5
        assert float((f[f > 0] - 1 / q).abs().max()) < 1e-12
    assert not factors([1, 2], 3, 9, 1.0).any() and bool((factors([1, 2], 3, 9, 2.0 ** -18) == 1).all())
    # rows and columns differ, another stream or key is another mask
    f = factors([7, 8], 64, 64, 0.5)
    assert not torch.equal(f[0], f[1])
    assert all(not torch.equal(f, factors(s, 64, 64, 0.5)) for s in ([7, 9], [8, 8], [7 + 2 ** 32, 8], [7, 8 + 2 ** 32]))
    assert torch.equal(f[5:9], factors([7, 8], 4, 64, 0.5, first=5))


def test_reference_is_torchs_gradient_and_agrees_with_differences():
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    n, c, o, k, rank = 14, 10, 9, 3, 4
    x, down, up = r(n, c).requires_grad_(), r(k, rank, c).requires_grad_(), r(k, o, rank).requires_grad_()
    scale, dy, seed = 1 + r(k), r(n, o), [3, 4]
    offsets, ids = [1, 4, 4, 9, 12], [2, 1, -1, 2]
    of = torch.tensor([-1] + [2] * 3 + [-1] * 5 + [2] * 3 + [-1] * 2)
    f = factors(seed, n, c, 0.25)

    def run(x, down, up):
        h = torch.einsum("ni,nri->nr", x * f, down[of.clamp(min=0)])
        y = torch.einsum("nr,nor->no", h, up[of.clamp(min=0)]) * scale[of.clamp(min=0)][:, None]
        return torch.where((of >= 0)[:, None], y, torch.zeros(()).double()), h

    y, h = run(x, down, up)
    want = torch.autograd.grad(y, (x, down, up), dy)
    ref = Adapters(x, down, up, scale, offsets, ids, 0.25, seed)
    ref.dtype = torch.float32
    torch.testing.assert_close(ref.forward()[0][0], y.detach())
    hid = torch.where((of >= 0)[:, None], h.detach(), torch.zeros(()).double())
    torch.testing.assert_close(ref.forward()[1][0], hid)
    for got, wt in zip(ref.backward(dy, hid), want):
        torch.testing.assert_close(got[0], wt)
    # a difference along a direction
    d = [r(*t.shape) for t in (x, down, up)]
    at = lambda t: float((run(*(a.detach() + t * b for a, b in zip((x, down, up), d)))[0] * dy).sum())  # noqa: E731
    t = 1e-4
    slope = (at(t) - at(-t)) / (2 * t)
    assert abs(slope - sum(float((a * b).sum()) for a, b in zip(want, d))) < 1e-5 * abs(slope) + 1e-6


def test_host_validation_dropout(spc):
    nat = spc._native
    L = nat.lib()
    fake = 1 << 12  # aligned, never dereferenced: validation fails first

    def run(n=4, c=64, dtype=nat.BF16, x=fake, y=fake, xs=64, p=0.5, seed=fake, res=None, rs=0):
        return L.spc_dropout(None, dtype, x, xs, n, c, p, seed, res, rs, y)

    assert run(n=0) == nat.OK
    assert run(n=-1) == run(n=1 << 31) == run(c=0) == run(c=1 << 31) == nat.BAD_SHAPE
    assert run(xs=-1) == run(rs=-1) == nat.BAD_SHAPE
    assert b"columns" in L.spc_last_error()
    for bad in (dict(dtype=nat.Q8_0), dict(p=-0.1), dict(p=1.01), dict(p=float("nan")), dict(x=None), dict(y=None),
                dict(seed=None), dict(seed=fake + 4), dict(x=fake + 1), dict(res=fake + 1), dict(y=fake + 2, dtype=nat.F32)):
        assert run(**bad) == nat.BAD_ARG, bad


def test_host_validation_lora(spc):
    nat = spc._native
    L = nat.lib()
    fake = 1 << 12

    def params(**kw):
        d = dict(down=fake, up=fake, scale=fake, offsets=fake, adapters=fake, seed=fake, n_adapters=3, n_items=2,
                 in_features=64, out_features=48, rank=8, p=0.1)
        d.update(kw)
        return nat.LoraParams(**d)

    def fwd(n=4, dtype=nat.BF16, x=fake, xs=64, base=fake, bs=48, y=fake, hidden=fake, ws=fake, wsb=1 << 30, **kw):
        return L.spc_lora(None, dtype, x, xs, n, ctypes.byref(params(**kw)), base, bs, y, hidden, ws, wsb)

    def bwd(n=4, dtype=nat.BF16, dy=fake, dys=48, x=fake, hidden=fake, base=fake, bs=64, dx=fake, dd=fake, du=fake,
            ws=fake, wsb=1 << 30, **kw):
        return L.spc_lora_backward(None, dtype, dy, dys, x, 64, hidden, n, ctypes.byref(params(**kw)), base, bs, dx, dd,
                                   du, ws, wsb)

    assert fwd(n=0) == nat.OK and bwd(dx=None, dd=None, du=None) == nat.OK
    for run in (fwd, bwd):
        for bad in (dict(n=-1), dict(n=1 << 31), dict(rank=0), dict(rank=129), dict(in_features=0),
                    dict(out_features=0), dict(in_features=(1 << 24) + 1), dict(n_adapters=0), dict(n_adapters=65536),
                    dict(n_items=0), dict(n_items=65536)):
            assert run(**bad) == nat.BAD_SHAPE, bad
        for bad in (dict(dtype=nat.Q8_0), dict(p=-1.0), dict(p=float("nan")), dict(x=None), dict(down=None), dict(up=None),
                    dict(seed=None), dict(offsets=None, n_items=3), dict(adapters=None), dict(offsets=fake + 4),
                    dict(adapters=fake + 2), dict(scale=fake + 2), dict(down=fake + 1), dict(base=fake + 1), dict(bs=-1),
                    dict(hidden=fake + 2), dict(x=fake + 1)):
            assert run(**bad) == nat.BAD_ARG, bad
    assert fwd(y=None) == fwd(y=fake + 1) == nat.BAD_ARG
    assert bwd(dy=None) == bwd(hidden=None) == bwd(dys=-1) == bwd(du=fake + 1) == nat.BAD_ARG
    # few wide rows: the forward pass in two kernels; the backward pass's shares
    for b, n, wide in ((0, 8, 8192), (1, 5000, 64)):
        need = L.spc_lora_workspace_bytes(nat.BF16, n, 2, 3, wide, 48, 64, b)
        assert need > 0
        kw = dict(n=n, in_features=wide, rank=64, **({"xs": wide} if b == 0 else {}))
        for bad in (dict(wsb=need - 1), dict(ws=None), dict(ws=fake + 4)):
            assert (fwd, bwd)[b](**kw, **bad) == nat.BAD_ARG
    assert b"workspace" in L.spc_last_error()
    for items in (1, 7, 65535):  # no rows: an answer, not a division
        assert all(L.spc_lora_workspace_bytes(nat.F16, 0, items, 2, 64, 48, 8, b) >= 0 for b in (0, 1))
    assert L.spc_lora_workspace_bytes(nat.BF16, 4, 1, 1, 64, 48, 129, 0) == 0
    assert L.spc_lora_workspace_bytes(nat.Q8_0, 4, 1, 1, 64, 48, 8, 0) == 0
    assert L.spc_lora_workspace_bytes(nat.BF16, 4, 0, 1, 64, 48, 8, 1) == 0
    assert L.spc_lora_workspace_bytes(nat.BF16, 4, 1, 0, 64, 48, 8, 1) == 0


def test_cpu_tensors_are_rejected(spc):
    nat = spc._native
    x, s = torch.zeros((4, 64)), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="GPU only"):
        nat.dropout(x, 0.1, s)
    with pytest.raises(RuntimeError, match="GPU only"):
        nat.lora(x, torch.zeros(1, 4, 64), torch.zeros(1, 8, 4))
    with pytest.raises(RuntimeError, match="GPU only"):
        nat.lora_backward(torch.zeros(4, 8), x, torch.zeros(4, 4), torch.zeros(1, 4, 64), torch.zeros(1, 8, 4))


def test_modules_without_a_gpu(spc):
    """Construction, state and refusals need none; a call does."""
    torch.manual_seed(1)
    lin = spc.sparse.Q4Linear(64, 20)
    x = torch.randn(3, 64)
    want = lin(x)
    assert list(lin.state_dict()) == ["weight", "bias"] and not lin.has_adapters
    lin.add_adapters(3, 4, alpha=8, dropout=0.1)
    assert lin.adapter_down.shape == (3, 4, 64) and lin.adapter_up.shape == (3, 20, 4)
    assert lin.adapter_scale.tolist() == [2.0] * 3 and not lin.adapter_up.any() and lin.adapter_down.any()
    assert torch.equal(lin(x), want)
    with pytest.raises(RuntimeError, match="GPU only"):
        lin(x, torch.zeros(3, dtype=torch.int32))
    for bad in (dict(count=0, rank=4), dict(count=1, rank=0), dict(count=1, rank=129), dict(count=1, rank=4, dropout=1.5)):
        with pytest.raises(ValueError):
            lin.add_adapters(**bad)
    assert lin.has_adapters
    lin.add_adapters(1, 2)
    assert lin.adapter_down.shape == (1, 2, 64) and lin.adapter_scale.tolist() == [1.0]
    lin.drop_adapters()
    assert list(lin.state_dict()) == ["weight", "bias"]
    t = spc.sparse.SparseTensor(x, torch.tensor([[0, i, 0, 0] for i in range(3)], dtype=torch.int32))
    drop = spc.sparse.SparseDropout(0.5)
    with pytest.raises(RuntimeError, match="GPU only"):
        drop(t)
    assert drop.eval()(t) is t and torch.equal(drop(t, t).feats, x + x)
    with pytest.raises(ValueError):
        spc.sparse.SparseDropout(1.5)
