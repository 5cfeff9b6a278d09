"""Layer norm: what is refused on the host, before any device work, and the
64-bit reference of the GPU tests against torch's own autograd."""
import ctypes

import pytest
import torch

from norm_reference import Reference


def test_reference_is_torchs_gradient():
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    n, c, nb = 12, 10, 3
    x, w, b = (r(n, c).requires_grad_(), (1 + r(c)).requires_grad_(), r(c).requires_grad_())
    sc, sh, dy = r(nb, c).requires_grad_(), r(nb, c).requires_grad_(), r(n, c)
    item = torch.tensor([0] * 5 + [1] * 1 + [2] * 6)
    y = torch.nn.functional.layer_norm(x, (c,), w, b, 1e-6) * (1 + sc[item]) + sh[item]
    y = torch.nn.functional.silu(y)
    want = torch.autograd.grad(y, (x, w, b, sc, sh), dy)
    ref = Reference(x, w, b, 1e-6, sc, sh, item, True)
    ref.dtype = torch.float32
    torch.testing.assert_close(ref.forward()[0], y.detach())
    for got, wt in zip(ref.backward(dy, 1), want):
        torch.testing.assert_close(got[0], wt)


def test_host_validation(spc):
    nat = spc._native
    L = nat.lib()
    fake = 1 << 12  # aligned, never dereferenced: validation fails first

    def fwd(n=4, c=64, dtype=nat.BF16, x=fake, y=fake, stride=64, **kw):
        p = nat.LayerNormParams(eps=kw.pop("eps", 1e-6), n_batch=kw.pop("n_batch", 1), **kw)
        return L.spc_layer_norm(None, dtype, x, stride, n, c, ctypes.byref(p), y, None)

    assert fwd(n=0) == nat.OK
    assert fwd(c=0) == nat.BAD_SHAPE and fwd(c=8193) == nat.BAD_SHAPE and fwd(n=-1) == nat.BAD_SHAPE
    assert fwd(n=1 << 31) == nat.BAD_SHAPE and fwd(stride=-1) == nat.BAD_SHAPE
    assert b"8192" in L.spc_last_error()
    assert fwd(dtype=nat.Q8_0) == nat.BAD_ARG
    assert fwd(eps=-1.0) == nat.BAD_ARG and fwd(eps=float("nan")) == nat.BAD_ARG
    assert fwd(x=None) == nat.BAD_ARG and fwd(y=None) == nat.BAD_ARG
    assert fwd(x=fake + 1) == nat.BAD_ARG and fwd(y=fake + 1) == nat.BAD_ARG
    assert fwd(gamma=fake, param_dtype=7) == nat.BAD_ARG
    assert fwd(gamma=fake + 2, param_dtype=nat.F32) == nat.BAD_ARG
    mod = dict(scale=fake, shift=fake, mod_stride=64)
    assert fwd(scale=fake) == nat.BAD_ARG
    assert fwd(**mod, n_batch=0) == nat.BAD_ARG and fwd(**mod, n_batch=65536) == nat.BAD_ARG
    assert fwd(**mod, n_batch=2) == nat.BAD_ARG                       # no offsets
    assert fwd(**mod, n_batch=2, offsets=fake + 4) == nat.BAD_ARG
    assert fwd(offsets=fake) == nat.BAD_ARG
    assert b"offsets" in L.spc_last_error()

    def bwd(ws=fake, wsb=1 << 30, dgamma=None, dscale=None, stats=fake, dy=fake, dys=64, **kw):
        p = nat.LayerNormParams(eps=0.0, n_batch=1, **kw)
        return L.spc_layer_norm_backward(None, nat.BF16, dy, dys, fake, 64, stats, 4, 64,
                                         ctypes.byref(p), fake, dgamma, None, dscale, None, ws, wsb)

    assert bwd(dgamma=fake) == nat.BAD_ARG                            # no gamma given
    assert bwd(dscale=fake, gamma=fake) == nat.BAD_ARG
    assert bwd(dy=None) == nat.BAD_ARG and bwd(stats=None) == nat.BAD_ARG
    assert bwd(dys=-1) == nat.BAD_ARG and bwd(stats=fake + 2) == nat.BAD_ARG
    need = L.spc_layer_norm_backward_workspace_bytes(nat.BF16, 4, 64, 1)
    assert need >= 3 * 2 * 64 * 4
    assert bwd(dgamma=fake, gamma=fake, wsb=need - 1) == nat.BAD_ARG
    assert bwd(dgamma=fake, gamma=fake, ws=None) == nat.BAD_ARG
    assert b"workspace" in L.spc_last_error()
    assert L.spc_layer_norm_backward_workspace_bytes(nat.BF16, 4, 8193, 1) == 0
    assert L.spc_layer_norm_backward_workspace_bytes(nat.BF16, 4, 64, 0) == 0


def test_cpu_tensors_are_rejected(spc):
    nat = spc._native
    x = torch.zeros((4, 64))
    with pytest.raises(RuntimeError, match="GPU only"):
        nat.layer_norm(x)
    with pytest.raises(RuntimeError, match="GPU only"):
        nat.layer_norm_backward(x, x, torch.zeros((4, 2)))
