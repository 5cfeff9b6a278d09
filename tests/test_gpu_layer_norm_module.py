"""SparseLayerNorm32 as a module: what may be captured, forward-mode
differentiation."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _tensor(spc, dev, feats):
    n = feats.shape[0]
    coords = torch.stack([torch.zeros(n), torch.arange(n) % 9, torch.arange(n) // 9, torch.zeros(n)], 1)
    return spc.sparse.SparseTensor(feats, coords.to(torch.int32).to(dev))


def test_capture_beside_graphs_of_other_operators(spc, dev):
    """A capture is refused while another operator's eager graph of its leaves
    is alive, and works once it is gone; leaves that the capture shares with
    other operators, and two captures of the same leaves, are as eager."""
    ln = spc.sparse.SparseLayerNorm32(64).to(dev)
    x = torch.randn(50, 64, device=dev, requires_grad=True)
    dy = torch.randn(50, 64, device=dev)
    t = _tensor(spc, dev, x.detach())
    leaves = [x, ln.weight, ln.bias]

    def run(xs):
        return ln(t.replace(ln(t.replace(xs)).feats + xs)).feats

    torch.autograd.grad(run(x), leaves, dy)
    torch.cuda.synchronize()
    keep = (ln.weight * 2).sum()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            run(x)
    torch.cuda.synchronize()
    del keep
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = run(x)
            graphs.append((g, y, torch.autograd.grad(y, leaves, dy)))
    x2 = x.detach().clone().requires_grad_()
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(50, 64, device=dev) + i)
            x2.copy_(x)
        dy.copy_(torch.randn(50, 64, device=dev))
        for g, _, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = run(x2)
        grads = torch.autograd.grad(want, [x2, ln.weight, ln.bias], dy)
        for _, y, got in graphs:
            assert torch.equal(y, want) and all(torch.equal(p, q) for p, q in zip(got, grads))


@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad])
@pytest.mark.parametrize("which", ["x", "weight", "scale"])
def test_forward_mode_is_refused(spc, dev, which, mode):
    """A tangent is not dropped in silence; calls without one work."""
    fw = torch.autograd.forward_ad
    ln = spc.sparse.SparseLayerNorm32(64).to(dev).requires_grad_(False)
    x, mod = torch.randn(6, 64, device=dev), torch.randn(1, 64, device=dev)
    want = ln(_tensor(spc, dev, x), mod, mod).feats
    with mode(), fw.dual_level():
        assert torch.equal(ln(_tensor(spc, dev, x), mod, mod).feats, want)
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        a, m = dual(x) if which == "x" else x, dual(mod) if which == "scale" else mod
        if which == "weight":
            w = ln.weight
            del ln.weight
            ln.weight = dual(w.detach())
        with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
            ln(_tensor(spc, dev, a), m, mod)
