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


def test_training_after_inference_mode(spc, dev):
    """What a first call in inference mode keeps (offsets, laid out weights)
    serves a training pass."""
    sp = spc.sparse
    ln, lin = sp.SparseLayerNorm32(64).to(dev), sp.Q4Linear(32, 128).to(dev)
    x = torch.randn(50, 64, device=dev)
    coords = torch.tensor([[0, i, 0, 0] for i in range(20)] + [[1, i, 0, 0] for i in range(30)],
                          dtype=torch.int32, device=dev)
    emb = torch.randn(2, 32, device=dev)
    t = sp.SparseTensor(x, coords)
    with torch.inference_mode():
        lin.quantize_q4_0()
        want = ln(t, *lin(emb).chunk(2, 1), silu=True).feats
    emb.requires_grad_()
    y = ln(t, *lin(emb).chunk(2, 1), silu=True).feats
    assert torch.equal(y, want)
    y.square().sum().backward()
    assert bool(emb.grad.isfinite().all()) and float(emb.grad.abs().max()) > 0
    assert bool(ln.weight.grad.isfinite().all()) and bool(lin.bias.grad.isfinite().all())
