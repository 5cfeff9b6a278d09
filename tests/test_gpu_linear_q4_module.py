"""Q4Linear as a module: streams, state, forward-mode differentiation."""
import pytest
import torch

from norm_reference import check
from q4_reference import gradient, product, random_blocks

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("load", ["blocks", "quantize"])
def test_blocks_loaded_on_another_stream(spc, dev, load):
    """Blocks that a busy stream has still to write are waited for before the
    first call, on another stream, lays them out."""
    lin = spc.sparse.Q4Linear(1024, 512, bias=False).to(dev)
    blocks = random_blocks(512, 1024, 5)
    weight, src = lin.weight.detach().clone(), blocks.to(dev)
    big = torch.randn(8192, 8192, device=dev)
    x = torch.randn(3, 1024, generator=torch.Generator().manual_seed(1)).to(dev).requires_grad_()
    with torch.no_grad():
        lin.weight.zero_()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s), torch.no_grad():
        for _ in range(4):
            big = big @ big * 1e-4
        if load == "blocks":
            late = torch.zeros_like(src)
            late.copy_(src)
            lin.load_q4_0(late)
        else:
            lin.weight.copy_(weight)
            blocks = lin.quantize_q4_0()
    y = lin(x)
    dy = torch.ones_like(y)
    y.backward(dy)
    torch.cuda.synchronize()
    blocks = blocks.cpu().view(512, 32, 18)
    check("y", y, *product(x, blocks), torch.float32)
    check("dx", x.grad, *gradient(dy, blocks), torch.float32)


@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad])
def test_forward_mode_is_refused(spc, dev, mode):
    fw = torch.autograd.forward_ad
    lin = spc.sparse.Q4Linear(64, 32).to(dev).requires_grad_(False)
    lin.quantize_q4_0()
    x = torch.randn(2, 64, device=dev)
    want = lin(x)
    with mode(), fw.dual_level():
        assert torch.equal(lin(x), want)
        with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
            lin(fw.make_dual(x, torch.ones_like(x)))


def test_weights_at_any_element_are_quantised(spc, dev):
    """A parameter that is a view into a flat buffer."""
    flat = torch.randn(64 * 96 + 3, generator=torch.Generator().manual_seed(1)).to(dev)
    lin = spc.sparse.Q4Linear(96, 64, bias=False).to(dev)
    want = spc._native.q4_0_quantize(flat[3:].clone().view(64, 96))
    lin.weight.data = flat[3:].view(64, 96)
    assert torch.equal(lin.quantize_q4_0(), want)
    assert torch.equal(spc._native.q4_0_quantize(flat[3:]), want)
