"""Adapters at the edges of what a call may be: no rows, the largest counts of items
and adapters, adapters that most rows name."""
import pytest
import torch

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
