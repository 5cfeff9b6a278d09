"""Adapters at the edges of what a call may be: no rows, the largest counts of items
and adapters, adapters that most rows name."""
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
