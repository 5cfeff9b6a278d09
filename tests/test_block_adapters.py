"""SparseResBlock3d with adapters: what its modulation may be, and what is refused,
without a GPU (the modulation runs on the CPU, the block's norm then asks for one)."""
import pytest
import torch
import torch.nn as nn


def _block(spc, cin=32, cout=64):
    torch.manual_seed(0)
    block = spc.blocks.SparseResBlock3d(cin, 48, cout)
    coords = torch.tensor([[b, i, 0, 0] for b in range(2) for i in range(3)], dtype=torch.int32)
    x = spc.sparse.SparseTensor(torch.randn(6, cin), coords)
    return block, x, torch.randn(2, 48)


class Wrapped(nn.Module):
    """What a checkpoint's or a compiler's wrapper looks like: no children to unpack."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, *args):
        return self.inner(*args)


def test_modulation_may_be_any_module(spc):
    """A wrapped modulation, or one of another length, reaches the block's norm."""
    block, x, emb = _block(spc)
    for module in (Wrapped(block.emb_layers), nn.Sequential(nn.SiLU(), nn.Dropout(0.0), block.emb_layers[1]),
                   block.emb_layers[1]):
        block.emb_layers = module
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU only"):
            block(x, emb)


def test_modulation_is_called_with_its_hooks(spc):
    """Adapters go through the modulation's own call, whose hooks see them, and
    through a wrapper."""
    block, x, emb = _block(spc)
    which = torch.tensor([0, -1], dtype=torch.int32)
    block.emb_layers[1].add_adapters(1, 4)
    seen = []
    block.emb_layers.register_forward_pre_hook(lambda m, args: seen.append(len(args)))
    plain = block.emb_layers(emb)
    for module in (block.emb_layers, Wrapped(block.emb_layers)):
        block.emb_layers = module
        # (the Linear's adapters are the GPU's)
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU only"):
            block(x, emb, which)
    assert seen == [1, 2, 2]
    block.emb_layers = spc.blocks._Modulation(nn.SiLU(), Wrapped(block.emb_layers.inner[1]))
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU only"):
        block.emb_layers(emb, which)
    block.emb_layers = Wrapped(block.emb_layers)
    assert torch.equal(block.emb_layers(emb), plain)


@pytest.mark.parametrize("where", ["emb_layers", "skip_connection"])
def test_adapters_that_need_a_gradient_are_refused(spc, where):
    """The block gives none: a call that would leave them without it, in training or
    not, frozen convs or not, raises before any work; without adapters, under no_grad
    and with frozen adapters nothing changes."""
    block, x, emb = _block(spc)
    which = torch.tensor([0, -1], dtype=torch.int32)
    lin = block.emb_layers[1] if where == "emb_layers" else block.skip_connection
    lin.add_adapters(1, 4)
    for train in (True, False):
        block.train(train)
        for frozen in (False, True):
            block.conv1.requires_grad_(not frozen), block.conv2.requires_grad_(not frozen)
            with pytest.raises(RuntimeError, match="no gradients"):
                block(x, emb, which)
            with pytest.raises(RuntimeError, match="GPU only"):
                block(x, emb)
            with torch.no_grad(), pytest.raises(RuntimeError, match="GPU only"):
                block(x, emb, which)
    lin.adapter_down.requires_grad_(False)
    with pytest.raises(RuntimeError, match="no gradients"):
        block(x, emb, which)
    lin.adapter_up.requires_grad_(False)
    with pytest.raises(RuntimeError, match="GPU only"):
        block(x, emb, which)
