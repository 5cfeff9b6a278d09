"""Q4Linear's adapters as module state, without a GPU."""
import pytest
import torch
import torch.nn as nn


@pytest.mark.parametrize("cast", [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.to(torch.float16),
                                  lambda m: m.to("cpu", torch.bfloat16), lambda m: m.double()])
@pytest.mark.parametrize("outer", [False, True])
def test_scale_keeps_its_bits(spc, cast, outer):
    """alpha / rank stays what it is, F32, when the module's dtype changes, once and
    again, of itself or of a module around it."""
    lin = spc.sparse.Q4Linear(32, 8)
    lin.add_adapters(2, 10, alpha=16)
    want = torch.tensor([1.6, 1.6])
    assert torch.equal(lin.adapter_scale, want)
    whole = nn.Sequential(lin) if outer else lin
    cast(whole)
    assert lin.adapter_down.dtype == lin.weight.dtype != torch.float32
    assert lin.adapter_scale.dtype == torch.float32 and torch.equal(lin.adapter_scale, want)
    assert torch.equal(whole.float().state_dict()[("0." if outer else "") + "adapter_scale"], want)
    lin.drop_adapters()
    assert cast(whole) is whole and not lin.has_adapters


def test_scale_on_meta(spc):
    lin = spc.sparse.Q4Linear(32, 8)
    lin.add_adapters(2, 10, alpha=16)
    lin.half().to("meta")
    assert lin.adapter_scale.is_meta and lin.adapter_scale.dtype == torch.float32
    lin.to_empty(device="cpu")
    assert lin.adapter_scale.dtype == torch.float32 and lin.adapter_down.dtype == torch.float16


def test_more_adapters_than_a_call_takes_are_refused(spc):
    """When they are added, not by the first call; what was there stays."""
    lin = spc.sparse.Q4Linear(8, 8)
    lin.add_adapters(65_535, 1)
    with pytest.raises(ValueError, match="65535"):
        lin.add_adapters(65_536, 1)
    assert lin.adapter_down.shape == (65_535, 1, 8)
