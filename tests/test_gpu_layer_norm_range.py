"""The row layer norm and its gradient where their values end: items without
rows, SiLU far from zero, rows that are not finite, the most items."""
import pytest
import torch

from norm_reference import Reference, check

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf"), 3e38])
@pytest.mark.parametrize("offsets", [[0, 4, 4, 30], [0, 0, 30, 30], [10, 10, 20, 20]])
def test_coefficients_that_no_row_meets(spc, dev, offsets, value):
    """What an empty item's scale and shift hold reaches no gradient, and its
    own are zeros, under an infinite weight too."""
    nat = spc._native
    n, c, nb = 30, 72, 3
    x, dy = _randn(1, n, c).to(dev), _randn(2, n, c).to(dev)
    w, b = (1 + 0.2 * _randn(3, c)).to(dev), (0.2 * _randn(4, c)).to(dev)
    sc, sh = _randn(5, nb, c).to(dev), _randn(6, nb, c).to(dev)
    kw = dict(offsets=torch.tensor(offsets, device=dev), silu=True)
    _, st = nat.layer_norm(x, w, b, scale=sc, shift=sh, return_stats=True, **kw)
    want = nat.layer_norm_backward(dy, x, st, w, b, scale=sc, shift=sh, **kw)
    empty = [i for i in range(nb) if offsets[i] == offsets[i + 1]]
    sc[empty], sh[empty] = value, value
    y, st = nat.layer_norm(x, w, b, scale=sc, shift=sh, return_stats=True, **kw)
    got = nat.layer_norm_backward(dy, x, st, w, b, scale=sc, shift=sh, **kw)
    assert bool(y.isfinite().all()) and all(torch.equal(p, q) for p, q in zip(got, want))
    assert bool((got[3][empty] == 0).all()) and bool((got[4][empty] == 0).all())
    w[:] = float("inf")
    ds = nat.layer_norm_backward(dy, x, st, w, b, scale=sc, shift=sh, **kw)[3]
    assert bool((ds[empty] == 0).all())
