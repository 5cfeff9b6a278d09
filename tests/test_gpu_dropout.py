"""spc_dropout against its 64-bit form (lora_reference): every width, stride and
alignment, probabilities 0 to 1, values that are not finite, long rows, streams,
graphs, refusals."""
import pytest
import torch

from lora_reference import dropout, factors, threshold
from norm_reference import check

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SEED = [0x123456789ABCDEF, -77]


def _seed(dev, seed=SEED):
    return torch.tensor(seed, dtype=torch.int64, device=dev)


def _rows(n, c, dt, dev, salt=0):
    return torch.randn(n, c, generator=torch.Generator().manual_seed(n + 7 * c + salt)).to(DT[dt]).to(dev)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("n,c", [(1, 1), (1, 8), (3, 7), (5, 101), (333, 192), (2, 8191), (1000, 16), (70, 1030)])
@pytest.mark.parametrize("dt", list(DT))
def test_dropout(spc, dev, dt, n, c, residual):
    x = _rows(n, c, dt, dev)
    r = _rows(n, c, dt, dev, 1) if residual else None
    y = spc._native.dropout(x, 0.3, _seed(dev), residual=r)
    check(f"dropout {dt} {n}x{c}", y, *dropout(x, 0.3, SEED, r))
    if not residual:
        assert torch.equal((y == 0).cpu(), ((factors(SEED, n, c, 0.3) == 0) | (x.cpu() == 0)))


@pytest.mark.parametrize("p", [0.0, 2.0 ** -18, 2.0 ** -16, 0.1, 1 / 3, 0.5, 0.999, 1 - 2.0 ** -16, 1 - 2.0 ** -18, 1.0])
@pytest.mark.parametrize("dt", list(DT))
def test_probabilities(spc, dev, dt, p):
    x, r = _rows(65, 72, dt, dev), _rows(65, 72, dt, dev, 1)
    small = x * 2.0 ** -8 if dt == "f16" else x   # (kept values grow 65,536-fold at most)
    for res in (None, r):
        y = spc._native.dropout(small, p, _seed(dev) if threshold(p) or p else None, residual=res)
        check(f"p {p} {dt}", y, *dropout(small, p, SEED, res))


@pytest.mark.parametrize("dt", list(DT))
def test_strides_and_alignment(spc, dev, dt):
    """Column ranges at any element, repeated rows, one column, a transposed view."""
    wide = _rows(40, 300, dt, dev)
    for x in (wide[:, 3:104], wide[:, 1:257], wide[::3, 5:69], wide[:1].expand(40, 300), wide[:, 7:8],
              wide[:, :64].t(), wide[4:5, 9:]):
        r = wide[:x.shape[0], 150:150 + x.shape[1]] if x.shape[1] <= 150 and x.shape[0] <= 40 else None
        check(f"view {tuple(x.shape)} {x.stride()}", spc._native.dropout(x, 0.4, _seed(dev), residual=r),
              *dropout(x, 0.4, SEED, r))


@pytest.mark.parametrize("dt", list(DT))
def test_values_that_are_not_finite(spc, dev, dt):
    """A dropped value counts as zero whatever it is; a kept one stays what it is."""
    x = _rows(64, 40, dt, dev)
    x[::3] = float("nan")
    x[1::3] = float("inf")
    f = factors(SEED, 64, 40, 0.5).to(dev)
    y = spc._native.dropout(x, 0.5, _seed(dev)).double()
    assert not y[f == 0].any()
    kept = x.double() * f
    assert torch.equal(y[f > 0].isnan(), kept[f > 0].isnan()) and torch.equal(y[f > 0].isinf(), kept[f > 0].isinf())


@pytest.mark.parametrize("dt", list(DT))
def test_in_place(spc, dev, dt):
    x, r = _rows(50, 77, dt, dev), _rows(50, 77, dt, dev, 1)
    want = spc._native.dropout(x, 0.2, _seed(dev), residual=r)
    for out in (x, r):
        a, b = x.clone(), r.clone()
        got = spc._native.dropout(a, 0.2, _seed(dev), residual=b, out=a if out is x else b)
        assert torch.equal(got, want) and got.data_ptr() == (a if out is x else b).data_ptr()


def test_more_elements_than_32_bits_count(spc, dev):
    """2^32 elements and some: the last rows are as a call of their own would
    have them."""
    n, c = (1 << 22) + 3, 1024
    x = torch.ones((n, c), dtype=torch.bfloat16, device=dev)
    spc._native.dropout(x, 0.5, _seed(dev), out=x)
    for first in (0, (1 << 22) - 2, n - 5):
        want = factors(SEED, 5, c, 0.5, first=first)
        assert torch.equal(x[first:first + 5].double().cpu(), want)


def test_more_groups_than_threads(spc, dev):
    """Of an odd number a row, so that a thread's next one begins elsewhere in its row."""
    n, c = (1 << 28) // 3 + 1000, 17
    x = _rows(1, c, "bf16", dev).expand(n, c)
    y = spc._native.dropout(x, 0.25, _seed(dev))
    for first in (0, n - 1003, n - 5):   # 2^28 groups of eight end in row n - 1000
        want = x[:5].double().cpu() * factors(SEED, 5, c, 0.25, first=first)
        # the factor's and the product's F32 steps, 2 x 2^-24, then the rounding of y
        check(f"rows from {first}", y[first:first + 5], want, want.abs() * 2.0 ** -23, torch.bfloat16)


def test_other_streams_graphs_and_two_seeds(spc, dev):
    """A replayed graph takes the seed that the tensor then holds, with eager
    work between the replays."""
    nat = spc._native
    x, seed = _rows(129, 333, "bf16", dev), _seed(dev)
    r = _rows(129, 333, "bf16", dev, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = nat.dropout(x, 0.3, seed, residual=r)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, nat.dropout(x, 0.3, seed, residual=r))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        z = nat.dropout(nat.dropout(x, 0.3, seed, residual=r), 0.5, seed)
    for i in range(4):
        seed.copy_(torch.tensor([i, 5 - i]))
        x.copy_(_rows(129, 333, "bf16", dev, 10 + i))
        g.replay()
        torch.cuda.synchronize()
        want = nat.dropout(nat.dropout(x, 0.3, torch.tensor([i, 5 - i], device=dev), residual=r), 0.5, seed)
        assert torch.equal(z, want)


def test_refusals(spc, dev):
    nat = spc._native
    x, s = _rows(4, 16, "f32", dev), _seed(dev)
    assert nat.dropout(x[:0], 0.5, s).shape == (0, 16) and nat.dropout(x[:, :0], 0.5, s).shape == (4, 0)
    for args, kw in [((x, 1.5, s), {}), ((x, float("nan"), s), {}), ((x, 0.5, None), {}), ((x, 0.5, s[:1]), {}),
                     ((x, 0.5, s.int()), {}), ((x[0], 0.5, s), {}), ((x, 0.5, s), {"residual": x[:2]}),
                     ((x, 0.5, s), {"residual": x.half()}), ((x, 0.5, s), {"out": x.half()}),
                     ((x, 0.5, s), {"out": torch.empty(16, 4, device=dev).t()}), ((x, 0.5, s.cpu()), {})]:
        with pytest.raises(ValueError):
            nat.dropout(*args, **kw)
    flat = torch.zeros(200, device=dev)
    with pytest.raises(ValueError, match="apart"):
        nat.dropout(flat[4:68].view(4, 16), 0.5, s, out=flat[:64].view(4, 16))
    with pytest.raises(TypeError):
        nat.dropout(x.double(), 0.5, s)
