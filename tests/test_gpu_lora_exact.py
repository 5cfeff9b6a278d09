"""Adapters of whole numbers: hidden rows and u of 23 bits meet 16-bit operands
whose products cancel down to numbers that every type holds, so that the results
are exact if, and only if, no bit of h or u is lost.

Every partial sum is a whole number below 2^24 (at most 1000 products of 127 x 61
each, one pair of ranks or of rows with a nonzero operand), so F32 sums are exact
in any order, and the outputs lie within +-256, bf16's whole numbers."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


class Whole:
    def __init__(self, seed):
        self.g = torch.Generator().manual_seed(seed)

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi + 1, shape, generator=self.g).double()

    def twins(self, lo, hi, pairs, width):
        """[2 pairs, width]: rows 2 j and 2 j + 1 differ by one in a column."""
        a = self.ints(lo, hi - 1, pairs, width)
        b = a.clone()
        b[torch.arange(pairs), torch.randint(width, (pairs,), generator=self.g)] += 1
        return torch.stack([a, b], 1).reshape(2 * pairs, width)

    def signs(self, rows, pairs):
        """[rows, 2 pairs]: a row has s and -s at one pair's places, else zeros."""
        w = torch.zeros(rows, pairs, 2, dtype=torch.float64)
        s = 2 * self.ints(0, 1, rows) - 1
        w[torch.arange(rows), torch.arange(rows) % pairs] = torch.stack([s, -s], 1)
        return w.reshape(rows, 2 * pairs)


def _ranks(w, r, dim):
    """Zeros behind the pairs of an odd rank."""
    shape = list(w.shape)
    shape[dim] = r - shape[dim]
    return torch.cat([w, w.new_zeros(shape)], dim)


def _equal(name, got, want):
    wrong = int((got.detach().cpu().double() != want).sum())
    assert wrong == 0, f"{name}: {wrong} of {want.numel()} differ"


# few rows (the gradients gathered), tiles of 16, 32 and 64 rows, each count of rank tiles
SHAPES = [(2, 1000, 16, 16), (12, 600, 80, 7), (20, 513, 72, 128), (64, 900, 300, 33), (8, 9000, 40, 64), (700, 600, 136, 16),
          (640, 512, 600, 32), (642, 520, 130, 64), (600, 400, 72, 128), (12_300, 400, 40, 16), (12_300, 300, 24, 20),
          (12_300, 260, 40, 40), (12_300, 264, 40, 128), (24_600, 300, 40, 64)]


@pytest.mark.parametrize("n,c,o,r", SHAPES)
@pytest.mark.parametrize("dt", list(DT))
def test_hidden_rows_keep_every_bit(spc, dev, dt, n, c, o, r):
    w, t = Whole(n + c + o + r), DT[dt]
    x = w.ints(64, 127, n, c)
    x[:, 1000:] = 0                       # (sums below 2^23)
    down = _ranks(w.twins(32, 61, r // 2, min(c, 1000)), r, 0)
    down = torch.cat([down, w.ints(0, 9, r, c - down.shape[1])], 1)
    up = _ranks(w.signs(o, r // 2), r, 1)
    base = w.ints(-100, 100, n, o)
    h = x @ down.t()
    assert float(h.max()) > 2 ** 20 and float(h.max()) < 2 ** 24
    f = lambda v: v.to(t).to(dev)  # noqa: E731
    y, hid = spc._native.lora(f(x), f(down)[None], f(up)[None], f(base), return_hidden=True)
    _equal("hidden", hid, h)
    _equal("y", y, base + h @ up.t())


@pytest.mark.parametrize("n,c,o,r", SHAPES)
@pytest.mark.parametrize("dt", list(DT))
def test_gradients_keep_every_bit(spc, dev, dt, n, c, o, r):
    nat, w, t = spc._native, Whole(n + c + o + r), DT[dt]
    o, c = max(c, 300), o                 # (u sums many features of dy)
    f = lambda v: v.to(t).to(dev)  # noqa: E731
    dy = w.twins(64, 127, n // 2, min(o, 1000))
    dy = torch.cat([dy, torch.zeros(n, o - dy.shape[1], dtype=torch.float64)], 1)
    up = _ranks(w.twins(32, 61, r // 2, o), r, 0).t().contiguous()
    down = _ranks(w.signs(c, r // 2), r, 1).t().contiguous()
    x = w.signs(c, n // 2).t().contiguous()
    base = w.ints(-100, 100, n, c)
    u = dy @ up
    assert float(u.max()) > 2 ** 19 and float(u.max()) < 2 ** 24
    args = f(x), None, f(down)[None], f(up)[None], f(base)
    dx, dd, _ = nat.lora_backward(f(dy), *args, need=(True, True, False))
    _equal("dx", dx, base + u @ down)
    _equal("ddown", dd[0], u.t() @ x)
    # hidden rows of 24 bits, two neighbours' difference in each sum
    hidden = w.ints(2 ** 23, 2 ** 24 - 300, n // 2, r)
    hidden = torch.stack([hidden, hidden + w.ints(-100, 100, n // 2, r)], 1).reshape(n, r)
    few = w.signs(o, n // 2).t().contiguous()
    _, _, du = nat.lora_backward(f(few), f(x), hidden.float().to(dev), *args[2:4], need=(False, False, True))
    _equal("dup", du[0], few.t() @ hidden)
