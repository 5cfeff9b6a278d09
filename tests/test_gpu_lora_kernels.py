"""Each kernel of the adapters and of their gradients (lora_routes), with and
without dropout, against the 64-bit form at small sizes that select it."""
import pytest

from test_gpu_lora import DT, Case

pytestmark = pytest.mark.gpu

# rows, items, adapters, in, out, rank
CASES = [
    # gradients: a block's waves along columns, ranks and rows
    (400, 1, 1, 400, 1000, 16), (400, 1, 1, 1000, 400, 9), (300, 2, 2, 200, 150, 16), (330, 1, 1, 40, 60, 7),
    (400, 1, 1, 300, 260, 30), (350, 3, 2, 60, 50, 20), (350, 1, 1, 60, 40, 17), (300, 1, 1, 200, 300, 50), (300, 2, 1, 70, 500, 64),
    (260, 1, 1, 200, 400, 100), (260, 2, 2, 60, 300, 128), (350, 1, 1, 130, 700, 12), (400, 1, 1, 100, 300, 11), (200, 50, 40, 72, 136, 16),
    # gradients of few rows
    (20, 20, 3, 130, 72, 13), (20, 20, 20, 72, 130, 32), (24, 24, 2, 200, 90, 64), (20, 20, 2, 136, 72, 65), (30, 10, 3, 72, 200, 128),
    # hidden sums of wide rows in a launch of their own
    (8, 2, 2, 8192, 40, 16), (8, 8, 2, 8200, 40, 20), (8, 1, 1, 8192, 72, 64), (9, 3, 2, 8185, 40, 128), (1, 1, 1, 8192, 40, 100),
    # tiles of 32 and of 64 rows
    (12_300, 2, 2, 40, 72, 8), (12_300, 1, 1, 72, 33, 20), (12_300, 3, 2, 33, 40, 40), (12_300, 2, 2, 40, 24, 128),
    (24_600, 2, 2, 24, 40, 33),
]


@pytest.mark.parametrize("n,items,k,c,o,r", CASES)
@pytest.mark.parametrize("p", [0.0, 0.2])
@pytest.mark.parametrize("dt", list(DT))
def test_kernels(spc, dev, dt, p, n, items, k, c, o, r):
    # uneven items, one of none at the end if there are three, rows behind them
    off = [i * (n - 1) // items + (i % 2 if i < items and n > 4 * items else 0) for i in range(items + 1)]
    ids = [k - 1 - i % k if i != 2 else -1 for i in range(items)]
    Case(dev, dt, n, c, o, r, k=k, offsets=off, adapters=ids, p=p, base=p == 0).check(spc._native)
