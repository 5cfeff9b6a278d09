"""Dropout's mask, low-rank adapters and their gradients in 64 bits, with error
bounds for a computation with F32 sums.

u = 2^-24.  A matrix instruction adds up to 32 products to its accumulator with at
most 32 roundings, each at most 2 u (a cut) of the magnitudes so far; an addition
elsewhere is one u.  Products of two 16-bit values are exact, of two F32 values
off by u.  F32 hidden rows that meet 16-bit operands enter as two bf16 parts,
whose sum is off by at most 2^-17 of the value (two roundings of 2^-9, the second
of what the first left, so 2^-18, doubled for good measure where a part is
subnormal: 2^-133 absolute).  The dropout factor, the adapter's scale and the base
add a rounding each.  The output's own rounding is half a step.
"""
import numpy as np
import torch

from norm_reference import U, half_step

SPLIT = 2.0 ** -17
TINY = 2.0 ** -125   # parts and products at the end of F32's range


def philox(counter, key, rounds=7):
    """Philox4x32 of four uint64 arrays (32-bit values) and two 32-bit ints."""
    m0, m1, low, half = np.uint64(0xD2511F53), np.uint64(0xCD9E8D57), np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [np.asarray(v, np.uint64) for v in counter]
    k = list(key)
    for _ in range(rounds):
        p0, p1 = c[0] * m0, c[2] * m1
        c = [(p1 >> half) ^ c[1] ^ np.uint64(k[0]), p1 & low, (p0 >> half) ^ c[3] ^ np.uint64(k[1]), p0 & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return c


def threshold(p):
    return int(np.floor(p * 65536 + 0.5))


def factors(seed, rows, c, p, first=0):
    """float64 [rows, c]: 0 where dropped, 1 / (1 - p) elsewhere."""
    t = threshold(p)
    if t == 0:
        return torch.ones(rows, c, dtype=torch.float64)
    s = [int(v) % 2 ** 64 for v in seed]
    g = (c + 7) // 8
    k = np.arange(first * g, (first + rows) * g, dtype=np.uint64)
    full = lambda v: np.full_like(k, v)  # noqa: E731
    w = philox([k & np.uint64(0xFFFFFFFF), k >> np.uint64(32), full(s[1] % 2 ** 32), full(s[1] >> 32)],
               [s[0] % 2 ** 32, s[0] >> 32])
    bits = np.stack([np.stack([v & np.uint64(0xFFFF), v >> np.uint64(16)], -1) for v in w], -2)
    keep = bits.reshape(rows, 8 * g)[:, :c] >= t
    return torch.from_numpy(keep.astype(np.float64) * (65536 / (65536 - t) if t < 65536 else 0.0))


def adapter_of_rows(n, k, offsets=None, adapters=None):
    """int64 [n], -1 for rows without one."""
    ids = None if adapters is None else [int(v) for v in adapters]
    items = 1 if ids is None else len(ids)
    off = range(0, n + 1, max(n // items, 1)) if offsets is None else [int(v) for v in offsets]
    ids = [0] * (len(off) - 1) if ids is None else ids
    of = torch.full((n,), -1, dtype=torch.int64)
    for lo, hi, a in zip(off, off[1:], ids):
        if 0 <= a < k:
            of[max(lo, 0):max(min(hi, n), 0)] = a
    return of


def dropout(x, p, seed, residual=None):
    """(y, bound)."""
    f = factors(seed, *x.shape, p)
    v = torch.where(f > 0, x.detach().cpu().double() * f, torch.zeros(()).double())
    e = 2 * U * v.abs()
    if residual is not None:
        r = residual.detach().cpu().double()
        e = e + U * (v.abs() + r.abs())
        v = v + r
    return v, e + half_step(v.abs() + e, x.dtype)


class Adapters:
    """Everything in float64 on the CPU."""

    def __init__(self, x, down, up, scale=None, offsets=None, adapters=None, p=0.0, seed=None):
        f = lambda t: t.detach().cpu().double()  # noqa: E731
        self.dtype, self.exact = x.dtype, x.dtype != torch.float32
        self.down, self.up = f(down), f(up)
        self.k, self.r, self.c = self.down.shape
        self.o = self.up.shape[1]
        self.n = x.shape[0]
        self.of = adapter_of_rows(self.n, self.k, offsets, adapters)
        self.scale = torch.ones(self.k, dtype=torch.float64) if scale is None else f(scale)
        self.f = torch.ones_like(x, dtype=torch.float64, device="cpu") if not p else \
            factors(seed, self.n, self.c, p)
        on = (self.of >= 0)[:, None] & (self.f > 0)
        self.x = torch.where(on, f(x) * self.f, torch.zeros(()).double())

    # roundings on the way of a value into a sum of c products
    @staticmethod
    def _sum(c):
        return 2 * 32 + c // 8 + 40

    def _product(self, v, w, e_v, split):
        """(v @ w, bound) for rows v with errors e_v; split: F32 rows against
        16-bit operands."""
        m = v.abs() @ w.abs()
        e = e_v @ w.abs() + (self._sum(v.shape[1]) * 2 * U + (SPLIT if split else U)) * m
        return v @ w, e + v.shape[1] * TINY * (1 + w.abs().sum(0))

    def forward(self, base=None):
        """(y, bound), (hidden, bound)."""
        y = torch.zeros(self.n, self.o, dtype=torch.float64)
        ey = torch.zeros_like(y)
        h = torch.zeros(self.n, self.r, dtype=torch.float64)
        eh = torch.zeros_like(h)
        b = torch.zeros_like(y) if base is None else base.detach().cpu().double()
        y += b
        for a in range(self.k):
            on = self.of == a
            h[on], eh[on] = self._product(self.x[on], self.down[a].t(), 3 * U * self.x[on].abs(), False)
            z, e = self._product(h[on], self.up[a].t(), eh[on], self.exact)
            s = self.scale[a]
            y[on] = b[on] + s * z
            ey[on] = s.abs() * e + 3 * U * (s * z).abs() + 2 * U * b[on].abs()
        return (y, ey + half_step(y.abs() + ey, self.dtype)), (h, eh)

    def backward(self, dy, hidden, dx_base=None):
        """(dx, bound), (ddown, bound), (dup, bound), roundings included."""
        dy = torch.where((self.of >= 0)[:, None], dy.detach().cpu().double(), torch.zeros(()).double())
        dx = torch.zeros(self.n, self.c, dtype=torch.float64) if dx_base is None else \
            dx_base.detach().cpu().double().clone()
        ex = torch.zeros_like(dx)
        dd, ed = torch.zeros_like(self.down), torch.zeros_like(self.down)
        du, eu = torch.zeros_like(self.up), torch.zeros_like(self.up)
        h = None if hidden is None else hidden.detach().cpu().double()
        for a in range(self.k):
            on = self.of == a
            s = self.scale[a]
            u, e = self._product(dy[on], self.up[a], 0 * dy[on], False)
            u, e = s * u, s.abs() * e + 2 * U * (s * u).abs()
            z, ez = self._product(u, self.down[a], e, self.exact)
            z, ez = z * self.f[on], (ez + 3 * U * z.abs()) * self.f[on]
            ex[on] = ez + 2 * U * (dx[on].abs() + z.abs())
            dx[on] += z
            g, eg = self._product(self.x[on].t(), u, 3 * U * self.x[on].t().abs(), self.exact)
            dd[a] = g.t()
            ed[a] = (eg + self.x[on].t().abs() @ e + 3 * U * g.abs()).t()
            if h is not None:
                g, eg = self._product(dy[on].t(), h[on], 0 * dy[on].t(), self.exact)
                du[a], eu[a] = s * g, s.abs() * (eg + 3 * U * g.abs())
        return tuple((v, e + half_step(v.abs() + e, self.dtype)) for v, e in ((dx, ex), (dd, ed), (du, eu)))
