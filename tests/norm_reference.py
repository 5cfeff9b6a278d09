"""The row layer norm and its gradient in 64 bits, with error bounds for an F32
computation of them.

h = (x - mean) r, z = h a + k, y = z or silu(z); a = gamma (1 + scale_b), k =
beta (1 + scale_b) + shift_b.  u = 2^-24 is one F32 rounding (relative).

A sum of c values in F32 by lanes and a tree takes at most 32 + 8 + 2 additions
on any value's way, so the mean is off by at most 42 u X, X the row's largest
magnitude; the variance's sum likewise 45 u relative (squares of differences),
with the mean's error entering squared; r adds a square root, a division and an
addition.  Hence
    |dh| <= u (50 r X + 30 |h|),      |dz| <= |a| |dh| + u 4 (|h a| + |k|)
(the coefficients a, k carry three roundings).  silu has slope at most 1.1 and
the exponential behind it a relative error of at most u (|z| + 4), which times
z sg(z) (1 - sg(z)) stays below u (|z| + 4).  The output's own rounding is half
a step, eps / 2 relative, or half of the smallest subnormal.
"""
import torch

U = 2.0 ** -24
_TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def half_step(t, dtype):
    return t.abs() * (torch.finfo(dtype).eps / 2) * 1.01 + _TINY[dtype]


class Reference:
    """Everything in float64 on the CPU; item [n] is a row's batch item, -1 for
    none."""

    def __init__(self, x, weight=None, bias=None, eps=1e-6, scale=None, shift=None, item=None,
                 silu=False):
        f = lambda t: None if t is None else t.detach().cpu().double()  # noqa: E731
        self.dtype = x.dtype
        x, w, b, scale, shift = f(x), f(weight), f(bias), f(scale), f(shift)
        n, c = x.shape
        self.item = torch.zeros(n, dtype=torch.int64) if item is None else item
        self.on = (self.item >= 0)[:, None]
        it = self.item.clamp(min=0)
        self.x, self.silu, self.c = x, silu, c
        self.gamma = torch.ones(c, dtype=torch.float64) if w is None else w
        self.beta = torch.zeros(c, dtype=torch.float64) if b is None else b
        self.s1 = torch.ones((1, c), dtype=torch.float64) if scale is None else 1 + scale
        t = torch.zeros((1, c), dtype=torch.float64) if shift is None else shift
        self.a = self.gamma * self.s1[it]
        self.k = self.beta * self.s1[it] + t[it]
        mean = x.mean(1, keepdim=True)
        self.r = 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
        self.mean = mean
        self.h = (x - mean) * self.r
        self.z = self.h * self.a + self.k
        self.sg = torch.sigmoid(self.z)
        X = x.abs().amax(1, keepdim=True)
        self.e_h = U * (50 * self.r * X + 30 * self.h.abs())
        self.e_z = self.a.abs() * self.e_h + 4 * U * ((self.h * self.a).abs() + self.k.abs())

    def forward(self):
        """(y, bound)."""
        y, e = self.z, self.e_z
        if self.silu:
            y = self.z * self.sg
            e = 1.1 * e + U * (self.z.abs() + 4)
        e = e + half_step(y.abs() + e, self.dtype)
        zero = torch.zeros_like(y)
        return torch.where(self.on, y, zero), torch.where(self.on, e, zero)

    def backward(self, dy, rows_in_a_sum):
        """dx, dgamma, dbeta, dscale, dshift as (value, bound before the
        output's rounding); rows_in_a_sum: additions on a row's way into a
        parameter's sum."""
        dy = torch.where(self.on, dy.detach().cpu().double(), torch.zeros(()).double())
        dz, e_dz = dy, torch.zeros_like(dy)
        if self.silu:
            sl = self.sg * (1 + self.z * (1 - self.sg))
            # |silu''| <= 1/2; the sigmoid's relative error u (|z| + 4) in
            # sg (1 + z (1 - sg)), each sg or 1 - sg at most 1
            e_sl = 0.5 * self.e_z + U * (self.z.abs() + 4) * (2 + self.z.abs()) \
                * self.sg.clamp(min=1e-30) * (1.1 - self.sg).clamp(max=1) * 2 + 8 * U * (
                    self.sg * (1 + self.z.abs() * (1 - self.sg)))
            dz = dy * sl
            e_dz = dy.abs() * e_sl + U * dz.abs()
        g = dz * self.a
        e_g = e_dz * self.a.abs() + 4 * U * g.abs()
        m = lambda t: t.mean(1, keepdim=True)  # noqa: E731
        m1, m2 = m(g), m(g * self.h)
        e_m1 = m(e_g) + 45 * U * m(g.abs())
        e_m2 = m(e_g * self.h.abs() + g.abs() * self.e_h) + 46 * U * m((g * self.h).abs())
        dx = self.r * (g - m1 - self.h * m2)
        e_dx = self.r * (e_g + e_m1 + self.h.abs() * e_m2 + self.e_h * m2.abs()) \
            + 35 * U * self.r * (g.abs() + m1.abs() + (self.h * m2).abs())
        out = [(torch.where(self.on, dx, torch.zeros(()).double()), e_dx)]
        nb = self.s1.shape[0]
        A, eA, B, eB = [], [], [], []
        dzh, e_dzh = dz * self.h, e_dz * self.h.abs() + dz.abs() * self.e_h
        steps = rows_in_a_sum * U
        for i in range(nb):
            p = self.item == i
            A.append(dzh[p].sum(0)), eA.append(e_dzh[p].sum(0) + steps * dzh[p].abs().sum(0))
            B.append(dz[p].sum(0)), eB.append(e_dz[p].sum(0) + steps * dz[p].abs().sum(0))
        A, eA, B, eB = map(torch.stack, (A, eA, B, eB))
        s = self.s1.abs()
        k = 1 + (nb + 4) * U
        out.append(((self.s1 * A).sum(0), k * (s * eA).sum(0) + (nb + 4) * U * (s * A.abs()).sum(0)))
        out.append(((self.s1 * B).sum(0), k * (s * eB).sum(0) + (nb + 4) * U * (s * B.abs()).sum(0)))
        ga, be = self.gamma.abs(), self.beta.abs()
        out.append((self.gamma * A + self.beta * B,
                    ga * eA + be * eB + 4 * U * (ga * A.abs() + be * B.abs())))
        out.append((B, eB))
        return out


def check(name, got, want, bound, dtype=None):
    """|got - want| <= bound (+ the rounding to dtype)."""
    got, want = got.detach().cpu().double(), want
    if dtype is not None:
        bound = bound + half_step(want.abs() + bound, dtype)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{name}: non-finite"
    over = (got - want).abs() - bound
    worst = float(((got - want).abs() / (bound + 1e-300)).max()) if got.numel() else 0.0
    print(f"[parity] {name}: worst error / bound = {worst:.3f}", flush=True)
    assert bool((over <= 0).all()), f"{name}: {int((over > 0).sum())} beyond the bound, worst {worst:.2f}"
