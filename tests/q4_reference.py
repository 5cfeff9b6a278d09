"""Q4_0 blocks and their products in 64 bits, with error bounds for the
kernels' F32 sums.

u = 2^-24.  A matrix instruction adds 32 exact products to its accumulator with
at most 32 roundings, each at most 2 u (a cut) of the magnitudes so far.  Under
16-bit rows the weights enter as 16 + q beside a sum of -24, so a block's
magnitudes are at most sum |x| d (31 + 24 + 24).  F32 rows enter as three parts
that add up exactly, so three instructions each, on the weights themselves.
"""
import numpy as np
import torch

from norm_reference import U


def random_blocks(out, inp, seed):
    """uint8 [out, inp / 32, 18]: scales of both signs and all q."""
    g = np.random.default_rng(seed)
    d = (g.standard_normal((out, inp // 32)) * 0.01).astype(np.float16)
    b = np.empty((out, inp // 32, 18), np.uint8)
    b[..., :2] = d[..., None].view(np.uint8)
    b[..., 2:] = g.integers(0, 256, (out, inp // 32, 16))
    return torch.from_numpy(b)


def parts(blocks):
    """(d [out, in / 32], q - 8 [out, in]) in float64."""
    b = blocks.cpu().numpy()
    d = np.ascontiguousarray(b[..., :2]).view(np.float16)[..., 0].astype(np.float64)
    q = np.concatenate([b[..., 2:] & 15, b[..., 2:] >> 4], -1).astype(np.float64) - 8
    return torch.from_numpy(d), torch.from_numpy(q.reshape(b.shape[0], -1))


def dequant(blocks):
    d, q = parts(blocks)
    return q * d.repeat_interleave(32, 1)


def product(x, blocks, bias=None):
    """(y, bound before the output's rounding) for x [m, in]."""
    f32 = x.dtype == torch.float32
    x = x.detach().cpu().double()
    w = dequant(blocks)
    d = parts(blocks)[0].abs().repeat_interleave(32, 1)
    y = x @ w.t()
    e = 2 * 96 * U * (x.abs() @ w.abs().t()) if f32 else 2 * 32 * U * 79 * (x.abs() @ d.t())
    e = e + (w.shape[1] // 32 + 12) * U * (x.abs() @ w.abs().t())
    if bias is not None:
        bias = bias.detach().cpu().double()
        y = y + bias
        e = e + 2 * U * (y.abs() + bias.abs())
    return y, e


def gradient(dy, blocks):
    """(dx, bound before the output's rounding) for dy [m, out].

    F32 rows: dy d rounded once (u), three parts as above.  f16 rows: the weights
    exactly, as f16(w) and the rest, two instructions a group of 32.  bf16 rows:
    the weights rounded to f16 (2^-11 of each; subnormal ones are multiples of
    their scale's last bit, so exact), without what lies below 2^-28 of the row's
    largest value."""
    f32 = dy.dtype == torch.float32
    bf16 = dy.dtype == torch.bfloat16
    dy = dy.detach().cpu().double()
    w = dequant(blocks)
    # eight waves share the summed features: instructions on one accumulator
    chain = (3 if f32 else 1 if bf16 else 2) * (-(-w.shape[0] // 128) // 8 + 1) * 4
    e = ((U if f32 else 2.0 ** -11 if bf16 else 0.0) + 2 * (32 + chain + 12) * U) * (dy.abs() @ w.abs())
    if bf16 and dy.numel():
        e = e + 2.0 ** -28 * dy.abs().amax(1, keepdim=True) * w.abs().sum(0)
    return dy @ w, e
