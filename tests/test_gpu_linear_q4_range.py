"""4-bit products of rows whose values lie far apart: what a value contributes
does not depend on the largest one of its row.

u = 2^-24; a matrix instruction adds 32 exact products with at most 32 roundings
of 2 u each (a cut) of the magnitudes so far, a chain of instructions on one
accumulator one more each; see q4_reference."""
import pytest
import torch

from norm_reference import U, check
from q4_reference import dequant, random_blocks

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _gradient(dy, blocks):
    """(dx, bound before the output's rounding), relative to sum |dy w| alone: a
    value on zero weights adds nothing to it.  F32 rows times the scale round
    once (u); bf16 rows meet f16(w), 2^-11 at most.  Up to three operands, eight
    waves or more; parts of F32 products below 2^-126 count as zero (2^-122 an
    element, q4_reference)."""
    d, w = dy.detach().cpu().double(), dequant(blocks)
    weights = {torch.float32: U, torch.bfloat16: 2.0 ** -11, torch.float16: 0.0}[dy.dtype]
    chain = 3 * (-(-w.shape[0] // 128) // 8 + 1) * 4
    e = (weights + 2 * (32 + chain + 16) * U) * (d.abs() @ w.abs())
    return d @ w, e + (w.shape[0] * 2.0 ** -122 if dy.dtype == torch.float32 else 0.0)


# blocks of 4, 8, 16 and 32 rows, of one and two column tiles, eight and sixteen waves
@pytest.mark.parametrize("out,inp,m", [
    (256, 64, 1), (2500, 96, 1), (2500, 96, 7), (16_500, 32, 4), (16_500, 64, 30), (300, 8256, 3),
    (300, 4096, 6), (300, 4096, 16), (300, 4096, 30), (8200, 4096, 13), (16_500, 4096, 16),
    (300, 2048, 90), (300, 8256, 40)])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_gradient_under_large_values_on_zero_weights(spc, dev, dt, out, inp, m):
    """Rows whose large values stand where every weight is zero: the others'
    products are the result, down to a type's last binade."""
    blocks = random_blocks(out, inp, out + inp)
    dead = torch.randperm(out, generator=torch.Generator().manual_seed(1))[:out // 50 + 1]
    blocks[dead, :, 2:] = 0x88
    bwd = spc._native.pack_q4_0(blocks.to(dev), out_features=out, in_features=inp, transpose=True)
    dy = torch.randn(m, out, generator=torch.Generator().manual_seed(2))
    for large, scale in [(1e4, 1e-4)] + ([] if dt == "f16" else [(1e30, 1e-3), (1e37, 1e-20)]):
        x = dy * scale
        x[:, dead] = large
        x = x.to(DT[dt]).to(dev)
        check(f"dx {dt} {large} over {scale}", spc._native.linear_q4_0_input_grad(x, bwd),
              *_gradient(x, blocks), DT[dt])



@pytest.mark.parametrize("out,inp,m", [(16_500, 32, 4), (16_500, 4096, 16), (2600, 8256, 8), (2600, 8256, 40)])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_gradient_before_large_values_on_zero_weights(spc, dev, dt, out, inp, m):
    """Large values at a row's end only: what was summed before they were met
    stays."""
    blocks = random_blocks(out, inp, out)
    blocks[-3:, :, 2:] = 0x88
    bwd = spc._native.pack_q4_0(blocks.to(dev), out_features=out, in_features=inp, transpose=True)
    for large, scale in [(1e5, 1e-5), (1e20, 1e-10), (3e38, 1e-20), (3e38, 1e-30)]:
        x = torch.randn(m, out, generator=torch.Generator().manual_seed(2)) * scale
        x[:, -3:] = large
        x = x.to(DT[dt]).to(dev)
        check(f"dx {dt} {large} after {scale}", spc._native.linear_q4_0_input_grad(x, bwd),
              *_gradient(x, blocks), DT[dt])


@pytest.mark.parametrize("out,inp,m", [(2600, 8256, 4), (16_500, 2048, 7), (2600, 8256, 16), (2600, 2048, 60)])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_rows_do_not_depend_on_each_other(spc, dev, dt, out, inp, m):
    """Bit for bit, whatever range the rows beside them have."""
    blocks = random_blocks(out, inp, out + m)
    bwd = spc._native.pack_q4_0(blocks.to(dev), out_features=out, in_features=inp, transpose=True)
    dy = torch.randn(m, out, generator=torch.Generator().manual_seed(m)).to(DT[dt]).to(dev)
    want = spc._native.linear_q4_0_input_grad(dy, bwd)
    dy[1::4, ::3] *= 2.0 ** -20 if dt == "f16" else 2.0 ** -60
    dy[2::4, out // 2:] *= 2.0 ** 10 if dt == "f16" else 2.0 ** 40
    dy[3, out - 1] = float("inf")
    got = spc._native.linear_q4_0_input_grad(dy, bwd)
    assert torch.equal(got[::4], want[::4])

def _product(x, blocks):
    """(y, bound before the output's rounding), relative to sum |x w| alone: a
    block's 32 products x (q - 8) are exact, in one matrix instruction (F32 rows:
    three), then one addition a block and the waves'."""
    d, w = x.detach().cpu().double(), dequant(blocks)
    steps = (96 if x.dtype == torch.float32 else 32) * 2 + w.shape[1] // 32 + 17
    return d @ w.t(), steps * U * (d.abs() @ w.abs().t())


@pytest.mark.parametrize("out,inp,m", [
    (64, 128, 1), (64, 128, 16), (190, 416, 30), (4100, 64, 17), (20, 16_416, 13), (8300, 64, 40),
    (2100, 96, 100)])
@pytest.mark.parametrize("dt,large", [("f16", 6e4), ("bf16", 2.0 ** 20), ("bf16", 2e37), ("bf16", 3e38),
                                      ("f32", 2.0 ** 20), ("f32", 3e38)])
def test_product_under_large_values_on_zero_weights(spc, dev, dt, large, out, inp, m):
    """A large value that meets zero weights only leaves no trace, in its
    block's sums or elsewhere; on other weights it is a term like any."""
    blocks = random_blocks(out, inp, out + inp)
    blocks[:, :, 2] = blocks[:, :, 2] & 0xf0 | 8          # weight 0 of every block: zero
    fwd = spc._native.pack_q4_0(blocks.to(dev), out_features=out, in_features=inp)
    x = torch.randn(m, inp, generator=torch.Generator().manual_seed(3))
    x[:, ::32] = torch.where(torch.arange(m)[:, None] % 2 == 0, large, -large)
    x = x.to(DT[dt]).to(dev)
    check(f"y {dt} {large}", spc._native.linear_q4_0(x, fwd), *_product(x, blocks), DT[dt])
    x[:, 5] = large                                       # and on weights of every size
    y, bound = _product(x, blocks)
    got = spc._native.linear_q4_0(x, fwd)
    fits = y.abs() + bound < torch.finfo(DT[dt]).max * 0.99
    check(f"y {dt} {large} met", torch.where(fits.to(dev), got, 0), torch.where(fits, y, 0),
          torch.where(fits, bound, 0), DT[dt])


@pytest.mark.parametrize("m", [1, 513])
def test_bias_gradient_of_the_widest_linear(spc, dev, m):
    """2^27 features, as many as the products take, by one kernel and by two
    (rows that repeat: the sums are exact)."""
    o = 1 << 27
    row = torch.randint(-128, 128, (1, o), device=dev, dtype=torch.int16).to(torch.bfloat16)
    db = spc._native.linear_q4_0_bias_grad(row.expand(m, o))
    assert bool((db == row[0].float() * m).all())


def test_elements_past_32_bits(spc, dev):
    """Rows further apart than 2^31 elements, and outputs of more than 2^32."""
    nat = spc._native
    blocks = random_blocks(4128, 32, 7)
    fwd = nat.pack_q4_0(blocks.to(dev), out_features=4128, in_features=32)
    wide = random_blocks(16, 4128, 8)
    bwd = nat.pack_q4_0(wide.to(dev), out_features=16, in_features=4128, transpose=True)
    ld = (1 << 31) + 8
    far = torch.empty(2 * ld + 32, dtype=torch.bfloat16, device=dev).as_strided((3, 32), (ld, 1))
    far.copy_(torch.randn(3, 32, generator=torch.Generator().manual_seed(1)))
    check("y far", nat.linear_q4_0(far, fwd), *_product(far, blocks), torch.bfloat16)
    check("dx far", nat.linear_q4_0_input_grad(far[:, :16], bwd), *_gradient(far[:, :16], wide),
          torch.bfloat16)
    del far
    m = 65_535 * 16
    assert m * 4128 > 1 << 32
    x = torch.randn(m, 32, device=dev).bfloat16()
    rows = [0, 1, 31, m // 2 + 5, 1_040_448, 1_040_449, m - 17, m - 1]   # (1,040,447.8: element 2^32)
    y = nat.linear_q4_0(x, fwd)
    check("y", y[rows], *_product(x[rows], blocks), torch.bfloat16)
    db = nat.linear_q4_0_bias_grad(y)
    for cols in (slice(0, 2), slice(4126, 4128)):
        want = y[:, cols].double()
        # a thread's 64 rows of a block's 2,048, lanes, waves, then 512 blocks' sums
        check("dbias", db[cols], want.sum(0).cpu(), 2.0 ** -24 * 200 * want.abs().sum(0).cpu(),
              torch.float32)
    del y
    dx = nat.linear_q4_0_input_grad(x[:, :16], bwd)
    check("dx", dx[rows], *_gradient(x[rows, :16], wide), torch.bfloat16)


@pytest.mark.parametrize("out,inp,m", [(130, 1024, 1), (1024, 192, 6), (1000, 1024, 16), (1024, 4096, 30),
                                       (70, 96, 200)])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_sums_of_whole_numbers_are_exact(spc, dev, dt, out, inp, m):
    """Rows of whole numbers up to 128 and scales +-2^-6 .. 2^-3: every sum over
    1,024 features stays below 2^23 of its last bit, so nothing may be lost before
    the output's rounding."""
    nat = spc._native
    blocks = random_blocks(out, inp, out + m)
    g = torch.Generator().manual_seed(out)
    d = 2.0 ** torch.randint(-6, -2, (out, inp // 32), generator=g) * (
        2 * torch.randint(0, 2, (out, inp // 32), generator=g) - 1)
    blocks[..., :2] = d.half()[..., None].view(torch.uint8)
    w = dequant(blocks)
    kw = dict(out_features=out, in_features=inp)
    fwd, bwd = nat.pack_q4_0(blocks.to(dev), **kw), nat.pack_q4_0(blocks.to(dev), transpose=True, **kw)
    x, dy = (torch.randint(-128, 129, (m, k), generator=g).to(DT[dt]) for k in (min(inp, 1024), out))
    x = torch.cat([x, torch.zeros(m, inp - x.shape[1], dtype=DT[dt])], 1)
    assert torch.equal(nat.linear_q4_0(x.to(dev), fwd).cpu(), (x.double() @ w.t()).to(DT[dt]))
    assert torch.equal(nat.linear_q4_0_input_grad(dy.to(dev), bwd).cpu(), (dy.double() @ w).to(DT[dt]))
    assert torch.equal(nat.linear_q4_0_bias_grad(dy.to(dev)).cpu(), dy.float().sum(0))


def test_f32_rows_keep_24_bits(spc, dev):
    """One value of a row against weights that are powers of two: the product is
    that value's, all 24 bits of it."""
    nat = spc._native
    blocks = random_blocks(64, 128, 3)
    blocks[..., :2] = torch.tensor([0.125]).half().view(torch.uint8)
    q = torch.tensor([0, 4, 6, 7, 8, 9, 10, 12])          # q - 8: -8, -4, -2, -1, 0, 1, 2, 4
    pick = q[torch.randint(0, 8, (2, 64, 4, 16), generator=torch.Generator().manual_seed(1))]
    blocks[..., 2:] = (pick[0] | pick[1] << 4).to(torch.uint8)
    w = dequant(blocks)
    kw = dict(out_features=64, in_features=128)
    fwd, bwd = nat.pack_q4_0(blocks.to(dev), **kw), nat.pack_q4_0(blocks.to(dev), transpose=True, **kw)
    for n, run, weights in ((128, lambda t: nat.linear_q4_0(t, fwd), w.t()),
                            (64, lambda t: nat.linear_q4_0_input_grad(t, bwd), w)):
        v = torch.randn(n, generator=torch.Generator().manual_seed(n)) * 10.0 ** torch.linspace(-25, 25, n)
        assert torch.equal(run(torch.diag(v).to(dev)).cpu().double(), v.double()[:, None] * weights)
