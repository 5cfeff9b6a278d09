"""Products with Q4_0 weights (nat.linear_q4_0, nat.linear_q4_0_input_grad,
Q4Linear, SparseLinear, SparseResBlock3d's modulation) against 64 bits.  Bounds:
tests/q4_reference.py."""
import importlib

import numpy as np
import pytest
import torch

from norm_reference import Reference, check
from q4_reference import dequant, gradient, parts, product, random_blocks

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SHAPES = [(1, 32), (16, 32), (17, 64), (15, 96), (50, 160), (128, 128), (129, 256), (256, 1024),
          (531, 3872), (2048, 512), (33, 8192)]


def _both(nat, blocks, dev):
    out, groups, _ = blocks.shape
    b = blocks.to(dev)
    kw = dict(out_features=out, in_features=32 * groups)
    return nat.pack_q4_0(b, **kw), nat.pack_q4_0(b, transpose=True, **kw)


def _randn(shape, seed, dt, dev):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dt).to(dev)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("out,inp", [(1, 32), (17, 64), (50, 160), (300, 384)])
def test_unit_rows_give_the_weights(spc, dev, dt, out, inp):
    """Rows of the identity: d (q - 8) is exact in F32, so every weight comes
    back at its place bit for bit (rounded once to 16-bit outputs; the gradient
    of bf16 rows takes them as f16)."""
    nat = spc._native
    blocks = random_blocks(out, inp, out + inp)
    fwd, bwd = _both(nat, blocks, dev)
    w = dequant(blocks)
    y = nat.linear_q4_0(torch.eye(inp, dtype=DT[dt], device=dev), fwd)
    assert torch.equal(y.cpu(), w.t().to(DT[dt]))
    dx = nat.linear_q4_0_input_grad(torch.eye(out, dtype=DT[dt], device=dev), bwd)
    assert torch.equal(dx.cpu(), (w.half() if dt == "bf16" else w).to(DT[dt]))


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("out,inp", SHAPES)
def test_shapes(spc, dev, dt, out, inp):
    nat = spc._native
    blocks = random_blocks(out, inp, out * 7 + inp)
    fwd, bwd = _both(nat, blocks, dev)
    for m in (1, 3):
        x = _randn((m, inp), m, DT[dt], dev)
        bias = _randn((out,), 5, torch.float32, dev)
        check(f"y {dt} {m}x{inp}->{out}", nat.linear_q4_0(x, fwd, bias), *product(x, blocks, bias), DT[dt])
        dy = _randn((m, out), m + 9, DT[dt], dev)
        check(f"dx {dt} {m}x{out}->{inp}", nat.linear_q4_0_input_grad(dy, bwd), *gradient(dy, blocks),
              DT[dt])


@pytest.mark.parametrize("m", [1, 2, 4, 5, 7, 15, 16, 17, 31, 33, 48, 63, 64, 65, 130, 1000])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_rows(spc, dev, dt, m):
    nat = spc._native
    out, inp = 190, 416
    blocks = random_blocks(out, inp, 3)
    fwd, bwd = _both(nat, blocks, dev)
    x, dy = _randn((m, inp), m, DT[dt], dev), _randn((m, out), m + 1, DT[dt], dev)
    check(f"y m={m}", nat.linear_q4_0(x, fwd), *product(x, blocks), DT[dt])
    check(f"dx m={m}", nat.linear_q4_0_input_grad(dy, bwd), *gradient(dy, blocks), DT[dt])


def test_no_rows(spc, dev):
    fwd, bwd = _both(spc._native, random_blocks(20, 64, 1), dev)
    assert spc._native.linear_q4_0(torch.empty((0, 64), device=dev), fwd).shape == (0, 20)
    assert spc._native.linear_q4_0_input_grad(torch.empty((0, 20), device=dev), bwd).shape == (0, 64)


@pytest.mark.parametrize("bdt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_bias_types(spc, dev, dt, bdt):
    nat = spc._native
    blocks = random_blocks(77, 96, 2)
    fwd, _ = _both(nat, blocks, dev)
    x = _randn((5, 96), 1, DT[dt], dev)
    bias = _randn((78,), 2, DT[bdt], dev)[1:]
    check("y", nat.linear_q4_0(x, fwd, bias), *product(x, blocks, bias), DT[dt])


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_strides(spc, dev, dt):
    """Rows at any stride and element, broadcast rows, transposed storage."""
    nat = spc._native
    out, inp = 100, 160
    blocks = random_blocks(out, inp, 4)
    fwd, bwd = _both(nat, blocks, dev)
    base = _randn((12, 400), 1, DT[dt], dev)
    for c0, step in [(0, 1), (8, 2), (1, 1), (3, 3)]:
        x, dy = base[::step, c0:c0 + inp], base[::step, c0 + 2:c0 + 2 + out]
        check(f"y +{c0} /{step}", nat.linear_q4_0(x, fwd), *product(x, blocks), DT[dt])
        check(f"dx +{c0} /{step}", nat.linear_q4_0_input_grad(dy, bwd), *gradient(dy, blocks), DT[dt])
    x = base[:1, :inp].expand(20, inp)
    check("broadcast", nat.linear_q4_0(x, fwd), *product(x, blocks), DT[dt])
    t = _randn((inp, 9), 2, DT[dt], dev).t()
    check("transposed", nat.linear_q4_0(t, fwd), *product(t, blocks), DT[dt])


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_infinite_rows_stay_alone(spc, dev, dt):
    nat = spc._native
    fwd, bwd = _both(nat, random_blocks(40, 96, 4), dev)
    x, dy = _randn((20, 96), 1, DT[dt], dev), _randn((20, 40), 2, DT[dt], dev)
    y, dx = nat.linear_q4_0(x, fwd), nat.linear_q4_0_input_grad(dy, bwd)
    x[3, 5], x[7, 0], dy[2, 39], dy[9, 1] = float("inf"), float("nan"), float("-inf"), float("nan")
    y2, dx2 = nat.linear_q4_0(x, fwd), nat.linear_q4_0_input_grad(dy, bwd)
    keep = torch.ones(20, dtype=torch.bool, device=dev)
    keep[3] = keep[7] = False
    assert torch.equal(y2[keep], y[keep]) and bool(y2[~keep].isnan().all())
    keep = torch.ones(20, dtype=torch.bool, device=dev)
    keep[2] = keep[9] = False
    assert torch.equal(dx2[keep], dx[keep]) and not bool(dx2[~keep].isfinite().any())


def test_large_and_small_magnitudes(spc, dev):
    """F32 rows at the ends of the exponent: the three parts keep 24 bits."""
    nat = spc._native
    blocks = random_blocks(64, 128, 6)
    fwd, bwd = _both(nat, blocks, dev)
    x, dy = _randn((4, 128), 1, torch.float32, dev), _randn((4, 64), 2, torch.float32, dev)
    for s in (1e30, 1e-20):
        check(f"y {s}", nat.linear_q4_0(x * s, fwd), *product(x * s, blocks), torch.float32)
        check(f"dx {s}", nat.linear_q4_0_input_grad(dy * s, bwd), *gradient(dy * s, blocks),
              torch.float32)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("out,inp", [(2500, 96), (2051, 15_456)])
def test_gradient_rows_of_any_range(spc, dev, dt, out, inp):
    """Rows whose magnitudes lie anywhere and change along the row by 2^20 and
    more: zeros first, growing, falling, single large and single tiny values."""
    nat = spc._native
    blocks = random_blocks(out, inp, 8)
    _, bwd = _both(nat, blocks, dev)
    g = torch.Generator().manual_seed(3)
    dy = torch.randn(19, out, generator=g)
    n = torch.arange(out)
    dy[0] = 0
    dy[1, :2000] = 0
    dy[2] *= 2.0 ** (n / 60 - 20)                 # grows 2^41
    dy[3] *= 2.0 ** (20 - n / 60)
    dy[4] *= torch.where(n % 128 == 5, 1e6, 1e-6)
    dy[5] *= 1e30
    dy[6] *= 1e-30
    dy[7] *= 1e-38                                # bf16 and F32 subnormals among them
    dy[8] = 0
    dy[8, out - 1] = 3e38
    dy[9] = 0
    dy[9, 1300] = 1e-39
    dy[10, 1200:1400] *= 1e9
    dy[11] *= 2.0 ** (n % 130 - 65).float()       # every group spans 2^130
    dy[12] *= 3.0 ** (n // 128 % 20 - 10).float()
    dy = dy.to(DT[dt]).to(dev)
    dx, bound = gradient(dy, blocks)
    if dt == "f32":
        # parts of dy d below 2^-126 count as zero: of an element's three cuts
        # (each below 2^-7 of the one before) less than 2^-125 in all, times |q - 8|
        # <= 8
        bound = bound + out * 2.0 ** -122
    got = nat.linear_q4_0_input_grad(dy, bwd)
    check(f"any range {dt}", got, dx, bound, DT[dt])
    # strided rows, at an odd element; alone, a row is as among the others up to
    # the order of its sums
    wide = torch.cat([dy[:, :1], dy, dy[:, :3]], 1)
    check(f"any range {dt} strided", nat.linear_q4_0_input_grad(wide[:, 1:out + 1], bwd), dx, bound,
          DT[dt])
    check(f"any range {dt} row", nat.linear_q4_0_input_grad(dy[4:5], bwd), dx[4:5], bound[4:5], DT[dt])
    dy[3, 7], dy[5, out - 1] = float("inf"), float("nan")
    bad = nat.linear_q4_0_input_grad(dy, bwd)
    keep = [i for i in range(19) if i not in (3, 5)]
    assert torch.equal(bad[keep], got[keep]) and not bool(bad[[3, 5]].isfinite().any())


def test_quantize(spc, dev):
    """d is the largest value over -8 in f16; every q is within half a step (and
    the F32 product's rounding, 2^-20 of a step) of its weight or at an end."""
    nat = spc._native
    w = torch.randn(70, 160, generator=torch.Generator().manual_seed(1)) * 0.05
    w[3, 32:64] = 0
    w[4, :32] = 0.25
    b = nat.q4_0_quantize(w.to(dev)).cpu().view(70, 5, 18)
    d, q = parts(b)
    g = w.view(70, 5, 32)
    top = g.gather(2, g.abs().argmax(2, keepdim=True))[..., 0]
    assert torch.equal(d, (top / -8).half().double())
    step = d.abs().repeat_interleave(32, 1)
    err = (w.double() - q * d.repeat_interleave(32, 1)).abs()
    inside = err <= step * (0.5 + 2.0 ** -20)
    end = (q == 7) | (q == -8)
    assert bool((inside | end).all())
    # past an end: the largest value is -8 d up to d's rounding (2^-11 of 8
    # steps), values of the other sign reach 7 d of at most 8 d
    assert bool((err <= step * (1 + 8 * 2.0 ** -10))[end].all())
    assert bool((q[3, 32:64] == 0).all()) and bool((b[3, 1, :2] == 0).all())


def test_equal_calls_streams_and_graphs(spc, dev):
    nat = spc._native
    fwd, bwd = _both(nat, random_blocks(256, 512, 4), dev)
    x, dy = _randn((9, 512), 1, torch.bfloat16, dev), _randn((9, 256), 2, torch.bfloat16, dev)

    def step():
        return nat.linear_q4_0(x, fwd), nat.linear_q4_0_input_grad(dy, bwd)

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(4):
        x.copy_(torch.randn(9, 512, device=dev) * (i + 1))
        dy.copy_(torch.randn(9, 256, device=dev))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, step()))


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("out,inp,m", [
    (8200, 64, 3), (8200, 64, 9), (16_500, 32, 16),             # long sums of the gradient
    (40, 8224, 2), (20, 16_416, 13),                            # and of the forward pass
    (1040, 96, 7), (2100, 96, 11), (4100, 64, 17), (4100, 64, 30), (64, 4128, 31), (70, 128, 200)])
def test_row_tiles(spc, dev, dt, out, inp, m):
    """Row counts around the blocks' 4, 8, 16 and 32 rows, where the columns are
    few, many, or the summed features long."""
    nat = spc._native
    blocks = random_blocks(out, inp, m)
    fwd, bwd = _both(nat, blocks, dev)
    x, dy = _randn((m, inp), 1, DT[dt], dev), _randn((m, out), 2, DT[dt], dev)
    check("y", nat.linear_q4_0(x, fwd), *product(x, blocks), DT[dt])
    check("dx", nat.linear_q4_0_input_grad(dy, bwd), *gradient(dy, blocks), DT[dt])


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,o", [(0, 5), (1, 1), (3, 33), (31, 130), (512, 64), (513, 31), (5000, 130),
                                 (262_200, 3)])
def test_bias_gradient(spc, dev, dt, m, o):
    """Column sums of strided rows, in every dtype of the bias, a captured one too."""
    nat = spc._native
    dy = _randn((m, o + 3), m + o, dt, dev)[:, 1:1 + o]
    ref = dy.cpu().double()
    # additions one behind another: a thread's rows, a wave's two lanes and the
    # sixteen waves, and the second pass over at most 512 blocks' sums
    per = max(512, -(-m // 512))
    steps = -(-per // 32) + 17 + 33
    bound = steps * 2.0 ** -24 * ref.abs().sum(0)
    for bdt in (torch.float32, torch.float16, torch.bfloat16, torch.float64):
        db = nat.linear_q4_0_bias_grad(dy, bdt)
        assert db.dtype == bdt
        check(f"dbias {bdt}", db, ref.sum(0), bound, torch.float32 if bdt == torch.float64 else bdt)
    if m:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = nat.linear_q4_0_bias_grad(dy, dt)
        for i in range(3):
            dy.copy_(torch.randn(m, o, device=dev) + i)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, nat.linear_q4_0_bias_grad(dy, dt))


def test_refusals(spc, dev):
    nat = spc._native
    blocks = random_blocks(20, 64, 1).to(dev)
    fwd, bwd = _both(nat, blocks, dev)
    x = torch.zeros((2, 64), device=dev)
    for call in [lambda: nat.linear_q4_0(x, bwd), lambda: nat.linear_q4_0_input_grad(x[:, :20], fwd),
                 lambda: nat.linear_q4_0(x[:, :32], fwd), lambda: nat.linear_q4_0(x[0], fwd),
                 lambda: nat.linear_q4_0(x, fwd, x[0]),
                 lambda: nat.linear_q4_0(x, fwd, torch.zeros(20)),
                 lambda: nat.linear_q4_0_input_grad(x, bwd),
                 lambda: nat.pack_q4_0(blocks, out_features=20, in_features=48),
                 lambda: nat.pack_q4_0(blocks, out_features=21, in_features=64),
                 lambda: nat.pack_q4_0(blocks.int(), out_features=20, in_features=64),
                 lambda: spc.sparse.Q4Linear(48, 4).load_q4_0(blocks),
                 lambda: spc.sparse.Q4Linear(48, 4).to(dev).quantize_q4_0(),
                 lambda: spc.sparse.Q4Linear(64, 21).load_q4_0(blocks)]:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        nat.linear_q4_0(x.double(), fwd)
    lin = spc.sparse.Q4Linear(64, 20)
    lin.load_q4_0(blocks)
    with pytest.raises(RuntimeError, match="GPU only"):
        lin(torch.zeros((2, 64)))


def test_module(spc, dev):
    """Q4Linear: leading dimensions, gradients of rows and bias, weights swapped
    and dropped, the float parameter out of it."""
    lin = spc.sparse.Q4Linear(96, 50).to(dev)
    x = _randn((2, 3, 96), 1, torch.float32, dev)
    plain = torch.nn.functional.linear(x, lin.weight, lin.bias)
    assert torch.equal(lin(x), plain)
    blocks = lin.quantize_q4_0().cpu().view(50, 3, 18)
    x.requires_grad_()
    y = lin(x)
    assert y.shape == (2, 3, 50)
    x2 = x.detach().reshape(6, 96)
    check("y", y.reshape(6, 50), *product(x2, blocks, lin.bias), torch.float32)
    dy = _randn((2, 3, 50), 2, torch.float32, dev)
    y.backward(dy)
    check("dx", x.grad.reshape(6, 96), *gradient(dy.reshape(6, 50), blocks), torch.float32)
    db = dy.cpu().double().sum((0, 1))
    check("dbias", lin.bias.grad, db, 6 * 2.0 ** -24 * dy.cpu().double().abs().sum((0, 1)),
          torch.float32)
    assert lin.weight.grad is None
    with torch.no_grad():
        assert torch.equal(lin(x), y) and torch.equal(lin(x[0, 0]), y[0, 0])
    y = lin(x)
    lin.load_q4_0(blocks)
    with pytest.raises(RuntimeError, match="replaced"):
        y.sum().backward()
    lin.drop_q4_0()
    assert torch.equal(lin(x), plain)


def test_blocks_dropped_under_a_queued_product(spc, dev):
    """The laid out weights outlive products that other streams have queued."""
    lin = spc.sparse.Q4Linear(1024, 1024, bias=False).to(dev)
    blocks = lin.quantize_q4_0()
    x = _randn((3, 1024), 1, torch.bfloat16, dev)
    big = torch.randn(8192, 8192, device=dev)
    out = torch.empty_like(big)
    for drop in (lin.drop_q4_0, lambda: lin.load_q4_0(blocks)):
        lin.load_q4_0(blocks)
        with torch.no_grad():
            want = lin(x)
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        with torch.cuda.stream(s), torch.no_grad():
            for _ in range(4):
                torch.mm(big, big, out=out)
            y = lin(x)
        size = lin._q4_operand(x.device, False).data.numel()
        drop()
        junk = [torch.full((size,), 0x3c, dtype=torch.uint8, device=dev) for _ in range(4)]
        s.synchronize()
        assert torch.equal(y, want)
        del junk


def test_first_call_in_a_capture_is_refused(spc, dev):
    lin = spc.sparse.Q4Linear(64, 32).to(dev)
    lin.quantize_q4_0()
    x = torch.randn(2, 64, device=dev)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="before capturing"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            with torch.no_grad():
                lin(x)
    torch.cuda.synchronize()
    with torch.no_grad():
        want = lin(x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = lin(x)
    for _ in range(3):
        x.copy_(torch.randn(2, 64, device=dev))
        g.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            assert torch.equal(y, lin(x))
    assert want.shape == y.shape


def _coords(counts, dev):
    rows = []
    for i, k in enumerate(counts):
        r = torch.arange(k)
        rows.append(torch.stack([torch.full_like(r, i), r % 9, r // 9 % 9, r // 81], 1))
    return torch.cat(rows).to(torch.int32).to(dev)


def test_modulated_norm_trains_through_4_bit_weights(spc, dev):
    """The operators as a training step runs them: the embedding through a
    4-bit Linear to scale and shift, the modulated norm with SiLU, and the
    gradient of everything back to the embedding.  Each stage against 64 bits
    on what the stage before it gave."""
    sp = spc.sparse
    c, e, counts = 96, 64, [70, 2, 130]
    n = sum(counts)
    lin = sp.Q4Linear(e, 2 * c).to(dev)
    blocks = lin.quantize_q4_0().cpu().view(2 * c, e // 32, 18)
    ln = sp.SparseLayerNorm32(c).to(dev)
    x = _randn((n, c), 1, torch.float32, dev).requires_grad_()
    emb = _randn((3, e), 2, torch.float32, dev).requires_grad_()
    dy = _randn((n, c), 3, torch.float32, dev)
    t = sp.SparseTensor(x, _coords(counts, dev))
    act = torch.nn.functional.silu(emb)
    act.retain_grad()
    mod = lin(act)
    mod.retain_grad()
    scale, shift = mod.chunk(2, 1)
    ln(t, scale, shift, silu=True).feats.backward(dy)
    check("modulation", mod, *product(act, blocks, lin.bias), torch.float32)
    item = torch.repeat_interleave(torch.arange(3), torch.tensor(counts))
    ref = Reference(x, ln.weight, ln.bias, 1e-6, scale, shift, item, True)
    (dx, bx), (dw, bw), (db, bb), (ds, bs), (dh, bh) = ref.backward(dy, 60)
    check("dx", x.grad, dx, bx, torch.float32)
    check("dweight", ln.weight.grad, dw, bw, torch.float32)
    check("dbias", ln.bias.grad, db, bb, torch.float32)
    check("dmod", mod.grad, torch.cat([ds, dh], 1), torch.cat([bs, bh], 1), torch.float32)
    check("dact", act.grad, *gradient(mod.grad, blocks), torch.float32)
    z = emb.detach().cpu().double()
    sg = torch.sigmoid(z)
    want = act.grad.cpu().double() * (sg * (1 + z * (1 - sg)))
    check("demb", emb.grad, want, 2.0 ** -20 * want.abs() + 2.0 ** -22 * act.grad.cpu().double().abs(),
          torch.float32)


@pytest.mark.parametrize("cin,cout", [(64, 64), (64, 96)])
def test_res_block_on_4_bit_modulation(spc, dev, cin, cout):
    """SparseResBlock3d with its modulation Linear on Q4_0 blocks against the
    same block holding their values: the Linears' outputs are one bf16 rounding
    apart (a step of a modulation where a sum ends near a border), so the
    blocks agree to the parity bar of the block's own tests."""
    sp = spc.sparse
    coords = torch.from_numpy(spc.workloads.random_voxels(3000, 20, batches=2, seed=5)).to(dev)
    torch.manual_seed(1)
    blk = spc.blocks.SparseResBlock3d(cin, 128, cout).to(dev)
    with torch.no_grad():
        for p in blk.conv2.parameters():
            p.normal_(0, 0.02)
    lin = blk.emb_layers[1]
    assert set(blk.state_dict()) >= {"emb_layers.1.weight", "emb_layers.1.bias"}
    blocks = lin.quantize_q4_0().cpu().view(2 * cout, 4, 18)
    blk = blk.to(torch.bfloat16)
    blk.norm1.float()
    x = _randn((coords.shape[0], cin), 1, torch.bfloat16, dev)
    emb = _randn((2, 128), 2, torch.bfloat16, dev)
    with torch.no_grad():
        y4 = blk(sp.SparseTensor(x, coords), emb).feats
        lin.drop_q4_0()
        lin.weight.data = dequant(blocks).float().to(dev)
        lin.bias.data = lin.bias.data.float()
        y = blk(sp.SparseTensor(x, coords), emb.float()).feats
    err = float((y4.float() - y.float()).abs().max() / y.float().abs().max())
    print(f"[parity] 4-bit modulation {cin}->{cout}: max_rel={err:.3e}", flush=True)
    assert err <= 2e-2


def test_sparse_linear_and_gguf(spc, dev, tmp_path):
    from gguf_writer import f32_bytes, write_gguf

    gg = importlib.import_module(spc.__name__ + ".gguf")
    sp = spc.sparse
    blocks = random_blocks(40, 64, 3)
    bias = np.linspace(-1, 1, 40).astype(np.float32)
    p = str(tmp_path / "m.gguf")
    write_gguf(p, [], [("blk.emb_layers.1.weight", "Q4_0", (64, 40), blocks.numpy().tobytes()),
                       ("blk.emb_layers.1.bias", "F32", (40,), f32_bytes(bias))])
    lin = sp.SparseLinear(64, 40)
    with gg.GGUFReader(p) as r:
        gg.load_linear(lin, r, "blk.emb_layers.1")
    lin = lin.to(dev)
    coords = _coords([30], dev)
    x = _randn((30, 64), 1, torch.bfloat16, dev)
    t = sp.SparseTensor(x, coords)
    with torch.no_grad():
        y = lin(t)
    assert y.coords is t.coords
    check("y", y.feats, *product(x, blocks, torch.from_numpy(bias)), torch.bfloat16)
