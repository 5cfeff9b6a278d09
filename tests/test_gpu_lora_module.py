"""Adapters of Q4Linear / SparseLinear and SparseDropout as modules: against the
64-bit forms, together as a training step and as serving use them, what may be
captured, what is refused."""
import pytest
import torch

from lora_reference import Adapters, dropout, factors
from norm_reference import U, check, half_step
from q4_reference import dequant, product

pytestmark = pytest.mark.gpu


def _tensor(spc, dev, feats, sizes=None):
    n = feats.shape[0]
    sizes = [n] if sizes is None else sizes
    item = torch.repeat_interleave(torch.arange(len(sizes)), torch.tensor(sizes))
    at = torch.cat([torch.arange(k) for k in sizes])
    coords = torch.stack([item, at % 9, at // 9, 0 * at], 1)
    return spc.sparse.SparseTensor(feats, coords.to(torch.int32).to(dev))


def _linear(spc, dev, cls, i, o, count, rank, dtype=torch.float32, q4=False, **kw):
    torch.manual_seed(i + o + rank)
    lin = getattr(spc.sparse, cls)(i, o).to(dev, dtype)
    blocks = lin.quantize_q4_0().cpu().reshape(o, i // 32, 18) if q4 else None
    lin.add_adapters(count, rank, **kw)
    with torch.no_grad():
        lin.adapter_up.normal_(std=0.1)
    return lin, blocks


def _ids(dev, *v):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _base(x, lin, blocks):
    """The projection alone in 64 bits and its bound before rounding."""
    if blocks is not None:
        return product(x, blocks, lin.bias)
    x, w, b = x.detach().cpu().double(), lin.weight.detach().cpu().double(), lin.bias.detach().cpu().double()
    y = x @ w.t() + b
    # a library product: F32 sums of exact products, a rounding a term at most
    return y, 2 * (w.shape[1] + 4) * U * (x.abs() @ w.abs().t() + b.abs())


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_linear_of_single_rows(spc, dev, dt, q4):
    """A batch's modulation Linear, an adapter a row: the projection rounded to the
    rows' type, then the adapters on top."""
    lin, blocks = _linear(spc, dev, "Q4Linear", 64, 96, 3, 8, dt, q4, alpha=16)
    x = torch.randn(6, 64, generator=torch.Generator().manual_seed(1)).to(dt).to(dev)
    ids = _ids(dev, 2, -1, 0, 1, 2, 7)
    with torch.no_grad():
        y = lin(x, ids)
        plain = lin(x)
    base, e = _base(x, lin, blocks)
    check("base", plain, base, e + half_step(base.abs() + e, dt))
    ref = Adapters(x, lin.adapter_down, lin.adapter_up, lin.adapter_scale, None, ids)
    # (the base as it was rounded)
    check("adapted", y, *ref.forward(plain)[0])
    assert torch.equal(y[[1, 5]], plain[[1, 5]])
    assert torch.equal(lin(x.view(6, 1, 64), ids).view(6, 96), y)
    assert torch.equal(lin.eval()(x[:2].repeat_interleave(5, 0).view(2, 5, 64), ids[:2])[:, 3], y[:2])


@pytest.mark.parametrize("q4", [False, True])
def test_gradients(spc, dev, q4):
    """Rows, bias and adapters of a SparseLinear over two items, as the 64-bit form
    has them, and against differences."""
    lin, blocks = _linear(spc, dev, "SparseLinear", 64, 96, 2, 8, q4=q4)
    x = torch.randn(70, 64, device=dev, requires_grad=True)
    t, ids = _tensor(spc, dev, x.detach(), [30, 40]), _ids(dev, 1, 0)
    dy = torch.randn(70, 96, device=dev)
    y = lin(t.replace(x), ids).feats
    grads = torch.autograd.grad(y, [x, lin.adapter_down, lin.adapter_up, lin.bias], dy)
    ref = Adapters(x, lin.adapter_down, lin.adapter_up, lin.adapter_scale, [0, 30, 70], ids)
    hidden = ref.forward()[1][0]
    w = dequant(blocks) if blocks is not None else lin.weight.detach().cpu().double()
    d = dy.cpu().double()
    # the projection's own gradient: F32 sums of products, three roundings a term at most
    e_base = (3 * 2 * (96 + 40)) * U * (d.abs() @ w.abs())
    (dx, e), (dd, ed), (du, eu) = ref.backward(dy, hidden, d @ w)
    check("dx", grads[0], dx, e + e_base)
    check("ddown", grads[1], dd, ed)
    # (hidden rows are F32 here, off by their own bound)
    e_h = ref.forward()[1][1]
    extra = torch.stack([(d[ref.of == a].abs().t() @ e_h[ref.of == a]) for a in range(2)])
    check("dup", grads[2], du, eu + extra)
    check("dbias", grads[3], d.sum(0), 80 * U * d.abs().sum(0))


def test_training_pass_with_dropout(spc, dev):
    """A frozen 4-bit Linear with adapters behind a norm, dropout in front of them
    and of the residual branch: gradients equal those of the same pass built of the
    functions, and an evaluation pass has no dropout."""
    sp, nat = spc.sparse, spc._native
    lin, _ = _linear(spc, dev, "SparseLinear", 64, 64, 2, 8, torch.bfloat16, True, dropout=0.2)
    lin.weight.requires_grad_(False), lin.bias.requires_grad_(False)
    ln, drop = sp.SparseLayerNorm32(64).to(dev), sp.SparseDropout(0.1)
    x = torch.randn(90, 64, device=dev).bfloat16().requires_grad_()
    t, ids = _tensor(spc, dev, x.detach(), [50, 40]), _ids(dev, 0, 1)
    torch.manual_seed(11)
    y = drop(lin(ln(t.replace(x)), ids), t.replace(x)).feats
    dy = torch.randn_like(y)
    leaves = [x, ln.weight, lin.adapter_down, lin.adapter_up]
    got = torch.autograd.grad(y, leaves, dy)
    torch.manual_seed(11)
    s1, s2 = sp.dropout_seed(dev), sp.dropout_seed(dev)
    off = torch.tensor([0, 50, 90], device=dev)
    kw = dict(scale=lin.adapter_scale, offsets=off, adapters=ids, p=0.2, seed=s1)
    h, stats = nat.layer_norm(x.detach(), ln.weight, ln.bias, ln.eps, return_stats=True)
    base = nat.linear_q4_0(h, lin._q4_operand(h.device, False), lin.bias)
    z, hid = nat.lora(h, lin.adapter_down.detach(), lin.adapter_up.detach(), base, return_hidden=True, **kw)
    assert torch.equal(y, nat.dropout(z, 0.1, s2, residual=x.detach()))
    dz = nat.dropout(dy, 0.1, s2)
    dh, dd, du = nat.lora_backward(dz, h, hid, lin.adapter_down.detach(), lin.adapter_up.detach(),
                                   nat.linear_q4_0_input_grad(dz, lin._q4_operand(h.device, True)), **kw)
    dx, dw, _, _, _ = nat.layer_norm_backward(dh, x.detach(), stats, ln.weight, ln.bias)
    assert torch.equal(got[2], dd) and torch.equal(got[3], du) and torch.equal(got[1], dw)
    assert torch.equal(got[0], dx + dy)
    lin.eval(), drop.eval()
    with torch.no_grad():
        out = drop(lin(ln(t), ids), t).feats
    assert torch.equal(out, nat.lora(h, lin.adapter_down, lin.adapter_up, base, **{**kw, "p": 0.0}) + x)


def test_dropout_module(spc, dev):
    sp = spc.sparse
    drop = sp.SparseDropout(0.3)
    x = torch.randn(40, 24, device=dev, requires_grad=True)
    r = torch.randn(40, 24, device=dev, requires_grad=True)
    t = _tensor(spc, dev, x.detach())
    seed = torch.tensor([5, 6], device=dev)
    y = drop(t.replace(x), t.replace(r), seed).feats
    check("y", y, *dropout(x, 0.3, [5, 6], r))
    dy = torch.randn(40, 24, device=dev, requires_grad=True)
    dx, dr = torch.autograd.grad(y, [x, r], dy, create_graph=True)
    check("dx", dx, *dropout(dy, 0.3, [5, 6]))
    assert torch.equal(dr, dy)
    # again differentiable, linear as it is
    ddy, = torch.autograd.grad(dx, dy, torch.ones_like(dx))
    assert torch.equal(ddy.double().cpu().round(decimals=5), factors([5, 6], 40, 24, 0.3).round(decimals=5))
    a, b = drop(t).feats, drop(t).feats
    assert not torch.equal(a, b)
    torch.manual_seed(3)
    a = drop(t).feats
    torch.manual_seed(3)
    assert torch.equal(a, drop(t).feats)
    heads = t.replace(x.detach().view(40, 4, 6))
    assert torch.equal(drop(heads, seed=seed).feats.view(40, 24), drop(t, seed=seed).feats)
    drop.eval()
    assert drop(t) is t and torch.equal(drop(t, t.replace(r)).feats, x + r)
    y = sp.SparseDropout(0.0)(t, t)
    assert torch.equal(y.feats, 2 * t.feats)
    with pytest.raises(ValueError, match="residual"):
        drop.train()(t, t.replace(r[:, :3]))


@pytest.mark.parametrize("q4", [False, True])
def test_captured_training_pass(spc, dev, q4):
    """Replays draw new masks, each the one of an eager pass with its seeds; refused
    while an eager graph of the leaves is alive."""
    sp = spc.sparse
    lin, _ = _linear(spc, dev, "SparseLinear", 64, 96, 2, 8, q4=q4, dropout=0.25)
    drop = sp.SparseDropout(0.5)
    x = torch.randn(50, 64, device=dev, requires_grad=True)
    t, ids = _tensor(spc, dev, x.detach(), [20, 30]), _ids(dev, 1, 0)
    dy = torch.randn(50, 96, device=dev)
    leaves = [x, lin.adapter_down, lin.adapter_up, lin.bias]
    seeds = torch.tensor([[1, 2], [3, 4]], device=dev)
    # the module's seed from a tensor, so that an eager pass can repeat it
    draw, sp.dropout_seed = sp.dropout_seed, lambda device: seeds[0]
    try:
        def run(xs):
            return drop(lin(t.replace(xs), ids), seed=seeds[1]).feats

        torch.autograd.grad(run(x), leaves, dy)
        torch.cuda.synchronize()
        keep = (lin.adapter_up * 2).sum()
        with pytest.raises(RuntimeError, match="eager graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                run(x)
        torch.cuda.synchronize()
        del keep
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                y = run(x)
                graphs.append((g, y, torch.autograd.grad(y, leaves, dy)))
        x2 = x.detach().clone().requires_grad_()
        for i in range(4):
            with torch.no_grad():
                x.copy_(torch.randn(50, 64, device=dev) + i)
                x2.copy_(x)
            dy.copy_(torch.randn(50, 96, device=dev))
            seeds.copy_(torch.randint(1 << 40, (2, 2)))
            for g, _, _ in graphs:
                g.replay()
            torch.cuda.synchronize()
            want = run(x2)
            grads = torch.autograd.grad(want, [x2, *leaves[1:]], dy)
            for _, y, got in graphs:
                assert torch.equal(y, want) and all(torch.equal(p, q) for p, q in zip(got, grads))
    finally:
        sp.dropout_seed = draw
    # and drawn by the generator: another mask in each replay
    del want, grads
    g = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(g):
        y = drop(t).feats
    seen = []
    for _ in range(3):
        g.replay()
        seen.append(y.clone())
        (t.feats + 1).sum().item()
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_block_with_adapters(spc, dev):
    """A residual block's modulation and skip Linears with an adapter for each object
    equal a block whose weights hold the products; without the argument, and for
    objects without one, nothing changes."""
    torch.manual_seed(5)
    block = spc.blocks.SparseResBlock3d(32, 64, 64).to(dev)
    for p in block.conv2.parameters():
        torch.nn.init.normal_(p, std=0.02)
    c = torch.stack(torch.meshgrid(*[torch.arange(5)] * 3, indexing="ij"), -1).reshape(-1, 3)
    coords = torch.cat([torch.cat([torch.full((125, 1), b), c], 1) for b in range(2)]).int().to(dev)
    x = spc.sparse.SparseTensor(torch.randn(250, 32, device=dev), coords)
    emb = torch.randn(2, 64, device=dev)
    with torch.no_grad():
        want = block(x, emb).feats
        block.emb_layers[1].add_adapters(2, 4)
        block.skip_connection.add_adapters(2, 4, alpha=8)
        assert torch.equal(block(x, emb, _ids(dev, 1, 0)).feats, want)   # (up is zero)
        for lin in (block.emb_layers[1], block.skip_connection):
            lin.adapter_up.normal_(std=0.1)
        assert torch.equal(block(x, emb).feats, want)
        y = block(x, emb, _ids(dev, 1, -1)).feats
        assert torch.equal(y[125:], want[125:]) and not torch.equal(y[:125], want[:125])
        merged = spc.blocks.SparseResBlock3d(32, 64, 64).to(dev)
        merged.load_state_dict({k: v for k, v in block.state_dict().items() if "adapter" not in k})
        for a, b in ((merged.emb_layers[1], block.emb_layers[1]), (merged.skip_connection, block.skip_connection)):
            a.weight += b.adapter_scale[1] * (b.adapter_up[1] @ b.adapter_down[1])
        m = merged(x, emb).feats[:125]
    # (both in F32: sums of 27 x 64 products twice, an ulp of 2^-24 a term at most, so 4e-4)
    assert float((y[:125] - m).norm() / m.norm()) < 4e-4


def test_state_and_refusals(spc, dev):
    lin, _ = _linear(spc, dev, "Q4Linear", 64, 96, 2, 8, q4=True)
    x, ids = torch.randn(3, 64, device=dev), _ids(dev, 0, 1, -1)
    state = lin.state_dict()
    assert sorted(state) == ["adapter_down", "adapter_scale", "adapter_up", "bias", "weight"]
    with torch.no_grad():
        y = lin(x, ids)
        other = spc.sparse.Q4Linear(64, 96).to(dev)
        with pytest.raises(RuntimeError, match="Unexpected"):
            other.load_state_dict(state)
        other.add_adapters(2, 8)
        other.load_state_dict(state)
        other.load_q4_0(lin._q4)
        assert torch.equal(other(x, ids), y)
        other.half()
        assert other(x.half(), ids).dtype == torch.float16
        empty = lin(x[:0], ids[:0])
        assert empty.shape == (0, 96)
        lin.drop_adapters()
        with pytest.raises(RuntimeError, match="add_adapters"):
            lin(x, ids)
    lin.add_adapters(2, 8)
    for bad in (ids[:2], ids[None], ids.long()):
        with pytest.raises(ValueError):
            lin(x, bad)
    with pytest.raises(ValueError):
        lin(x[:, :32], ids)
    fw = torch.autograd.forward_ad
    with fw.dual_level(), pytest.raises((RuntimeError, NotImplementedError), match="forward"):
        lin(fw.make_dual(x, torch.ones_like(x)), ids)
    with fw.dual_level(), pytest.raises((RuntimeError, NotImplementedError), match="forward"):
        t = _tensor(spc, dev, x)
        spc.sparse.SparseDropout(0.5)(t.replace(fw.make_dual(x, torch.ones_like(x))))


def test_autocast_and_other_streams(spc, dev):
    lin, _ = _linear(spc, dev, "Q4Linear", 64, 96, 2, 8)
    x, ids = torch.randn(5, 64, device=dev), _ids(dev, 0, 1, -1, 1, 0)
    with torch.autocast("cuda", torch.bfloat16):
        y = lin(x, ids)
    assert y.dtype == torch.bfloat16
    y.float().sum().backward()
    assert lin.adapter_up.grad.dtype == torch.float32 and float(lin.adapter_up.grad.abs().max()) > 0
    want = lin(x, ids)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = lin(x, ids)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
