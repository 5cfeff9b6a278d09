"""Q4_0 Linears: host checks, module bookkeeping and the GGUF loader (no GPU)."""
import importlib

import numpy as np
import pytest
import torch

from gguf_writer import bf16_bytes, f32_bytes, write_gguf
from q4_reference import dequant, gradient, parts, product, random_blocks


def test_reference_products():
    b = random_blocks(5, 64, 0)
    d, q = parts(b)
    assert q.min() >= -8 and q.max() <= 7
    raw = b.numpy()
    assert float(q[2, 33]) == float(raw[2, 1, 2 + 1] & 15) - 8       # byte 1, low half
    assert float(q[2, 32 + 17]) == float(raw[2, 1, 2 + 1] >> 4) - 8  # byte 1, high half
    w = dequant(b)
    assert torch.equal(w[2, 32:64], q[2, 32:64] * d[2, 1])
    x, dy = torch.randn(3, 64), torch.randn(3, 5)
    torch.testing.assert_close(product(x, b)[0], x.double() @ w.t())
    torch.testing.assert_close(gradient(dy, b)[0], dy.double() @ w)


def test_host_validation(spc):
    nat = spc._native
    L = nat.lib()
    fake = 1 << 12
    assert L.spc_linear_q4_0_packed_bytes(16, 128, 0) == 16 * 128 * 18 // 32
    assert L.spc_linear_q4_0_packed_bytes(17, 32, 0) == 2 * 16 * 128 * 18 // 32   # padded tiles
    assert L.spc_linear_q4_0_packed_bytes(128, 32, 1) == 128 * 32 * 18 // 32
    for out, inp in ((0, 32), (1, 0), (1, 33), (-1, 32), (1 << 31, 32), (1, 1 << 31)):
        assert L.spc_linear_q4_0_packed_bytes(out, inp, 0) == 0
        assert L.spc_linear_q4_0_pack(None, fake, out, inp, 0, fake) == nat.BAD_SHAPE
    assert L.spc_linear_q4_0_pack(None, None, 16, 32, 0, fake) == nat.BAD_ARG
    assert L.spc_linear_q4_0_pack(None, fake, 16, 32, 0, fake + 8) == nat.BAD_ARG
    assert L.spc_q4_0_quantize(None, fake, 33, fake) == nat.BAD_ARG
    assert L.spc_q4_0_quantize(None, fake + 4, 32, fake) == nat.BAD_ARG
    assert L.spc_q4_0_quantize(None, None, 0, None) == nat.OK

    def run(fn, dtype=nat.BF16, x=fake, stride=64, m=1, w=fake, y=fake):
        if fn == "y":
            return L.spc_linear_q4_0(None, dtype, x, stride, m, w, 64, 64, None, 0, y)
        return L.spc_linear_q4_0_input_grad(None, dtype, x, stride, m, w, 64, 64, y)

    for fn in ("y", "dx"):
        assert run(fn, m=0, x=None, w=None, y=None) == nat.OK
        assert run(fn, m=-1) == nat.BAD_SHAPE and run(fn, m=65535 * 16 + 1) == nat.BAD_SHAPE
        assert run(fn, stride=-1) == nat.BAD_SHAPE
        assert run(fn, dtype=nat.Q8_0) == nat.BAD_ARG
        assert run(fn, x=None) == nat.BAD_ARG and run(fn, w=None) == nat.BAD_ARG
        assert run(fn, x=fake + 1) == nat.BAD_ARG and run(fn, w=fake + 8) == nat.BAD_ARG
        assert run(fn, y=fake + 2, dtype=nat.F32) == nat.BAD_ARG
        assert b"misaligned" in L.spc_last_error()
    assert L.spc_linear_q4_0(None, nat.BF16, fake, 64, 1, fake, 64, 64, fake, 9, fake) == nat.BAD_ARG
    assert L.spc_linear_q4_0(None, nat.BF16, fake, 64, 1, fake, 64, 64, fake + 2, 0, fake) == nat.BAD_ARG


def test_cpu_tensors_are_rejected(spc):
    nat = spc._native
    b = random_blocks(20, 64, 1)
    with pytest.raises(RuntimeError, match="GPU only"):
        nat.pack_q4_0(b, out_features=20, in_features=64)
    with pytest.raises(RuntimeError, match="GPU only"):
        nat.q4_0_quantize(torch.zeros(32))


def test_module_is_nn_linear_until_blocks_are_loaded(spc):
    torch.manual_seed(4)
    plain = torch.nn.Linear(64, 20)
    torch.manual_seed(4)
    lin = spc.sparse.Q4Linear(64, 20)
    assert isinstance(lin, torch.nn.Linear) and list(lin.state_dict()) == list(plain.state_dict())
    x = torch.randn(3, 64)
    assert torch.equal(lin(x), plain(x))
    lin.load_q4_0(random_blocks(20, 64, 1))
    assert list(lin.state_dict()) == list(plain.state_dict())
    with pytest.raises(RuntimeError, match="GPU only"):
        lin(x)
    lin.drop_q4_0()
    assert torch.equal(lin(x), plain(x))
    for bad in (torch.zeros(720 - 18, dtype=torch.uint8), torch.zeros(720, dtype=torch.int8)):
        with pytest.raises(ValueError):
            lin.load_q4_0(bad)


def test_gguf_linear(spc, orc, tmp_path):
    gg = importlib.import_module(spc.__name__ + ".gguf")
    rng = np.random.default_rng(0)
    w = rng.standard_normal((40, 64)).astype(np.float32)
    bias = rng.standard_normal(40).astype(np.float32)
    blocks = random_blocks(40, 64, 3)
    q8 = orc.q8_0_quantize(w)
    p = str(tmp_path / "m.gguf")
    write_gguf(p, [], [
        ("f.weight", "F32", (64, 40), f32_bytes(w)), ("f.bias", "F32", (40,), f32_bytes(bias)),
        ("h.weight", "BF16", (64, 40), bf16_bytes(w)),
        ("q4.weight", "Q4_0", (64, 40), blocks.numpy().tobytes()),
        ("q4.bias", "BF16", (40,), bf16_bytes(bias)),
        ("q8.weight", "Q8_0", (64, 40), q8.tobytes()),
        ("t.weight", "F32", (40, 64), f32_bytes(w)),
        ("b.weight", "F32", (64, 40), f32_bytes(w)), ("b.bias", "F32", (39,), f32_bytes(bias[:39])),
    ])
    lin = spc.sparse.Q4Linear(64, 40)
    with gg.GGUFReader(p) as r:
        gg.load_linear(lin, r, "q4")
        assert torch.equal(lin._q4.view(40, 2, 18), blocks)
        assert torch.equal(lin.bias.detach(), torch.from_numpy(bias).bfloat16().float())
        gg.load_linear(lin, r, "f")
        assert lin._q4 is None
        assert np.array_equal(lin.weight.detach().numpy(), w)
        assert np.array_equal(lin.bias.detach().numpy(), bias)
        plain = torch.nn.Linear(64, 40)
        gg.load_linear(plain, r, "h")
        assert torch.equal(plain.weight.detach(), torch.from_numpy(w).bfloat16().float())
        gg.load_linear(plain, r, "q8")
        assert float((plain.weight.detach() - torch.from_numpy(w)).abs().max()) < 0.02
        with pytest.raises(gg.GGUFError, match="Q4Linear"):
            gg.load_linear(plain, r, "q4")
        for name in ("t", "b"):
            before = lin.weight.detach().clone()
            with pytest.raises(gg.GGUFError):
                gg.load_linear(lin, r, name)
            assert torch.equal(lin.weight.detach(), before)
        with pytest.raises(gg.GGUFError):
            gg.load_linear(torch.nn.Linear(64, 40, bias=False), r, "f")
        with pytest.raises(KeyError):
            gg.load_linear(lin, r, "none")


def test_features_past_a_launch_are_refused(spc):
    """512 threads for every 16 or 32 columns have to stay below 2^32 threads."""
    L = spc._native.lib()
    top = 1 << 27
    for out, inp, t in ((top, 32, 0), (32, top, 1)):
        assert L.spc_linear_q4_0_packed_bytes(out, inp, t) > 0
    fake = 1 << 12
    for out, inp in ((top + 1, 32), (32, top + 32)):
        assert L.spc_linear_q4_0_packed_bytes(out, inp, 0) == 0
        assert L.spc_linear_q4_0_pack(None, fake, out, inp, 0, fake) == spc._native.BAD_SHAPE
        assert L.spc_linear_q4_0(None, 0, fake, inp, 1, fake, out, inp, None, 0,
                                 fake) == spc._native.BAD_SHAPE


def test_bias_gradient_validation(spc):
    nat = spc._native
    L = nat.lib()
    fake = 1 << 12
    need = L.spc_linear_q4_0_bias_grad_workspace_bytes
    assert need(0, 8) == need(512, 8) == need(-1, 8) == 0
    assert need(513, 8) == 2 * 8 * 4 and need(65535 * 16, 8) == 512 * 8 * 4

    def run(dt=nat.BF16, dy=fake, stride=8, m=4, o=8, bdt=nat.F32, out=fake, ws=None, nbytes=0):
        return L.spc_linear_q4_0_bias_grad(None, dt, dy, stride, m, o, bdt, out, ws, nbytes)

    assert run(m=-1) == run(m=65535 * 16 + 1) == run(o=0) == run(stride=-1) == nat.BAD_SHAPE
    assert run(dt=nat.Q8_0) == run(bdt=nat.Q8_0) == run(dy=None) == run(out=None) == nat.BAD_ARG
    assert run(dy=fake + 1) == run(out=fake + 2) == run(m=513) == nat.BAD_ARG
    assert run(m=513, ws=fake, nbytes=63) == run(m=513, ws=fake + 1, nbytes=64) == nat.BAD_ARG


def test_captures_take_fresh_accumulators_only(spc, monkeypatch):
    """What a capture makes of leaves that an eager graph of any operator still
    holds, and of those it has met itself."""
    held, sp = spc.sparse._eager_leaves, spc.sparse

    def capture(stream):
        monkeypatch.setattr(sp.torch.cuda, "is_current_stream_capturing", lambda: stream is not None)
        monkeypatch.setattr(sp.torch.cuda, "current_stream",
                            lambda *a: type("Stream", (), {"cuda_stream": stream}))

    a, b = torch.zeros(3, requires_grad=True), torch.zeros(3, requires_grad=True)
    y = a * 2                                 # an eager graph of another operator
    capture(7)
    with pytest.raises(RuntimeError, match="eager graph"):
        held(a, b)
    with pytest.raises(RuntimeError, match="eager graph"):
        held(a)                               # again: the first refusal left nothing behind
    del y
    keep = held(a, b), a * 2, b * 3
    assert held(a, a) and held(b)             # met before in this capture
    capture(8)                                # their graph is alive, on another stream
    with pytest.raises(RuntimeError, match="eager graph"):
        held(a)
    capture(7)
    assert held(a, None, torch.zeros(3), a * 2)
    del keep
    capture(None)
    keep = held(a), a * 2                     # an eager graph of ours
    capture(7)
    with pytest.raises(RuntimeError, match="eager graph"):
        held(b, a)
    del keep
    assert held(a)


def test_a_state_dict_does_not_load_behind_blocks(spc):
    """A weight that would not be read is refused; the module's own state, a
    state without the weight, and any after drop_q4_0 load as into nn.Linear."""
    net = torch.nn.Sequential(spc.sparse.Q4Linear(64, 20), torch.nn.SiLU(), spc.sparse.SparseLinear(64, 20))
    net[0].load_q4_0(random_blocks(20, 64, 1))
    own, other = net.state_dict(), torch.nn.Sequential(
        torch.nn.Linear(64, 20), torch.nn.SiLU(), torch.nn.Linear(64, 20)).state_dict()
    net.load_state_dict({k: v.clone() for k, v in own.items()})
    with pytest.raises(RuntimeError, match=r"0\.weight: Q4_0 blocks .* drop_q4_0"):
        net.load_state_dict(other)
    with pytest.raises(RuntimeError, match="drop_q4_0"):
        net.load_state_dict(other, strict=False)
    other["0.bias"] = other["0.bias"] + 1
    net.load_state_dict({k: v for k, v in other.items() if k != "0.weight"}, strict=False)
    assert torch.equal(net[0].bias, other["0.bias"]) and net[0]._q4 is not None
    assert torch.equal(net[2].weight, other["2.weight"])
    net[0].drop_q4_0()
    net.load_state_dict(other)
    assert torch.equal(net[0].weight, other["0.weight"])
