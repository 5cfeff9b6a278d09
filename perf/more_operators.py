"""Low-rank adapters with their gradients and counter-based dropout, as they are
timed.

kind          what it is
  lora        lora: base + scale_a (dropout(x) down_a^T) up_a^T, a the adapter of
              the row's batch item (a request), beside a shared projection's
              output; in training with dropout and the hidden rows kept
  lora_grad   lora_backward: the gradients of the rows (added to the projection's
              own), and of every adapter's down and up
  dropout     dropout: a mask computed from (seed, row, column), with or without
              the residual it is added to

Items are contiguous row ranges (a batch's layout); some name no adapter, and
rows may lie behind the last item.  Widths are those of the flow model's Linears
and of large ones, ranks what adapters have.  Features differ in scale by
channel, adapters are as after some training.
"""
from __future__ import annotations

import importlib.util
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False   # True: the package's operators; False: elementary torch operations

_NAME = "sam3d_amd"
_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_MAX_BYTES = 62_710 * 2048 * 2        # rows x (inputs + outputs) of the largest adapters' case
_MAX_PRODUCTS = 62_710 * 2048 * 16    # times the rank
_MAX_ELEMENTS = 62_710 * 1024         # of dropout


def _native():
    """sam-3d-objects-ggml_amd/_native (the folder's name is no identifier)."""
    if _NAME not in sys.modules:
        root = Path.cwd() / "sam-3d-objects-ggml_amd"
        spec = importlib.util.spec_from_file_location(_NAME, root / "__init__.py",
                                                      submodule_search_locations=[str(root)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[_NAME] = mod
        spec.loader.exec_module(mod)
    return sys.modules[_NAME]._native


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def _lora(kind, dtype, rows, inputs, outputs, rank, *, items=1, adapters=1, base=True, p=0.0,
          behind=0):
    """behind: rows behind the last item, which belong to none."""
    return {"kind": kind, "dtype": dtype, "rows": rows, "inputs": inputs, "outputs": outputs,
            "rank": rank, "items": items, "adapters": adapters, "base": base, "p": p,
            "behind": behind}


def _drop(dtype, rows, width, p, residual):
    return {"kind": "dropout", "dtype": dtype, "rows": rows, "width": width, "p": p,
            "residual": residual}


def listed():
    def named(name, case):
        return {"name": name, **case}

    return [
        # one object's modulation Linear while serving: launches and latency
        named("lora_token", _lora("lora", "bf16", 1, 1024, 2048, 16)),
        # 64 requests of one row each, sixteen adapters among them, some without
        named("lora_requests", _lora("lora", "bf16", 64, 1024, 4096, 16, items=64, adapters=16)),
        # few requests through a large Linear: the adapters' bytes
        named("lora_large", _lora("lora", "f16", 8, 8192, 16_384, 64, items=8, adapters=8)),
        # four objects' feature rows, each its own adapter
        named("lora_objects", _lora("lora", "bf16", 62_710, 1024, 1024, 16, items=4, adapters=4)),
        # the training pass of the output block's skip Linear, hidden rows kept
        named("lora_train", _lora("lora", "bf16", 11_774, 2048, 1024, 32, items=4, adapters=2, p=0.1)),
        # widths and a rank that no vector divides, reference precision, no base
        named("lora_odd", _lora("lora", "f32", 5003, 101, 77, 5, items=3, adapters=2, base=False,
                                behind=10)),
        # a batch's modulation rows in training
        named("grad_token", _lora("lora_grad", "f16", 7, 1024, 2048, 8, items=7, adapters=2, p=0.05)),
        # the largest: four objects' rows, added to the projection's own gradient
        named("grad_objects", _lora("lora_grad", "bf16", 62_710, 1024, 1024, 16, items=4, adapters=2,
                                    p=0.1)),
        # reference-precision training at the mesh decoder's width
        named("grad_f32", _lora("lora_grad", "f32", 21_766, 768, 768, 8, base=False)),
        # a small object's rows
        named("drop_small", _drop("f16", 333, 192, 0.1, False)),
        # four objects' rows onto their residual
        named("drop_large", _drop("bf16", 62_710, 1024, 0.1, True)),
        # a width that no vector divides
        named("drop_odd", _drop("f32", 21_766, 101, 0.5, False)),
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["lora", "lora", "lora_grad", "dropout"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "dropout":
        width = rng.choice([size(1, 4096), 8 * size(1, 512)])
        most = max(1, min(200_000, _MAX_ELEMENTS * 2 // _SIZE[dtype] // width))
        return _drop(dtype, size(1, most), width, round(rng.uniform(0.0, 0.6), 3), rng.random() < 0.5)
    few = rng.random() < 0.4
    inputs, outputs = (rng.choice([size(8, 8192 if few else 2048), 64 * size(1, 128 if few else 32)])
                       for _ in range(2))
    rank = rng.choice([4, 8, 16, 16, 32, 64, 128, size(1, 128)])
    most = min(_MAX_BYTES // (_SIZE[dtype] * (inputs + outputs)),
               _MAX_PRODUCTS // ((inputs + outputs) * rank), 62_710)
    rows = size(1, 128 if few else most)
    # requests of one row each, or a batch of objects
    items = rows if few and rng.random() < 0.6 else min(rows, rng.choice([1, 1, 2, 4, 7]))
    adapters = min(items, size(1, 32))
    behind = rng.choice([0, 0, rows // 8])
    items = min(items, rows - behind)
    p = 0.0 if kind == "lora" and rng.random() < 0.5 else round(rng.uniform(0.0, 0.5), 3)
    return _lora(kind, dtype, rows, inputs, outputs, rank, items=items,
                 adapters=min(adapters, items), base=rng.random() < 0.7, p=p, behind=behind)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _bounds(case):
    """Row offsets of the items: uneven, every item with at least one row."""
    n, k = case["rows"] - case["behind"], case["items"]
    return [0] + [i + (n - k) * (2 * i + (i % 2)) // (2 * k + 1) for i in range(1, k)] + [n]


def _chosen(case):
    """The items' adapters, -1 for none: out of order, every fifth without."""
    k = case["adapters"]
    return [-1 if i % 5 == 4 else (5 * i + 2) % k for i in range(case["items"])]


def prepare(case, seed):
    dev = torch.device("cuda")
    dt = _DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    def rows(n, c):
        x = normal(n, c)
        x *= 0.5 + normal(c).abs()
        return x.to(dt)

    s = {"case": case}
    words = torch.randint(-2 ** 62, 2 ** 62, (2,), generator=gen, device=dev)
    if case["kind"] == "dropout":
        n, c = case["rows"], case["width"]
        s["seed"] = words
        s["x"] = rows(n, c)
        s["residual"] = normal(n, c).to(dt) if case["residual"] else None
        return s
    n, i, o, r, k = (case[a] for a in ("rows", "inputs", "outputs", "rank", "adapters"))
    s["seed"] = words if case["p"] else None
    s["bounds"], s["chosen"] = _bounds(case), _chosen(case)     # as the host knows them
    s["offsets"] = torch.tensor(s["bounds"], dtype=torch.int64, device=dev)
    s["adapters"] = torch.tensor(s["chosen"], dtype=torch.int32, device=dev)
    s["x"] = rows(n, i)
    s["down"] = (normal(k, r, i) * i ** -0.5).to(dt)
    s["up"] = (normal(k, o, r) * 0.1 * r ** -0.5).to(dt)
    s["scale"] = 1.0 + 0.5 * torch.rand(k, generator=gen, device=dev)
    s["base"] = None
    if case["kind"] == "lora":
        if case["base"]:
            s["base"] = normal(n, o).to(dt)     # the projection's output
        return s
    s["dy"] = normal(n, o).to(dt)
    if case["base"]:
        s["base"] = normal(n, i).to(dt)         # the projection's gradient of the rows
    # what the forward pass kept
    s["hidden"] = torch.zeros((n, r), device=dev)
    for lo, hi, a in _segments(s):
        for j in range(lo, hi, 8192):
            e = min(hi, j + 8192)
            s["hidden"][j:e] = _dropped(s, s["x"][j:e].float(), j) @ s["down"][a].float().t()
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
_M0, _M1, _W0, _W1 = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85
_LOW = 0xFFFFFFFF


def _keeps(seed, rows, c, threshold, first=0):
    """The mask of `rows` rows from row `first` on: seven rounds of the Philox
    generator of four 32-bit words (Salmon et al., 2011) on the counter
    (number of the eight columns' group, seed[1]), keyed by seed[0]; 16 bits an
    element, kept from the threshold on."""
    groups = (c + 7) // 8
    k = torch.arange(first * groups, (first + rows) * groups, device=seed.device)
    key, stream = seed[0], seed[1]
    a, b = k & _LOW, k >> 32
    x, y = (stream & _LOW).expand_as(k), ((stream >> 32) & _LOW).expand_as(k)
    k0, k1 = key & _LOW, (key >> 32) & _LOW
    for _ in range(7):
        u, v = a * _M0, x * _M1     # (their low 64 bits, whatever the sign)
        a, b, x, y = (((v >> 32) & _LOW) ^ b ^ k0, v & _LOW, ((u >> 32) & _LOW) ^ y ^ k1, u & _LOW)
        k0, k1 = (k0 + _W0) & _LOW, (k1 + _W1) & _LOW
    w = torch.stack([a, b, x, y], 1)
    w = torch.stack([w & 0xFFFF, w >> 16], 2)
    return w.view(rows, 8 * groups)[:, :c] >= threshold


def _threshold(p):
    return math.floor(p * 65536 + 0.5)


def _dropped(s, x, first):
    """dropout of float32 rows that begin at row `first`."""
    t = _threshold(s["case"]["p"])
    if t == 0:
        return x
    keep = _keeps(s["seed"], x.shape[0], x.shape[1], t, first)
    return torch.where(keep, x * (65536 / (65536 - t)), torch.zeros((), device=x.device))


def _segments(s):
    """(first row, end, adapter) of the items that name one."""
    return [(lo, hi, a) for lo, hi, a in zip(s["bounds"], s["bounds"][1:], s["chosen"]) if a >= 0]


def _plain_lora(s):
    c, x = s["case"], s["x"]
    y = x.new_zeros((c["rows"], c["outputs"])) if s["base"] is None else s["base"].clone()
    hidden = torch.zeros((c["rows"], c["rank"]), device=x.device) if c["p"] else None
    for lo, hi, a in _segments(s):
        h = _dropped(s, x[lo:hi].float(), lo) @ s["down"][a].float().t()
        z = (h @ s["up"][a].float().t()) * s["scale"][a]
        if s["base"] is not None:
            z = z + s["base"][lo:hi].float()
        y[lo:hi] = z.to(x.dtype)
        if hidden is not None:
            hidden[lo:hi] = h
    return y if hidden is None else (y, hidden)


def _plain_lora_grad(s):
    x, dy = s["x"], s["dy"]
    dx = torch.zeros_like(x) if s["base"] is None else s["base"].clone()
    ddown = torch.zeros(s["down"].shape, device=x.device)
    dup = torch.zeros(s["up"].shape, device=x.device)
    for lo, hi, a in _segments(s):
        g = dy[lo:hi].float() * s["scale"][a]
        u = g @ s["up"][a].float()
        z = _dropped(s, u @ s["down"][a].float(), lo)
        if s["base"] is not None:
            z = z + s["base"][lo:hi].float()
        dx[lo:hi] = z.to(x.dtype)
        ddown[a] += u.t() @ _dropped(s, x[lo:hi].float(), lo)
        dup[a] += g.t() @ s["hidden"][lo:hi]
    return dx, ddown.to(x.dtype), dup.to(x.dtype)


def _plain_dropout(s):
    y = _dropped(s, s["x"].float(), 0)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def run(state):
    s, kind, p = state, state["case"]["kind"], state["case"]["p"]
    if own:
        nat = _native()
        if kind == "dropout":
            return nat.dropout(s["x"], p, s["seed"], residual=s["residual"])
        if kind == "lora":
            return nat.lora(s["x"], s["down"], s["up"], s["base"], scale=s["scale"],
                            offsets=s["offsets"], adapters=s["adapters"], p=p, seed=s["seed"],
                            return_hidden=p > 0)
        return nat.lora_backward(s["dy"], s["x"], s["hidden"], s["down"], s["up"], s["base"],
                                 scale=s["scale"], offsets=s["offsets"], adapters=s["adapters"],
                                 p=p, seed=s["seed"])
    if kind == "dropout":
        return _plain_dropout(s)
    return _plain_lora(s) if kind == "lora" else _plain_lora_grad(s)


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its values in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    e = _SIZE[case["dtype"]]
    if case["kind"] == "dropout":
        m = case["rows"] * case["width"]
        return {"bytes": m * e * (3 if case["residual"] else 2), "flops": 2 * m}
    n, i, o, r = (case[k] for k in ("rows", "inputs", "outputs", "rank"))
    ids, off = _chosen(case), _bounds(case)
    on = sum(hi - lo for lo, hi, a in zip(off, off[1:], ids) if a >= 0)     # rows that meet an adapter
    used = len({a for a in ids if a >= 0}) * r * (i + o) * e
    if case["kind"] == "lora":
        return {"bytes": on * i * e + n * o * e * (2 if case["base"] else 1) + used
                + (4 * n * r if case["p"] else 0),
                "flops": 2 * on * r * (i + o)}
    return {"bytes": on * (i + o) * e + 4 * on * r + n * i * e * (2 if case["base"] else 1) + used
            + case["adapters"] * r * (i + o) * e,
            "flops": 4 * on * r * (i + o)}


def _mask64(seed, rows, c, p):
    """The factor of every element: 0 or 1 / (1 - p), p in 65536ths."""
    t = int(p * 65536 + 0.5)
    if t == 0:
        return None
    seed = seed.cpu().numpy().view(np.uint64)
    k = np.arange(rows * (-(-c // 8)), dtype=np.uint64)
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    ctr = [k & low, k >> half, np.full_like(k, seed[1] & low), np.full_like(k, seed[1] >> half)]
    key = [int(seed[0]) & 0xFFFFFFFF, int(seed[0]) >> 32]
    for i in range(7):
        k0, k1 = (np.uint64((w + i * b) % 2 ** 32) for w, b in zip(key, (0x9E3779B9, 0xBB67AE85)))
        p0, p1 = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(p1 >> half) ^ ctr[1] ^ k0, p1 & low, (p0 >> half) ^ ctr[3] ^ k1, p0 & low]
    words = np.stack(ctr, 1).astype(np.uint32).view(np.uint16).reshape(rows, -1)[:, :c]
    return torch.from_numpy((words >= t).astype(np.float64) * (1 / (1 - t / 65536)))


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if s["seed"] is not None:
        factor = _mask64(s["seed"], x.shape[0], x.shape[1], case["p"])
        factor = None if factor is None else factor.to(x.device)
    else:
        factor = None
    if factor is not None:
        x = x * factor
    if case["kind"] == "dropout":
        return x if s["residual"] is None else x + s["residual"].double()
    # the adapter of every row, and all rows of an adapter at once
    item = torch.bucketize(torch.arange(case["rows"], device=x.device), s["offsets"], right=True) - 1
    of = torch.cat([s["adapters"].long(), item.new_tensor([-1])])[item]
    down, up, scale = s["down"].double(), s["up"].double(), s["scale"].double()
    width = case["outputs"] if case["kind"] == "lora" else case["inputs"]
    out = x.new_zeros((case["rows"], width)) if s["base"] is None else s["base"].double()
    first, second = [], []
    hidden = x.new_zeros((case["rows"], case["rank"]))
    for a in range(case["adapters"]):
        rows = (of == a).nonzero().squeeze(1)
        if case["kind"] == "lora":
            h = x[rows] @ down[a].t().contiguous()
            hidden[rows] = h
            out[rows] += scale[a] * (h @ up[a].t().contiguous())
            continue
        g = s["dy"][rows].double()
        u = scale[a] * (g @ up[a])
        z = u @ down[a]
        out[rows] += z if factor is None else z * factor[rows]
        first.append(u.t().contiguous() @ x[rows])
        second.append(scale[a] * (g.t().contiguous() @ s["hidden"][rows].double()))
    if case["kind"] == "lora":
        return (out, hidden) if case["p"] else out
    return out, torch.stack(first), torch.stack(second)
