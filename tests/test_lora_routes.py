"""Every kernel of the adapters is launched by a test, in every dtype."""
import re
from pathlib import Path

import pytest

import lora_routes
from test_gpu_lora_kernels import CASES

CSRC = Path(__file__).resolve().parent.parent / "sam-3d-objects-ggml_amd" / "csrc"


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_cases_name_every_kernel(dt):
    seen = set()
    for n, items, k, c, o, r in CASES:
        for p in (0.0, 0.2):
            seen |= lora_routes.forward(dt, n, items, c, o, r, p) | lora_routes.backward(dt, n, items, k, c, o, r, p)
    assert seen == lora_routes.ALL


def test_all_is_what_the_sources_instantiate():
    t = (CSRC / "lora_kernel.h").read_text()
    tiles = {tuple(map(int, m)) for m in re.findall(r"lora_back_out_kernel<DT, (\d), (\d), (\d)><<<", t)}
    assert tiles == set(lora_routes.TILES)
    assert {tuple(map(int, m)) for m in re.findall(r"lora_back_in_kernel<DT, (\d), (\d), (\d), DROP><<<", t)} == tiles
    assert {m for m in re.findall(r"lora_forward_mode<DT, (\d), ([\dM* ]+)>\(", t)} == {
        *[(str(rt), mt) for rt in (1, 2, 4, 8) for mt in ("1", "M")], ("4", "2 * M")}


@pytest.mark.parametrize("dt,name", [("bf16", "BF16"), ("f32", "F32")])
def test_routes_agree_with_the_workspaces(spc, dt, name):
    """The mirror's two forms of each pass are the library's: hidden sums, or shares of u alone,
    are workspace."""
    L, nat = spc._native.lib(), spc._native
    for n, items, k, c, o, r in CASES:
        if min(c, o) < 8:
            continue
        ws = [L.spc_lora_workspace_bytes(getattr(nat, name), n, items, k, c, o, r, b) for b in (0, 1)]
        assert (ws[0] > 0) == any(f[2] == "hidden" for f in lora_routes.forward(dt, n, items, c, o, r, 0.0))
        gathered = any(f[0] == "gathered" for f in lora_routes.backward(dt, n, items, k, c, o, r, 0.0))
        shares = [-(-i * n * r // 64) * 256 for i in range(1, 9)]   # (F32, rounded up to 256 bytes)
        assert (ws[1] in shares) == gathered
