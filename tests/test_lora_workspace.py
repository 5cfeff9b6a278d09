"""What the adapters' gradients ask for as workspace, without a GPU."""
import pytest

# (rows, items, adapters, in, out, rank)
MANY = [(65_535, 65_535, 1, 1024, 1024, 16), (4096, 4096, 1, 4096, 4096, 64), (62_710, 1024, 8, 1024, 1024, 128),
        (140_000, 65_535, 8, 4096, 4096, 128), (1 << 20, 65_535, 64, 64, 16_384, 8)]


@pytest.mark.parametrize("n,items,k,c,o,r", MANY)
def test_backward_workspace_does_not_grow_with_the_items(spc, n, items, k, c, o, r):
    """u in shares of at least 128 outputs (64 of F32 rows), slots of 2^29 bytes for
    each weight (one slot, if that is more), and F32 sums of both (slots are of whole
    tiles and rounded up to 256 bytes): not a slot an item, 275 GB of the fourth."""
    L, nat = spc._native.lib(), spc._native
    for dt, size, cols in ((nat.BF16, 2, 128), (nat.F16, 2, 128), (nat.F32, 4, 64)):
        u = 4 * n * r * -(-o // cols)
        sums = 4 * k * r * (c + o)
        need = L.spc_lora_workspace_bytes(dt, n, items, k, c, o, r, 1)
        assert 0 < need <= u + 2 * (1 << 29) + sums + 4096


@pytest.mark.parametrize("n,items,k", [(1920, 64, 64), (1024, 64, 64), (8192, 1024, 1024), (1024, 256, 32)])
def test_route_does_not_trust_the_bank(spc, n, items, k):
    """Rows that may all be one adapter's (some 14 us for each 32 of them, one after the
    other, where they are gathered) take the tiles, whose workspace has the sums'
    slots, whatever the number of adapters in the bank."""
    L, nat = spc._native.lib(), spc._native
    need = [L.spc_lora_workspace_bytes(nat.BF16, n, items, a, 1024, 1024, 16, 1) for a in (1, k)]
    assert need[0] == need[1] > 4 * 2 * items * 1024 * 16
