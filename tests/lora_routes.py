"""Which kernels a call of nat.lora or nat.lora_backward runs: the host's rules of
csrc/lora.hip and csrc/lora_kernel.h, so that a test can say that none is left out."""


def _up(a, b):
    return -(-a // b)


def rank_tiles(r):
    return 1 if r <= 16 else 2 if r <= 32 else 4 if r <= 64 else 8


def forward(dt, n, items, c, o, r, p):
    """{(rank tiles, row tiles, what, dropout)}"""
    c, o, rt = max(c, 8), max(o, 8), rank_tiles(r)
    mt = 2 if n // items >= 32 and n >= 384 * 32 else 1
    if rt == 4 and n // items >= 64 and n >= 384 * 64:
        mt = 4
    busy = max(1, _up(n, 16 * mt), min(items, n))
    if mt > 1 or busy >= 256 or c * (16 + r) * (4 if dt == "f32" else 2) <= 200_000:
        return {(rt, mt, "both", p > 0)}
    return {(rt, 1, "hidden", p > 0), (rt, 1, "y", False)}


def _waves(dt, r, width):
    """(a wave's rank tiles, waves along ranks, along columns)"""
    along = 1 if r <= 16 else 2 if r <= 32 else 4
    tiles, w = _up(width, 64 if dt == "f32" else 128), 4 // along
    if w == 4 and (tiles - 1) % 4 < 2:
        w = 2
    return 2 if r > 64 else 1, along, 1 if tiles == 1 else w


def backward(dt, n, items, k, c, o, r, p):
    c, o, rt = max(c, 8), max(o, 8), rank_tiles(r)
    if n <= min(32 * items, min(items, k) * (32 + items // 2), 180 + 2 * items):
        return {("gathered", 4 * rt, p > 0)}
    out, rows = _waves(dt, r, o), _waves(dt, r, c)
    used = {("over dy", *out), ("over x", *rows, p > 0)}
    cols = 64 if dt == "f32" else 128
    shares, along = _up(o, out[2] * cols), 4 // (rows[1] * rows[2])
    held = 1 if along > 2 or rt == 8 else 2 if along == 2 or rt > 1 else 4
    if shares > held:
        used.add("u added first")

    def chunks(width, w):
        blocks, tile = _up(width, w[2] * cols), 32 * (4 // (w[1] * w[2]))
        most = max(1, 512 // blocks)
        per = _up(_up(n, most - min(items, most // 2)), tile) * tile
        return n // per + items + 3

    used.add(("sums", 4 if max(chunks(o, out), chunks(c, rows)) <= 32 * k else 16))
    return used


TILES = [(1, 1, 4), (1, 1, 2), (1, 1, 1), (1, 2, 2), (1, 2, 1), (1, 4, 1), (2, 4, 1)]
ALL = ({(rt, mt, "both", d) for rt in (1, 2, 4, 8) for mt in (1, 2, 4) for d in (False, True) if mt < 4 or rt == 4}
       | {(rt, 1, "hidden", d) for rt in (1, 2, 4, 8) for d in (False, True)} | {(rt, 1, "y", False) for rt in (1, 2, 4, 8)}
       | {("gathered", 4 * rt, d) for rt in (1, 2, 4, 8) for d in (False, True)}
       | {("over dy", *t) for t in TILES} | {("over x", *t, d) for t in TILES for d in (False, True)}
       | {"u added first", ("sums", 4), ("sums", 16)})
