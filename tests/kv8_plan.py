"""How an attention call over 8-bit pages is split, restated from the rules beside kv8_attn_plan: for
tests to say which paths a size takes."""

NWAVES, CHIP, RING_MOST = 8, 256, 128


def up(a, b):
    return (a + b - 1) // b


def plan(n_heads, n_kv, M, n, n_sel, ring_rows, mass):
    """dict of the split; batch: pages a block takes before it asks for their numbers again."""
    n_list, units, nv = n_sel or n, up(ring_rows, 64), M * (n_heads // n_kv)
    tiles, rows = up(nv // M if n_sel else nv, 16), M if n_sel else 1
    visits = n_list * n_kv
    most = 300 if tiles == 1 else 2500 if tiles == 2 else 3500 if tiles <= 4 else 1 << 62
    shared = visits * rows * up(tiles, NWAVES) <= most
    pair = 2 if not shared and tiles > 2 else 1
    wave = (2 if tiles > NWAVES and visits > 1400 else 1) if shared else min(tiles, 2)
    cols = rows * up(tiles, wave * (NWAVES if shared else pair))
    share = CHIP // (cols * n_kv)
    upr = up(units, max(share, RING_MOST))
    ring_parts = up(units, upr)
    parts = min(max(1, share // 2, share - ring_parts), n_list if shared else up(n_list, NWAVES // pair))
    upp = up(n_list, parts) if parts else 0
    total = ring_parts + (up(n_list, upp) if parts else 0)
    off = 0
    for size in (n_kv * nv * total * 512, n_kv * nv * total * 8, (n_kv * nv * n + 16) * 8 if mass else 0):
        if size:
            off = up(off, 256) * 256 + size
    return dict(shared=shared, pair=pair, tiles=wave, cols=cols, upr=upr, ring_parts=ring_parts, upp=upp,
                parts=total, batch=64 if shared else 64 * NWAVES // pair, bytes=off)
