"""How mi_hist_attn cuts a call over long histories, asked of the library, and histories whose attention counts positions."""
import ctypes

import numpy as np


def cut_of(dtype, lens, width, page, heads, group, tokens, dim):
    """The cut of a call whose page table has room for more than 1024 positions.  The number of workgroups follows from the
    workspace the library asks for; the rest restates the rules of the kernel: units of 128 positions, runs of equal length,
    and whole rows to a workgroup (units of several 128, runs of one) where runs are up to 8 units and the chip holds them."""
    from recommendation_amd import _lib
    c = _lib.HistCacheC(kv=4096, exps=4096 if dtype == _lib.MI_DT_E4M3 else None, n_pages=8, n_heads=heads, page_size=page,
                        dim=dim, dtype=dtype)
    rows = tokens * group
    RT = 2 if rows > 16 and dim <= 128 else 1
    tiles = -(-rows // (16 * RT))
    NR = 4 if tiles >= 3 else tiles
    NG = -(-tiles // NR)
    slot = min(rows, NR * 16 * RT)
    ws = _lib.load().mi_hist_attn_workspace_bytes(ctypes.byref(c), len(lens), tokens, heads * group, width)
    blocks = ws // (2 * slot * (dim * 4 + 8) + 16)
    assert blocks > 0 and ws == blocks * 2 * slot * dim * 4 + -(-blocks * 2 * slot * 8 // 16) * 16 + blocks * 16
    HG = heads * NG

    def units(unit):
        return sum(max(1, -(-max(0, n) // unit)) for n in lens) * HG

    run, unit = -(-units(128) // blocks), 128
    aligned = 1 < run <= 8 and 2 * HG * len(lens) <= blocks
    if aligned:
        unit *= run
        while units(unit) > blocks:
            unit += 128
    return dict(RT=RT, NR=NR, NG=NG, blocks=blocks, run=run, aligned=aligned, part=unit if aligned else run * 128)


def depth_of(cut, n):
    """Additions that follow each other in a sum over n positions: those of the longest part, then one a part."""
    return min(n, cut['part']) + -(-n // cut['part']) + 1


def lengths_for(rng, users, shortest, longest):
    """Uniform lengths, the longest, an empty and a negative one and a single event among them."""
    x = rng.integers(shortest, longest + 1, size=users)
    x[0] = longest
    if users > 4:
        x[users // 2], x[-1], x[users // 3] = 0, 1, -2
    return x.tolist()


def counting_rows(rng, n, heads, dim, most=24):
    """Value rows of +1 and -1 (channel 0: +1 alone) whose sums over positions 0 .. any end stay within +-most, and these sums
    [n + 1, heads, dim].  With equal keys attention gives sums / length: whole numbers over a known one, so that a position
    lost, added or taken twice shows in every cache type, however long the history."""
    rows, sums = np.empty((n, heads, dim)), np.zeros((n + 1, heads, dim))
    for j in range(n):
        step = np.where(rng.random((heads, dim)) < 0.5, 1.0, -1.0)
        rows[j] = np.where(np.abs(sums[j]) >= most, -np.sign(sums[j]), step)
        sums[j + 1] = sums[j] + rows[j]
    rows[:, :, 0] = 1.0
    sums[:, :, 0] = np.arange(n + 1)[:, None]
    return rows, sums


# users, shortest, longest, heads, query heads a head, tokens, dim; whether runs are whole rows, and their least length
CUTS = [
    (30, 2000, 9000, 1, 2, 3, 64, True, 2), (12, 300, 8191, 2, 4, 16, 128, True, 2), (20, 1000, 8000, 2, 2, 75, 32, True, 4),
    (20, 1000, 5000, 1, 1, 20, 256, True, 2), (40, 500, 6000, 2, 1, 8, 32, True, 2),
    (150, 0, 1500, 4, 1, 33, 64, False, 3), (100, 0, 1500, 2, 2, 75, 128, False, 3), (150, 0, 1400, 3, 2, 4, 256, False, 9),
    (700, 0, 1400, 2, 2, 4, 32, False, 9), (150, 0, 3400, 2, 2, 65, 64, False, 9), (300, 0, 3000, 2, 2, 4, 128, False, 9),
    (200, 0, 1500, 4, 2, 20, 256, False, 9), (400, 0, 1300, 3, 1, 150, 32, False, 9), (60, 0, 40000, 1, 2, 1, 32, False, 9),
    (1, 40000, 40000, 1, 2, 1, 32, False, 1)]
