"""Rotary positions of several axes in 64 bits, pair by pair from their definition:
what the tests compare with."""
import numpy as np


def pairs(sections, order, own):
    """(axis, column of the table) of each pair that turns."""
    if order == "blocks":
        out = [(a, i) for a, n in enumerate(sections) for i in range(n)]
    else:
        out, given = [], [0] * len(sections)
        while sum(given) < sum(sections):
            for a, n in enumerate(sections):
                if given[a] < n:
                    out.append((a, given[a]))
                    given[a] += 1
    return out if own else [(a, p) for p, (a, _) in enumerate(out)]


def turn(x, pos, table, sections, order, own, half):
    """x [rows, heads, dim], pos [axes, rows], table [n_pos, columns, 2]."""
    x = np.asarray(x, np.float64)
    y, shares = x.copy(), pairs(sections, order, own)
    used = [a for a, n in enumerate(sections) if n]
    bad = np.any((pos[used] < 0) | (pos[used] >= len(table)), axis=0)
    for i, (axis, col) in enumerate(shares):
        a, b = (i, len(shares) + i) if half else (2 * i, 2 * i + 1)
        cs = table[np.where(bad, 0, pos[axis]), col].astype(np.float64)[:, None]
        y[..., a] = x[..., a] * cs[..., 0] - x[..., b] * cs[..., 1]
        y[..., b] = x[..., a] * cs[..., 1] + x[..., b] * cs[..., 0]
    y[bad] = np.nan
    return y
