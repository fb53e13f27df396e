"""float64 restatement of the row operators' number formats (8-bit checkpoints, 4-bit microscaled product): numpy on the CPU, test
infrastructure only."""
import numpy as np

GRID8 = np.array([k * 2.0 ** -9 for k in range(8)] + [(8 + k) * 2.0 ** (e - 3) for e in range(-6, 9) for k in range(8)][:-1])      # e4m3: 0 .. 448
GRID4 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])                                                                        # e2m1


def nearest_even(v, grid):
    """Index of the grid value nearest to |v|; a tie goes to the even index (the code whose last bit is clear)."""
    a = np.abs(v)
    hi = np.clip(np.searchsorted(grid, a), 1, len(grid) - 1)
    lo = hi - 1
    dh, dl = grid[hi] - a, a - grid[lo]
    return np.where((dh < dl) | ((dh == dl) & (hi % 2 == 0)), hi, lo)


def quantise(x, kind):
    """x [rows, n] -> (index into the grid, sign, biased exponent per row and group, restored values), groups of 32 along the rows."""
    grid, step_over = (GRID8, lambda top, s: top > 464.0 * s) if kind == 8 else (GRID4, lambda top, s: top >= 7.0 * s)
    x = np.asarray(x, dtype=np.float64)
    rows, n = x.shape
    groups = (n + 31) // 32
    pad = np.zeros((rows, groups * 32))
    pad[:, :n] = x
    g = pad.reshape(rows, groups, 32)
    top = np.abs(g).max(-1)
    bad = ~np.isfinite(top)
    byte = np.full(top.shape, 16, dtype=np.int64)      # 2^-111, the smallest scale
    for _ in range(260):
        up = ~bad & step_over(np.where(bad, 0, top), np.ldexp(1.0, (byte - 127)))
        if not up.any():
            break
        byte = byte + up
    s = np.ldexp(1.0, byte - 127)[..., None]
    t = np.where(bad[..., None], 0.0, g) / s
    idx = nearest_even(t, grid)
    val = np.where(bad[..., None], np.nan, np.copysign(grid[idx], t) * s)
    byte = np.where(bad, 255, byte)
    return (idx.reshape(rows, -1)[:, :n], np.signbit(t).reshape(rows, -1)[:, :n], byte, val.reshape(rows, -1)[:, :n])


def codes8(x):
    idx, sign, byte, val = quantise(x, 8)
    return (idx + 128 * sign).astype(np.uint8), byte.astype(np.uint8), val
