"""Microscaled 4-bit rows by their definition, in float64 (numpy), for the tests.

MX: blocks of 32, s = 2^(floor(log2 bmax) - 2) in [2^-127, 2^125], g = 1 (0 for a zero row).
NV: blocks of 16, g = f32(amax / 2688), s = e4m3(bmax / f32(6 g)), d = f32(s g); a row whose
amax is below 2^-100 is zeros with g = 0.  code = e2m1(x / s or d).  Roundings to nearest,
ties to even, of exact quotients, saturating; a row with a NaN or infinity has g = NaN."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BLOCK = {"mx": 32, "nv": 16}


def pad_dim(dim):
    return -(-dim // 128) * 128


def nearest_on(grid, y):
    """Index of the nearest entry of an ascending grid (ties to the even index), saturating."""
    mid = 0.5 * (grid[1:] + grid[:-1])
    i = np.searchsorted(mid, y, side="left")     # mid[i - 1] < y <= mid[i]
    tie = (i < len(mid)) & (y == mid[np.minimum(i, len(mid) - 1)]) & (i % 2 == 1)
    return i + tie


def e4m3_grid():
    b = np.arange(127)  # up to 448, byte 126
    e, m = b >> 3, b & 7
    return np.where(e > 0, (8 + m) * 2.0 ** (e - 10.0), m * 2.0 ** -9)


E4M3 = e4m3_grid()


def quantise(x, fmt):
    """x [n, dim] -> (codes uint8 [n, dp], scale bytes uint8 [n, blocks], g float32 [n])."""
    x = np.asarray(x, dtype=np.float64)
    n, dim = x.shape
    dp, block = pad_dim(dim), BLOCK[fmt]
    fine = np.isfinite(x).all(1)
    b = np.zeros((n, dp))
    b[:, :dim] = np.where(fine[:, None], x, 0.0)
    b = b.reshape(n, dp // block, block)
    top = np.abs(b).max(2)
    amax = top.max(1)
    if fmt == "mx":
        live = amax > 0
        e = np.clip(np.frexp(top)[1] - 3, -127, 125)
        e = np.where(top > 0, e, -127)
        bits = e + 127
        unit = np.ldexp(1.0, e)
        g = np.where(live, np.float32(1), np.float32(0))
    else:
        live = amax >= 2.0 ** -100
        g = np.where(live, amax / 2688.0, 0.0).astype(np.float32)
        h = (np.float64(6.0) * g).astype(np.float32).astype(np.float64)
        bits = nearest_on(E4M3, top / np.where(live, h, 1.0)[:, None])
        unit = (E4M3[bits] * g[:, None].astype(np.float64)).astype(np.float32).astype(np.float64)
    live = live & fine
    ok = live[:, None] & (unit > 0)
    y = np.abs(b) / np.where(ok, unit, 1.0)[:, :, None]
    codes = nearest_on(GRID, y) + 8 * (b < 0)
    codes = np.where(ok[:, :, None], codes, 0)
    bits = np.where(live[:, None], bits, 0)
    g = np.where(fine, g, np.float32(np.nan)).astype(np.float32)
    return codes.reshape(n, dp).astype(np.uint8), bits.astype(np.uint8), g


def values(codes, bits, fmt):
    """Rows in units of g, float64 (exact)."""
    v = np.where(codes >= 8, -GRID[codes & 7], GRID[codes & 7])
    s = np.ldexp(1.0, bits.astype(np.int32) - 127) if fmt == "mx" else E4M3[bits]
    return v * np.repeat(s, BLOCK[fmt], axis=1)


def store_scales(bits, n_slots):
    """Scale bytes [n, blocks] in the store's layout (n <= n_slots; the rest zero)."""
    n, nb = bits.shape
    tiles, atoms = -(-n_slots // 128), nb // 4
    full = np.zeros((tiles * 128, nb), np.uint8)
    full[:n] = bits
    return full.reshape(tiles, 4, 32, atoms, 4).transpose(0, 3, 2, 1, 4).reshape(-1)


def row_scales(flat, n, atoms):
    """The inverse: the store's scale bytes -> [n, 4 * atoms]."""
    t = flat.reshape(-1, atoms, 32, 4, 4).transpose(0, 3, 2, 1, 4)
    return t.reshape(-1, 4 * atoms)[:n]


def products(q, rows, fmt):
    """(f64 scores [nq, n] as f64((sum g_r) g_t), sum of |terms|) of raw queries and rows."""
    qc, qb, qg = quantise(q, fmt)
    rc, rb, rg = quantise(rows, fmt)
    a, b = values(qc, qb, fmt), values(rc, rb, fmt)
    with np.errstate(invalid="ignore", over="ignore"):
        s = (a @ b.T) * rg.astype(np.float64) * qg.astype(np.float64)[:, None]
        m = (np.abs(a) @ np.abs(b).T) * rg.astype(np.float64) * qg.astype(np.float64)[:, None]
    return s, m


def best(scores, k):
    """The k best per query by (float32 score desc, id asc), -1 / -inf past the NaN ones."""
    with np.errstate(over="ignore"):
        s = scores.astype(np.float32) + np.float32(0)
    s = np.where(np.isnan(s), -np.inf, s).astype(np.float32)
    nq, n = s.shape
    order = np.argsort(-s, axis=1, kind="stable")[:, :k]
    v = np.take_along_axis(s, order, 1)
    ids = np.where(v > -np.inf, order, -1).astype(np.int32)
    pad = ((0, 0), (0, k - ids.shape[1]))
    return (np.pad(ids, pad, constant_values=-1),
            np.pad(v, pad, constant_values=-np.inf).astype(np.float32))
