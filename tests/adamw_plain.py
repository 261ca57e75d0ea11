"""AdamW with 32-bit and 8-bit moments in 64 bits on the CPU: what the tests of optim.AdamW's operators compare with.
Written from the formulas, with tables of what the codes stand for; nothing of the package is used."""
import numpy as np

BLOCK = 64
M_TABLE = np.array([(a & 7) * 2.0 ** -9 if a < 8 else 2.0 ** ((a >> 3) - 7) * (1 + (a & 7) / 8) for a in range(127)])
V_TABLE = np.array([0.0] + [2.0 ** (c >> 3) * (1 + (c & 7) / 8) for c in range(1, 256)])


def row_length(shape):
    return shape[1] if len(shape) == 2 and 1 <= shape[1] <= BLOCK else 0


def blocks_of(shape):
    """Block index of every element (flattened) and the number of blocks."""
    n = int(np.prod(shape))
    row = row_length(shape) or BLOCK
    return np.arange(n) // row, (shape[0] if row_length(shape) else -(-n // BLOCK))


def decode(mcode, vcode, exponents, shape):
    where, _ = blocks_of(shape)
    xm, xv = exponents[where, 0].astype(np.float64), exponents[where, 1].astype(np.float64)
    c, v = mcode.reshape(-1).astype(np.int64), vcode.reshape(-1).astype(np.int64)
    m = np.append(M_TABLE, 480.0)[c % 128] * np.where(c >= 128, -1.0, 1.0) * 2.0 ** (np.maximum(xm, 9) - 135)
    v = V_TABLE[v] * 2.0 ** (np.maximum(xv, 32) - 158)
    m[xm == 255] = np.nan
    v[xv == 255] = np.nan
    return m.reshape(shape), v.reshape(shape)


def _mix(x):
    x = np.uint32(x) if np.isscalar(x) else x.astype(np.uint32)
    with np.errstate(over="ignore"):
        x = (x ^ (x >> np.uint32(16))) * np.uint32(0x6A09E667)
        x = (x ^ (x >> np.uint32(15))) * np.uint32(0xBB67AE85)
    return x ^ (x >> np.uint32(16))


def noise(n, seed, tensor, step):
    """The 32 random bits of elements 0..n-1."""
    return noise_at(np.arange(n, dtype=np.int64), seed, tensor, step)


def noise_at(i, seed, tensor, step):
    with np.errstate(over="ignore"):
        key = _mix(_mix(np.uint32(seed & 0xFFFFFFFF) + np.uint32(0x9E3779B1) * np.uint32(tensor)) + np.uint32(step))
    h = _mix((i >> 2).astype(np.uint32) ^ key).astype(np.uint64)
    turn = (8 * (i & 3)).astype(np.uint64)
    return ((h << turn) | (h >> (np.uint64(32) - turn))) & np.uint64(0xFFFFFFFF)


def encode(m, v, bits, shape):
    """(mcode, vcode, exponents) and how near each element's rounding was to the other code, in units of a code step."""
    where, count = blocks_of(shape)
    m, v = m.reshape(-1), v.reshape(-1)
    chance = [((bits & np.uint64(0xFFFF)).astype(np.float64) + 0.5) / 65536, ((bits >> np.uint64(16)).astype(np.float64) + 0.5) / 65536]
    codes, xs, margins = [], [], []
    for x, table, top, low, unit_of, r in ((np.abs(m), M_TABLE, 1.75, 9, 135, chance[0]), (v, V_TABLE, 1.875, 32, 158, chance[1])):
        largest = np.zeros(count)
        bad = np.zeros(count, bool)
        np.logical_or.at(bad, where, ~np.isfinite(x) | (np.abs(x) > 3.4028235e38))
        np.maximum.at(largest, where, np.where(np.isfinite(x), x, 0.0))
        mant, e = np.frexp(largest)
        e = np.where(largest > 0, e - 1 + (2 * mant > top), -1000)
        xb = np.clip(e + 127, low, 254)
        y = np.where(bad[where], 0.0, x) / 2.0 ** (xb[where] - unit_of)
        i = np.clip(np.searchsorted(table, y, side="right") - 1, 0, len(table) - 2)
        share = (y - table[i]) / (table[i + 1] - table[i])
        c = i + (share + r >= 1)
        if table is V_TABLE:
            c = np.where((y > 0) & (c < 1), 1, c)
        codes.append(np.where(bad[where], 0, c))
        xs.append(np.where(bad, 255, xb))
        margins.append(np.abs(share + r - 1))
    codes[0] = np.where((m < 0) & ~(np.isnan(m)), codes[0] + 128, codes[0])
    codes[0] = np.where(xs[0][where] == 255, 0, codes[0])
    return (codes[0].astype(np.uint8).reshape(shape), codes[1].astype(np.uint8).reshape(shape),
            np.stack(xs, 1).astype(np.uint8).reshape(-1, 2), [x.reshape(shape) for x in margins])


def update(p, g, m, v, *, step, lr, betas, eps, weight_decay, scale=1.0, missed=None):
    """p, m, v after the step, in 64 bits; ``missed``: steps that each row missed."""
    b1, b2 = betas
    if missed is not None:
        d = np.maximum(missed, 0).astype(np.float64)[:, None]
        m, v = m * b1 ** d, v * b2 ** d
    g = g * scale
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    with np.errstate(invalid="ignore", divide="ignore"):
        p = p * (1 - lr * weight_decay) - lr * (m / (1 - b1 ** step)) / (np.sqrt(v / (1 - b2 ** step)) + eps)
    return p, m, v


def error_bounds(p0, p, g, m0, m, v, *, step, lr, betas, eps, weight_decay):
    """Bounds of the errors of p, m, v computed in float32 (half a spacing, u = 2^-24 relative, for every rounding).

    m' = m + (1-b1)(g - m): g carries the clip's product (u|g|), the decay of a late row 3u|m| (a power and a product), the
    difference and the constant a rounding each, the fused sum one: (1-b1)(4u|g| + 3u|m|) + 3u|m| + u|m'|.
    v': sums of positive terms, each with at most 8 roundings (g twice, the products, the constants, the decay): 8u v'.
    step = rate m' / (sqrt(v') root + eps): m' as above, sqrt 4u + 1u, rate and root (constants) and three operations: 12u of
    it, hardware's square root and reciprocal (one unit in the last place = 2u each) among them.
    p': the constant, the product and the sum: u each of |p|, |p| and |p'| plus u of the step."""
    u = 2.0 ** -24
    b1, b2 = betas
    em = (1 - b1) * (4 * u * np.abs(g) + 3 * u * np.abs(m0)) + 3 * u * np.abs(m0) + 2 * u * np.abs(m)
    ev = 8 * u * v + 2.0 ** -149
    rate, denom = lr / (1 - b1 ** step), np.sqrt(v / (1 - b2 ** step)) + eps
    change = rate * np.abs(m) / denom
    ep = 16 * u * change + rate * em / denom + u * (2 * np.abs(p0) + np.abs(p)) + 2.0 ** -149
    return ep, em + 2.0 ** -149, ev
