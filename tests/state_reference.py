"""The optimizer-state operators in float64 numpy, restated from the definitions in
``include/thorn_b200.h``, with bounds on what fp32 arithmetic may change.

A code may differ from the float64 one only where the float64 value lies within the fp32
error of the border between two codes (the rounding fraction included), and a scale only
where the block's maximum lies within it of 448 times a power of two.
"""
import numpy as np

M32, M64 = (1 << 32) - 1, (1 << 64) - 1
BLOCK = 128
# values of the codes 0..126, and of the negative ones
GRID = np.array([(c & 7) * 2.0 ** -9 if c < 8 else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 7) for c in range(127)])


def key_of(seed):
    z = (seed + 0x9E3779B97F4A7C15) & M64
    z = ((z ^ (z >> 32)) * 0x6A09E667F3BCC909) & M64
    z = ((z ^ (z >> 29)) * 0xBB67AE8584CAA73B) & M64
    return z ^ (z >> 32)


def _fold(a, b):
    t = a * b
    return (t >> np.uint64(32)) ^ (t & np.uint64(M32))


def fractions(n, seed, run=0, start=0):
    """The rounding fraction in [0, 1) of n elements of run ``run`` from ``start`` (a multiple of 4)."""
    key = key_of(seed)
    q = np.arange(-(-n // 4), dtype=np.uint64) + np.uint64(start // 4)
    a = ((q & np.uint64(M32)) * np.uint64(0x9E3779B9) + np.uint64(key & M32)) & np.uint64(M32)
    hi = ((q >> np.uint64(32)) + np.uint64(run)) & np.uint64(M32)
    x = _fold(a, a ^ np.uint64(key >> 32) ^ hi)
    r = _fold(x, x ^ np.uint64(0xBB67AE85))
    out = np.zeros((q.size, 4))
    for lane in range(4):
        half = (r >> np.uint64(16 * (lane // 2))) & np.uint64(0xFFFF)
        for bit in range(16):
            w = 2.0 ** -(bit + 1) if lane % 2 else 2.0 ** (bit - 16)
            out[:, lane] += w * ((half >> np.uint64(bit)) & np.uint64(1)).astype(np.float64)
    return out.reshape(-1)[:n]


def scale_bytes(x):
    """Scale byte of every block of the flat array x."""
    nb = -(-x.size // BLOCK)
    v = np.zeros(nb * BLOCK)
    v[:x.size] = np.abs(x)
    top = v.reshape(nb, BLOCK).max(1) if nb else np.zeros(0)
    out = np.zeros(nb, dtype=np.int64)
    for i, t in enumerate(top):
        if not np.isfinite(t):
            out[i] = 255
        elif t > 0:
            k = int(np.floor(np.log2(t))) - 10
            while t > 448.0 * 2.0 ** k:
                k += 1
            out[i] = max(0, k + 127)
    return out


def read(codes, bytes_):
    """Values of a flat 8-bit state (codes and scale bytes as uint8)."""
    c = codes.astype(np.int64)
    v = np.where((c & 127) == 127, np.nan, GRID[np.minimum(c & 127, 126)]) * np.where(c & 128, -1.0, 1.0)
    s = np.where(bytes_.astype(np.int64) == 255, np.nan, 2.0 ** (bytes_.astype(np.float64) - 127))
    return v * np.repeat(s, BLOCK)[:c.size]


def check_state(x, err, codes, bytes_, frac, positive, what):
    """Checks the codes and scale bytes that a kernel wrote for float64 values ``x`` known to
    ``err`` (absolute, per element), with rounding fractions ``frac``."""
    want = scale_bytes(x)
    got = bytes_.astype(np.int64)
    for i in np.nonzero(want != got)[0]:  # only at a border
        blk = slice(i * BLOCK, (i + 1) * BLOCK)
        ok = {int(b) for s in (-1, 1) for b in scale_bytes(np.maximum(np.abs(x[blk]) + s * err[blk], 0))}
        assert got[i] in ok, (what, "scale", i, got[i], want[i], np.abs(x[blk]).max())
    ok_blocks = np.repeat(got < 255, BLOCK)[:x.size]
    size = np.repeat(2.0 ** (got - 127.0), BLOCK)[:x.size]
    y = np.abs(x) / size
    e = err / size
    if positive:
        some = np.repeat([np.abs(x[i * BLOCK:(i + 1) * BLOCK]).max() > 0 for i in range(got.size)], BLOCK)[:x.size]
        y = np.where(some, np.maximum(y, 2.0 ** -9), y)

    def rounded(t):
        t = np.clip(t, 0.0, 448.0)
        i = np.clip(np.searchsorted(GRID, t, side="right") - 1, 0, 125)
        gap = GRID[i + 1] - GRID[i]
        return np.where((t - GRID[i]) / gap + frac >= 1.0, GRID[i + 1], GRID[i])

    with np.errstate(invalid="ignore"):
        lo, hi = rounded(y - e), rounded(y + e)
    c = codes.astype(np.int64)
    mag = GRID[np.minimum(c & 127, 126)]
    bad = ok_blocks & ~((mag >= lo) & (mag <= hi))
    assert not bad.any(), (what, "codes", int(bad.sum()), np.nonzero(bad)[0][:5], mag[bad][:5], y[bad][:5])
    sign = np.where(c & 128, -1.0, 1.0)
    wrong = ok_blocks & (mag > 0) & (np.abs(x) > err) & (sign != np.sign(x))
    assert not wrong.any(), (what, "sign")
    return read(codes, bytes_)


def adamw(p, g, m, v, *, lr, step, betas, eps, wd, degenerate=False):
    """(p, m, v, u) of one step from float64 arrays."""
    b1, b2 = betas
    m = m + (g - m) * (1 - b1)
    v = b2 * v + (1 - b2) * g * g
    num, root = m / (1 - b1 ** step), np.sqrt(v / (1 - b2 ** step))
    if degenerate:
        u = m
    else:
        with np.errstate(divide="ignore", invalid="ignore"):
            u = np.arctan2(num, root) if eps == 0 else num / (root + eps)
    if wd > 0:
        u = np.where(u * p >= 0, u + wd * p, u)
    return p - lr * u, m, v, u
