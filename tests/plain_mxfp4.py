"""Plain implementations of the microscaled 4-bit format and its products, in numpy and 64 bits."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
CHUNK = 8704


def addresses(rows, k):
    """(byte of the codes, shift within it, byte of the scale) of every element of a packed [rows, k] matrix."""
    chunks = -(-k // 128)
    r, c = np.arange(rows)[:, None], np.arange(k)[None, :]
    base = (r // 128 * chunks + c // 128) * CHUNK
    within = c % 8
    nibble = np.where(within % 2 == 0, within // 2, 4 + within // 2)
    code = base + c % 128 // 32 * 2048 + r % 128 * 16 + c % 32 // 8 * 4 + nibble // 2
    scale = base + 8192 + r % 32 * 16 + r % 128 // 32 * 4 + c % 128 // 32
    return code, 4 * (nibble % 2) + 0 * r, scale


def values(data, rows, k):
    """What a packed matrix stands for, [rows, k] in 64 bits; `data`: its bytes."""
    data = np.asarray(data).reshape(-1)
    code, shift, scale = addresses(rows, k)
    c = data[code].astype(np.int64) >> shift & 15
    s = data[scale].astype(np.float64)
    with np.errstate(invalid="ignore"):
        return np.where(s == 255, np.nan, GRID[c & 7] * np.where(c & 8, -1.0, 1.0) * 2.0 ** (s - 127))


def scales_and_codes(x):
    """The scale byte and the code of every element of x [rows, k] (float32 values): the largest magnitude's exponent less 2,
    and the nearest grid value, of two equally near ones the even code."""
    x = np.asarray(x, dtype=np.float64)
    rows, k = x.shape
    wide = np.zeros((rows, -(-k // 32) * 32))
    wide[:, :k] = x
    wide = wide.reshape(rows, -1, 32)
    bad = ~np.isfinite(wide).all(2)
    clean = np.where(np.isfinite(wide), wide, 0.0)
    top = np.abs(clean).max(2)
    s = np.where(top > 0, np.maximum(np.frexp(np.where(top > 0, top, 1.0))[1] - 1 - 2 + 127, 0), 0)
    a = np.abs(clean) * 2.0 ** (127.0 - s)[..., None]
    best, code = np.full(a.shape, np.inf), np.zeros(a.shape, dtype=np.int64)
    for c in (0, 2, 4, 6, 1, 3, 5, 7):
        off = np.abs(a - GRID[c])
        code, best = np.where(off < best, c, code), np.minimum(off, best)
    code = code | np.where(np.signbit(clean), 8, 0)
    code[bad] = 0
    s[bad] = 255
    return s, code.reshape(rows, -1)[:, :k]


def pack(x):
    """The packed bytes of x [rows, k], uint8 [ceil(rows / 128), ceil(k / 128), 8704]."""
    rows, k = x.shape
    data = np.zeros((-(-rows // 128), -(-k // 128), CHUNK), dtype=np.uint8)
    s, codes = scales_and_codes(x)
    code_at, shift, scale_at = addresses(rows, k)
    flat = data.reshape(-1)
    np.bitwise_or.at(flat, code_at, (codes << shift).astype(np.uint8))
    flat[scale_at] = np.repeat(s, 32, axis=1)[:, :k].astype(np.uint8)
    return data


def unit(name, g, u, params=(0.0, 0.0)):
    """act(g) * u in 64 bits."""
    if name == "relu":
        return np.maximum(g, 0) * u
    if name == "relu_squared":
        return np.maximum(g, 0) ** 2 * u
    if name == "gelu_tanh":
        return 0.5 * g * (1 + np.tanh(0.7978845608028654 * (g + 0.044715 * g ** 3))) * u
    if name == "clamped_swish":
        g, u = np.minimum(g, params[0]), np.clip(u, -params[0], params[0])
        return g / (1 + np.exp(-params[1] * g)) * (u + 1)
    return g / (1 + np.exp(-g)) * u
