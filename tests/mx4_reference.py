"""Plain numpy forms, in 64 bits, of the 4-bit block format and of the gated block norm, for their tests."""
import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)


def quantize(x):
    """x [rows, K] -> (codes [rows, 16 nb] uint8, scale bytes [rows, nb] uint8), from the definition: the largest
    magnitude's exponent, then the nearest magnitude, ties to the even code."""
    x = np.asarray(x, np.float64)
    rows, k = x.shape
    nb = -(-k // 32)
    b = np.zeros((rows, nb * 32))
    b[:, :k] = x
    b = b.reshape(rows, nb, 32)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    top = np.abs(b).max(-1)
    _, e = np.frexp(top)  # top = f 2^e, f in [0.5, 1)
    s = np.where(top > 0, np.maximum(e - 3, -127), -127)
    a = np.abs(b) / np.exp2(s.astype(np.float64))[..., None]
    code = np.zeros(a.shape, np.uint8)
    for i in range(7):
        mid = (E2M1[i] + E2M1[i + 1]) / 2
        code += (a >= mid) if i % 2 else (a > mid)
    code |= (np.signbit(b).astype(np.uint8) << 3)
    code[bad] = 0
    sb = np.where(bad, 255, s + 127).astype(np.uint8)
    code = code.reshape(rows, nb * 16, 2)
    return code[..., 0] | (code[..., 1] << 4), sb


def round_to(x, sb):
    """x [rows, K] in 64 bits rounded to the values of blocks with the scale bytes sb [rows, nb]."""
    f = np.repeat(np.exp2(sb.astype(np.float64) - 127), 32, 1)[:, :x.shape[1]]
    a = np.abs(x) / f
    code = np.zeros(a.shape, int)
    for i in range(7):
        mid = (E2M1[i] + E2M1[i + 1]) / 2
        code += (a >= mid) if i % 2 else (a > mid)
    return np.copysign(E2M1[code] * f, x)


def values(codes, sb, k):
    """The values [rows, k] in 64 bits."""
    c = np.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1)
    v = np.where(c & 8, -1.0, 1.0) * E2M1[c & 7]
    f = np.where(sb == 255, np.nan, np.exp2(sb.astype(np.float64) - 127))
    return (v * np.repeat(f, 32, 1)[:, :v.shape[1]])[:, :k]


def tile_scales(sb):
    """Scale bytes [rows, nb] -> the tiles of 128 rows x 4 blocks, one byte at a time."""
    rows, nb = sb.shape
    kt = -(-nb // 4)
    out = np.zeros(-(-rows // 128) * kt * 512, np.uint8)
    r, b = np.meshgrid(np.arange(rows), np.arange(nb), indexing="ij")
    out[((r // 128) * kt + b // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4] = sb
    return out


def untile_scales(tiles, rows, nb):
    kt = -(-nb // 4)
    r, b = np.meshgrid(np.arange(rows), np.arange(nb), indexing="ij")
    return tiles[((r // 128) * kt + b // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4]


def norm(v, kind, w, b, eps):
    """kind 0 nothing, 1 LayerNorm, 2 RMSNorm; returns (norm(v), |v|'s size in units of its spread per row)."""
    if kind == 0:
        return v, np.zeros((len(v), 1))
    m = v.mean(-1, keepdims=True) if kind == 1 else 0.0
    r = 1 / np.sqrt(((v - m) ** 2).mean(-1, keepdims=True) + eps)
    y = (v - m) * r
    if w is not None:
        y = y * w
    if b is not None:
        y = y + b
    return y, np.abs(v).mean(-1, keepdims=True) * r
