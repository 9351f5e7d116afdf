"""Microscaled matrices in plain numpy, 64 bits: the formats' elements, quantisation by search over them, the memory
layout element by element (include/kq4.h kq4_mx_bytes), and the products with bounds of what fp32 sums may be off."""
import numpy as np

F32 = np.float32


def elements(bits):
    """The non-negative elements by their codes: e2m1, e2m3."""
    if bits == 4:
        return np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    return np.array([m / 8 if e == 0 else (8 + m) * 2.0 ** (e - 4) for e in range(4) for m in range(8)])


def decode(codes, bits):
    """Codes (one per element) as float64."""
    el = elements(bits)
    half = len(el)
    return el[codes % half] * np.where(codes >= half, -1.0, 1.0)


def scale_values(b):
    v = np.exp2(b.astype(np.float64) - 127)
    return np.where(b == 255, np.nan, v)


def values(codes, scales, bits):
    """float64 [rows][cols] of codes [rows][cols] (one per element) and scale bytes [rows][cols / 32]."""
    with np.errstate(invalid="ignore"):
        return decode(codes, bits) * np.repeat(scale_values(scales), 32, 1)


def quantize(x, bits):
    """(codes [rows][cols], scale bytes [rows][cols / 32]) of fp32 x, by the definition."""
    el = elements(bits)
    n, cols = x.shape
    x = x.astype(np.float64).reshape(n, -1, 32)
    over = (el[-1] + 8) / 2                                      # halfway to the element after the largest
    finite = np.isfinite(x).all(2)
    amax = np.where(finite, np.abs(np.where(np.isfinite(x), x, 0)).max(2), 0)
    e = np.full(amax.shape, -127)
    for k in range(-127, 128):                                   # a tie goes to the even code, the one past the last
        e[amax * 2.0 ** -k >= over] = k + 1
    y = np.abs(np.where(np.isfinite(x), x, 0)) * np.exp2(-e.astype(np.float64))[:, :, None]
    mid = (el[1:] + el[:-1]) / 2
    code = np.zeros(y.shape, np.int64)
    for i, m in enumerate(mid):
        code += (y > m) if i % 2 == 0 else (y >= m)
    code += np.signbit(x) * len(el)
    code[~finite] = 0
    b = np.where(finite, e + 127, 255)
    return code.reshape(n, cols).astype(np.uint8), b.astype(np.uint8)


def row_major(codes, bits):
    """Codes as a checkpoint holds them."""
    if bits == 4:
        return codes[:, 0::2] | (codes[:, 1::2] << 4)
    b = np.unpackbits(codes[:, :, None], axis=2, count=6, bitorder="little")
    return np.packbits(b.reshape(codes.shape[0], -1), axis=1, bitorder="little")


def dims(rows, cols):
    return -(-rows // 16), -(-cols // 128), -(-cols // 512)


def matrix(codes, scales, bits):
    """The bytes of a microscaled matrix, tile by tile."""
    n, cols = codes.shape
    nt, kt, kq = dims(n, cols)
    c = np.zeros((16 * nt, 128 * kt), np.uint8)
    c[:n, :cols] = codes
    c = row_major(c, bits)
    s = np.zeros((16 * nt, 16 * kq), np.uint8)
    s[:n, :cols // 32] = scales
    width, out = 16 * bits, []                                   # bytes of a tile's row: 4 blocks
    for g in range(0, nt, 8):
        for k in range(kt):
            for t in range(g, min(g + 8, nt)):
                tile = c[16 * t:16 * t + 16, width * k:width * (k + 1)].reshape(16, 4, -1).transpose(1, 0, 2)
                out += [tile[:, :, :16].tobytes(), tile[:, :, 16:].tobytes()]
    for g in range(0, nt, 8):
        for q in range(kq):
            for t in range(g, min(g + 8, nt)):
                tile = s[16 * t:16 * t + 16, 16 * q:16 * q + 16]
                out.append(tile.reshape(16, 4, 4).transpose(2, 0, 1).tobytes())
    return np.frombuffer(b"".join(out), np.uint8)


def random_weights(rng, rows, cols, spread=2):
    """(codes, scale bytes): every code, scales over 2^(2 * spread)."""
    return (rng.integers(0, 16, (rows, cols), np.uint8),
            rng.integers(120 - spread, 121 + spread, (rows, cols // 32)).astype(np.uint8))


# How far a kernel's fp32 sum may be off, relative to the sum of the terms' magnitudes: a matrix instruction takes in 128 columns
# exactly but for the alignment and one rounding of its result, at most 2^-23 of the magnitudes (truncation), and the waves' and
# splits' sums and the residual are added with 2^-24 each, at most 64 of them. 2^-126 times the columns: terms that vanish.
def bound(mags, cols):
    return mags * ((-(-cols // 128)) * 2.0 ** -23 + 64 * 2.0 ** -24) + cols * 2.0 ** -126


def product(xv, wv, res=None):
    """(out, bound) of x [n][cols] and w [rows][cols] in 64 bits."""
    out, mags = xv @ wv.T, np.abs(xv) @ np.abs(wv).T
    if res is not None:
        out, mags = out + res, mags + np.abs(res)
    return out, bound(mags, xv.shape[1])


def gated(xv, gv, uv):
    """(silu(x . g) * (x . u), bound). silu' lies in [-0.1, 1.1]; exp, the quotient and two products add under 2^-20."""
    (g, eg), (u, eu) = product(xv, gv), product(xv, uv)
    silu = g / (1 + np.exp(-g))
    out = silu * u
    return out, 1.1 * eg * (np.abs(u) + eu) + (np.abs(silu)) * eu + np.abs(out) * 2.0 ** -20 + 2.0 ** -120


def acts(rng, n, cols):
    """fp32 rows as hidden states are: normal, some channels large, blocks of all magnitudes."""
    gain = np.where(rng.random(cols) < 0.02, 30.0, 1.0)
    return (rng.standard_normal((n, cols)) * gain * np.exp2(rng.integers(-3, 4, (n, 1)))).astype(F32)
