"""Microscaled 4-bit matrices on the CPU, from the definition (in 64 bits but for one FP32 product): the quantiser, the packed form, the values it stands for."""
import numpy as np

MXFP4, NVFP4 = 8, 9
BLOCK = {MXFP4: 32, NVFP4: 16}
LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def e4m3_value(byte):
    byte = np.asarray(byte).astype(np.int64) & 0x7F
    e, m = byte >> 3, byte & 7
    v = np.where(e > 0, (1 + m / 8.0) * 2.0 ** (e - 7.0), m / 8.0 * 2.0 ** -6)
    return np.where(byte == 0x7F, np.nan, v)


E4M3 = e4m3_value(np.arange(127))


def nearest(table, num, den):
    """Index of the entry of an ascending table nearest to num / den (den > 0), ties to the even index; halfway points times den are exact in
    64 bits for the tables and denominators used here."""
    mids = (table[1:] + table[:-1]) / 2
    at = np.zeros(np.broadcast(num, den).shape, np.int64)
    for i, m in enumerate(mids):
        at += np.where((num > m * den) | ((num == m * den) & (i % 2 == 1)), 1, 0)
    return at


def matrix_scale(amax):
    """The power of two 2^t with the smallest t for which amax <= 2688 * 2^t, t from -110 to 117."""
    if not (amax > 0) or not np.isfinite(amax):
        return 1.0
    t = -110
    while t < 117 and amax > 2688.0 * 2.0 ** t:
        t += 1
    return 2.0 ** t


def quantize(x, fmt, amax=None):
    """(codes, scale bytes, matrix scale) of a 2-D array; codes up to the end of the last block of a row."""
    rows, cols = x.shape
    bs = BLOCK[fmt]
    blocks = -(-cols // bs)
    v = np.zeros((rows, blocks * bs))
    v[:, :cols] = x
    sign = np.signbit(v).astype(np.uint8) << 3
    bad = ~np.isfinite(v).reshape(rows, blocks, bs).all(axis=2)
    finite = np.where(np.isfinite(v), v, 0.0)
    v = np.abs(finite).reshape(rows, blocks, bs)
    m = v.max(axis=2)
    if fmt == MXFP4:
        g = 1.0
        e = np.frexp(np.where(m > 0, m, 1.0))[1] - 1 - 2
        e = np.where(m > 0, np.maximum(e, -127), -127)
        byte, s = e + 127, 2.0 ** e
        byte = np.where(bad, 255, byte)
    else:
        g = matrix_scale((np.abs(finite).max() if finite.size else 0.0) if amax is None else float(amax))
        p = (m / g).astype(np.float32) * np.float32(1 / 6)             # (the definition: an FP32 product)
        byte = nearest(E4M3, p.astype(np.float64), np.ones_like(m))
        s = E4M3[byte] * g
        byte = np.where(bad, 127, byte)
    codes = np.where(s[..., None] > 0, nearest(LEVELS, v, s[..., None]), 0).reshape(rows, -1).astype(np.uint8) | sign
    codes = np.where(np.repeat(bad, bs, axis=1), 0, codes)
    return codes, byte.astype(np.uint8), g


def sizes(rows, cols, fmt):
    ld = -(-cols // 32) * 16
    at = -(-(128 + rows * ld) // 128) * 128
    return ld, at, -(-rows // 128), -(-cols // (4 * BLOCK[fmt]))


def packed_bytes(rows, cols, fmt):
    _, at, groups, quads = sizes(rows, cols, fmt)
    return at + groups * quads * 512


def pack(codes, byte, g, fmt, cols, fill=0):
    """The packed form; `fill` stands in scale bytes of rows behind the last one."""
    rows, blocks = byte.shape
    ld, at, groups, quads = sizes(rows, cols, fmt)
    out = np.zeros(at + groups * quads * 512, np.uint8)
    out[:4] = np.array([g], np.float32).view(np.uint8)
    wide = np.zeros((rows, 2 * ld), np.uint8)
    wide[:, : codes.shape[1]] = codes
    out[128: 128 + rows * ld] = (wide[:, 0::2] | (wide[:, 1::2] << 4)).reshape(-1)
    full = np.full((groups * 128, quads * 4), fill, np.uint8)
    full[:rows] = 0
    full[:rows, :blocks] = byte
    for r in range(groups * 128):
        for b in range(quads * 4):
            out[at + ((r // 128) * quads + b // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4] = full[r, b]
    return out


def values(codes, byte, g, fmt, cols):
    rows, blocks = byte.shape
    codes = codes[:, : blocks * BLOCK[fmt]]
    v = np.where(codes > 7, -1.0, 1.0) * LEVELS[codes & 7]
    s = e4m3_value(byte) if fmt == NVFP4 else np.where(byte == 255, np.nan, 2.0 ** (byte.astype(np.float64) - 127))
    return ((v.reshape(rows, blocks, -1) * s[..., None]).reshape(rows, -1) * float(np.float32(g)))[:, :cols]


def random_parts(rng, rows, cols, fmt, exact=True):
    """Codes and scales of a matrix.  exact: scales 1, 2 and 4 and a matrix scale 1, so that every value is a multiple of 0.5 up to 24."""
    bs = BLOCK[fmt]
    blocks = -(-cols // bs)
    codes = rng.integers(0, 16, (rows, blocks * bs)).astype(np.uint8)
    codes[:, cols:] = 0
    if exact:
        e = rng.integers(0, 3, (rows, blocks))
        byte = (e + 127 if fmt == MXFP4 else (e + 7) << 3).astype(np.uint8)
        return codes, byte, 1.0
    byte = (rng.integers(117, 130, (rows, blocks)) if fmt == MXFP4 else rng.integers(40, 120, (rows, blocks))).astype(np.uint8)
    return codes, byte, (1.0 if fmt == MXFP4 else 0.37)
