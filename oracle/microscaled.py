"""Microscaled number formats in float64 (numpy): quantisation, expansion, products, RMS norm.

Restates the definitions of ``include/ancha_b200.h`` (``ancha_mx_*``) with explicit value grids; the
reference project has no counterpart. Test infrastructure only.
"""
from __future__ import annotations

import numpy as np

BLOCK = {"mxf8": 32, "mxf4": 32, "nvf4": 16}
# Non-negative element values in code order. E4M3: bias 7, subnormals of 2^-9, code 127 is NaN.
E4M3 = np.array([m / 8 * 2.0 ** -6 for m in range(8)]
                + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:-1])
E2M1 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
GRID = {"mxf8": E4M3, "mxf4": E2M1, "nvf4": E2M1}


def nearest(t, grid):
    """Codes of the grid values nearest to t >= 0, ties to the even code, saturating."""
    t = np.asarray(t, np.float64)
    hi = np.minimum(np.searchsorted(grid, t), len(grid) - 1)
    lo = np.maximum(hi - 1, 0)
    up, down = grid[hi] - t, t - grid[lo]
    return np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)


def blocks(v, fmt):
    """Rows cut into blocks, zeros behind the end: [rows, blocks, block]."""
    b = BLOCK[fmt]
    rows, cols = v.shape
    z = np.zeros((rows, -(-cols // b) * b))
    z[:, :cols] = v
    return z.reshape(rows, -1, b)


def scale_codes(amax, fmt, g=1.0):
    """Scale codes of blocks whose largest magnitudes are amax (finite)."""
    amax = np.asarray(amax, np.float64)
    if fmt == "nvf4":
        return nearest(np.minimum(amax / (6 * g), 448), E4M3)
    most, power = (464, 8) if fmt == "mxf8" else (7, 2)
    _, e = np.frexp(amax)
    e = np.where(amax > 0, e - 1 - power, -127)
    r = amax / 2.0 ** e
    e = e + ((r > most) if fmt == "mxf8" else (r >= most))
    return np.maximum(e, -127) + 127


def scale_values(codes, fmt, g=1.0):
    codes = np.asarray(codes)
    if fmt == "nvf4":
        return np.append(E4M3, np.nan)[codes] * g
    return np.where(codes == 255, np.nan, 2.0 ** (codes.astype(np.float64) - 127))


def quantize(v, fmt, g=1.0):
    """(element codes with sign bit [rows, cols], scale codes [rows, blocks]) of float64 rows."""
    z = blocks(v, fmt)
    bad = ~np.isfinite(z).all(-1)
    a = np.where(bad, 0, np.abs(np.where(np.isfinite(z), z, 0)).max(-1))
    codes = scale_codes(a, fmt, g)
    s = scale_values(codes, fmt, g)
    with np.errstate(divide="ignore", invalid="ignore"):
        t = np.where((s > 0)[..., None] & ~bad[..., None], np.abs(z) / s[..., None], 0)
    e = nearest(t, GRID[fmt])
    sign = 128 if fmt == "mxf8" else 8
    e = np.where(np.signbit(z) & ~bad[..., None] & (s > 0)[..., None], e | sign, e)
    codes = np.where(bad, 127 if fmt == "nvf4" else 255, codes)
    return e.reshape(v.shape[0], -1)[:, :v.shape[1]], codes


def element_values(codes, fmt):
    n = 128 if fmt == "mxf8" else 8
    grid = np.append(GRID[fmt], np.nan) if fmt == "mxf8" else GRID[fmt]
    return np.where(codes >= n, -1.0, 1.0) * grid[codes % n]


def expand(elements, codes, fmt, g=1.0):
    """Values of element codes [rows, cols] with scale codes [rows, blocks]."""
    s = np.repeat(scale_values(codes, fmt, g), BLOCK[fmt], axis=1)[:, :elements.shape[1]]
    return element_values(elements, fmt) * s


def unpack(data, fmt, cols):
    """Element codes of stored bytes [rows, ld]."""
    data = np.asarray(data)
    if fmt == "mxf8":
        return data[:, :cols].astype(np.int64)
    return np.stack((data & 15, data >> 4), -1).reshape(data.shape[0], -1)[:, :cols].astype(np.int64)


def pack(elements, fmt):
    """Stored bytes of element codes, rows filled with zeros to a multiple of 16 bytes."""
    e = np.asarray(elements, np.uint8)
    per = 1 if fmt == "mxf8" else 2
    width = -(-e.shape[1] // (16 * per)) * 16 * per
    z = np.zeros((e.shape[0], width), np.uint8)
    z[:, :e.shape[1]] = e
    return z if fmt == "mxf8" else z[:, 0::2] | (z[:, 1::2] << 4)


def tile(codes):
    """Scale codes [rows, blocks] in the stored order, by the address formula of the header."""
    rows, nb = codes.shape
    kt = -(-nb // 4)
    out = np.zeros(-(-rows // 128) * kt * 512, np.uint8)
    r, b = np.meshgrid(np.arange(rows), np.arange(nb), indexing="ij")
    out[((r // 128) * kt + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4] = codes
    return out


def untile(data, rows, nb):
    kt = -(-nb // 4)
    r, b = np.meshgrid(np.arange(rows), np.arange(nb), indexing="ij")
    return np.asarray(data).reshape(-1)[((r // 128) * kt + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4]


def rms_norm(s, gain, eps):
    s = np.asarray(s, np.float64)
    return s / np.sqrt((s ** 2).mean(-1, keepdims=True) + eps) * gain
