"""Microscaled 4-bit floating point rows in float64 numpy: quantisation, packing and the values that packed rows stand for
(the layout of include/h3_c.h, H3K_FP4_MX and H3K_FP4_NV) -- TEST INFRASTRUCTURE ONLY."""
import numpy as np

MX, NV = 0, 1
BLOCK = {MX: 32, NV: 16}
VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)


def e4m3_values():
    """The 127 nonnegative e4m3 numbers by code (0x7f is a NaN)."""
    b = np.arange(127)
    return np.where(b < 8, b / 8 * 2.0 ** -6, (1 + (b & 7) / 8) * 2.0 ** ((b >> 3) - 7.0))


def nearest(x, values):
    """Index of the nearest of ascending `values` to each x >= 0, ties to the even index, the last one past the end."""
    hi = np.clip(np.searchsorted(values, x), 1, len(values) - 1)
    lo = hi - 1
    below, above = x - values[lo], values[hi] - x
    return np.where((above < below) | ((above == below) & (hi % 2 == 0)), hi, lo)


def exponent(x):
    """floor(log2 x); -1000 for 0."""
    m, e = np.frexp(x)
    return np.where(x > 0, e - 1, -1000)


def quantise(x, f):
    """x [rows][K] -> (codes, scale bytes [rows][blocks], row scale [rows], quotients before rounding)."""
    x = np.asarray(x, np.float64)
    rows, K = x.shape
    b = x.reshape(rows, K // BLOCK[f], BLOCK[f])
    fine = np.isfinite(b)
    most = np.where(fine, np.abs(b), 0).max(2)
    row = np.ones(rows)
    if f == MX:
        e = np.maximum(exponent(most) - 2, -127)
        bad = ~fine.all(2)
        bytes_ = np.where(bad, 255, e + 127)
        unit = 2.0 ** e
        bad = np.broadcast_to(bad[..., None], b.shape)
    else:
        g = 2.0 ** np.maximum(exponent(most.max(1, initial=0)) - 10, -126)
        bad_row = ~fine.all((1, 2))
        row = np.where(bad_row, np.nan, g)
        v = e4m3_values()
        bytes_ = nearest(most / g[:, None] / 6, v)
        unit = v[bytes_] * g[:, None]
        bytes_ = np.where(bad_row[:, None], 0, bytes_)
        bad = np.broadcast_to(bad_row[:, None, None], b.shape)
    q = np.where((unit[..., None] > 0) & ~bad, np.where(fine, b, 0) / np.where(unit > 0, unit, 1)[..., None], 0)
    codes = nearest(np.abs(q), VALUES)
    codes = codes + 8 * (np.signbit(q) & (codes > 0))
    return codes.reshape(rows, K).astype(np.uint8), bytes_.astype(np.uint8), row, q.reshape(rows, K)


def pack(codes, bytes_):
    """(packed codes [rows][K / 2], scale tiles as one byte array)."""
    rows, n = bytes_.shape
    full = np.zeros((-(-rows // 128) * 128, -(-n // 4) * 4), np.uint8)
    full[:rows, :n] = bytes_
    tiles = full.reshape(-1, 4, 32, full.shape[1] // 4, 4).transpose(0, 3, 2, 1, 4)
    return codes[:, 0::2] | (codes[:, 1::2] << 4), np.ascontiguousarray(tiles).reshape(-1)


def unpack(packed, tiles, f):
    packed = np.asarray(packed, np.uint8)
    rows, K = packed.shape[0], packed.shape[1] * 2
    codes = np.stack([packed & 15, packed >> 4], 2).reshape(rows, K)
    n = K // BLOCK[f]
    kt = -(-n // 4)
    bytes_ = np.asarray(tiles, np.uint8).reshape(-1, kt, 32, 4, 4).transpose(0, 3, 2, 1, 4).reshape(-1, kt * 4)
    return codes, bytes_[:rows, :n]


def values(codes, bytes_, row, f):
    """The numbers that codes [rows][K] and scale bytes stand for (float64)."""
    v = VALUES[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    b = bytes_.astype(np.int64)
    if f == MX:
        unit = np.where(b == 255, np.nan, 2.0 ** (b - 127.0))
    else:
        unit = np.where(b == 127, np.nan, e4m3_values()[np.minimum(b, 126)])
    return v * np.repeat(unit, BLOCK[f], 1) * (np.ones(len(codes)) if row is None else np.asarray(row, np.float64))[:, None]
