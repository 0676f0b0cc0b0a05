"""The 8-bit floating point product in 64 bits, from the format's definition (numpy only)."""
import numpy as np

BLOCK, MOST, TINY = 128, 448.0, 2.0 ** -100


def _table():
    codes = np.arange(256)
    sign, exponent, mantissa = np.where(codes & 0x80, -1.0, 1.0), (codes >> 3) & 15, codes & 7
    value = np.where(exponent == 0, mantissa * 2.0 ** -9, (8 + mantissa) * 2.0 ** (exponent - 10.0))
    value[(codes & 0x7F) == 0x7F] = np.nan
    return sign * value


VALUES = _table()


def encode(x):
    """Nearest code of f32 values within [-448, 448], ties to the even code; a NaN is one."""
    x = np.asarray(x, np.float32).astype(np.float64)
    size = np.minimum(np.abs(np.where(np.isnan(x), 0.0, x)), MOST)
    step = 2.0 ** np.maximum(np.floor(np.log2(np.maximum(size, 2.0 ** -30))) - 3, -9.0)
    rounded = np.rint(size / step) * step  # numpy rounds halves to even
    code = np.searchsorted(VALUES[:127], rounded).astype(np.uint8)
    assert np.array_equal(VALUES[code], rounded)
    code = np.where(np.signbit(x), code | 0x80, code).astype(np.uint8)
    return np.where(np.isnan(x), np.where(np.signbit(x), 0xFF, 0x7F), code).astype(np.uint8)


def quantize(x):
    """Codes and scales of f32 [rows, in_dim], with the definition's f32 operations."""
    x = np.asarray(x, np.float32)
    rows, dim = x.shape
    blocks = -(-dim // BLOCK)
    padded = np.zeros((rows, blocks * BLOCK), np.float32)
    padded[:, :dim] = x
    padded = padded.reshape(rows, blocks, BLOCK)
    with np.errstate(all="ignore"):
        most = np.fmax(np.fmax.reduce(np.abs(padded), axis=2), np.float32(TINY)).astype(np.float32)
        by, scale = (np.float32(MOST) / most).astype(np.float32), (most / np.float32(MOST)).astype(np.float32)
        codes = encode((padded * by[:, :, None]).astype(np.float32))
    return codes.reshape(rows, -1)[:, :dim].copy(), scale


def weights(rng, out_dim, in_dim):
    """Codes spread over the type and scales over three decades."""
    codes = rng.integers(0, 256, (out_dim, in_dim)).astype(np.uint8)
    codes[(codes & 0x7F) == 0x7F] = 0x3C
    scales = np.exp(rng.uniform(np.log(1e-4), np.log(1e-1), (-(-out_dim // BLOCK), -(-in_dim // BLOCK)))).astype(np.float32)
    return codes, scales


def dense(codes, scales, rows_a_scale):
    wide = np.repeat(np.repeat(scales.astype(np.float64), rows_a_scale, 0)[:codes.shape[0]], BLOCK, 1)[:, :codes.shape[1]]
    return VALUES[codes] * wide


def matmul(codes, scales, w_codes, w_scales):
    """(Y, the largest error that f32 sums may have): the matrix cores add a block's products in some order, the blocks' sums
    follow in another: every one of at most 128 + blocks additions is off by 2^-23 (half of that when it rounds, all of it
    when it cuts) of the sum of the absolute products, three more roundings by the scales."""
    x, w = dense(codes, scales, 1), dense(w_codes, w_scales, BLOCK)
    steps = BLOCK + -(-codes.shape[1] // BLOCK) + 4
    return x @ w.T, steps * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T)


def activate(y, kind):
    if kind == 1:
        return np.where(y < 0, 0.0, y)
    if kind == 2:
        return y / (1.0 + np.exp(-1.702 * y))
    if kind == 3:
        return 0.5 * y * (1.0 + np.tanh(0.7978845608028654 * (y + 0.044715 * y ** 3)))
    return y
