"""8-bit floating point in blocks of 128 on the host: codes, scales and values in numpy."""
import numpy as np


def blocks(n):
    return -(-n // 128)


def e4m3_values():
    """The value of every code byte."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c & 128, -v, v)


def e4m3_codes(q):
    """Codes of f32 quotients of at most 448 (and NaN): nearest, ties to the even mantissa."""
    q = np.asarray(q, np.float64)
    a = np.abs(np.where(np.isnan(q), 0, q))
    e = np.clip(np.floor(np.log2(np.maximum(a, 2.0 ** -30))), -6, 8)
    steps = np.round(a / 2.0 ** (e - 3))           # half to even; 16 steps are 8 of the next exponent
    up = steps >= 16
    e, steps = np.where(up, e + 1, e), np.where(up, 8, steps)
    code = np.where(steps < 8, steps, (e + 7) * 8 + steps - 8).astype(np.uint8)
    code = np.where(np.isnan(q), 127, code)
    return (code | (np.signbit(q).astype(np.uint8) << 7)).astype(np.uint8)


def per_value(scales, block_rows, rows, cols):
    return np.repeat(np.repeat(scales, block_rows, 0)[:rows], 128, 1)[:, :cols]


def quantize(x, block_rows):
    """x f32 [rows, cols] -> codes u8 [rows, cols], scales f32."""
    rows, cols = x.shape
    pad = np.zeros((-(-rows // block_rows) * block_rows, blocks(cols) * 128), np.float32)
    pad[:rows, :cols] = np.where(np.isnan(x), 0, np.abs(x))
    most = pad.reshape(pad.shape[0] // block_rows, block_rows, blocks(cols), 128).max((1, 3))
    with np.errstate(all="ignore"):
        scales = np.where(most > 0, np.maximum(most / np.float32(448), np.float32(2.0 ** -126)), np.float32(1)).astype(np.float32)
        q = x / per_value(scales, block_rows, rows, cols)
    return e4m3_codes(q), scales


def values(codes, scales, block_rows):
    return e4m3_values()[codes] * per_value(scales.astype(np.float64), block_rows, *codes.shape)
