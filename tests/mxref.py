"""The block-scaled formats in 64 bits, from their definition (include/lyth_b200.h): numpy, element by
element, sharing nothing with the library. x is float64 (exact widenings of the stored values)."""
import numpy as np

FP8, FP4, NVFP4 = 0, 1, 2
BLOCK = {FP8: 32, FP4: 32, NVFP4: 16}
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
E4M3 = np.array([(i % 8) * 2.0 ** -9 if i < 8 else (1 + (i % 8) / 8) * 2.0 ** (i // 8 - 7) for i in range(127)], np.float64)


def padded(fmt, cols):
    w = 4 * BLOCK[fmt]
    return -(-cols // w) * w


def nearest(levels, v):
    """Index of the level nearest to v >= 0, ties to the even index, beyond the last: the last."""
    hi = np.clip(np.searchsorted(levels, v), 1, len(levels) - 1)
    up, down = levels[hi] - v, v - levels[hi - 1]
    return np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)


def quantize(fmt, x, g=1.0):
    """(codes as integers rows x k, scale bytes rows x blocks)."""
    rows, cols = x.shape
    k, b = padded(fmt, cols), BLOCK[fmt]
    w = np.zeros((rows, k))
    w[:, :cols] = x
    w = w.reshape(rows, k // b, b)
    bad = ~np.isfinite(w).all(2)
    w = np.where(bad[:, :, None], 0.0, w)
    top = np.abs(w).max(2)
    if fmt == NVFP4:
        byte = nearest(E4M3, top / (6 * g))
        scale = E4M3[byte] * g
    else:
        e = np.frexp(top)[1] - 1  # floor(log2 top) for top > 0
        byte = np.where(top > 0, np.maximum(e + 127 - (8 if fmt == FP8 else 2), 0), 0)
        scale = np.ldexp(1.0, byte - 127)
    levels = E4M3 if fmt == FP8 else E2M1
    safe = np.where(scale > 0, scale, 1.0)[:, :, None]
    ratio = np.where(scale[:, :, None] > 0, np.abs(w) / safe, 0.0)
    codes = nearest(levels, ratio) | np.where(np.signbit(w), 0x80 if fmt == FP8 else 8, 0)
    codes = np.where(bad[:, :, None], 0, codes).reshape(rows, k)
    return codes, np.where(bad, 0x7F if fmt == NVFP4 else 0xFF, byte)


def pack(fmt, codes):
    if fmt == FP8:
        return codes.astype(np.uint8)
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def unpack(fmt, packed):
    if fmt == FP8:
        return packed.astype(np.int64)
    out = np.empty((packed.shape[0], packed.shape[1] * 2), np.int64)
    out[:, 0::2] = packed & 15
    out[:, 1::2] = packed >> 4
    return out


def scale_at(rows, blocks):
    """Where the scale of row r, block b lies: rows x blocks byte offsets."""
    r, b = np.arange(rows)[:, None], np.arange(blocks)[None, :]
    return ((r // 128) * (blocks // 4) + b // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4


def tile(scales, fill=0):
    rows, blocks = scales.shape
    out = np.full(-(-rows // 128) * (blocks // 4) * 512, fill, np.uint8)
    out[scale_at(rows, blocks)] = scales
    return out


def values(fmt, codes, scales, g=1.0):
    """float64 rows x k of integer codes and scale bytes."""
    rows, k = codes.shape
    if fmt == FP8:
        mag = np.append(E4M3, np.nan)[codes & 127]
        sign = np.where(codes >= 128, -1.0, 1.0)
    else:
        mag, sign = E2M1[codes & 7], np.where(codes >= 8, -1.0, 1.0)
    if fmt == NVFP4:
        s = np.append(E4M3, np.nan)[scales & 127]
    else:
        s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return sign * mag * np.repeat(s, BLOCK[fmt], axis=1) * g


def random_operand(fmt, rows, cols, rng, spread=6):
    """Codes and scales as a quantised normal matrix has them: (packed, tiled, float64 values of
    rows x k); zero behind cols; the scale bytes of rows behind the last hold NaN scales."""
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-spread, spread + 1, (rows, 1)).astype(np.float64))
    codes, scales = quantize(fmt, x.astype(np.float32).astype(np.float64), 1.0)
    return pack(fmt, codes), tile(scales, 0x7F if fmt == NVFP4 else 0xFF), values(fmt, codes, scales)
