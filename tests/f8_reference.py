"""8-bit matrices in numpy, from their definition: e4m3's 256 values, the conversion with block
scales (bit for bit), the norm and the block-scaled product in 64 bits."""
from __future__ import annotations

import numpy as np

BLOCK = 128
EPS32 = 2.0 ** -24   # half a step of fp32, relative


def _values():
    out = np.empty(256)
    for code in range(256):
        exponent, mantissa = (code >> 3) & 15, code & 7
        v = (8 + mantissa) * 2.0 ** (exponent - 10) if exponent else mantissa * 2.0 ** -9
        out[code] = np.nan if code & 0x7F == 0x7F else v
        if code & 0x80:
            out[code] = -out[code]
    return out


VALUES = _values()                                    # by code
_FINITE = VALUES[:0x7F]                               # 0 .. 448, rising
_MIDDLE = (_FINITE[1:] + _FINITE[:-1]) / 2


def encode(x) -> np.ndarray:
    """The e4m3 codes nearest to x (|x| below 464), ties to the even code; NaN gives 0x7F."""
    x = np.asarray(x, dtype=np.float64)
    a = np.abs(np.where(np.isnan(x), 0.0, x))
    assert np.all(a < 464.0)
    up = np.searchsorted(_MIDDLE, a, side="left")     # the number of midpoints below a
    tie = (up < len(_MIDDLE)) & (_MIDDLE[np.minimum(up, len(_MIDDLE) - 1)] == a)
    code = np.where(tie, up + (up & 1), up)           # a lies on the midpoint of up and up + 1
    code = code | np.where(np.signbit(x), 0x80, 0)
    return np.where(np.isnan(x), 0x7F, code).astype(np.uint8)


def blocks(n: int) -> int:
    return -(-n // BLOCK)


def quantize(x: np.ndarray, block_rows: int = 1):
    """(codes, scales) of a float32 matrix: s = max(top / 448, 2^-126), the scale fl(s), the codes
    nearest to x / s (448 x and top are exact in 64 bits, and their quotient is never rounded across
    a border between codes). Blocks with a NaN or an infinity are NaN throughout, or hold NaN and
    zeros under an infinite scale."""
    x = np.asarray(x, dtype=np.float32)
    rows, cols = x.shape
    mb, nb = -(-rows // block_rows), blocks(cols)
    scales = np.empty((mb, nb), np.float32)
    codes = np.empty((rows, cols), np.uint8)
    with np.errstate(all="ignore"):
        for j in range(nb):
            part = x[:, j * BLOCK:(j + 1) * BLOCK]
            top = np.abs(part).max(axis=1) if cols else np.zeros(rows, np.float32)
            top = np.array([np.max(top[i * block_rows:(i + 1) * block_rows]) for i in range(mb)],
                           np.float32)
            s = (top / np.float32(448)).astype(np.float32)
            s = np.where(s < np.float32(2.0 ** -126), np.float32(2.0 ** -126), s)
            scales[:, j] = s
            tops = np.repeat(top.astype(np.float64), block_rows)[:rows, None]
            wide = part.astype(np.float64)
            codes[:, j * BLOCK:(j + 1) * BLOCK] = encode(
                np.where(tops < 448 * 2.0 ** -126, wide * 2.0 ** 126, wide * 448 / tops))
    return codes, scales


def quantize_exact(y: np.ndarray):
    """(codes, sure, scales) of a float64 matrix with a scale per row and 128 columns: the codes
    nearest to y / s, where that is no closer to a border between two codes than 2^-40 of it
    (elsewhere either may come), and s."""
    y = np.asarray(y, dtype=np.float64)
    rows, cols = y.shape
    codes, sure = np.empty((rows, cols), np.uint8), np.empty((rows, cols), bool)
    scales = np.empty((rows, blocks(cols)))
    with np.errstate(all="ignore"):
        for j in range(blocks(cols)):
            part = y[:, j * BLOCK:(j + 1) * BLOCK]
            s = np.abs(part).max(axis=1) / 448
            s = np.where(s < 2.0 ** -126, 2.0 ** -126, s)
            scales[:, j] = s
            v = part / s[:, None]
            at = slice(j * BLOCK, (j + 1) * BLOCK)
            codes[:, at] = encode(v)
            a = np.minimum(np.abs(np.where(np.isnan(v), 0.0, v)), 448.0)
            i = np.minimum(np.searchsorted(_MIDDLE, a), len(_MIDDLE) - 1)
            away = np.minimum(np.abs(_MIDDLE[i] - a), np.abs(_MIDDLE[np.maximum(i - 1, 0)] - a))
            sure[:, at] = away > 2.0 ** -40 * a
    return codes, sure, scales


def dequantize(codes: np.ndarray, scales: np.ndarray, block_rows: int = 1) -> np.ndarray:
    """What the codes stand for, in 64 bits (exact)."""
    rows, cols = codes.shape
    s = np.repeat(scales.astype(np.float64), block_rows, axis=0)[:rows]
    return VALUES[codes] * np.repeat(s, BLOCK, axis=1)[:, :cols]


def rms_norm(t: np.ndarray, weight=None, eps: float = 1e-6) -> np.ndarray:
    """In 64 bits, eps as the fp32 number that the call gets."""
    t = np.asarray(t, dtype=np.float64)
    with np.errstate(all="ignore"):
        y = t / np.sqrt((t * t).mean(axis=-1, keepdims=True) + float(np.float32(eps)))
        return y if weight is None else y * np.asarray(weight, dtype=np.float64)


def product(a, a_scales, b, b_scales):
    """(a b^T, sum of |a b|) in 64 bits from codes and scales."""
    x, y = dequantize(a, a_scales, 1), dequantize(b, b_scales, BLOCK)
    return x @ y.T, np.abs(x) @ np.abs(y).T


def product_bound(magnitude: np.ndarray, k: int) -> np.ndarray:
    """How far a product may be from the exact one: the 128 products of a block are exact and
    summed in fp32 (at most 128 roundings, each at most 2^-24 of the sum of magnitudes), the two
    scales' product rounds once, and each block's multiply-add once."""
    return (BLOCK + 2 + blocks(k)) * EPS32 * magnitude


def silu(x: np.ndarray) -> np.ndarray:
    x = np.asarray(x, dtype=np.float64)
    with np.errstate(over="ignore"):
        return x / (1 + np.exp(-x))
