"""Q4_0 in plain numpy, for the tests of the 4-bit caches: the quantizer's fp32
operations one by one, and the values that a block stands for in 64 bits."""
import numpy as np

BYTES = 18  # of a block of 32: fp16 d, then 16 bytes, byte j the levels of elements j (low) and j + 16 (high)


def quantize(x: np.ndarray) -> np.ndarray:
    """F32 (..., n) -> bytes (..., n / 32 * 18)."""
    x = np.ascontiguousarray(x, np.float32)
    b = x.reshape(-1, 32)
    mag = b.view(np.uint32) & np.uint32(0x7FFFFFFF)  # ordered as the magnitudes, NaN last
    m = b[np.arange(len(b)), mag.argmax(1)]          # the first of equal ones
    with np.errstate(all="ignore"):
        d = m * np.float32(-0.125)
        inv = np.where(d != 0, np.float32(1) / d, np.float32(0)).astype(np.float32)
        v = (b * inv[:, None]).astype(np.float32) + np.float32(8.5)
        q = np.floor(np.where(np.isnan(v), 0, np.clip(v, 0, 15))).astype(np.uint8)
        out = np.empty((len(b), BYTES), np.uint8)
        out[:, :2] = d.astype(np.float16).view(np.uint8).reshape(-1, 2)
    out[:, 2:] = q[:, :16] | q[:, 16:] << 4
    return out.reshape(*x.shape[:-1], -1)


def dequantize(c: np.ndarray) -> np.ndarray:
    """bytes (..., blocks * 18) -> float64 (..., blocks * 32)."""
    b = np.ascontiguousarray(c).reshape(-1, BYTES)
    d = b[:, :2].copy().view(np.float16).astype(np.float64)
    q = np.concatenate([b[:, 2:] & 15, b[:, 2:] >> 4], 1).astype(np.float64) - 8
    with np.errstate(invalid="ignore"):
        v = q * d
    return v.reshape(*c.shape[:-1], -1)
