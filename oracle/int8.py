"""8-bit integer rows and weights with a scale for each row and channel in 64 bits (numpy): the oracle of the kernels, test infrastructure only."""
import numpy as np

SMALLEST = 2.0**-100


def quantise(x, zero_points=False):
    """x (rows, K) -> codes (rows, K), scales (rows) and zero points (rows).  A scale is a number of 32 bits, so it is made in 32 bits: the span and its part are one rounding each."""
    x = np.asarray(x, np.float64)
    with np.errstate(all="ignore"):
        bad = ~np.isfinite(x).all(1)
        safe = np.where(bad[:, None], 0, x)
        if zero_points:
            high, low = np.maximum(safe.max(1), 0), np.minimum(safe.min(1), 0)
            span = (high.astype(np.float32) - low.astype(np.float32)).astype(np.float64)
        else:
            low, span = np.zeros(len(x)), np.abs(safe).max(1)
        bad |= np.isinf(span)
        scale = np.maximum((np.where(bad, 0, span).astype(np.float32) / np.float32(255 if zero_points else 127)), np.float32(SMALLEST)).astype(np.float64)
        # (a quotient of two numbers of 24 bits that is not halfway between whole numbers differs from there by more than 2^-33 of itself: 64 bits tell)
        whole = np.round(safe / scale[:, None])
        zero = np.where(bad, 0, -128 - np.round(low / scale)) if zero_points else np.zeros(len(x))
        codes = np.clip(whole + zero[:, None], -128 if zero_points else -127, 127)
    codes = np.where(bad[:, None], 0, codes)
    return codes.astype(np.int8), np.where(bad, np.nan, scale), zero.astype(np.int32)


def values(codes, scales, zeros=0):
    return (codes.astype(np.float64) - np.reshape(zeros, (-1, 1))) * np.reshape(scales, (-1, 1))


def silu(x):
    return x / (1 + np.exp(-x))
