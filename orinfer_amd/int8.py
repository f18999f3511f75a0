"""Rows and weights in 8-bit integers with an fp32 scale, and if wanted a zero point, for each row.

A row has s = max |x| / 127 and codes q = x / s; with zero points s = (high - low) / 255 over low = min(x, 0) and high = max(x, 0), z = round(-low / s) - 128 and codes round(x / s) + z within
[-128, 127].  q stands for (q - z) s.  Quotients round to the nearest whole number, ties to the even one; a scale is at least 2^-100.  A row with an infinity or NaN, or whose range leaves fp32,
has the scale NaN and codes 0.
"""
import functools

import torch

from .lib import Kernel

STEP = 128   # K of a step of the products, which take K padded to pairs of steps
MOST_K = 65536  # that a product adds exactly
DTYPES = {torch.float16: "float16", torch.bfloat16: "bfloat16", torch.float32: "float32"}


def dtype_name(dtype):
    if dtype not in DTYPES:
        raise ValueError(f"dtype must be float16, bfloat16 or float32, not {dtype}")
    return DTYPES[dtype]


def padded(k):
    """Bytes from one stored row to the next: an odd multiple of 128 (at even distances rows meet in few channels of the L2)."""
    return (steps(k) | 1) * STEP


def steps(k):
    """Steps that the products take of K."""
    return -(-k // (2 * STEP)) * 2


@functools.lru_cache(maxsize=256)
def _kernel(symbol, **variant):
    return Kernel(symbol, **variant)


def quantize(x, zero_points=False):
    """x (..., K) of fp16, bf16 or fp32 values on the GPU -> codes (..., K) int8, scales (...) fp32 and, with zero points, those (...) int32.
    The codes are a view of rows that lie padded(K) apart.  Weights (N, K) quantise alike, a scale to a channel."""
    if not x.is_cuda:
        raise ValueError("quantize takes a tensor on the GPU")
    k = x.shape[-1] if x.ndim else 0
    if k == 0:
        raise ValueError("quantize needs at least one column")
    x = x.contiguous()
    lead, rows = x.shape[:-1], x.numel() // k
    codes = torch.empty((*lead, padded(k)), dtype=torch.int8, device=x.device)
    scales = torch.empty(lead, dtype=torch.float32, device=x.device)
    zeros = torch.empty(lead, dtype=torch.int32, device=x.device) if zero_points else None
    if rows:
        with torch.cuda.device(x.device):
            # (a launch takes 2^24 rows)
            most, kernel = 1 << 24, _kernel("int8_token_quantization", K=k, input_dtype=dtype_name(x.dtype), zero_points=bool(zero_points))
            flat, q, s = x.view(rows, k), codes.view(rows, -1), scales.view(rows)
            for first in range(0, rows, most):
                part = slice(first, min(first + most, rows))
                kernel(Q=q[part], S=s[part], X=flat[part], rows=part.stop - first, **({"Z": zeros.view(rows)[part]} if zero_points else {}))
    else:
        dtype_name(x.dtype)
    return (codes[..., :k], scales, zeros) if zero_points else (codes[..., :k], scales)
