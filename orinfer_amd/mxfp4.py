"""Microscaled 4-bit floating point (MXFP4): weights and rows as tensors, and the layout that the products read.

A row is cut into blocks of 32 along K.  A block has one power of two, kept as a byte e for 2^(e - 127) (255: the whole block is NaN), and 32 codes of a
sign, two exponent and one mantissa bits (0, 0.5, 1, 1.5, 2, 3, 4, 6), two to a byte with the even element in the low half.  A matrix (N, K) is two uint8
tensors: codes (N, K / 2) and exponents (N, K / 32).
"""
import functools

import torch

from .lib import Kernel

BLOCK = 32   # elements to a power
STEP = 256   # K of a tile; the products take rows padded to an odd multiple of it
DTYPES = {torch.float16: "float16", torch.bfloat16: "bfloat16", torch.float32: "float32"}


def dtype_name(dtype):
    if dtype not in DTYPES:
        raise ValueError(f"dtype must be float16, bfloat16 or float32, not {dtype}")
    return DTYPES[dtype]


def padded(k, pad=STEP):
    """K as rows are stored: whole blocks (pad 32), or an odd multiple of 256 (pad 256: for the products; at even distances rows meet in few channels of the L2)."""
    if pad not in (BLOCK, STEP):
        raise ValueError("pad must be 32 or 256")
    return -(-k // BLOCK) * BLOCK if pad == BLOCK else (-(-k // STEP) | 1) * STEP


@functools.lru_cache(maxsize=256)
def _kernel(symbol, **variant):
    return Kernel(symbol, **variant)


def quantize(x, scale="floor", pad=BLOCK):
    """x (..., K) of fp16, bf16 or fp32 values on the GPU -> codes (..., KP / 2), exponents (..., KP / 32), KP = padded(K, pad), zeros behind K up to a
    multiple of 32 (pad 256: of 256; what lies behind that is not written and not read).
    scale: "floor" takes the power of two of a block's largest magnitude (what is above 6 of its units saturates), "ceil" the smallest that nothing saturates with.
    Blocks with an infinity or NaN become NaN."""
    if not x.is_cuda:
        raise ValueError("quantize takes a tensor on the GPU")
    k = x.shape[-1]
    if k == 0:
        raise ValueError("quantize needs at least one column")
    x = x.contiguous()
    rows = x.numel() // k
    lead = x.shape[:-1]
    codes = torch.empty((*lead, padded(k, pad) // 2), dtype=torch.uint8, device=x.device)
    exponents = torch.empty((*lead, padded(k, pad) // BLOCK), dtype=torch.uint8, device=x.device)
    if rows:
        with torch.cuda.device(x.device):
            _kernel("mxfp4_quantization", K=k, input_dtype=dtype_name(x.dtype), scale=scale, pad=pad)(Q=codes, S=exponents, X=x, rows=rows)
    return codes, exponents


def dequantize(codes, exponents, k, dtype=torch.float16, pad=BLOCK):
    """What codes and exponents stand for, (..., k) of `dtype` (exact in bf16 and fp32, infinite above their range, which bytes 253 and 254 reach; fp16 rounds what it cannot hold)."""
    if not codes.is_cuda or codes.device != exponents.device:
        raise ValueError("dequantize takes two tensors on one GPU")
    if (codes.dtype != torch.uint8 or exponents.dtype != torch.uint8 or codes.shape[-1] != padded(k, pad) // 2 or exponents.shape[-1] != padded(k, pad) // BLOCK
            or codes.shape[:-1] != exponents.shape[:-1]):
        raise ValueError(f"need uint8 codes (..., {padded(k, pad) // 2}) and exponents (..., {padded(k, pad) // BLOCK}) for K = {k}")
    codes, exponents = codes.contiguous(), exponents.contiguous()
    out = torch.empty((*codes.shape[:-1], k), dtype=dtype, device=codes.device)
    if out.numel():
        with torch.cuda.device(codes.device):
            _kernel("mxfp4_dequantization", K=k, output_dtype=dtype_name(dtype), pad=pad)(Q=codes, S=exponents, Y=out, rows=out.numel() // k)
    return out


def tiles(codes, exponents, paired=False):
    """Weights (..., N, K / 2), (..., N, K / 32) laid out for the products: 16 channels x 256 K are 2048 bytes of codes, [block][channel][16 bytes], and 128 bytes of
    exponents, [channel][block & 1][block >> 1]; tiles of the same channels lie along K behind one another.  N is padded to 16 and K to 256 with zeros.
    paired: the upper half of the N rows are the up channels of the gate channels in the lower half (SwiGLU); tiles of the two halves take turns."""
    codes, exponents = torch.as_tensor(codes), torch.as_tensor(exponents)
    *lead, n, half_k = codes.shape
    k = 2 * half_k
    if codes.dtype != torch.uint8 or exponents.dtype != torch.uint8:
        raise ValueError("codes and exponents are uint8")
    if n == 0 or k == 0 or k % BLOCK or tuple(exponents.shape) != (*lead, n, k // BLOCK):
        raise ValueError(f"codes (..., N, K / 2) of K = {k} and exponents {tuple(exponents.shape)} do not go together: K is a multiple of 32, exponents (..., N, K / 32)")
    if paired and n % 2:
        raise ValueError("paired weights have as many up channels as gate channels")

    def rows(t):
        if paired:
            t = t.unflatten(-2, (2, n // 2))
        t = torch.nn.functional.pad(t, (0, 0, 0, -t.shape[-2] % 16))
        t = t.unflatten(-2, (-1, 16))
        return t.transpose(-4, -3).flatten(-4, -3) if paired else t  # (..., tiles, 16, columns)

    steps = -(-k // STEP)
    codes = torch.nn.functional.pad(rows(codes), (0, 128 * steps - half_k)).unflatten(-1, (steps, 8, 16))          # (..., tiles, 16, steps, 8, 16)
    exponents = torch.nn.functional.pad(rows(exponents), (0, 8 * steps - k // BLOCK)).unflatten(-1, (steps, 4, 2))  # (..., tiles, 16, steps, 4, 2)
    codes = codes.movedim(-4, -2).contiguous()                               # (..., tiles, steps, 8, 16, 16)
    exponents = exponents.movedim(-4, -3).transpose(-1, -2).contiguous()     # (..., tiles, steps, 16, 2, 4)
    return codes, exponents
