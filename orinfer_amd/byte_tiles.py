"""The layout of weights that are multiplied as they are stored, 8-bit integers or 16-bit values: tiles of 16 channels x 128 bytes of K."""
import torch

STEP = 128  # bytes of K of a tile
PAIR = 256  # K is padded to


def _by_16(t, axis, paired):
    """Axis `axis` (negative) of N channels as (tiles, 16), padded with zeros to four tiles; paired: tiles of the lower and of the upper half of the channels take turns."""
    n = t.shape[axis]
    if paired:
        t = t.unflatten(axis, (2, n // 2))
    pad = [0] * (2 * (-axis - 1)) + [0, -t.shape[axis] % (32 if paired else 64)]
    t = torch.nn.functional.pad(t, pad).unflatten(axis, (-1, 16))
    return t.transpose(axis - 2, axis - 1).flatten(axis - 2, axis - 1) if paired else t


def _check_paired(n, paired):
    if paired and n % 2:
        raise ValueError("paired weights have as many up channels as gate channels")


def tiles(weight, paired=False):
    """Weights (..., N, K) of int8, fp16 or bf16 laid out for the products, uint8: 16 channels x 128 bytes of K are 2048 bytes, [piece of 16 bytes][channel][16]; the tiles of the same K
    lie behind one another.  N is padded to 64 and K to 256 bytes with zeros.
    paired: the upper half of the N rows are the up channels of the gate channels in the lower half (SwiGLU); tiles of the two halves take turns."""
    weight = torch.as_tensor(weight)
    if weight.ndim < 2 or weight.dtype not in (torch.int8, torch.float16, torch.bfloat16):
        raise ValueError(f"weights are int8, float16 or bfloat16 (..., N, K), not {weight.dtype} {tuple(weight.shape)}")
    n, k = weight.shape[-2:]
    if n == 0 or k == 0:
        raise ValueError("weights have at least one channel and one column")
    _check_paired(n, paired)
    width = k * weight.element_size()
    rows = _by_16(weight.contiguous().view(torch.uint8), -2, paired)  # (..., tiles, 16, bytes)
    steps = -(-width // PAIR) * (PAIR // STEP)
    rows = torch.nn.functional.pad(rows, (0, STEP * steps - width)).unflatten(-1, (steps, 8, 16))  # (..., tiles, 16, steps, 8, 16)
    return rows.movedim((-3, -5, -2, -4), (-5, -4, -3, -2)).contiguous()                          # (..., steps, tiles, 8, 16, 16)


def channels(values, paired=False):
    """What the channels have, (..., N), in the order of the tiles, (..., tiles, 16), padded with zeros."""
    values = torch.as_tensor(values).detach()
    _check_paired(values.shape[-1], paired)
    return _by_16(values, -1, paired).contiguous()
