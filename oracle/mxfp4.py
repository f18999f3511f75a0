"""MXFP4 and the router by scores in 64 bits (numpy): the oracle of the kernels, test infrastructure only."""
import numpy as np

MAGNITUDES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
VALUES = np.concatenate([MAGNITUDES, -MAGNITUDES])


def quantise(x, ceil=False, pad=32):
    """x (..., K) -> codes (..., KP / 2) and exponents (..., KP / 32), uint8."""
    x = np.asarray(x, np.float64)
    k = x.shape[-1]
    wide = np.zeros((*x.shape[:-1], -(-k // 32) * 32 if pad == 32 else (-(-k // 256) | 1) * 256))  # (for the products an odd multiple of 256)
    wide[..., :k] = x
    blocks = wide.reshape(*x.shape[:-1], -1, 32)
    largest = np.abs(blocks).max(-1)
    bad = ~np.isfinite(largest)
    safe = np.where(bad, 0, largest)
    mantissa, exponent = np.frexp(safe)  # safe = mantissa * 2^exponent, mantissa in [1/2, 1)
    power = np.where(safe == 0, -127, exponent - 3 + ((mantissa > 0.75) & ceil))
    power = np.clip(power, -127, 127)
    scaled = np.where(bad[..., None], 0, blocks) / np.exp2(power.astype(np.float64))[..., None]
    size = np.minimum(np.abs(scaled), 6.0)
    step = np.where(size < 2, 0.5, np.where(size < 4, 1.0, 2.0))
    value = np.round(size / step) * step  # (numpy rounds halves to even; even multiples of a step have even codes)
    code = np.searchsorted(MAGNITUDES, value).astype(np.uint8)
    code |= (np.signbit(scaled).astype(np.uint8) << 3)
    code = np.where(bad[..., None], 0, code).astype(np.uint8).reshape(*x.shape[:-1], -1)
    return code[..., 0::2] | (code[..., 1::2] << 4), np.where(bad, 255, power + 127).astype(np.uint8)


def values(codes, exponents):
    """What codes (..., K / 2) and exponents (..., K / 32) stand for."""
    codes, exponents = np.asarray(codes), np.asarray(exponents)
    nibbles = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    power = np.where(exponents == 255, np.nan, np.exp2(exponents.astype(np.float64) - 127))
    return VALUES[nibbles] * np.repeat(power, 32, -1)


def silu(x):
    return x / (1 + np.exp(-x))


def routes(logits, top_k, scoring="softmax", bias=None, groups=1, top_groups=None, group_best=2, renormalize=True, scale=1.0):
    """-> ids (M, top_k), weights (M, top_k) in 64 bits."""
    logits = np.clip(np.asarray(logits, np.float64), -np.finfo(np.float32).max, np.finfo(np.float32).max)
    known = ~np.isnan(logits)
    m, experts = logits.shape
    top_groups = groups if top_groups is None else top_groups
    with np.errstate(all="ignore"):
        if scoring == "sigmoid":
            score = 1 / (1 + np.exp(-logits))
        else:
            largest = np.where(known, logits, -np.inf).max(1, keepdims=True)
            score = np.exp(logits - largest)
            score = score / np.where(known, score, 0).sum(1, keepdims=True)
        choice = score + (0 if bias is None else np.asarray(bias, np.float64))
    is_open = known & (choice > -np.inf)
    ids, weights = np.zeros((m, top_k), np.int64), np.zeros((m, top_k))
    size = experts // groups
    for row in range(m):
        best = []
        for g in range(groups):
            mine = [choice[row, e] for e in range(g * size, (g + 1) * size) if is_open[row, e]]
            best.append(sum(sorted(mine, reverse=True)[:group_best]) if mine else -np.inf)
        kept = set(sorted(range(groups), key=lambda g: (-best[g], g))[:top_groups])
        candidates = [e for e in range(experts) if e // size in kept]
        candidates.sort(key=lambda e: (not is_open[row, e], -choice[row, e] if is_open[row, e] else 0, e))
        ids[row] = candidates[:top_k]
        s = np.array([score[row, e] if is_open[row, e] else 0.0 for e in ids[row]])
        total = s.sum() if renormalize else 1.0
        weights[row] = s / total * scale if total > 0 else 0
    return ids, weights
