"""Head norms with rotation, the paged 8-bit cache and attention over it, from their definitions in 64 bits (NumPy, loops)."""
from __future__ import annotations

import numpy as np

TINY = 2.0 ** -64


def e4m3_values() -> np.ndarray:
    """What the 256 codes stand for (NaN for 0x7f and 0xff)."""
    codes = np.arange(256)
    exponent, fraction = (codes >> 3) & 15, codes & 7
    size = np.where(exponent == 0, fraction * 2.0 ** -9, (1 + fraction / 8.0) * 2.0 ** (exponent - 7.0))
    size[codes & 127 == 127] = np.nan
    return np.where(codes & 128, -size, size)


def e4m3(x: np.ndarray) -> np.ndarray:
    """Nearest value, ties to even, the largest for what is beyond it."""
    size = np.maximum(np.abs(x), 2.0 ** -6)
    step = 2.0 ** (np.floor(np.log2(np.where(np.isfinite(size), size, 1.0))) - 3)
    return np.clip(np.where(np.isinf(x), x, np.round(x / step) * step), -448.0, 448.0)


def head_norm_rotary(x, weight, normalize, positions, frequencies, interleaved=False, epsilon=1e-6):
    """x [rows, heads, D] -> float64."""
    y = x.astype(np.float64)
    if normalize:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + epsilon)
    if weight is not None:
        y = y * weight.astype(np.float64)
    if frequencies is None:
        return y
    half = len(frequencies)
    first = np.arange(0, 2 * half, 2) if interleaved else np.arange(half)
    second = first + 1 if interleaved else first + half
    angle = positions.astype(np.float64)[:, None] * frequencies.astype(np.float64)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    out = y.copy()
    out[..., first] = y[..., first] * c - y[..., second] * s
    out[..., second] = y[..., second] * c + y[..., first] * s
    return out


def append(codes, scales, x, row_offsets, lengths, table):
    """x [rows, heads, D] into the pages; codes as values [pages, heads, P, D].  Returns (codes, scales, touched), `touched` 2 for
    slots of new tokens, 1 for codes that were rounded again."""
    codes, scales = codes.astype(np.float64).copy(), scales.astype(np.float64).copy()
    touched = np.zeros(codes.shape[:3], dtype=np.int8)
    page_tokens = codes.shape[2]
    for s, length in enumerate(lengths):
        at, end = max(0, length - (row_offsets[s + 1] - row_offsets[s])), length
        row = row_offsets[s + 1] - (end - at)
        while at < end:
            page, slot = table[s][at // page_tokens], at % page_tokens
            many = min(page_tokens - slot, end - at)
            part = x[row:row + many].transpose(1, 0, 2)
            size = np.where(np.isfinite(part), np.abs(part), 0.0).max(axis=(1, 2))
            with np.errstate(divide="ignore"):
                needed = np.maximum(2.0 ** np.ceil(np.log2(size / 448.0)), TINY)
            for h in range(codes.shape[1]):
                new = max(needed[h], scales[page, h]) if slot else needed[h]
                if slot and new > scales[page, h]:
                    codes[page, h, :slot] = e4m3(codes[page, h, :slot] * (scales[page, h] / new))
                    touched[page, h, :slot] = 1
                codes[page, h, slot:slot + many] = part[h] / new        # not rounded: the caller counts the rounding
                touched[page, h, slot:slot + many] = 2
                scales[page, h] = new
            row, at = row + many, at + many
    return codes, scales, touched


def attention(q, k, v, scale, first_position, window=0):
    """q [n, heads, D] at positions first_position ..; k, v [kv heads, tokens, D].  Returns (output, sum p |v|), 0 for rows that see nothing."""
    n, heads, _ = q.shape
    group = heads // k.shape[0]
    out, size = np.zeros(q.shape), np.zeros(q.shape)
    for i in range(n):
        position = first_position + i
        begin = max(0, position - window + 1) if window else 0
        end = min(position + 1, k.shape[1])
        if end <= begin:
            continue
        for h in range(heads):
            keys, values = k[h // group, begin:end], v[h // group, begin:end]
            scores = keys @ q[i, h].astype(np.float64) * scale
            p = np.exp(scores - scores.max())
            p /= p.sum()
            out[i, h], size[i, h] = p @ values, p @ np.abs(values)
    return out, size
