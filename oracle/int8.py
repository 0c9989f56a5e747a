"""The int8 cache with a scale for every (block, KV head), restated in numpy. TEST INFRASTRUCTURE ONLY.

The reference plans a quantised KV cache (liteinfer docs/roadmap.md, section
2.5) and has no code for it. Written from the format's definition, one block
and one head at a time, in the float dtype asked for (float32 gives the very
codes and scales that a store holds, float64 the values without their
intermediate roundings):

    old   = 0 if the block's first slot is written, else its scale
    new   = max(old, largest magnitude of the rows / 127, 2^-126)
    rows  -> clip(rint(x * (1 / new)), -127, 127)
    other rows of the block -> rint(code * (old * (1 / new))), if new > old

and a value that is not finite (or a scale that is NaN already) makes the
scale NaN and the rows' codes 0.
"""

from __future__ import annotations

import numpy as np

LEAST = 2.0 ** -126


def append(codes: np.ndarray, scales: np.ndarray, slots: np.ndarray, rows: np.ndarray, dtype=np.float32):
    """(codes, scales) after rows [tokens, heads, dim] went to `slots`; slots outside the store are skipped.

    codes [num_slots, heads, dim] (int8 values), scales [num_blocks, heads].
    """
    codes, scales = codes.copy(), scales.astype(dtype)
    block = codes.shape[0] // scales.shape[0]
    by_block: dict[int, dict[int, int]] = {}
    for t, slot in enumerate(np.asarray(slots).reshape(-1).tolist()):
        if 0 <= slot < codes.shape[0]:
            by_block.setdefault(slot // block, {})[slot % block] = t  # a later token replaces an earlier one
    for b, tokens in by_block.items():
        for h in range(codes.shape[1]):
            old = dtype(0) if 0 in tokens else scales[b, h]
            largest = dtype(max(np.abs(rows[t, h].astype(dtype)).max() for t in tokens.values()))
            if any(not np.isfinite(rows[t, h]).all() for t in tokens.values()) or np.isnan(old):
                scales[b, h] = np.nan
                for o in tokens:
                    codes[b * block + o, h] = 0
                continue
            step = largest * dtype(1.0 / 127.0) if dtype is np.float32 else largest / 127
            new = max(old, step, dtype(LEAST))
            inv = dtype(1) / new
            if new > old:
                for o in range(block):
                    if o not in tokens:
                        codes[b * block + o, h] = np.rint(codes[b * block + o, h].astype(dtype) * (old * inv))
            for o, t in tokens.items():
                codes[b * block + o, h] = np.clip(np.rint(rows[t, h].astype(dtype) * inv), -127, 127)
            scales[b, h] = new
    return codes, scales


def dequantize(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """float64 values a store stands for, [num_slots, heads, dim]."""
    block = codes.shape[0] // scales.shape[0]
    return codes.astype(np.float64) * np.repeat(scales.astype(np.float64), block, axis=0)[..., None]


def rotate(x: np.ndarray, cos: np.ndarray, sin: np.ndarray, dtype=np.float32) -> np.ndarray:
    """x [..., tokens, heads, dim] rotated by tables [..., tokens, dim], every operation in `dtype`."""
    half = x.shape[-1] // 2
    x, cos, sin = x.astype(dtype), cos.astype(dtype)[..., None, :], sin.astype(dtype)[..., None, :]
    lo, hi = x[..., :half], x[..., half:]
    return np.concatenate((lo * cos[..., :half] - hi * sin[..., :half],
                           hi * cos[..., half:] + lo * sin[..., half:]), axis=-1)


def quantize_rows(x: np.ndarray, dtype=np.float32):
    """(codes int8 [..., k], scales [...]) of rows: scale = max(largest / 127, 2^-126), code = rint(x * (1 / scale))."""
    x = x.astype(dtype)
    largest = np.abs(x).max(axis=-1)
    step = largest * dtype(1.0 / 127.0) if dtype is np.float32 else largest / 127
    scales = np.maximum(step, dtype(LEAST))
    lost = ~np.isfinite(largest)
    codes = np.clip(np.rint(np.where(lost[..., None], 0, x) * (dtype(1) / scales)[..., None]), -127, 127)
    codes[lost] = 0
    return codes.astype(np.int8), np.where(lost, dtype(np.nan), scales).astype(dtype)


def linear(x: np.ndarray, codes: np.ndarray, scales: np.ndarray, dtype=np.float32) -> np.ndarray:
    """x [m, k] times the weight codes [n, k] * scales [n]: whole-number sums, then two products in `dtype`."""
    xc, xs = quantize_rows(x, dtype)
    # (Products and sums of whole numbers below 2^53: exact in float64.)
    sums = xc.astype(np.float64) @ codes.astype(np.float64).T
    return sums.astype(dtype) * xs[:, None] * scales.astype(dtype)
