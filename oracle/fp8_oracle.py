"""The 8-bit (e4m3) paged cache in numpy, in 64 bits: the tests' checker.

A cache is held as codes uint8 [blocks, bs, Hkv, D] and scale bytes uint8 [blocks, bs / 16, Hkv], one for
every 16 tokens and head; ``pack`` / ``unpack`` go between those and pages uint8
[blocks, Hkv, bs / 16, 16 * D + 16], ``store`` writes rows into them as the operator does.
"""

from __future__ import annotations

import numpy as np

from oracle import mxfp4_oracle as mo

# magnitudes of codes 0 to 126
GRID = np.array([m * 2.0 ** -9 for m in range(8)]
                + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:-1])
MIDDLE = (GRID[1:] + GRID[:-1]) / 2
NAN = 127


def codes_of(x):
    """The codes nearest to x: ties to even, at most 448, NaN for what is not finite."""
    x = np.asarray(x, dtype=np.float64)
    bad = ~np.isfinite(x)
    a = np.where(bad, 0.0, np.abs(x))
    code = np.searchsorted(MIDDLE, a, side="left")  # the first boundary that a does not pass
    code = np.where(np.isin(a, MIDDLE) & (code % 2 == 1), code + 1, code)
    return np.where(bad, NAN, code + 128 * (np.signbit(x) & ~bad)).astype(np.uint8)


def values_of(code):
    a = np.append(GRID, np.nan)[code % 128]
    return np.where(code >= 128, -a, a)


def scale_of(byte):
    return np.where(byte == 0, 0.0, np.exp2(byte.astype(np.float64) - 127))


def byte_for(a):
    """The scale byte that largest magnitudes a need."""
    a = np.asarray(a, dtype=np.float64)
    mantissa, exponent = np.frexp(np.where(a > 0, a, 1.0))  # 448 = 0.875 * 2^9
    return np.where(a > 0, np.clip(exponent - 9 + (mantissa > 0.875) + 127, 1, 246), 0).astype(np.uint8)


def encode(x):
    """Codes and scale bytes of x [blocks, bs, Hkv, D], every group quantised at once."""
    x = np.asarray(x, dtype=np.float64)
    nb, bs, hkv, d = x.shape
    groups = x.reshape(nb, bs // 16, 16, hkv, d)
    byte = byte_for(np.where(np.isfinite(groups), np.abs(groups), 0.0).max((2, 4)))
    unit = np.where(byte > 0, scale_of(byte), 1.0)
    return codes_of(groups / unit[:, :, None, :, None]).reshape(x.shape), byte


def decode(code, byte):
    """float64 [blocks, bs, Hkv, D]."""
    return values_of(code) * np.repeat(scale_of(byte), 16, 1)[..., None]


def store(code, byte, slots, x):
    """Rows x [T, Hkv, D] to slots [T] (-1: nowhere), in place."""
    bs = code.shape[1]
    x = np.asarray(x, dtype=np.float64)
    slots = np.asarray(slots)
    for g in np.unique(slots[slots >= 0] // 16):
        tokens = np.flatnonzero((slots >= 0) & (slots // 16 == g))
        block, group = divmod(int(g), bs // 16)
        new = x[tokens]
        need = byte_for(np.where(np.isfinite(new), np.abs(new), 0.0).max((0, 2)))
        fresh = bool((slots[tokens] % 16 == 0).any())
        old = byte[block, group].copy()
        now = need if fresh else np.maximum(old, need)
        here = code[block, group * 16:group * 16 + 16]  # a view
        if not fresh:
            for h in np.flatnonzero(now > old):
                shrink = scale_of(old[h]) / scale_of(now[h])
                kept = values_of(here[:, h])
                here[:, h] = codes_of(np.where(np.isnan(kept), np.nan, kept * shrink))
        unit = np.where(now > 0, scale_of(now), 1.0)
        here[slots[tokens] % 16] = codes_of(new / unit[:, None])
        byte[block, group] = now


def _place(d, value):
    """Byte of each (token, dim) in a group."""
    place = np.zeros((16, d), dtype=np.int64)
    for tok in range(16):
        for dim in range(d):
            start = dim // 64 * 64
            w, i = min(64, d - start), dim - start
            inner = (((tok // 8 * 8 + i // (w // 8)) * 4 + tok % 8 // 2) * (w // 8) + i % (w // 8)) * 2 + tok % 2
            place[tok, dim] = start * 16 + (inner if value else tok * w + i)
    return place


def pack(code, byte, value):
    nb, bs, hkv, d = code.shape
    out = np.zeros((nb, hkv, bs // 16, 16 * d + 16), dtype=np.uint8)
    out[..., _place(d, value)] = code.reshape(nb, bs // 16, 16, hkv, d).transpose(0, 3, 1, 2, 4)
    out[..., 16 * d] = byte.transpose(0, 2, 1)
    return out


def unpack(pages, value):
    nb, hkv, groups, size = pages.shape
    d = size // 16 - 1
    code = pages[..., _place(d, value)].transpose(0, 2, 3, 1, 4).reshape(nb, groups * 16, hkv, d)
    return np.ascontiguousarray(code), np.ascontiguousarray(pages[..., 16 * d].transpose(0, 2, 1))


def rows(pages, table, ctx, value):
    """float64 [ctx, Hkv, D] of one block-table row."""
    bs = pages.shape[2] * 16
    some = decode(*unpack(pages[np.asarray(table[:-(-ctx // bs)], dtype=np.int64)], value))
    return some.reshape(-1, *some.shape[2:])[:ctx]


def attention(q, key_pages, value_pages, table, ctx, scale):
    """Causal attention of q [n, Hq, D] at the end of a context, in float64.

    Returns the result and what rounding errors are measured against: the sum of p |v|, the largest key's sum
    of scale |q| |k|, and ctx times half the largest magnitude that the context's scales of V reach.
    """
    k, v = rows(key_pages, table, ctx, False), rows(value_pages, table, ctx, True)
    out, weight, size, _ = mo.attention(q, np.nan_to_num(k), np.nan_to_num(v), scale)
    floor = np.zeros_like(out)
    # a NaN reaches the rows that see its key: one of V its dim, one of K all
    n, group = q.shape[0], q.shape[1] // k.shape[1]
    for pos in np.flatnonzero(np.isnan(k).any((1, 2)) | np.isnan(v).any((1, 2))):
        sees = slice(max(0, pos - (ctx - n)), n)
        lost = np.isnan(v[pos]) | np.isnan(k[pos]).any(-1, keepdims=True)
        out[sees, np.repeat(lost, group, 0)] = np.nan
    if ctx:
        bs = key_pages.shape[2] * 16
        _, byte = unpack(value_pages[np.asarray(table[:-(-ctx // bs)], dtype=np.int64)], True)
        byte = byte.reshape(-1, byte.shape[-1])[:-(-ctx // 16)].max(0)
        reach = ctx * 224.0 * scale_of(byte)
        floor[:] = np.repeat(reach, q.shape[1] // len(reach))[None, :, None]
    return out, weight, size, floor
