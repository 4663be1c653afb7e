"""The 4-bit (MXFP4) paged cache in numpy, in 64 bits: the tests' checker.

``encode`` / ``decode`` go between rows [..., D] and (codes, scale bytes);
``pack`` / ``unpack`` between those and pages uint8
[blocks, Hkv, block_size / 16, D / 32 * 272].
"""

from __future__ import annotations

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
MIDDLE = (GRID[1:] + GRID[:-1]) / 2


def encode(x):
    """Codes uint8 [..., D] (one per element) and scale bytes uint8 [..., D / 32]."""
    x = np.asarray(x, dtype=np.float64)
    blocks = x.reshape(*x.shape[:-1], -1, 32)
    top = np.abs(blocks).max(-1)
    bad = ~np.isfinite(blocks).all(-1)
    top = np.where(bad, 1.0, top)
    exponent = np.frexp(np.where(top > 0, top, 1.0))[1] - 1 - 2
    exponent = np.maximum(exponent, -126)
    q = np.abs(np.where(bad[..., None], 0.0, blocks)) / np.exp2(exponent)[..., None]
    # the index of the first boundary that q does not reach; a tie goes to the even code
    code = np.searchsorted(MIDDLE, q, side="left")
    tie = np.isin(q, MIDDLE)
    code = np.where(tie & (code % 2 == 1), code + 1, code)
    code = (code + 8 * np.signbit(blocks)).astype(np.uint8)
    code = np.where(bad[..., None], 0, code).astype(np.uint8)
    byte = np.where(bad, 255, np.where(top > 0, exponent + 127, 0)).astype(np.uint8)
    return code.reshape(x.shape), byte


def decode(code, byte):
    """float64 [..., D]."""
    value = np.where(code >= 8, -GRID[code % 8], GRID[code % 8])
    scale = np.where(byte == 0, 0.0, np.exp2(byte.astype(np.float64) - 127))
    scale = np.where(byte == 255, np.nan, scale)
    blocks = value.reshape(*byte.shape, 32) * scale[..., None]
    return blocks.reshape(value.shape)


def pack(code, byte):
    """Pages of codes [blocks, bs, Hkv, D] and scales [blocks, bs, Hkv, D / 32]."""
    nb, bs, hkv, d = code.shape
    out = np.zeros((nb, hkv, bs // 16, d // 32 * 272), dtype=np.uint8)
    for tok in range(bs):
        g, t = divmod(tok, 16)
        for b in range(d // 32):
            for j in range(16):
                out[:, :, g, b * 256 + t * 16 + j] = (code[:, tok, :, b * 32 + 2 * j]
                                                      | code[:, tok, :, b * 32 + 2 * j + 1] << 4)
            out[:, :, g, d // 32 * 256 + t * (d // 32) + b] = byte[:, tok, :, b]
    return out


def unpack(pages):
    """(codes [blocks, bs, Hkv, D], scales [blocks, bs, Hkv, D / 32]) of pages."""
    nb, hkv, groups, size = pages.shape
    d = size // 272 * 32
    code = np.zeros((nb, groups * 16, hkv, d), dtype=np.uint8)
    byte = np.zeros((nb, groups * 16, hkv, d // 32), dtype=np.uint8)
    for tok in range(groups * 16):
        g, t = divmod(tok, 16)
        for b in range(d // 32):
            raw = pages[:, :, g, b * 256 + t * 16:b * 256 + t * 16 + 16]
            code[:, tok, :, b * 32:b * 32 + 32:2] = raw & 15
            code[:, tok, :, b * 32 + 1:b * 32 + 32:2] = raw >> 4
            byte[:, tok, :, b] = pages[:, :, g, d // 32 * 256 + t * (d // 32) + b]
    return code, byte


def rows(pages, table, ctx):
    """float64 [ctx, Hkv, D] of one block-table row."""
    bs = pages.shape[2] * 16
    code, byte = unpack(pages[np.asarray(table[:-(-ctx // bs)], dtype=np.int64)])
    return decode(code.reshape(-1, *code.shape[2:])[:ctx], byte.reshape(-1, *byte.shape[2:])[:ctx])


def attention(q, k, v, scale):
    """Causal attention of q [n, Hq, D], at the end of k / v [ctx, Hkv, D], in float64.

    Returns the result and what rounding errors are measured against: the sum of p |v|, the
    largest key's sum of scale |q| |k|, and ctx times the largest |v| of each block of 32.
    """
    n, hq, _ = q.shape
    ctx, hkv, d = k.shape
    out, weight, size, floor = (np.zeros((n, hq, d)) for _ in range(4))
    for h in range(hq if ctx else 0):
        kh, vh = k[:, h // (hq // hkv)], v[:, h // (hq // hkv)]
        x = q[:, h] @ kh.T * scale
        far = np.abs(q[:, h]) @ np.abs(kh).T * scale
        x = np.where(np.arange(ctx)[None] > np.arange(ctx - n, ctx)[:, None], -np.inf, x)
        top = x.max(-1, keepdims=True)
        p = np.exp(x - np.where(np.isneginf(top), 0, top))
        total = p.sum(-1, keepdims=True)
        p /= np.where(total == 0, 1, total)  # a row before the first key: zeros
        out[:, h] = p @ vh
        weight[:, h] = p @ np.abs(vh)
        size[:, h] = far.max(-1, keepdims=True)
        floor[:, h] = ctx * np.abs(vh).reshape(ctx, -1, 32).max((0, 2)).repeat(32)
    return out, weight, size, floor
