"""Decode where a product of partial results leaves fp32's range although the result does not.

The bound is that of test_mxfp4: it is relative to the scores and values, whatever their powers of two.
"""
import numpy as np
import pytest
import torch

import microinfer_b200 as mi
from oracle import mxfp4_oracle as mo
from tests.test_mxfp4 import DECODE_STEP, DTYPES, _close, _cuda, _table

gpu = pytest.mark.gpu


def _at(rng, nb, bs, hkv, d, power):
    """Pages of normal rows times 2^power, by way of their scale bytes."""
    code, byte = mo.encode(rng.standard_normal((nb, bs, hkv, d)))
    byte = np.where(byte == 0, 0, np.clip(byte.astype(int) + power, 1, 252)).astype(np.uint8)
    return mo.pack(code, byte)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("d,group", [(32, 4), (64, 7), (96, 2), (128, 4), (128, 8), (256, 4)])
@pytest.mark.parametrize("k_power,q_power,v_power", [
    (118, -118, 0), (104, -104, 0), (-110, 112, -100), (0, 0, 110), (0, 0, 124), (118, -118, 124), (0, 0, -122)])
def test_decode_over_the_whole_range_of_scales(cuda_device, name, d, group, k_power, q_power, v_power):
    """Scores of ordinary size from keys and queries of 2^+-118, values up to fp32's end; sequences within a warp,
    over warps and over CTAs."""
    ctxs, bs, hkv = [9000, 1, 40, 700], 16, 2
    rng = np.random.default_rng(d + group)
    dtype = DTYPES[name]
    nb = sum(-(-c // bs) for c in ctxs)
    kp, vp = _at(rng, nb, bs, hkv, d, k_power), _at(rng, nb, bs, hkv, d, v_power)
    table = _table(rng, ctxs, nb, bs)
    query = _cuda(np.ldexp(rng.standard_normal((len(ctxs), hkv * group, d)), q_power), cuda_device, dtype)
    got = mi.paged_decode_mxfp4(query, _cuda(kp, cuda_device), _cuda(vp, cuda_device), _cuda(table, cuda_device),
                                torch.tensor(ctxs, dtype=torch.int32, device=cuda_device))
    mi.check_device_status(cuda_device)
    q = query.double().cpu().numpy()
    parts = [mo.attention(q[r:r + 1], mo.rows(kp, table[r], c), mo.rows(vp, table[r], c), d ** -0.5)
             for r, c in enumerate(ctxs)]
    _close(got, *[np.concatenate(x) for x in zip(*parts)], dtype, DECODE_STEP[dtype])


@gpu
@pytest.mark.parametrize("d", [64, 128])
def test_decode_of_blocks_of_very_different_size(cuda_device, d):
    """The query is zero where the keys are large, and its largest elements meet keys as small."""
    rng = np.random.default_rng(d)
    ctx, bs = 200, 16
    kc, kb = mo.encode(rng.standard_normal((13, bs, 1, d)))
    kb = np.clip(kb.astype(int) + 112, 1, 252).astype(np.uint8)
    kb[..., 0] = rng.integers(20, 24, kb[..., 0].shape)  # 2^-107 to 2^-104
    kp, vp = mo.pack(kc, kb), _at(rng, 13, bs, 1, d, 0)
    table = _table(rng, [ctx], 13, bs)
    q = rng.standard_normal((1, 4, d)) * 2.0 ** 104
    q[..., 32:] = 0
    query = _cuda(q, cuda_device, torch.float32)
    got = mi.paged_decode_mxfp4(query, _cuda(kp, cuda_device), _cuda(vp, cuda_device), _cuda(table, cuda_device),
                                torch.tensor([ctx], dtype=torch.int32, device=cuda_device))
    want = mo.attention(query.double().cpu().numpy(), mo.rows(kp, table[0], ctx), mo.rows(vp, table[0], ctx), d ** -0.5)
    _close(got, *want, torch.float32, DECODE_STEP[torch.float32])
