"""The 4-bit cache's attention at scores and softmax scales at the ends of fp32's range."""

import numpy as np
import pytest
import torch

import microinfer_b200 as mi
from oracle import mxfp4_oracle as mo
from tests.test_mxfp4 import DTYPES, _cuda

gpu = pytest.mark.gpu
LOG2E = np.float32(np.log2(np.e))


def _attend(device, query, kp, vp, ctx, scale, way):
    nb = kp.shape[0]
    pool = _cuda(kp, device), _cuda(vp, device)
    table = torch.arange(nb, dtype=torch.int32, device=device)[None]
    if way == "decode":
        got = mi.paged_decode_mxfp4(query, *pool, table, torch.tensor([ctx], dtype=torch.int32, device=device), scale=scale)
    else:
        n = query.shape[0]
        cu_q, cu_k = (torch.tensor([0, x], dtype=torch.int32, device=device) for x in (n, ctx))
        got = mi.paged_prefill_mxfp4(query, *pool, cu_q, cu_k, table, max_seqlen_q=n, total_k=ctx, scale=scale)
    mi.check_device_status(device)
    return got


# rows of a prefill large enough for the dense kernel at head_dim 128 in 16 bits, and few rows
WAYS = [("decode", 1), ("prefill", 2), ("prefill", 1280)]


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("way,rows", WAYS)
@pytest.mark.parametrize("power,ahead", [(18, 4), (22, 4), (24, 4), (25, 4), (26, 8), (27, 0), (27, 16), (28, 0), (28, 16), (31, 0)])
@pytest.mark.parametrize("off", [1.0, 1.3])
def test_scores_a_step_apart(cuda_device, name, d, way, rows, power, ahead, off):
    """Runs of keys whose largest score is in turn 2^power and `ahead` above it, a few steps of fp32 at most: p stays within f16, so
    results lie between the values, which are 1 and 4."""
    ctx, run = 1280, 32 if way == "decode" else 64
    nb = ctx // 16
    high = np.arange(nb) * 16 // run % 2 == 1
    k, v = np.zeros((nb, 16, 1, d)), np.ones((nb, 16, 1, d))
    k[..., 0] = 1.0
    k[high, 3, 0, 1] = 1.0
    v[high] = 4.0
    kp, vp = mo.pack(*mo.encode(k)), mo.pack(*mo.encode(v))
    query = np.zeros((rows, 1, d))
    query[:, 0, 0], query[:, 0, 1] = 1.0, ahead * 2.0 ** -power
    scale = np.float32(2.0 ** power) / LOG2E
    while float(scale * LOG2E) % 4 or float(scale * LOG2E) < 2.0 ** power:
        scale = np.nextafter(scale, np.float32(np.inf))
    # off: scores that are no fp32 numbers
    got = _attend(cuda_device, _cuda(query, cuda_device, DTYPES[name]), kp, vp, ctx, float(scale) * off, way)
    assert bool(torch.isfinite(got).all()) and bool((got >= 1 - 2.0 ** -7).all()) and bool((got <= 4 + 2.0 ** -5).all())
