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


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("way,rows", WAYS)
def test_softmax_scale_of_zero_with_large_keys(cuda_device, name, d, way, rows):
    """Every visible key weighs the same, however large its product with the query."""
    rng = np.random.default_rng(d)
    ctx = 1280
    nb = ctx // 16
    code, byte = mo.encode(rng.standard_normal((nb, 16, 1, d)))
    power = 108 if name != "f16" or way == "decode" else 14  # prefill's K is fp16 there
    kp = mo.pack(code, np.where(byte == 0, 0, byte + power).astype(np.uint8))
    vp = mo.pack(*mo.encode(rng.standard_normal((nb, 16, 1, d))))
    query = _cuda(rng.standard_normal((rows, 2, d)), cuda_device, DTYPES[name])
    got = _attend(cuda_device, query, kp, vp, ctx, 0.0, way).double().cpu().numpy()
    v = mo.rows(vp, np.arange(nb), ctx)[:, 0]
    seen = np.arange(ctx - rows, ctx) + 1
    want = np.cumsum(v, 0)[seen - 1] / seen[:, None]
    size = np.cumsum(np.abs(v), 0)[seen - 1] / seen[:, None]
    u = torch.finfo(DTYPES[name]).eps / 2
    # p is 1, exact in every type; scores off by 2^-20 at most; the result is rounded once
    assert (np.abs(got - want[:, None]) <= u * np.abs(want[:, None]) + (2.0 ** -18 + ctx * 2.0 ** -24) * size[:, None]).all()


@gpu
@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("way,rows", WAYS)
def test_softmax_scale_that_is_nan(cuda_device, name, way, rows):
    rng = np.random.default_rng(3)
    kp, vp = (mo.pack(*mo.encode(rng.standard_normal((80, 16, 1, 128)))) for _ in range(2))
    query = _cuda(rng.standard_normal((rows, 2, 128)), cuda_device, DTYPES[name])
    assert bool(torch.isnan(_attend(cuda_device, query, kp, vp, 1280, float("nan"), way)).all())


@gpu
@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [5, 300])
def test_softmax_scale_of_zero_with_large_keys_in_16_and_32_bits(cuda_device, name, d, rows):
    rng = np.random.default_rng(d)
    q, k, v = (torch.from_numpy(rng.standard_normal((rows, 1, d))).to(cuda_device, DTYPES[name]) for _ in range(3))
    cu = torch.tensor([0, rows], dtype=torch.int32, device=cuda_device)
    got = mi.varlen_prefill(q, k * 2.0 ** 108, v, cu, cu, max_seqlen_q=rows, scale=0.0).double().cpu()
    v = v.double().cpu()
    count = torch.arange(1, rows + 1, dtype=torch.float64)[:, None, None]
    want, size = v.cumsum(0) / count, v.abs().cumsum(0) / count
    u = torch.finfo(DTYPES[name]).eps / 2
    assert bool(((got - want).abs() <= u * want.abs() + (2.0 ** -18 + rows * 2.0 ** -24) * size).all())
