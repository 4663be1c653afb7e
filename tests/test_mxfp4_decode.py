"""Decode over block tables with pages that are none."""

import numpy as np
import pytest
import torch

import microinfer_b200 as mi
from microinfer_b200 import _lib
from oracle import mxfp4_oracle as mo
from tests.test_mxfp4 import DECODE_STEP, DTYPES, _close, _cuda, _pages, _table

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d,bs", [(64, 16), (128, 16), (128, 48), (96, 32), (256, 16)])
def test_pages_that_are_none_are_left_out(cuda_device, name, d, bs):
    """They and no others, whether they come first or second in a unit of 32 keys, at an end, or are all of them."""
    rng = np.random.default_rng(d + bs)
    dtype = DTYPES[name]
    ctxs = [16 * bs, 3 * bs + 5, 40 * bs, 2 * bs, bs, 2 * bs - 3]
    gone = [[0, 3], [3], [1, 7, 8, 20, 39], [0, 1], [], [0]]
    nb = sum(-(-c // bs) for c in ctxs)
    kp, vp = _pages(rng, nb, bs, 2, d)
    table = _table(rng, ctxs, nb, bs)
    broken = table.copy()
    for r, cols in enumerate(gone):
        broken[r, cols] = [-1, nb, 1 << 30, -1, nb + 3][:len(cols)]
    query = _cuda(rng.standard_normal((len(ctxs), 8, d)), cuda_device, dtype)
    got = mi.paged_decode_mxfp4(query, _cuda(kp, cuda_device), _cuda(vp, cuda_device), _cuda(broken, cuda_device),
                                torch.tensor(ctxs, dtype=torch.int32, device=cuda_device))
    assert mi.read_device_status(cuda_device) == _lib.DEV_BAD_BLOCK
    q = query.double().cpu().numpy()
    parts = []
    for r, c in enumerate(ctxs):
        keep = ~np.isin(np.arange(c) // bs, gone[r])
        parts.append(mo.attention(q[r:r + 1], mo.rows(kp, table[r], c)[keep], mo.rows(vp, table[r], c)[keep], d ** -0.5))
    assert bool((got[3] == 0).all())
    _close(got, *[np.concatenate(x) for x in zip(*parts)], dtype, DECODE_STEP[dtype])
