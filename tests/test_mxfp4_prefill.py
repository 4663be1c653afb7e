"""Prefill over the 4-bit cache where the query's type, the layout or a page gets in the way; the bounds are test_mxfp4's."""

import numpy as np
import pytest
import torch

import microinfer_b200 as mi
from oracle import mxfp4_oracle as mo
from tests.test_mxfp4 import PREFILL_STEP, _close, _cuda, _pages, _table

gpu = pytest.mark.gpu
LARGE = [140, 150, 1, 137, 144]  # with 8 kv heads of 128, 2 query heads each: 120 tiles of 128 rows


@gpu
@pytest.mark.parametrize("d,large", [(64, False), (96, False), (256, False), (128, False)])
def test_prefill_keys_past_fp16(cuda_device, d, large):
    """Keys of 2^14 to 2^24, met by queries small enough for ordinary scores."""
    q_lens, ctxs = (LARGE, [140, 200, 9, 137, 300]) if large else ([86], [90])
    hkv, group = (8, 2) if large else (1, 3)
    rng = np.random.default_rng(d)
    nb = sum(-(-c // 16) for c in ctxs)
    kp, vp = _pages(rng, nb, 16, hkv, d)
    code, byte = mo.unpack(kp)
    table = _table(rng, ctxs, nb, 16)
    for i, pos in enumerate([0, 5, 6, 17, 40, 63, 64, 70, 85]):
        byte[table[0, pos // 16], pos % 16, 0, i % (d // 32)] = 127 + [14, 15, 20, 24][i % 4]
    kp = mo.pack(code, byte)
    q = rng.standard_normal((sum(q_lens), hkv * group, d))
    q[:q_lens[0], :group] *= 2.0 ** -22
    q[:q_lens[0], :group, ::5] = 0  # an infinite key would make a NaN of these
    query = _cuda(q, cuda_device, torch.float16)
    cu_q, cu_k = (torch.tensor([0, *np.cumsum(x)], dtype=torch.int32, device=cuda_device) for x in (q_lens, ctxs))
    got = mi.paged_prefill_mxfp4(query, _cuda(kp, cuda_device), _cuda(vp, cuda_device), cu_q, cu_k,
                                 _cuda(table, cuda_device), max_seqlen_q=max(q_lens), total_k=sum(ctxs))
    mi.check_device_status(cuda_device)
    q, at = query.double().cpu().numpy(), np.cumsum([0, *q_lens])
    parts = [mo.attention(q[at[r]:at[r + 1]], mo.rows(kp, table[r], c), mo.rows(vp, table[r], c), d ** -0.5)
             for r, c in enumerate(ctxs)]
    _close(got, *[np.concatenate(x) for x in zip(*parts)], torch.float16, PREFILL_STEP[torch.float16])
