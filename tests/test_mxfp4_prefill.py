"""Prefill over the 4-bit cache where the query's type, the layout or a page gets in the way; the bounds are test_mxfp4's."""

import numpy as np
import pytest
import torch

import microinfer_b200 as mi
from microinfer_b200 import _lib
from oracle import mxfp4_oracle as mo
from tests.test_mxfp4 import DTYPES, PREFILL_STEP, _close, _close_or_past, _cuda, _pages, _prefill_case, _table

gpu = pytest.mark.gpu
LARGE = [140, 150, 1, 137, 144]  # with 8 kv heads of 128, 2 query heads each: 120 tiles of 128 rows


@gpu
@pytest.mark.parametrize("d,large", [(64, False), (96, False), (256, False), (128, False), (128, True)])
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


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
def test_gathered_scale_of_zero(cuda_device, name):
    """Every key that a row sees weighs the same, masked ones nothing; rows before the first key are zeros."""
    hkv, group, d = (8, 2, 128) if name != "f32" else (2, 2, 160)
    got, free, want, dtype = _prefill_case(cuda_device, name, hkv, group, d, 16, LARGE, [140, 200, 9, 130, 300], scale=0.0)
    for x in (got, free):
        _close(x, *want, dtype, PREFILL_STEP[dtype])


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
def test_16_bit_prefill_with_a_scale_of_zero(cuda_device, name):
    dtype = DTYPES[name]
    query, k, v = (torch.randn(200, h, 128, device=cuda_device).to(dtype) for h in (16, 8, 8))
    cu = torch.tensor([0, 200], dtype=torch.int32, device=cuda_device)
    want = (v.double().cumsum(0) / torch.arange(1, 201, device=cuda_device)[:, None, None]).repeat_interleave(2, 1)
    # p is one for every key: what is left is the sum in fp32 and one rounding
    bound = torch.finfo(dtype).eps / 2 * want.abs() + 200 * 2.0 ** -23 * v.double().abs().max()
    got = mi.varlen_prefill(query, k, v, cu, cu, max_seqlen_q=200, scale=0.0)
    assert bool(((got.double() - want).abs() <= bound).all())
    pages_k, pages_v = (torch.cat([t, t[:8]]).view(13, 16, 8, 128) for t in (k, v))
    table = torch.arange(13, dtype=torch.int32, device=cuda_device)[None]
    got = mi.paged_prefill(query, pages_k, pages_v, cu, cu, table, max_seqlen_q=200, scale=0.0)
    assert bool(((got.double() - want).abs() <= bound).all())
    mi.check_device_status(cuda_device)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
def test_gathered_nan_blocks_reach_only_rows_that_see_them(cuda_device, name):
    def edit(kp, vp, table):
        kc, kb = mo.unpack(kp)
        vc, vb = mo.unpack(vp)
        vb[table[0, 60 // 16], 60 % 16, 0, 1] = 255  # position 60 of 140, row 60
        kb[table[1, 180 // 16], 180 % 16, 0, 0] = 255  # position 180 of 200, row 130 of 150
        kp[:], vp[:] = mo.pack(kc, kb), mo.pack(vc, vb)

    got, free, _, _ = _prefill_case(cuda_device, name, 8, 2, 128, 16, LARGE, [140, 200, 9, 137, 300], edit=edit)
    for x in (got, free):
        nan = torch.isnan(x).cpu()
        assert bool(nan[60:140, :2, 32:64].all()) and int(nan[:140].sum()) == 80 * 2 * 32
        assert bool(nan[140 + 130:290, :2].all()) and int(nan[140:290].sum()) == 20 * 2 * 128
        assert not bool(nan[290:].any())


@gpu
def test_gathered_values_past_fp16(cuda_device):
    def edit(kp, vp, table):
        code, byte = mo.unpack(vp)
        for i, pos in enumerate([5, 6, 17, 40, 63, 64, 70, 129]):
            byte[table[0, pos // 16], pos % 16, 0, i % 4] = 127 + [14, 15, 20, 40][i % 4]
        vp[:] = mo.pack(code, byte)

    got, free, want, dtype = _prefill_case(cuda_device, "f16", 8, 2, 128, 16, LARGE, [140, 200, 9, 137, 300], edit=edit)
    for x in (got, free):
        _close_or_past(x, *want, dtype, PREFILL_STEP[dtype])
    assert bool(torch.isfinite(got[:5]).all())


@gpu
@pytest.mark.parametrize("name,hkv,group,d,q_lens,ctxs", [
    ("bf16", 8, 2, 128, LARGE, [140, 200, 9, 137, 300]), ("f16", 8, 4, 128, LARGE, [140, 200, 9, 137, 300]),
    ("f32", 2, 2, 160, [40, 3], [50, 900]), ("bf16", 2, 4, 96, [40, 1], [50, 3000]), ("f32", 2, 4, 96, [1], [3000])])
def test_results_over_the_query(cuda_device, name, hkv, group, d, q_lens, ctxs):
    rng = np.random.default_rng(50)
    dtype = DTYPES[name]
    nb = sum(-(-c // 16) for c in ctxs)
    kp, vp = _pages(rng, nb, 16, hkv, d)
    table = _cuda(_table(rng, ctxs, nb, 16), cuda_device)
    query = _cuda(rng.standard_normal((sum(q_lens), hkv * group, d)), cuda_device, dtype)
    cu_q, cu_k = (torch.tensor([0, *np.cumsum(x)], dtype=torch.int32, device=cuda_device) for x in (q_lens, ctxs))
    args = (_cuda(kp, cuda_device), _cuda(vp, cuda_device), cu_q, cu_k, table)
    want = mi.paged_prefill_mxfp4(query, *args, max_seqlen_q=max(q_lens))
    for _ in range(3):
        over = query.clone()
        assert mi.paged_prefill_mxfp4(over, *args, max_seqlen_q=max(q_lens), out=over) is over
        assert torch.equal(over, want)
    mi.check_device_status(cuda_device)


@gpu
@pytest.mark.parametrize("name,hkv,d", [("bf16", 8, 128), ("f16", 8, 128), ("f32", 2, 160)])
def test_gathered_bad_pages(cuda_device, name, hkv, d):
    """Twice the same finite result with the allocator's memory full of NaN, and the other sequences untouched."""
    rng = np.random.default_rng(40)
    dtype = DTYPES[name]
    q_lens, ctxs = LARGE, [140, 200, 9, 137, 300]
    nb = sum(-(-c // 16) for c in ctxs)
    kp, vp = _pages(rng, nb, 16, hkv, d)
    table = _table(rng, ctxs, nb, 16)
    broken = table.copy()
    broken[1, 3], broken[4, 0], broken[4, 7] = nb + 5, -1, 1 << 30
    query = _cuda(rng.standard_normal((sum(q_lens), 2 * hkv, d)), cuda_device, dtype)
    cu_q, cu_k = (torch.tensor([0, *np.cumsum(x)], dtype=torch.int32, device=cuda_device) for x in (q_lens, ctxs))
    pages = _cuda(kp, cuda_device), _cuda(vp, cuda_device)

    def call(t):
        for n in (sum(ctxs) * hkv * d, 2 * sum(ctxs) * hkv * d + 4096):
            for _ in range(3):
                torch.full((n,), float("nan"), dtype=dtype, device=cuda_device)
        return mi.paged_prefill_mxfp4(query, *pages, cu_q, cu_k, _cuda(t, cuda_device), max_seqlen_q=max(q_lens),
                                      total_k=sum(ctxs))

    good = call(table)
    assert mi.read_device_status(cuda_device) == 0
    got = call(broken)
    assert mi.read_device_status(cuda_device) == _lib.DEV_BAD_BLOCK
    again = call(broken)
    mi.read_device_status(cuda_device)
    assert bool(torch.isfinite(got).all()) and torch.equal(got, again)
    at = np.cumsum([0, *q_lens])
    for r in (0, 2, 3):
        assert torch.equal(got[at[r]:at[r + 1]], good[at[r]:at[r + 1]])
    # keys of pages that are none are left out; in fp32 above head_dim 128 they count as zeros
    q = query.double().cpu().numpy()
    for r, cols in ((1, [3]), (4, [0, 7])):
        k, v = mo.rows(kp, table[r], ctxs[r]), mo.rows(vp, table[r], ctxs[r])
        gone = np.isin(np.arange(ctxs[r]) // 16, cols)
        k[gone], v[gone] = 0, 0
        rows = q[at[r]:at[r + 1]]
        x = np.einsum("qhd,khd->hqk", rows, k.repeat(2, 1)) * d ** -0.5
        hidden = np.arange(ctxs[r])[None] > np.arange(ctxs[r] - len(rows), ctxs[r])[:, None]
        x[:, hidden | gone if d == 128 else hidden] = -np.inf
        p = np.exp(x - x.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        want = np.einsum("hqk,khd->qhd", p, v.repeat(2, 1))
        weight = np.einsum("hqk,khd->qhd", p, np.abs(v).repeat(2, 1))
        size = np.einsum("qhd,khd->qhk", np.abs(rows), np.abs(k).repeat(2, 1)).max(-1, keepdims=True) * d ** -0.5
        _close(got[at[r]:at[r + 1]], want, weight, size, 0 * want, dtype, PREFILL_STEP[dtype])


@gpu
@pytest.mark.parametrize("name,hkv,d", [("bf16", 8, 128), ("f16", 8, 128), ("f32", 2, 160)])
def test_gathered_context_past_the_table(cuda_device, name, hkv, d):
    """A context longer than its block-table row is flagged; what it does see gives the same every time."""
    rng = np.random.default_rng(41)
    dtype = DTYPES[name]
    q_lens, ctxs = LARGE, [140, 200, 9, 137, 300]
    nb = sum(-(-c // 16) for c in ctxs)
    kp, vp = _pages(rng, nb, 16, hkv, d)
    table = _table(rng, ctxs, nb, 16)
    query = _cuda(rng.standard_normal((sum(q_lens), 2 * hkv, d)), cuda_device, dtype)
    cu_q, cu_k = (torch.tensor([0, *np.cumsum(x)], dtype=torch.int32, device=cuda_device) for x in (q_lens, ctxs))
    pages = _cuda(kp, cuda_device), _cuda(vp, cuda_device)

    def call(width):
        for n in (sum(ctxs) * hkv * d, 2 * sum(ctxs) * hkv * d + 4096):
            for _ in range(3):
                torch.full((n,), float("nan"), dtype=dtype, device=cuda_device)
        return mi.paged_prefill_mxfp4(query, *pages, cu_q, cu_k, _cuda(table[:, :width], cuda_device), max_seqlen_q=max(q_lens))

    good = call(table.shape[1])
    assert mi.read_device_status(cuda_device) == 0
    got = call(14)  # 224 positions
    assert mi.read_device_status(cuda_device) & _lib.DEV_BAD_BLOCK
    again = call(14)
    mi.read_device_status(cuda_device)
    assert bool(torch.isfinite(got).all()) and torch.equal(got, again)
    end = sum(q_lens[:4])
    assert torch.equal(got[:end], good[:end])
    first = 224 - (300 - 144)  # rows of the last sequence that see nothing past the table
    want = mo.attention(query[end:].double().cpu().numpy(), mo.rows(kp, table[4], 300), mo.rows(vp, table[4], 300), d ** -0.5)
    _close(got[end:end + first], *[x[:first] for x in want], dtype, PREFILL_STEP[dtype])


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
def test_gathered_keys_of_little_weight(cuda_device, name):
    """One key takes nearly everything and its value is zero: the rest, each about 2^-20 of it, decides the result.
    p is lifted by 2^7 in fp16, so half its smallest step is 2^-32 of the largest p, a key at most."""
    dtype = DTYPES[name]
    hkv, d, q_lens = 8, 128, LARGE
    ctxs = [3000] * 5
    rng = np.random.default_rng(80)
    nb = 5 * 188
    kc, kb = mo.encode(rng.standard_normal((nb, 16, hkv, d)) * 0.01)
    vc, vb = mo.encode(rng.standard_normal((nb, 16, hkv, d)) + 1.0)
    table = _table(rng, ctxs, nb, 16)
    kc[table[:, 3], 5], kb[table[:, 3], 5] = 2, 127  # all 1.0
    vc[table[:, 3], 5], vb[table[:, 3], 5] = 0, 0
    kp, vp = mo.pack(kc, kb), mo.pack(vc, vb)
    query = _cuda(np.full((sum(q_lens), 2 * hkv, d), 1.0), cuda_device, dtype)
    cu_q, cu_k = (torch.tensor([0, *np.cumsum(x)], dtype=torch.int32, device=cuda_device) for x in (q_lens, ctxs))
    scale = 14.0 / d  # the sink is exp(14) = 2^20 above the others
    got = mi.paged_prefill_mxfp4(query, _cuda(kp, cuda_device), _cuda(vp, cuda_device), cu_q, cu_k, _cuda(table, cuda_device),
                                 max_seqlen_q=max(q_lens), total_k=sum(ctxs), scale=scale)
    mi.check_device_status(cuda_device)
    q, at = query.double().cpu().numpy(), np.cumsum([0, *q_lens])
    parts = [mo.attention(q[at[r]:at[r + 1]], mo.rows(kp, table[r], c), mo.rows(vp, table[r], c), scale)
             for r, c in enumerate(ctxs)]
    want, weight, size, floor = (np.concatenate(x) for x in zip(*parts))
    assert 0.0001 < np.abs(want).max() < 0.1
    _close(got, want, weight, size, 4 * floor, dtype, PREFILL_STEP[dtype])
