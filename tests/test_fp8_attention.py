"""Decode and prefill over the 8-bit cache against the formula in 64 bits (bounds: fp8_support.py), and runs of the
operators together."""

import numpy as np
import pytest
import torch

import microinfer_b200 as mi
from microinfer_b200 import _lib
from oracle import fp8_oracle as fo
from tests.fp8_support import (
    DECODE_STEP,
    DTYPES,
    PREFILL_STEP,
    close,
    cuda,
    decode_case,
    pages,
    prefill_case,
    table_of,
)

gpu = pytest.mark.gpu
DENSE_LOST = 2.0 ** -31


def _place(pos, table, bs=16):
    """(page, group, token) of a position."""
    return int(table[pos // bs]), pos % bs // 16, pos % 16


def _set_code(page, value, where, head, dim, code):
    block, group, tok = where
    d = page.shape[-1] // 16 - 1
    page[block, head, group, fo._place(d, value)[tok, dim]] = code


def _set_byte(page, block, group, head, byte):
    page[block, head, group, page.shape[-1] - 16] = byte


# ---------------------------------------------------------------------------
# decode
# ---------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hkv,group,d,bs", [
    (8, 2, 128, 16), (2, 7, 64, 64), (1, 16, 128, 32), (4, 1, 64, 16), (2, 5, 128, 256), (1, 12, 64, 16),
    (1, 4, 96, 32), (2, 3, 32, 16), (1, 2, 256, 16), (2, 8, 160, 16), (1, 1, 128, 16), (1, 17, 64, 48)])
def test_decode_matches_the_formula(cuda_device, name, hkv, group, d, bs):
    ctxs = [1, 2, 15, 16, 17, 0, 31, 33, 129, 300, 257]
    got, want = decode_case(cuda_device, name, hkv, group, d, bs, ctxs)
    mi.check_device_status(cuda_device)
    close(got, *want, DECODE_STEP[DTYPES[name]])
    assert bool((got[5] == 0).all())  # no key: zeros


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("ctxs", [[5000], [4096, 1, 0, 2777], [1], [0], [0, 0, 16], [20000, 3]])
@pytest.mark.parametrize("hkv,group,d,bs", [(2, 4, 128, 16), (1, 8, 64, 64)])
def test_decode_splits_long_contexts(cuda_device, name, ctxs, hkv, group, d, bs):
    got, want = decode_case(cuda_device, name, hkv, group, d, bs, ctxs)
    mi.check_device_status(cuda_device)
    close(got, *want, DECODE_STEP[DTYPES[name]])


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("group", [1, 6, 9])
def test_decode_every_head_dim(cuda_device, name, d, group):
    """Long and short contexts of every head_dim, scales far apart, sequences that cross CTAs."""
    ctxs = [7000, 0, 1, 31, 33, 1500]
    got, want = decode_case(cuda_device, name, 2, group, d, 32, ctxs, spread=6.0)
    mi.check_device_status(cuda_device)
    assert bool((got[1] == 0).all())
    close(got, *want, DECODE_STEP[DTYPES[name]])


@gpu
@pytest.mark.parametrize("count,most", [(400, 90), (2500, 20)])
def test_decode_many_sequences(cuda_device, count, most):
    """More sequences than CTAs, and more than one launch takes."""
    ctxs = np.random.default_rng(9).integers(0, most, count).tolist()
    got, want = decode_case(cuda_device, "bf16", 2, 4, 64, 16, ctxs)
    mi.check_device_status(cuda_device)
    close(got, *want, DECODE_STEP[torch.bfloat16])


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("spread,scale", [(4.0, None), (8.0, None), (0.5, 3.0), (0.5, 0.0), (0.5, -0.2)])
def test_decode_uneven_scales_and_sharp_softmax(cuda_device, name, spread, scale):
    """Groups of V whose scales differ by up to 2^46; scores far apart, all equal, and with the sign turned."""
    got, want = decode_case(cuda_device, name, 2, 4, 128, 16, [700, 40, 16, 1], seed=3, spread=spread, scale=scale)
    mi.check_device_status(cuda_device)
    close(got, *want, DECODE_STEP[DTYPES[name]])


@gpu
@pytest.mark.parametrize("prefill", [False, True])
@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_large_values_with_no_weight(cuda_device, name, prefill):
    """Groups whose keys get no weight carry V of 2^40, the ones with weight V of 2^-30: nothing is lost."""
    rng = np.random.default_rng(2)
    d, ctx = 64, 130
    code = fo.codes_of(np.abs(rng.standard_normal((9, 16, 1, d))) + 0.5)
    heavy = np.arange(9) % 3 == 1
    kp = fo.pack(code, np.where(heavy, 127, 60).astype(np.uint8)[:, None, None], False)
    vp = fo.pack(fo.codes_of(rng.standard_normal((9, 16, 1, d))), np.where(heavy, 97, 167).astype(np.uint8)[:, None, None], True)
    table = np.arange(9, dtype=np.int32)[None]
    query = cuda(np.abs(rng.standard_normal((1, 4, d))) + 0.5, cuda_device, DTYPES[name])
    want = fo.attention(query.double().cpu().numpy(), kp, vp, table[0], ctx, 6.0)
    args = cuda(kp, cuda_device), cuda(vp, cuda_device)
    lens = torch.tensor([ctx], dtype=torch.int32, device=cuda_device)
    if prefill:
        cu = torch.tensor([0, 1], dtype=torch.int32, device=cuda_device)
        got = mi.paged_prefill_fp8(query, *args, cu, cu * ctx, cuda(table, cuda_device), max_seqlen_q=1, scale=6.0)
    else:
        got = mi.paged_decode_fp8(query, *args, cuda(table, cuda_device), lens, scale=6.0)
    close(got, *want, DECODE_STEP[DTYPES[name]], lost=0.0)  # what the large ones lose of p is nothing


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("k_byte,q_power,v_byte", [(246, -100, 246), (1, 90, 1), (246, 0, 127), (127, -120, 200), (20, 20, 10)])
def test_decode_and_prefill_over_the_whole_range_of_scales(cuda_device, name, k_byte, q_power, v_byte):
    if name == "f16":  # q, and the results of a small or large V, do not reach further
        q_power, v_byte = max(-14, min(8, q_power)), max(118, min(130, v_byte))
    rng = np.random.default_rng(abs(q_power) + k_byte)
    d, ctx = 64, 70
    dtype = DTYPES[name]
    kb = np.clip(k_byte - rng.integers(0, 3, (5, 1, 1)), 1, 246).astype(np.uint8)
    vb = np.clip(v_byte - rng.integers(0, 3, (5, 1, 1)), 1, 246).astype(np.uint8)
    kp = fo.pack(fo.codes_of(30 * rng.standard_normal((5, 16, 1, d))), kb, False)
    vp = fo.pack(fo.codes_of(30 * rng.standard_normal((5, 16, 1, d))), vb, True)
    query = cuda(rng.standard_normal((3, 3, d)) * 2.0 ** q_power, cuda_device, dtype)
    scale = float(np.float32(2.0 ** np.clip(127 - k_byte - q_power - 6, -100, 100)))  # scores of about 1
    table = np.arange(5, dtype=np.int32)[None]
    pool = cuda(kp, cuda_device), cuda(vp, cuda_device)
    want = fo.attention(query.double().cpu().numpy(), kp, vp, table[0], ctx, scale)
    cu = torch.tensor([0, 3], dtype=torch.int32, device=cuda_device)
    ck = torch.tensor([0, ctx], dtype=torch.int32, device=cuda_device)
    got = mi.paged_prefill_fp8(query, *pool, cu, ck, cuda(table, cuda_device), max_seqlen_q=3, scale=scale)
    close(got, *want, PREFILL_STEP[dtype])
    step = mi.paged_decode_fp8(query[2:], *pool, cuda(table, cuda_device), ck[1:], scale=scale)
    close(step, *(x[2:] for x in want), DECODE_STEP[dtype])
    mi.check_device_status(cuda_device)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
def test_decode_many_keys_of_little_weight(cuda_device, name):
    """One key takes nearly everything and its value is zero: the rest of a long context, each key about 2^-20
    of it, decides the result."""
    ctx, d = 9000, 64
    rng = np.random.default_rng(22)
    nb = ctx // 16 + 2
    k = rng.standard_normal((nb, 16, 1, d)) * 0.01
    v = rng.standard_normal((nb, 16, 1, d)) + 1.0
    table = table_of(rng, [ctx], nb, 16)
    k[table[0, 3], 5], v[table[0, 3], 5] = 1.0, 0.0
    kp, vp = fo.pack(*fo.encode(k), False), fo.pack(*fo.encode(v), True)
    query = cuda(np.full((1, 4, d), 1.0), cuda_device, DTYPES[name])
    scale = 14.0 / d  # the sink is exp(14) = 2^20 above the others
    got = mi.paged_decode_fp8(query, cuda(kp, cuda_device), cuda(vp, cuda_device), cuda(table, cuda_device),
                              torch.tensor([ctx], dtype=torch.int32, device=cuda_device), scale=scale)
    want = fo.attention(np.full((1, 4, d), 1.0), kp, vp, table[0], ctx, scale)
    assert 0.001 < np.abs(want[0]).max() < 0.1
    close(got, *want, DECODE_STEP[DTYPES[name]])


@gpu
@pytest.mark.parametrize("prefill", [False, True])
@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 256])
def test_what_lies_past_the_context_is_ignored(cuda_device, name, d, prefill):
    """Codes past the context are NaN, scales of groups and pages past it the largest; columns past it bad ids."""
    ctxs = [5, 16, 21, 40]

    def edit(kp, vp, table):
        for page, value in ((kp, False), (vp, True)):
            code, byte = fo.unpack(page, value)
            tokens, groups = (np.zeros(x.shape[:2], dtype=bool) for x in (code, byte))
            for r, c in enumerate(ctxs):
                for pos in range(c):
                    block, group, tok = _place(pos, table[r])
                    tokens[block, tok] = groups[block, group] = True
            code[~tokens] = 127
            byte[~groups] = 255
            page[:] = fo.pack(code, byte, value)
        if not prefill:
            for r, c in enumerate(ctxs):
                table[r, -(-c // 16):] = 1 << 30

    if prefill:
        got, _, want = prefill_case(cuda_device, name, 2, 2, d, 16, [1, 16, 3, 30], ctxs, edit=edit)
        close(got, *want, PREFILL_STEP[DTYPES[name]])
    else:
        got, want = decode_case(cuda_device, name, 2, 2, d, 16, ctxs, edit=edit)
        close(got, *want, DECODE_STEP[DTYPES[name]])
    mi.check_device_status(cuda_device)


@gpu
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_decode_nan_codes_and_zero_groups(cuda_device, d, name):
    """A NaN of V is NaN in its dim of its sequence alone, one of K in all of them; groups of scale 0 are zeros, whatever
    their codes."""
    rng = np.random.default_rng(d)
    kp, vp = pages(rng, 12, 16, 1, d)
    _set_code(vp, True, (2, 0, 5), 0, d - 3, 127)
    _set_code(kp, False, (9, 0, 0), 0, 7, 255)
    _set_byte(vp, 6, 0, 0, 0)
    _set_byte(kp, 5, 0, 0, 0)
    table = np.arange(12, dtype=np.int32).reshape(3, 4)
    query = torch.randn(3, 4, d, device=cuda_device).to(DTYPES[name])
    got = mi.paged_decode_fp8(query, cuda(kp, cuda_device), cuda(vp, cuda_device), cuda(table, cuda_device),
                              torch.full((3,), 60, dtype=torch.int32, device=cuda_device))
    nan = torch.isnan(got)
    assert bool(nan[0, :, d - 3].all()) and int(nan[0].sum()) == 4
    assert not bool(nan[1].any()) and bool(nan[2].all())
    want = fo.attention(query[1:2].double().cpu().numpy(), kp, vp, table[1], 60, d ** -0.5)
    close(got[1:2], *want, DECODE_STEP[DTYPES[name]])


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
def test_decode_query_values_of_any_size(cuda_device, name):
    """Queries of very small and large magnitude, a zero row, and rows that are not finite."""
    rng = np.random.default_rng(5)
    dtype = DTYPES[name]
    kp, vp = pages(rng, 6, 16, 1, 64)
    sizes = {"f16": [2.0 ** -14, 2.0 ** 9, 0.0, 1.0], "bf16": [2.0 ** -100, 2.0 ** 90, 0.0, 1.0],
             "f32": [2.0 ** -100, 2.0 ** 90, 0.0, 1.0]}[name]
    table = np.array([[0, 1, 2]] * 4, dtype=np.int32)
    query = cuda(rng.standard_normal((4, 4, 64)) * np.array(sizes)[:, None, None], cuda_device, dtype)
    query[3, 1, 5] = float("nan")
    query[3, 2, 6] = float("inf")
    pool = cuda(kp, cuda_device), cuda(vp, cuda_device)
    got = mi.paged_decode_fp8(query, *pool, cuda(table, cuda_device),
                              torch.full((4,), 40, dtype=torch.int32, device=cuda_device))
    q = query.double().cpu().numpy()
    k, v = fo.rows(kp, table[0], 40, False), fo.rows(vp, table[0], 40, True)
    for r in (0, 2, 3):
        heads = [0, 3] if r == 3 else [0, 1, 2, 3]
        close(got[r:r + 1, heads], *fo.attention(q[r:r + 1, heads], kp, vp, table[0], 40, 0.125), DECODE_STEP[dtype])
    if name == "f16":
        close(got[1:2], *fo.attention(q[1:2], kp, vp, table[0], 40, 0.125), DECODE_STEP[dtype])
    else:  # scores of 2^90: the largest takes everything
        best = np.argmax(q[1] @ k[:, 0].T, -1)
        assert np.array_equal(got[1].double().cpu().numpy(), cuda(v[best, 0], cuda_device, dtype).double().cpu().numpy())
    assert bool(torch.isnan(got[3, 1:3]).all())


@gpu
@pytest.mark.parametrize("name,d,bs", [("bf16", 128, 16), ("bf16", 64, 64), ("f32", 96, 32)])
def test_decode_flags_bad_pages_and_lengths(cuda_device, name, d, bs):
    """Pages that are none are left out and flagged; a length past the table's columns is clamped to them, a negative
    one is none."""
    rng = np.random.default_rng(6)
    kp, vp = pages(rng, 5, bs, 1, d)
    query = torch.randn(2, 4, d, device=cuda_device).to(DTYPES[name])
    args = (query, cuda(kp, cuda_device), cuda(vp, cuda_device))

    def run(table, lens):
        return mi.paged_decode_fp8(*args, torch.tensor(table, dtype=torch.int32, device=cuda_device),
                                   torch.tensor(lens, dtype=torch.int32, device=cuda_device))

    got = run([[0, 7, 2], [-1, 3, 4]], [2 * bs + 5, 3 * bs - 1])
    assert mi.read_device_status(cuda_device) == _lib.DEV_BAD_BLOCK
    q = query.double().cpu().numpy()
    for r, (named, ctx) in enumerate((([0, 2], bs + 5), ([3, 4], 2 * bs - 1))):
        close(got[r:r + 1], *fo.attention(q[r:r + 1], kp, vp, np.array(named), ctx, d ** -0.5), DECODE_STEP[DTYPES[name]])
    full = run([[0, 3], [1, 2]], [2 * bs, 2 * bs])
    assert mi.read_device_status(cuda_device) == 0
    long = run([[0, 3], [1, 2]], [100000, -5])
    assert mi.read_device_status(cuda_device) == _lib.DEV_BAD_BLOCK
    assert torch.equal(long[0], full[0]) and bool((long[1] == 0).all())


@gpu
@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_decode_views_and_out(cuda_device, name):
    """A query that is a view, int64 tables, an output given by the caller, a table without columns."""
    rng = np.random.default_rng(7)
    dtype = DTYPES[name]
    ctxs = [30, 9, 64]
    kp, vp = pages(rng, 9, 16, 2, 64)
    table = cuda(table_of(rng, ctxs, 9, 16), cuda_device)
    lens = torch.tensor(ctxs, dtype=torch.int32, device=cuda_device)
    pool = cuda(kp, cuda_device), cuda(vp, cuda_device)
    query = torch.randn(3, 12, 64, device=cuda_device).to(dtype)[:, 2:10]
    want = mi.paged_decode_fp8(query.contiguous(), *pool, table, lens)
    out = torch.empty(3, 8, 64, dtype=dtype, device=cuda_device)
    assert mi.paged_decode_fp8(query, *pool, table.long(), lens.long(), out=out) is out
    assert torch.equal(out, want)  # the same order of sums, whatever the strides
    none = mi.paged_decode_fp8(query, *pool, table[:, :0], lens)
    assert bool((none == 0).all())
    assert mi.paged_decode_fp8(query[:0], *pool, table[:0], lens[:0]).shape == (0, 8, 64)


@gpu
def test_cache_past_32_bit_offsets(cuda_device):
    """Pages that lie more than 4 GiB into the pool are stored, gathered and attended to."""
    hkv, d, bs = 8, 128, 64
    nb = (1 << 32) // (hkv * 4 * 2064) + 40
    kt = torch.zeros(nb, hkv, 4, 2064, dtype=torch.uint8, device=cuda_device)
    vt = torch.zeros_like(kt)
    rng = np.random.default_rng(8)
    table = np.array([[nb - 1, nb - 7] + list(range(nb - 30, nb - 20))], dtype=np.int32)
    for ctx in (100, 700):  # the two ways of finding groups
        pos = np.arange(ctx)
        slots = table[0, pos // bs].astype(np.int64) * bs + pos % bs
        rows = cuda(rng.standard_normal((2, ctx, hkv, d)), cuda_device, torch.bfloat16)
        mi.store_kv_fp8(kt, vt, cuda(slots, cuda_device), rows[0], rows[1])
        tt = cuda(table, cuda_device)
        some = [t[nb - 40:].cpu().numpy() for t in (kt, vt)]
        near = table[0] - (nb - 40)
        want = [fo.rows(some[0], near, ctx, False), fo.rows(some[1], near, ctx, True)]
        for got, w, x in zip(mi.gather_paged_kv_fp8(kt, vt, tt, [ctx]), want, rows):
            assert np.array_equal(got.double().cpu().numpy(), w)
            assert float((got - x).abs().max()) < 0.3  # 2^-4 of values below 4.5
        assert int(kt[:nb - 40].max()) == 0
        query = cuda(rng.standard_normal((1, 16, d)), cuda_device, torch.bfloat16)
        got = mi.paged_decode_fp8(query, kt, vt, tt, torch.tensor([ctx], dtype=torch.int32, device=cuda_device))
        close(got, *fo.attention(query.double().cpu().numpy(), *some, near, ctx, d ** -0.5), DECODE_STEP[torch.bfloat16])
        cu = torch.tensor([0, 1], dtype=torch.int32, device=cuda_device)
        got = mi.paged_prefill_fp8(query, kt, vt, cu, cu * ctx, tt, max_seqlen_q=1)
        close(got, *fo.attention(query.double().cpu().numpy(), *some, near, ctx, d ** -0.5), PREFILL_STEP[torch.bfloat16])
    mi.check_device_status(cuda_device)


# ---------------------------------------------------------------------------
# prefill
# ---------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hkv,group,d,bs", [
    (8, 2, 128, 16), (2, 4, 64, 64), (1, 3, 96, 32), (2, 7, 128, 32), (1, 5, 64, 16), (1, 16, 64, 256), (4, 1, 128, 48)])
def test_prefill_matches_the_formula(cuda_device, name, hkv, group, d, bs):
    q_lens, ctxs = [1, 40, 7, 130, 1], [90, 40, 135, 201, 1]
    got, free, want = prefill_case(cuda_device, name, hkv, group, d, bs, q_lens, ctxs)
    for x in (got, free):  # the bound on the contexts only decides the split over the keys
        close(x, *want, PREFILL_STEP[DTYPES[name]], lost=DENSE_LOST)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("group", [1, 5])
def test_prefill_every_head_dim(cuda_device, name, d, group):
    """Chunks of one token and of several tiles, a context split over its keys; in shapes that are computed
    from the pages also a context shorter than its chunk, whose first rows see no key."""
    short = d != 128 or name == "f32"
    q_lens, ctxs = [140, 1, 3, 20, 9], [140, 3000, 3, 77, 5 if short else 9]
    got, free, want = prefill_case(cuda_device, name, 2, group, d, 32, q_lens, ctxs)
    if short:
        assert bool((got[164:168] == 0).all())
    for x in (got, free):
        close(x, *want, PREFILL_STEP[DTYPES[name]], lost=DENSE_LOST)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("q_lens,ctxs", [([3], [5000]), ([64], [2000]), ([1, 17], [4097, 63]), ([33], [33])])
def test_prefill_small_chunks_over_long_contexts(cuda_device, name, d, q_lens, ctxs):
    got, free, want = prefill_case(cuda_device, name, 2, 4, d, 16, q_lens, ctxs)
    for x in (got, free):
        close(x, *want, PREFILL_STEP[DTYPES[name]])


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("spread,scale", [(0.5, 2.0), (0.5, 0.0), (0.5, -0.3), (5.0, None)])
def test_prefill_scales(cuda_device, name, spread, scale):
    got, _, want = prefill_case(cuda_device, name, 1, 3, 64, 16, [50, 20], [70, 150], scale=scale, spread=spread)
    close(got, *want, PREFILL_STEP[DTYPES[name]])


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("large", [False, True])
def test_prefill_nan_codes_reach_only_rows_that_see_them(cuda_device, name, d, large):
    """A NaN value of a key in the chunk: NaN in its dim for the rows from it on; a NaN key: those rows alone.
    `large`: enough tiles for the dense kernel, where it takes the shape."""
    def edit(kp, vp, table):
        _set_code(vp, True, _place(60, table[0]), 0, d - 5, 127)  # position 60 of 90, row 10 of 40
        _set_code(vp, True, _place(63, table[0]), 0, 2, 255)
        _set_code(kp, False, _place(80, table[0]), 0, 3, 127)     # position 80, row 30

    hkv, group = (16, 2) if large else (1, 3)
    more = [40] * 4 if large else []
    got, _, want = prefill_case(cuda_device, name, hkv, group, d, 16, [40, *more], [90, *more], edit=edit)
    nan = torch.isnan(got).cpu()
    seen = nan[:40, :group]
    assert not bool(seen[:10].any()) and bool(seen[30:].all())
    assert bool(seen[10:30, :, d - 5].all()) and bool(seen[13:30, :, 2].all()) and int(seen[10:30].sum()) == (20 + 17) * group
    assert int(nan.sum()) == int(seen.sum())
    keep = ~nan[:, :, 0].numpy() & ~nan[:, :, 2].numpy() & ~nan[:, :, d - 5].numpy()
    sub = [x[keep] for x in want]
    close(got[torch.from_numpy(keep).to(got.device)], *sub, PREFILL_STEP[DTYPES[name]], lost=DENSE_LOST)


@gpu
@pytest.mark.parametrize("operand", ["keys", "values"])
@pytest.mark.parametrize("hkv,d", [(16, 128), (1, 128), (1, 64)])
def test_prefill_in_fp16_of_what_fp16_does_not_hold(cuda_device, operand, hkv, d):
    """Groups that reach 2^17 to 2^40: their keys' scores and their values count, in the rows that see them."""
    def edit(kp, vp, table):
        for i, pos in enumerate((17, 40, 70)):
            if operand == "values":
                _set_byte(vp, table[0, pos // 16], 0, 0, 127 + [9, 12, 32][i])
            else:
                _set_byte(kp, table[0, pos // 16], 0, 0, 127 + [9, 12, 32][i])

    scale = d ** -0.5 if operand == "values" else 2.0 ** -36
    got, free, want = prefill_case(cuda_device, "f16", hkv, 2, d, 16, [86, 40, 40, 40], [90, 40, 40, 40], edit=edit, scale=scale)
    for x in (got, free):
        close(x, *want, PREFILL_STEP[torch.float16], lost=DENSE_LOST)
    if operand == "values":
        assert bool(torch.isfinite(got[0]).all())  # position 4: before the first of them


@gpu
@pytest.mark.parametrize("hkv,d", [(1, 64), (1, 128), (16, 128)])
def test_prefill_leaves_rows_of_no_sequence_and_leaves_out_bad_pages(cuda_device, hkv, d):
    rng = np.random.default_rng(31)
    kp, vp = pages(rng, 12, 16, hkv, d)
    q_lens, ctxs = [3, 5, 30, 40], [20, 43, 30, 40]
    rows = sum(q_lens) + 4
    query = torch.randn(rows, 2 * hkv, d, device=cuda_device, dtype=torch.float16)
    cu_q, cu_k = (torch.tensor([0, *np.cumsum(x)], dtype=torch.int32, device=cuda_device) for x in (q_lens, ctxs))
    table = np.array([[0, 1, -1], [2, 3, 4], [5, 6, -1], [7, 8, 9]], dtype=np.int32)
    out = torch.full_like(query, 7.0)
    pool = cuda(kp, cuda_device), cuda(vp, cuda_device)
    mi.paged_prefill_fp8(query, *pool, cu_q, cu_k, cuda(table, cuda_device), max_seqlen_q=40, out=out)
    mi.check_device_status(cuda_device)
    assert bool((out[-4:] == 7.0).all()) and not bool((out[:-4] == 7.0).all(-1).any())
    table[1, 1] = 12
    got = mi.paged_prefill_fp8(query, *pool, cu_q, cu_k, cuda(table, cuda_device), max_seqlen_q=40)
    assert mi.read_device_status(cuda_device) == _lib.DEV_BAD_BLOCK
    q = query[3:8].double().cpu().numpy()
    want = fo.attention(q, kp, vp, np.array([2, 4]), 27, d ** -0.5)  # rows at positions 38 to 42 of 43: all past page 1
    close(got[3:8], *want, PREFILL_STEP[torch.float16], lost=DENSE_LOST)
    keep = [i for i in range(rows - 4) if not 3 <= i < 8]
    assert torch.equal(got[keep], out[keep])
    # a context past the table's columns
    far = cu_k.clone()
    far[2:] += 40
    mi.paged_prefill_fp8(query, *pool, cu_q, far, cuda(table, cuda_device), max_seqlen_q=40)
    assert mi.read_device_status(cuda_device) & _lib.DEV_BAD_BLOCK


# ---------------------------------------------------------------------------
# runs of them together
# ---------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hkv,d,bs", [(2, 128, 16), (1, 64, 32), (2, 96, 16), (1, 256, 16)])
def test_a_prompt_in_chunks_then_tokens(cuda_device, name, hkv, d, bs):
    """CachedAttention on an 8-bit layer: two prefill chunks, then decode steps, then a fork by copy-on-write."""
    from microinfer_b200.layer.cached_attention import CachedAttention
    from microinfer_b200.layer.metadata import AttentionMetadata

    dtype = DTYPES[name]
    gen = torch.Generator().manual_seed(11)
    hq = 4 * hkv
    pool = mi.FP8KVCache(1, 12, bs, hkv, d, device=cuda_device)
    pool.keys.fill_(0x5a)  # a last owner's codes and scales
    pool.values.fill_(0x5a)
    attn = CachedAttention()
    attn.bind_cache(pool.layer(0))
    tables = [[3, 7, 1, 10], [0, 5, 2]]
    table = torch.full((2, 4), -1, dtype=torch.int32)
    for r, t in enumerate(tables):
        table[r, :len(t)] = torch.tensor(t)
    lens = [0, 0]
    state = [fo.unpack(p.cpu().numpy()[0], value) for p, value in ((pool.keys, False), (pool.values, True))]

    def step(new, prefill):
        q, k, v = (torch.randn(sum(new), h, d, generator=gen).to(dtype).to(cuda_device) for h in (hq, hkv, hkv))
        slots = []
        for r, n in enumerate(new):
            slots += [tables[r][pos // bs] * bs + pos % bs for pos in range(lens[r], lens[r] + n)]
            lens[r] += n
        for (code, byte), x in zip(state, (k, v)):
            fo.store(code, byte, slots, x.double().cpu().numpy())
        kp, vp = (fo.pack(*s, value) for s, value in zip(state, (False, True)))
        at = np.cumsum([0, *new])
        want = [fo.attention(q[at[r]:at[r + 1]].double().cpu().numpy(), kp, vp, tables[r], lens[r], d ** -0.5)
                for r in range(2)]
        fields = dict(slot_mapping=torch.tensor(slots, dtype=torch.int32, device=cuda_device),
                      block_tables=table.to(cuda_device))
        if prefill:
            cu_q, cu_k = (torch.tensor([0, *np.cumsum(x)], dtype=torch.int32, device=cuda_device) for x in (new, lens))
            meta = AttentionMetadata.build(is_prefill=True, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k,
                                           max_seqlen_q=max(new), max_seqlen_k=max(lens), **fields)
        else:
            meta = AttentionMetadata.build(is_prefill=False, validate_cache_write=False,
                                           context_lens=torch.tensor(lens, dtype=torch.int32, device=cuda_device),
                                           **fields)
        close(attn(q, k, v, meta), *(np.concatenate(x) for x in zip(*want)),
              (PREFILL_STEP if prefill else DECODE_STEP)[dtype], lost=DENSE_LOST)

    step([20, 9], True)
    step([23, 20], True)
    for _ in range(4):
        step([1, 1], False)
    # sequence 1 goes on in a private copy of its last page
    last = (lens[1] - 1) // bs
    pool.copy_blocks([(tables[1][last], 9)])
    for code, byte in state:
        code[9], byte[9] = code[tables[1][last]], byte[tables[1][last]]
    tables[1][last] = 9
    table[1, last] = 9
    step([1, 1], False)
    mi.check_device_status(cuda_device)


@gpu
def test_graphs_and_eager_calls_on_their_own_streams(cuda_device):
    """Captured steps (store, decode, prefill) replayed together on two streams, with an eager one beside them, share
    nothing."""
    rng = np.random.default_rng(12)
    ctxs = [3000, 17, 800]
    cases = []
    for _ in range(3):
        kp, vp = pages(rng, 260, 16, 2, 128)
        table = table_of(rng, ctxs, 260, 16)
        query = torch.randn(3, 8, 128, device=cuda_device, dtype=torch.bfloat16)
        lens = torch.tensor(ctxs, dtype=torch.int32, device=cuda_device)
        cu_k = torch.tensor([0, *np.cumsum(ctxs)], dtype=torch.int32, device=cuda_device)
        pos = np.arange(2000, 2700)
        slots = cuda((table[0, pos // 16].astype(np.int64) * 16 + pos % 16), cuda_device)
        rows = torch.randn(2, 700, 2, 128, device=cuda_device, dtype=torch.bfloat16)
        cases.append((query, cuda(kp, cuda_device), cuda(vp, cuda_device), cuda(table, cuda_device), lens, cu_k, slots, rows))
    cu_q = torch.arange(4, dtype=torch.int32, device=cuda_device)

    def run(c):
        mi.store_kv_fp8(c[1], c[2], c[6], *c[7])
        return (mi.paged_decode_fp8(*c[:5]),
                mi.paged_prefill_fp8(c[0], c[1], c[2], cu_q, c[5], c[3], max_seqlen_q=1, total_k=sum(ctxs)))

    want = [run(c) for c in cases]
    streams = [torch.cuda.Stream(cuda_device) for _ in range(3)]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for c, s in zip(cases[:2], streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(run(c))
        graphs.append(g)
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            third = run(cases[2])
        torch.cuda.synchronize()
        for got, w in zip([*outs, third], want):
            assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])
    mi.check_device_status(cuda_device)


@gpu
def test_under_torch_compile(cuda_device):
    rng = np.random.default_rng(13)
    kp, vp = pages(rng, 6, 16, 2, 64)
    kt, vt = cuda(kp, cuda_device), cuda(vp, cuda_device)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=cuda_device)
    lens = torch.tensor([20, 32], dtype=torch.int32, device=cuda_device)
    cu_q = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda_device)
    cu_k = torch.tensor([0, 20, 52], dtype=torch.int32, device=cuda_device)
    slots = torch.tensor([1 * 16 + 3, 3 * 16 + 15], dtype=torch.int32, device=cuda_device)
    heads_first = torch.randn(4, 2, 64, device=cuda_device, dtype=torch.bfloat16)
    k, v = (torch.randn(2, 2, 64, device=cuda_device, dtype=torch.bfloat16) for _ in range(2))

    def fn(x, k, v, kt, vt):
        q = x.transpose(0, 1)
        mi.store_kv_fp8(kt, vt, slots, k, v)
        a = mi.paged_decode_fp8(q, kt, vt, table, lens)
        b = mi.paged_prefill_fp8(q, kt, vt, cu_q, cu_k, table, max_seqlen_q=1)
        return a.view(2, 256), b.view(2, 256)

    want = fn(heads_first, k, v, kt.clone(), vt.clone())
    got = torch.compile(fn, fullgraph=True, backend="aot_eager")(heads_first, k, v, kt, vt)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("hkv,d", [(2, 64), (2, 96), (2, 128), (16, 128)])
def test_results_over_the_query_and_shared_pages(cuda_device, name, hkv, d):
    """`out` may be the query itself; rows of the table may name the same pages, and one page twice."""
    rng = np.random.default_rng(15)
    dtype = DTYPES[name]
    kp, vp = pages(rng, 40, 16, hkv, d)
    pool = cuda(kp, cuda_device), cuda(vp, cuda_device)
    one = rng.integers(0, 40, 200).astype(np.int32)
    one[7] = one[3]
    names = [one, one, one[::-1]]
    table = cuda(np.stack(names), cuda_device)
    lens = torch.tensor([3200, 3185, 1700], dtype=torch.int32, device=cuda_device)
    query = cuda(rng.standard_normal((3, 4 * hkv, d)), cuda_device, dtype)
    q = query.double().cpu().numpy()
    parts = [fo.attention(q[r:r + 1], kp, vp, names[r], int(c), d ** -0.5) for r, c in enumerate(lens.tolist())]
    want = [np.concatenate(x) for x in zip(*parts)]
    over = query.clone()
    assert mi.paged_decode_fp8(over, *pool, table, lens, out=over) is over
    close(over, *want, DECODE_STEP[dtype])
    over = query.clone()
    cu_q = torch.arange(4, dtype=torch.int32, device=cuda_device)
    cu_k = torch.cat([cu_q[:1], lens.cumsum(0).int()])
    mi.paged_prefill_fp8(over, *pool, cu_q, cu_k, table, max_seqlen_q=1, out=over)
    close(over, *want, PREFILL_STEP[dtype])
    mi.check_device_status(cuda_device)
