"""Attention over the 8-bit cache where its ways of computing could part: values that are nowhere finite, groups of scale 0,
scales and scores at the ends of the range (bounds: fp8_support.py).  Prefill's cases run in each of its ways."""

import numpy as np
import pytest
import torch

import microinfer_b200 as mi
from oracle import fp8_oracle as fo
from tests.fp8_support import DECODE_STEP, DTYPES, PREFILL_STEP, close, cuda, pages, prefill_case, table_of
from tests.test_fp8_attention import DENSE_LOST, _place, _set_byte, _set_code
from tests.test_fp8_prefill_ways import way  # noqa: F401  (a fixture)

gpu = pytest.mark.gpu


def _same(got, want, step, lost=DENSE_LOST):
    """NaN exactly where the formula has it, and the bound elsewhere."""
    nan = np.isnan(want[0])
    assert np.array_equal(torch.isnan(got).cpu().numpy(), nan)
    got = torch.where(torch.from_numpy(nan).to(got.device), torch.zeros_like(got), got)
    close(got, np.where(nan, 0.0, want[0]), *want[1:], step, lost=lost)


def _attend(device, query, kp, vp, tables, q_lens, ctxs, scale, decode=False):
    """The operators' result and the formula's."""
    cu_q, cu_k = (torch.tensor([0, *np.cumsum(x)], dtype=torch.int32, device=device) for x in (q_lens, ctxs))
    pool = cuda(kp, device), cuda(vp, device)
    table = cuda(np.asarray(tables, dtype=np.int32), device)
    if decode:
        got = mi.paged_decode_fp8(query, *pool, table, torch.tensor(ctxs, dtype=torch.int32, device=device), scale=scale)
    else:
        got = mi.paged_prefill_fp8(query, *pool, cu_q, cu_k, table, max_seqlen_q=max(q_lens), total_k=sum(ctxs), scale=scale)
    mi.check_device_status(device)
    q = query.double().cpu().numpy()
    at = np.cumsum([0, *q_lens])
    parts = [fo.attention(q[at[r]:at[r + 1]], kp, vp, tables[r], c, scale) for r, c in enumerate(ctxs)]
    return got, [np.concatenate(x) for x in zip(*parts)]


# ---------------------------------------------------------------------------
# values that are nowhere finite: their group's scale is 0
# ---------------------------------------------------------------------------
def _stored_rows_that_are_not_finite(device, dtype, d):
    """Pages as the store leaves them of rows of V without a finite element (but zeros), and tables and contexts."""
    rng = np.random.default_rng(d)
    hkv = 2
    kt = torch.zeros(14, hkv, 1, 16 * d + 16, dtype=torch.uint8, device=device)
    vt = torch.zeros_like(kt)
    tables = [[3, 1, 0, 5, 9, 7], [2, 4, 13], [6, -1, -1], [8, 10, 11]]
    tables = [t + [-1] * (6 - len(t)) for t in tables]
    q_lens, ctxs = [40, 33, 1, 40], [90, 33, 1, 40]
    k, v = (rng.standard_normal((sum(ctxs), hkv, d)) for _ in range(2))
    v[64:80, 0] = np.nan            # sequence 0: a whole group of head 0, beside finite ones
    v[16:32, 1] = 0.0               # zeros with one NaN among them, of head 1
    v[20, 1, 3] = np.inf
    v[90 + 32, :] = -np.inf         # sequence 1: the last group is one token
    v[90 + 33, 1] = np.nan          # sequence 2: the only key
    slots = np.concatenate([np.asarray(t)[np.arange(c) // 16] * 16 + np.arange(c) % 16 for t, c in zip(tables, ctxs)])
    mi.store_kv_fp8(kt, vt, cuda(slots, device), cuda(k, device, dtype), cuda(v, device, dtype))
    assert [int(vt[b, h, 0, 16 * d]) for b, h in ((9, 0), (1, 1), (13, 0), (13, 1), (6, 1))] == [0] * 5
    return kt.cpu().numpy(), vt.cpu().numpy(), tables, q_lens, ctxs


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
def test_prefill_of_values_that_are_nowhere_finite(cuda_device, way, name, d):  # noqa: F811
    """They are NaN in the rows that see them, and only there, though their group's scale is 0."""
    dtype = DTYPES[name]
    kp, vp, tables, q_lens, ctxs = _stored_rows_that_are_not_finite(cuda_device, dtype, d)
    query = cuda(np.random.default_rng(1).standard_normal((sum(q_lens), 4, d)), cuda_device, dtype)
    got, want = _attend(cuda_device, query, kp, vp, tables, q_lens, ctxs, d ** -0.5)
    nan = np.isnan(want[0])
    assert nan[:40, 2:, 3].all() and not nan[:14, :2].any() and nan[14:40, :2].all()
    assert nan[72].all() and not nan[40:72].any() and nan[73, 2:].all() and not nan[74:].any()
    _same(got, want, PREFILL_STEP[dtype])


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("where", [None, 0, 1403, 1950, 2047])
def test_prefill_of_zeros_with_one_nan(cuda_device, way, d, where):  # noqa: F811
    """Values that are zero throughout but for one that is NaN, or none: 128 groups of scale 0 to look through."""
    rng = np.random.default_rng(d)
    ctx, rows = 2048, 150
    kp, _ = pages(rng, ctx // 16, 16, 2, d)
    vp = np.zeros_like(kp)
    table = rng.permutation(ctx // 16).astype(np.int32)
    if where is not None:
        _set_code(vp, True, _place(where, table), 1, d - 7, 127)
    query = cuda(rng.standard_normal((rows, 4, d)), cuda_device, torch.bfloat16)
    got, _ = _attend(cuda_device, query, kp, vp, [table], [rows], [ctx], d ** -0.5)
    nan = torch.isnan(got)
    if where is None:
        assert bool((got == 0).all())
        return
    first = max(0, where - (ctx - rows))
    assert bool(nan[first:, 2:, d - 7].all()) and int(nan.sum()) == 2 * (rows - first)
    assert bool((got[~nan] == 0).all())


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("decode", [False, True])
def test_values_that_are_nowhere_finite(cuda_device, name, d, decode):
    """The same in decode, and in prefill of every type by the way that it chooses."""
    dtype = DTYPES[name]
    kp, vp, tables, q_lens, ctxs = _stored_rows_that_are_not_finite(cuda_device, dtype, d)
    if decode:
        q_lens = [1] * 4
    query = cuda(np.random.default_rng(2).standard_normal((sum(q_lens), 4, d)), cuda_device, dtype)
    got, want = _attend(cuda_device, query, kp, vp, tables, q_lens, ctxs, d ** -0.5, decode)
    assert np.isnan(want[0]).any()
    _same(got, want, (DECODE_STEP if decode else PREFILL_STEP)[dtype])


# ---------------------------------------------------------------------------
# groups of scale 0 are zeros, whatever their codes
# ---------------------------------------------------------------------------
def _zero_groups(device, name, d, operand, decode):
    rng = np.random.default_rng(d)
    dtype = DTYPES[name]
    kp, vp = pages(rng, 6, 16, 1, d)
    (kp if operand == "keys" else vp)[..., 16 * d] = 0
    ctxs, q_lens = [70], [1 if decode else 20]
    # queries so large that 2^-127, taken for 0, would give scores
    query = rng.standard_normal((sum(q_lens), 4, d)) * (1.0 if operand == "values" or name == "f16" else 2.0 ** 120)
    got, want = _attend(device, cuda(query, device, dtype), kp, vp, [[0, 1, 2, 3, 4, 5]], q_lens, ctxs, 1.0, decode)
    if operand == "values":
        assert bool((got == 0).all())
    else:  # the mean of V
        close(got, *want, (DECODE_STEP if decode else PREFILL_STEP)[dtype], lost=DENSE_LOST)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("operand", ["keys", "values"])
def test_prefill_over_groups_of_scale_zero(cuda_device, way, name, d, operand):  # noqa: F811
    _zero_groups(cuda_device, name, d, operand, False)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("operand", ["keys", "values"])
@pytest.mark.parametrize("d,decode", [(64, True), (96, True), (96, False), (128, False)])
def test_attention_over_groups_of_scale_zero(cuda_device, name, operand, d, decode):
    _zero_groups(cuda_device, name, d, operand, decode)


# ---------------------------------------------------------------------------
# NaN beside large scores
# ---------------------------------------------------------------------------
def _nan_beside_large_scores(device, name, where):
    """Chunks of 16 rows (one warp's) whose row 5 has scores past 2^21, with a NaN in row 9 of q or in key 0."""
    rng = np.random.default_rng(16)
    dtype, d = DTYPES[name], 64
    kp, vp = pages(rng, 4, 16, 1, d)
    if where == "key":
        _set_code(kp, False, (0, 0, 0), 0, 11, 127)
    query = rng.standard_normal((16, 1, d)) * 2.0 ** -12
    query[5] = np.sign(query[5]) * 2.0 ** 10
    if where == "query":
        query[9, 0, 3] = np.nan
    got, want = _attend(device, cuda(query, device, dtype), kp, vp, [[0, 1]], [16], [16], 2.0 ** 12)
    if where == "key":  # every row sees it
        assert bool(torch.isnan(got).all())
        return
    assert bool(torch.isnan(got[9]).all())
    keep = [i for i in range(16) if i not in (5, 9)]  # row 5's one key is as good as any here
    assert bool(torch.isfinite(got[5]).all())
    close(got[keep], *(x[keep] for x in want), PREFILL_STEP[dtype], lost=DENSE_LOST)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("where", ["query", "key"])
def test_prefill_of_nan_beside_large_scores(cuda_device, way, name, where):  # noqa: F811
    _nan_beside_large_scores(cuda_device, name, where)


@gpu
@pytest.mark.parametrize("where", ["query", "key"])
def test_prefill_of_nan_beside_large_scores_in_fp32(cuda_device, where):
    _nan_beside_large_scores(cuda_device, "f32", where)


# ---------------------------------------------------------------------------
# the ends of the range in each way of prefill, at the dense kernel's head_dim
# ---------------------------------------------------------------------------
def _range_case(device, name, d, k_byte, q_power, v_byte, scale, decode=False):
    rng = np.random.default_rng(abs(q_power) + k_byte)
    kb = np.clip(k_byte - rng.integers(0, 3, (5, 1, 1)), 1, 246).astype(np.uint8)
    vb = np.clip(v_byte - rng.integers(0, 3, (5, 1, 1)), 1, 246).astype(np.uint8)
    kp = fo.pack(fo.codes_of(30 * rng.standard_normal((5, 16, 1, d))), kb, False)
    vp = fo.pack(fo.codes_of(30 * rng.standard_normal((5, 16, 1, d))), vb, True)
    n = 1 if decode else 3
    query = cuda(rng.standard_normal((n, 2, d)) * 2.0 ** q_power, device, DTYPES[name])
    return _attend(device, query, kp, vp, [[0, 1, 2, 3, 4]], [n], [70], float(np.float32(scale)), decode)


@gpu
@pytest.mark.parametrize("name,k_byte,q_power,v_byte", [
    ("bf16", 246, -100, 246), ("bf16", 1, 90, 1), ("bf16", 246, 0, 127), ("bf16", 127, -120, 200), ("bf16", 20, 20, 10),
    ("bf16", 230, 10, 60), ("f16", 246, -14, 130), ("f16", 105, 8, 127), ("f16", 20, 8, 118), ("f16", 111, 10, 120)])
def test_prefill_over_the_whole_range_of_scales(cuda_device, way, name, k_byte, q_power, v_byte):  # noqa: F811
    scale = 2.0 ** np.clip(127 - k_byte - q_power - 6, -100, 100)  # scores of about 1
    got, want = _range_case(cuda_device, name, 128, k_byte, q_power, v_byte, scale)
    close(got, *want, PREFILL_STEP[DTYPES[name]], lost=DENSE_LOST)


@gpu
@pytest.mark.parametrize("v_byte", [246, 190])
def test_prefill_of_large_values_over_a_long_context(cuda_device, way, v_byte):  # noqa: F811
    """Sums of p v are past fp32's range, their mean is not."""
    rng = np.random.default_rng(v_byte)
    d, ctx = 128, 3000
    nb = -(-ctx // 16)
    kp, vp = pages(rng, nb, 16, 1, d)
    codes = fo.codes_of(30 * np.abs(rng.standard_normal((nb, 16, 1, d))))
    vp = fo.pack(codes, np.full((nb, 1, 1), v_byte, dtype=np.uint8), True)
    query = cuda(rng.standard_normal((40, 2, d)), cuda_device, torch.bfloat16)
    got, want = _attend(cuda_device, query, kp, vp, [np.arange(nb)], [40], [ctx], d ** -0.5)
    close(got, *want, PREFILL_STEP[torch.bfloat16], lost=DENSE_LOST)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("spread,scale", [(0.5, 2.0), (0.5, 0.0), (0.5, -0.3), (5.0, None), (0.5, 2.0 ** -40)])
def test_prefill_scales(cuda_device, way, name, spread, scale):  # noqa: F811
    got, free, want = prefill_case(cuda_device, name, 2, 4, 128, 16, [50, 20], [70, 150], scale=scale, spread=spread)
    for x in (got, free):
        close(x, *want, PREFILL_STEP[DTYPES[name]], lost=DENSE_LOST)


# ---------------------------------------------------------------------------
# the softmax's scale: 0, far below any other, not a number
# ---------------------------------------------------------------------------
SCALES = [(246, 0.0), (230, 2.0 ** -110), (246, 2.0 ** -126), (246, -2.0 ** -127), (127, float("nan"))]


def _softmax_scale(device, name, d, k_byte, scale, decode):
    got, want = _range_case(device, name, d, k_byte, 0, 127, scale, decode)
    if np.isnan(scale):
        assert bool(torch.isnan(got).all())
    else:
        close(got, *want, (DECODE_STEP if decode else PREFILL_STEP)[DTYPES[name]], lost=DENSE_LOST)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("k_byte,scale", SCALES)
def test_prefill_of_any_softmax_scale(cuda_device, way, name, d, k_byte, scale):  # noqa: F811
    _softmax_scale(cuda_device, name, d, k_byte, scale, False)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("decode", [False, True])
@pytest.mark.parametrize("k_byte,scale", SCALES)
def test_any_softmax_scale(cuda_device, name, decode, k_byte, scale):
    _softmax_scale(cuda_device, name, 96, k_byte, scale, decode)


# ---------------------------------------------------------------------------
# what is done over
# ---------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("distance", [12, 13, 16, 40])
def test_prefill_of_scales_that_fall_from_tile_to_tile(cuda_device, way, d, distance):  # noqa: F811
    """V's scales fall by 2^distance between the first tile of keys and the next ones: the keys behind count."""
    def edit(kp, vp, table):
        for pos in range(0, 700, 16):
            _set_byte(vp, table[0, pos // 16], 0, 0, 150 - (distance if pos >= 128 else 0))
        _set_code(vp, True, _place(5, table[0]), 0, 0, 0)

    got, free, want = prefill_case(cuda_device, "bf16", 1, 2, d, 16, [300, 30], [700, 30], edit=edit)
    for x in (got, free):
        close(x, *want, PREFILL_STEP[torch.bfloat16], lost=DENSE_LOST)


@gpu
@pytest.mark.parametrize("name,d", [("bf16", 64), ("f16", 128)])
def test_prefill_of_many_sequences_with_a_nan_each(cuda_device, way, name, d):  # noqa: F811
    rng = np.random.default_rng(d)
    count, hkv = 260, 2
    q_lens = rng.integers(1, 4, count)
    ctxs = (q_lens + rng.integers(0, 30, count)).tolist()
    nb = sum(-(-c // 16) for c in ctxs)
    kp, vp = pages(rng, nb, 16, hkv, d)
    tables = table_of(rng, ctxs, nb, 16)
    for r, c in enumerate(ctxs):
        if r % 7:
            _set_code(vp, True, _place(int(rng.integers(0, c)), tables[r]), r % hkv, r % d, 127)
    query = cuda(rng.standard_normal((int(q_lens.sum()), 2 * hkv, d)), cuda_device, DTYPES[name])
    got, want = _attend(cuda_device, query, kp, vp, tables, q_lens.tolist(), ctxs, d ** -0.5)
    _same(got, want, PREFILL_STEP[DTYPES[name]])


# ---------------------------------------------------------------------------
# scores of which fp32 has only every second or fourth whole number
# ---------------------------------------------------------------------------
def _steps_case(device, name, d, power, run, decode, ahead=4, off=1.0):
    """Runs of keys whose largest score is in turn 2^power and `ahead` above it, a few steps of fp32; V of the latter is 4, V's
    reference after the first, so that p goes in as it is: within f16."""
    ctx = 1280
    nb = ctx // 16
    high = np.arange(nb) * 16 // run % 2 == 1
    k, v = np.zeros((nb, 16, 1, d)), np.ones((nb, 16, 1, d))
    k[..., 0] = 1.0
    k[high, 3, 0, 1] = 1.0
    v[high] = 4.0
    kp, vp = fo.pack(*fo.encode(k), False), fo.pack(*fo.encode(v), True)
    rows = 1 if decode else 2
    query = np.zeros((rows, 1, d))
    query[:, 0, 0], query[:, 0, 1] = 1.0, ahead * 2.0 ** -power
    # a softmax scale whose product with log2(e) in fp32 is 2^power, or a few steps above
    scale = np.float32(2.0 ** power / np.log2(np.e))
    while float(scale * np.float32(np.log2(np.e))) % 4 or float(scale * np.float32(np.log2(np.e))) < 2.0 ** power:
        scale = np.nextafter(scale, np.float32(np.inf))
    got, want = _attend(device, cuda(query, device, DTYPES[name]), kp, vp, [np.arange(nb)], [rows], [ctx], float(scale) * off, decode)
    # scores are off by a step, two at most: p by 2^(2^(power - 22)) against the others, the mean stays between 1 and 4
    assert bool(torch.isfinite(got).all()) and bool((got >= 1 - 2.0 ** -7).all()) and bool((got <= 4 + 2.0 ** -5).all())
    if power <= 23 and off == 1:
        assert np.abs(got.double().cpu().numpy() - want[0]).max() < 3.0 * (2.0 ** 2.0 ** (power - 22) - 1)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("power", [18, 20, 22, 23, 24])
@pytest.mark.parametrize("off", [1.0, 1.3])  # the latter: scores that are no fp32 numbers
@pytest.mark.parametrize("d,run,decode", [(64, 32, True), (128, 32, True), (64, 64, False), (96, 64, False)])
def test_largest_scores_a_step_apart(cuda_device, name, power, d, run, decode, off):
    _steps_case(cuda_device, name, d, power, run, decode, off=off)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("d,run", [(64, 64), (64, 128), (128, 64), (128, 128)])
@pytest.mark.parametrize("off", [1.0, 1.3])
@pytest.mark.parametrize("power,ahead", [(18, 4), (20, 4), (22, 4), (23, 4), (24, 4), (24, 8), (26, 8), (27, 16), (28, 0), (31, 0)])
def test_prefill_of_largest_scores_a_step_apart(cuda_device, way, name, d, run, power, ahead, off):  # noqa: F811
    _steps_case(cuda_device, name, d, power, run, False, ahead, off)
