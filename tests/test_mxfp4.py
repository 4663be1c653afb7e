"""The 4-bit (MXFP4) paged cache: store, gather, decode, chunked prefill, and a run of them together.

Store and gather are exact (the scale is a power of two).  Attention is held to
    |got - want| <= u |want| + c * sum_k p_k |v_k|
with u half a step of the output type and c from the kernels' roundings:
  scores: fp32 sums of D products, off by at most D 2^-23 S with S = scale * sum |q||k|;
          that and the exponential's 2^-21 move p by as much, in the numerator and the sum;
  p:      rounded once to f16 before the tensor-core product (2^-11); fp32 carries the error in a second
          f16 (2^-22, within the exponential's term).
          f16 ends: p times a power of two that puts the sum above 2^12 and V's scale
          into [2^-7, 1] (at most 4 above the block's largest) loses at most half of 2^-24 a key,
          which is 2^-37 * 4 * 2^s_max * 6 of the result, and 2^s_max <= max|v| / 4 over the block:
          no more than ctx * 2^-34 max|v|.
Prefill rounds p to the query's type (half a step of it) and accumulates in the
same way; its K and V are the cache's values rounded to the query's type (bf16 holds them exactly).
"""

import ctypes

import numpy as np
import pytest
import torch

import microinfer_b200 as mi
from microinfer_b200 import _lib
from oracle import mxfp4_oracle as mo

gpu = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _bound(want, weight, size, floor, dtype, d, p_step):
    u = torch.finfo(dtype).eps / 2
    c = 2 * (d * 2.0 ** -23 * size + 2.0 ** -21) + p_step
    # below the smallest normal number the steps stay as they are there: half of one is u * smallest_normal
    return u * np.maximum(np.abs(want), torch.finfo(dtype).smallest_normal) + (c + u) * weight + floor * 2.0 ** -34


def _close(got, want, weight, size, floor, dtype, p_step):
    got = got.double().cpu().numpy()
    bound = _bound(want, weight, size, floor, dtype, got.shape[-1], p_step)
    off = np.abs(got - want)
    assert np.isfinite(got).all()
    worst = float(np.max(off / bound))
    assert worst <= 1, f"{worst:.3g} of the bound"


def _close_or_past(got, want, weight, size, floor, dtype, p_step):
    """As _close, for fp16 with results past its range: from 65520 on (half a step past 65504) a result has
    to be an infinity of the right sign; what may round either way leaves the comparison."""
    if dtype == torch.float16:
        slack = _bound(want, weight, size, floor, dtype, got.shape[-1], p_step)
        out = got.double().cpu().numpy()
        past, near = np.abs(want) - slack >= 65520, np.abs(want) + slack >= 65504
        assert np.array_equal(out[past], np.sign(want[past]) * np.inf)
        got = torch.from_numpy(np.where(near, want, out))
    _close(got, want, weight, size, floor, dtype, p_step)


DECODE_STEP = {torch.bfloat16: 2.0 ** -11, torch.float16: 2.0 ** -11, torch.float32: 0.0}


def _pages(rng, nb, bs, hkv, d, spread=0.5):
    """Random K and V pages by way of the oracle: rows of uneven size, V's by exp(+-2 spread)."""
    def one(by):
        size = np.exp(by * np.clip(rng.standard_normal((nb, bs, hkv, 1)), -2, 2))
        return mo.pack(*mo.encode(rng.standard_normal((nb, bs, hkv, d)) * size))
    return one(0.5), one(spread)


def _table(rng, ctxs, nb, bs, width=None):
    need = [-(-c // bs) for c in ctxs]
    assert sum(need) <= nb
    table = np.full((len(ctxs), width or max(1, max(need))), -1, dtype=np.int32)
    perm = rng.permutation(nb).astype(np.int32)
    at = 0
    for r, k in enumerate(need):
        table[r, :k] = perm[at:at + k]
        at += k
    return table


def _cuda(x, device, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x)).to(device)
    return t if dtype is None else t.to(dtype)


# ---------------------------------------------------------------------------
# host side
# ---------------------------------------------------------------------------
def test_oracle_round_trip_and_ties():
    x = np.array([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9, -0.2500001, -5.0, 0.0, -0.0] + [4.0] * 20])
    code, byte = mo.encode(x)
    assert byte.tolist() == [[127]]
    assert mo.decode(code, byte)[0, :12].tolist() == [0, 1, 1, 2, 2, 4, 4, 6, -0.5, -4, 0, 0]
    rng = np.random.default_rng(0)
    kp, _ = _pages(rng, 3, 32, 2, 64)
    code, byte = mo.unpack(kp)
    assert np.array_equal(mo.pack(code, byte), kp)
    again = mo.encode(mo.decode(code, byte))
    assert np.array_equal(mo.decode(*again), mo.decode(code, byte))  # values of the format are kept


def test_page_bytes_and_pool():
    lib = _lib.load()
    assert lib.mi_mxfp4_page_bytes(16, 128) == 1088
    assert lib.mi_mxfp4_page_bytes(64, 96) == 4 * 816
    for bs, d in ((8, 128), (24, 64), (16, 48), (16, 288), (0, 64)):
        assert lib.mi_mxfp4_page_bytes(bs, d) < 0
    pool = mi.MXFP4KVCache(2, 3, 32, 4, 128, device="cpu")
    assert pool.num_bytes == 2 * 2 * 3 * 4 * 2 * 1088
    layer = pool.layer(1)
    assert layer.block_size == 32 and layer.head_dim == 128
    with pytest.raises(ValueError, match="layer outside"):
        pool.layer(2)
    for bad in ((2, 3, 8, 4, 128), (2, 3, 16, 4, 40), (2, 3, 16, 4, 512), (0, 3, 16, 4, 64)):
        with pytest.raises(ValueError):
            mi.MXFP4KVCache(*bad, device="cpu")


def test_refusals_before_any_launch():
    pages = torch.zeros(4, 2, 1, 544, dtype=torch.uint8)
    rows = torch.zeros(3, 2, 64)
    slots = torch.zeros(3, dtype=torch.int32)
    table = torch.zeros(3, 1, dtype=torch.int32)
    lens = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensors"):
        mi.store_kv_mxfp4(pages, pages, slots, rows, rows)
    with pytest.raises(ValueError, match="uint8"):
        mi.store_kv_mxfp4(pages.int(), pages.int(), slots, rows, rows)
    with pytest.raises(ValueError, match="272"):
        mi.store_kv_mxfp4(pages[..., :512].contiguous(), pages[..., :512].contiguous(), slots, rows, rows)
    with pytest.raises(ValueError, match="contiguous"):
        mi.store_kv_mxfp4(pages[..., :272], pages[..., :272], slots, rows, rows)
    with pytest.raises(ValueError, match="heads"):
        mi.store_kv_mxfp4(pages, pages, slots, rows[:, :1].contiguous(), rows[:, :1].contiguous())
    with pytest.raises(ValueError, match="share a dtype"):
        mi.store_kv_mxfp4(pages, pages, slots, rows, rows.half())
    with pytest.raises(ValueError, match="dtype"):
        mi.store_kv_mxfp4(pages, pages, slots, rows.double(), rows.double())
    with pytest.raises(ValueError, match="one entry per token"):
        mi.store_kv_mxfp4(pages, pages, slots[:2], rows, rows)
    with pytest.raises(ValueError, match="int32 or int64"):
        mi.store_kv_mxfp4(pages, pages, slots.float(), rows, rows)
    query = torch.zeros(3, 4, 64)
    with pytest.raises(ValueError, match="CUDA tensors"):
        mi.paged_decode_mxfp4(query, pages, pages, table, lens)
    with pytest.raises(ValueError, match="head dimensions"):
        mi.paged_decode_mxfp4(query[..., :32], pages, pages, table, lens)
    with pytest.raises(ValueError, match="divisible"):
        mi.paged_decode_mxfp4(query[:, :3], pages, pages, table, lens)
    with pytest.raises(ValueError, match="one row per request"):
        mi.paged_decode_mxfp4(query, pages, pages, table[:2], lens)
    with pytest.raises(ValueError, match="one entry per request"):
        mi.paged_decode_mxfp4(query, pages, pages, table, lens[:2])
    with pytest.raises(ValueError, match="dtype"):
        mi.paged_decode_mxfp4(query.double(), pages, pages, table, lens)
    with pytest.raises(ValueError, match="out must"):
        mi.paged_decode_mxfp4(query, pages, pages, table, lens, out=query[:2])
    with pytest.raises(ValueError, match="num_requests"):
        mi.paged_prefill_mxfp4(query, pages, pages, lens, lens, table, max_seqlen_q=1)
    cu = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="max_seqlen_q"):
        mi.paged_prefill_mxfp4(query, pages, pages, cu, cu, table, max_seqlen_q=0)
    with pytest.raises(ValueError, match="CUDA tensors"):
        mi.gather_paged_kv_mxfp4(pages, pages, table, [1, 1, 1])


@pytest.mark.parametrize("shape", [(4, 0, 1, 544), (4, 2, 0, 544), (4, 2, 1, 0)])
def test_pages_without_heads_or_tokens_are_refused(shape):
    pages = torch.zeros(shape, dtype=torch.uint8)
    table, lens = torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="pages"):
        mi.paged_decode_mxfp4(torch.zeros(3, 4, 64), pages, pages, table, lens)
    with pytest.raises(ValueError, match="pages"):
        mi.gather_paged_kv_mxfp4(pages, pages, table, [1, 1, 1])


def test_fake_results_are_contiguous_like_the_real_ones():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        query = torch.empty(4, 3, 64).transpose(0, 1)
        pages = torch.empty(4, 2, 1, 544, dtype=torch.uint8)
        table, lens, cu = (torch.empty(n, dtype=torch.int32) for n in ((3, 1), 3, 4))
        ops = torch.ops.microinfer_b200
        for got in (ops.paged_decode_mxfp4(query, pages, pages, table, lens),
                    ops.paged_prefill_mxfp4(query, pages, pages, cu, cu, table, 1)):
            assert got.shape == query.shape and got.is_contiguous()


def test_c_entries_refuse_bad_arguments():
    lib = _lib.load()
    buf = ctypes.create_string_buffer(64)
    p = ctypes.cast(buf, ctypes.c_void_p)

    def store(dtype=2, bs=16, d=64, n=1, pages=p, index=0):
        return lib.mi_store_kv_mxfp4(pages, p, 4, bs, 2, d, p, index, p, p, dtype, 128, 128, n, None, None)

    assert store(n=0) == 0
    assert store(dtype=7) < 0 and store(bs=8) < 0 and store(d=48) < 0 and store(n=-1) < 0
    assert store(pages=None) < 0 and store(index=3) < 0

    def decode(hq=4, stride=2, n=1, ws=None, q=p, d=64):
        return lib.mi_paged_decode_mxfp4(p, q, p, p, 4, 16, hq, 2, d, 2, p, stride, p, n, 0.1, ws, 0, None, None)

    assert decode(n=0) == 0
    assert decode(hq=3) < 0 and decode(stride=-1) < 0 and decode(n=70000) < 0 and decode(q=None) < 0
    assert decode(d=320) < 0

    def gather(n=1, most=16, rows=16, dtype=2):
        return lib.mi_gather_paged_kv_mxfp4(p, p, p, p, 4, 16, 2, 64, dtype, p, 2, p, n, rows, most, None, None)

    assert gather(n=0) == 0 and gather(most=0) == 0 and gather(rows=0) == 0
    assert gather(n=-1) < 0 and gather(dtype=5) < 0 and gather(n=70000) < 0
    assert lib.mi_paged_decode_mxfp4_workspace_bytes(0, 8, 16, 4, 2, 64, 2, 100, 0) == 0


# ---------------------------------------------------------------------------
# store
# ---------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hkv,d,bs", [(1, 32, 16), (8, 128, 16), (2, 64, 64), (3, 96, 32), (20, 256, 16)])
@pytest.mark.parametrize("aligned", [True, False])
def test_store_is_exact(cuda_device, name, hkv, d, bs, aligned):
    rng = np.random.default_rng(hkv * 1000 + d + bs)
    dtype = DTYPES[name]
    nb, tokens = 7, 53
    kp, vp = _pages(rng, nb, bs, hkv, d)
    pad = 0 if aligned else 3  # a row stride that rules out 16-byte loads
    x = rng.standard_normal((2, tokens, hkv * d + pad)) * np.exp(3 * rng.standard_normal((2, tokens, 1)))
    x = _cuda(x, cuda_device, dtype)
    keys, values = (t[:, :hkv * d].unflatten(1, (hkv, d)) for t in x)
    slots = rng.permutation(nb * bs)[:tokens].astype(np.int64)
    slots[[3, 17]] = -1
    index = torch.int32 if aligned else torch.int64
    kt, vt = _cuda(kp, cuda_device), _cuda(vp, cuda_device)
    mi.store_kv_mxfp4(kt, vt, _cuda(slots, cuda_device, index), keys, values)
    torch.cuda.synchronize()
    mi.check_device_status(cuda_device)
    for pages, got, new in ((kp, kt, keys), (vp, vt, values)):
        code, byte = mo.unpack(pages)
        new_code, new_byte = mo.encode(new.double().cpu().numpy())
        for t, s in enumerate(slots):
            if s >= 0:
                code[s // bs, s % bs], byte[s // bs, s % bs] = new_code[t], new_byte[t]
        assert np.array_equal(got.cpu().numpy(), mo.pack(code, byte))


@gpu
def test_store_borders_and_values_that_are_not_finite(cuda_device):
    """Every multiple of 1/16 up to 8, both signs, at scales from the smallest to the largest; zero,
    denormal, infinite and NaN blocks."""
    grid = np.arange(0, 128) / 16
    lists = [np.concatenate([s * grid, [7.99] * 0]).reshape(4, 32) for s in (1, -1)]
    x = np.concatenate(lists)  # [8, 32]
    x[:, 31] = 7.75  # the same scale for every row
    rows = [x * 2.0 ** e for e in (-124, -20, 0, 3, 60, 124)]
    odd = np.zeros((8, 32))
    odd[1, 5] = 1e-40
    odd[2, 7] = -3.4e38
    odd[3, :] = 2.0 ** -126
    odd[4, 3] = np.inf
    odd[5, 9] = np.nan
    odd[6, :] = -0.0
    odd[7, 0] = 2.0 ** -149
    rows = np.concatenate([*rows, odd]).astype(np.float32).reshape(-1, 1, 32)
    tokens = len(rows)
    kp = np.zeros((-(-tokens // 16), 1, 1, 272), dtype=np.uint8)
    kt, vt = _cuda(kp, cuda_device), _cuda(kp, cuda_device)
    r = _cuda(rows, cuda_device)
    mi.store_kv_mxfp4(kt, vt, torch.arange(tokens, device=cuda_device), r, -r)
    code, byte = mo.encode(rows)
    got_code, got_byte = mo.unpack(kt.cpu().numpy())
    assert np.array_equal(got_byte.reshape(-1, 1, 1)[:tokens], byte)
    assert np.array_equal(got_code.reshape(-1, 1, 32)[:tokens], code)
    contexts = [tokens]
    table = torch.arange(len(kp), dtype=torch.int32, device=cuda_device)[None]
    k, v = mi.gather_paged_kv_mxfp4(kt, vt, table, contexts, dtype=torch.float32)
    want = mo.decode(code, byte)
    assert np.array_equal(k.double().cpu().numpy(), want, equal_nan=True)
    assert np.array_equal(v.double().cpu().numpy(), -want, equal_nan=True)


@gpu
def test_store_skips_and_flags_slots_outside_the_pool(cuda_device):
    kt = torch.full((2, 1, 1, 544), 7, dtype=torch.uint8, device=cuda_device)
    vt = kt.clone()
    rows = torch.ones(3, 1, 64, device=cuda_device)
    mi.store_kv_mxfp4(kt, vt, torch.tensor([-2, 32, -1], device=cuda_device), rows, rows)
    assert mi.read_device_status(cuda_device) == _lib.DEV_BAD_SLOT
    assert bool((kt == 7).all()) and bool((vt == 7).all())
    layer = mi.LayerMXFP4Cache(kt, vt)
    for bad in ([0, 32, 1], [-2, 0, 1], [5, 5, 1]):
        with pytest.raises(ValueError):
            layer.write_checked(torch.tensor(bad, device=cuda_device), rows, rows)
    assert bool((kt == 7).all())


# ---------------------------------------------------------------------------
# gather
# ---------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hkv,d,bs,ctxs", [
    (8, 128, 16, [1, 15, 16, 17, 0, 100]), (2, 64, 64, [130, 64, 63]), (1, 96, 256, [300]), (5, 256, 32, [33, 0, 1])])
def test_gather_is_exact(cuda_device, name, hkv, d, bs, ctxs):
    rng = np.random.default_rng(d + bs)
    dtype = DTYPES[name]
    nb = sum(-(-c // bs) for c in ctxs) + 2
    kp, vp = _pages(rng, nb, bs, hkv, d, spread=2.0)
    table = _table(rng, ctxs, nb, bs, width=max(-(-c // bs) for c in ctxs) + 1)
    args = (_cuda(kp, cuda_device), _cuda(vp, cuda_device), _cuda(table, cuda_device), ctxs)
    k, v = mi.gather_paged_kv_mxfp4(*args, dtype=dtype)
    out = torch.full_like(k, 3.0), torch.full_like(v, 3.0)
    cu = torch.tensor([0, *np.cumsum(ctxs)], dtype=torch.int32, device=cuda_device)
    mi.gather_paged_kv_mxfp4(*args, cu_seqlens_k=cu, out=out)
    mi.check_device_status(cuda_device)
    for got, again, pages in ((k, out[0], kp), (v, out[1], vp)):
        want = np.concatenate([mo.rows(pages, table[r], c) for r, c in enumerate(ctxs)])
        want = torch.from_numpy(want).to(dtype)
        assert torch.equal(got.cpu(), want) and torch.equal(again.cpu(), want)


@gpu
def test_gather_flags_bad_pages_and_stays_within_its_rows(cuda_device):
    rng = np.random.default_rng(1)
    kp, vp = _pages(rng, 4, 16, 1, 64)
    kt, vt = _cuda(kp, cuda_device), _cuda(vp, cuda_device)
    table = torch.tensor([[0, 9], [-1, 2]], dtype=torch.int32, device=cuda_device)
    out = torch.full((64, 1, 64), 5.0, device=cuda_device), torch.full((64, 1, 64), 5.0, device=cuda_device)
    mi.gather_paged_kv_mxfp4(kt, vt, table, [32, 32], out=out)
    assert mi.read_device_status(cuda_device) == _lib.DEV_BAD_BLOCK
    want = mo.rows(kp, [0], 16)
    assert np.array_equal(out[0][:16].double().cpu().numpy(), want)
    assert bool((out[0][16:48] == 5.0).all())
    # offsets that run past the output's rows
    cu = torch.tensor([0, 40, 100], dtype=torch.int32, device=cuda_device)
    table = torch.tensor([[0, 1, 2, 3]] * 2, dtype=torch.int32, device=cuda_device)
    big = torch.full((96, 1, 64), 5.0, device=cuda_device), torch.full((96, 1, 64), 5.0, device=cuda_device)
    mi.gather_paged_kv_mxfp4(kt, vt, table, [10, 40], cu_seqlens_k=cu, out=(big[0][:50], big[1][:50]))
    assert mi.read_device_status(cuda_device) == _lib.DEV_BAD_SLOT
    assert bool((big[0][50:] == 5.0).all())
    with pytest.raises(ValueError, match="longer than"):
        mi.gather_paged_kv_mxfp4(kt, vt, table, [65, 1])


# ---------------------------------------------------------------------------
# decode
# ---------------------------------------------------------------------------
def _decode_case(device, name, hkv, group, d, bs, ctxs, seed=0, scale=None, spread=0.5, edit=None):
    rng = np.random.default_rng(seed + d + bs + group)
    dtype = DTYPES[name]
    nb = sum(-(-max(c, 0) // bs) for c in ctxs) + 3
    kp, vp = _pages(rng, nb, bs, hkv, d, spread)
    table = _table(rng, [max(c, 0) for c in ctxs], nb, bs, width=max(1, max(-(-c // bs) for c in ctxs)) + 1)
    query = _cuda(rng.standard_normal((len(ctxs), hkv * group, d)), device, dtype)
    if edit is not None:
        edit(kp, vp, table)
    scale = d ** -0.5 if scale is None else scale
    got = mi.paged_decode_mxfp4(query, _cuda(kp, device), _cuda(vp, device), _cuda(table, device),
                                torch.tensor(ctxs, dtype=torch.int32, device=device), scale=scale)
    q = query.double().cpu().numpy()
    parts = [mo.attention(q[r:r + 1], mo.rows(kp, table[r], max(c, 0)), mo.rows(vp, table[r], max(c, 0)), scale)
             for r, c in enumerate(ctxs)]
    return got, [np.concatenate(x) for x in zip(*parts)], dtype


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hkv,group,d,bs", [
    (8, 2, 128, 16), (2, 7, 64, 64), (1, 16, 128, 32), (4, 1, 64, 16), (2, 5, 128, 256), (1, 12, 64, 16),
    (1, 4, 96, 32), (2, 3, 32, 16), (1, 2, 256, 16), (2, 8, 160, 16), (1, 1, 128, 16)])
def test_decode_matches_the_formula(cuda_device, name, hkv, group, d, bs):
    ctxs = [1, 2, 15, 16, 17, 0, 31, 33, 129, 300, 257]
    got, want, dtype = _decode_case(cuda_device, name, hkv, group, d, bs, ctxs)
    mi.check_device_status(cuda_device)
    _close(got, *want, dtype, DECODE_STEP[dtype])
    assert bool((got[5] == 0).all())  # no key: zeros


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("ctxs", [[5000], [4096, 1, 0, 2777], [1], [0], [0, 0, 16], [20000, 3]])
@pytest.mark.parametrize("hkv,group,d,bs", [(2, 4, 128, 16), (1, 8, 64, 64)])
def test_decode_splits_long_contexts(cuda_device, name, ctxs, hkv, group, d, bs):
    got, want, dtype = _decode_case(cuda_device, name, hkv, group, d, bs, ctxs)
    mi.check_device_status(cuda_device)
    _close(got, *want, dtype, DECODE_STEP[dtype])


@gpu
@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_decode_many_sequences(cuda_device, name):
    rng = np.random.default_rng(9)
    ctxs = rng.integers(0, 90, 400).tolist()
    got, want, dtype = _decode_case(cuda_device, name, 4, 4, 64, 16, ctxs)
    mi.check_device_status(cuda_device)
    _close(got, *want, dtype, DECODE_STEP[dtype])


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("spread,scale", [(4.0, None), (8.0, None), (0.5, 3.0), (0.5, 0.0), (0.5, -0.2)])
def test_decode_uneven_scales_and_sharp_softmax(cuda_device, name, spread, scale):
    """V rows whose scales differ by up to 2^46; scores far apart, all equal, and with the sign turned."""
    if name == "f16" and spread == 8.0:
        pytest.skip("the values are past fp16's range")
    got, want, dtype = _decode_case(cuda_device, name, 2, 4, 128, 16, [700, 40, 16, 1], seed=3, spread=spread,
                                    scale=scale)
    mi.check_device_status(cuda_device)
    _close(got, *want, dtype, DECODE_STEP[dtype])


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
def test_decode_large_values_with_no_weight(cuda_device, name):
    """Keys that get no weight carry V of 2^40, the ones with weight V of 2^-30: nothing is lost."""
    def edit(kp, vp, table):
        kc, kb = mo.unpack(kp)
        vc, vb = mo.unpack(vp)
        kc[:] &= 7  # positive keys; their size decides
        kc[..., :] = np.maximum(kc, 2)
        for r in range(table.shape[0]):
            for col, blk in enumerate(table[r]):
                if blk >= 0:
                    heavy = col % 3 == 1
                    kb[blk] = 127 if heavy else 60
                    vb[blk] = 97 if heavy else 167
        kp[:], vp[:] = mo.pack(kc, kb), mo.pack(vc, vb)

    rng = np.random.default_rng(2)
    dtype = DTYPES[name]
    ctxs, bs, d = [130, 48], 16, 128
    kp, vp = _pages(rng, 14, bs, 1, d)
    table = _table(rng, ctxs, 14, bs)
    edit(kp, vp, table)
    query = _cuda(np.abs(rng.standard_normal((2, 4, d))) + 0.5, cuda_device, dtype)
    got = mi.paged_decode_mxfp4(query, _cuda(kp, cuda_device), _cuda(vp, cuda_device), _cuda(table, cuda_device),
                                torch.tensor(ctxs, dtype=torch.int32, device=cuda_device), scale=6.0)
    q = query.double().cpu().numpy()
    parts = [mo.attention(q[r:r + 1], mo.rows(kp, table[r], c), mo.rows(vp, table[r], c), 6.0)
             for r, c in enumerate(ctxs)]
    want = [np.concatenate(x) for x in zip(*parts)]
    if name == "f16":  # 2^-30 is below fp16's smallest step: the result is its rounding
        assert bool((got.float().abs() <= 2.0 ** -24).all())
    else:
        _close(got, *want, dtype, DECODE_STEP[dtype])


@gpu
def test_decode_more_sequences_than_one_launch_takes(cuda_device):
    rng = np.random.default_rng(21)
    ctxs = rng.integers(0, 20, 2500).tolist()
    got, want, dtype = _decode_case(cuda_device, "bf16", 1, 4, 64, 16, ctxs)
    mi.check_device_status(cuda_device)
    _close(got, *want, dtype, DECODE_STEP[dtype])


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
def test_decode_many_keys_of_little_weight(cuda_device, name):
    """One key takes nearly everything and its value is zero: the rest of a long context, each key about 2^-20
    of it, decides the result."""
    ctx, d = 9000, 64
    rng = np.random.default_rng(22)
    nb = ctx // 16 + 2
    kc, kb = mo.encode(rng.standard_normal((nb, 16, 1, d)) * 0.01)
    vc, vb = mo.encode(rng.standard_normal((nb, 16, 1, d)) + 1.0)
    table = _table(rng, [ctx], nb, 16)
    sink = table[0, 3], 5
    kc[sink], kb[sink] = 2, 127  # all 1.0
    vc[sink], vb[sink] = 0, 0
    kp, vp = mo.pack(kc, kb), mo.pack(vc, vb)
    query = _cuda(np.full((1, 4, d), 1.0), cuda_device, DTYPES[name])
    scale = 14.0 / d  # the sink is exp(14) = 2^20 above the others
    got = mi.paged_decode_mxfp4(query, _cuda(kp, cuda_device), _cuda(vp, cuda_device), _cuda(table, cuda_device),
                                torch.tensor([ctx], dtype=torch.int32, device=cuda_device), scale=scale)
    want = mo.attention(np.full((1, 4, d), 1.0), mo.rows(kp, table[0], ctx), mo.rows(vp, table[0], ctx), scale)
    assert 0.001 < np.abs(want[0]).max() < 0.1
    _close(got, *want, DTYPES[name], DECODE_STEP[DTYPES[name]])


@gpu
@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_decode_ignores_what_lies_past_the_context(cuda_device, name):
    """Stale rows of the last page and pages past the context hold NaN scales; columns past it bad ids."""
    ctxs = [5, 16, 21, 40]

    def edit(kp, vp, table):
        for pages in (kp, vp):
            code, byte = mo.unpack(pages)
            used = np.zeros(byte.shape[:2], dtype=bool)
            for r, c in enumerate(ctxs):
                for pos in range(c):
                    used[table[r, pos // 16], pos % 16] = True
            byte[~used] = 255
            pages[:] = mo.pack(code, byte)
        for r, c in enumerate(ctxs):
            table[r, -(-c // 16):] = 1 << 30

    got, want, dtype = _decode_case(cuda_device, name, 2, 2, 128, 16, ctxs, edit=edit)
    mi.check_device_status(cuda_device)
    _close(got, *want, dtype, DECODE_STEP[dtype])


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
def test_decode_nan_blocks(cuda_device, name):
    """A NaN block of a key makes its heads' rows NaN, one of a value only its 32 elements."""
    bs, d, ctx = 16, 128, 50
    rng = np.random.default_rng(4)
    kp, vp = _pages(rng, 8, bs, 2, d)
    table = _table(rng, [ctx, ctx], 8, bs)
    kc, kb = mo.unpack(kp)
    vc, vb = mo.unpack(vp)
    kb[table[0, 1], 3, 0, 2] = 255
    vb[table[1, 2], 7, 1, 1] = 255
    kp, vp = mo.pack(kc, kb), mo.pack(vc, vb)
    query = _cuda(rng.standard_normal((2, 8, d)), cuda_device, DTYPES[name])
    got = mi.paged_decode_mxfp4(query, _cuda(kp, cuda_device), _cuda(vp, cuda_device), _cuda(table, cuda_device),
                                torch.tensor([ctx, ctx], dtype=torch.int32, device=cuda_device))
    nan = torch.isnan(got).cpu()
    assert bool(nan[0, :4].all()) and not bool(nan[0, 4:].any())
    assert bool(nan[1, 4:, 32:64].all()) and int(nan[1].sum()) == 4 * 32


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
def test_decode_query_values_of_any_size(cuda_device, name):
    """Queries of very small and large magnitude, a zero row, and rows that are not finite."""
    rng = np.random.default_rng(5)
    dtype = DTYPES[name]
    kp, vp = _pages(rng, 6, 16, 1, 64)
    sizes = {"f16": [2.0 ** -14, 2.0 ** 9, 0.0, 1.0], "bf16": [2.0 ** -100, 2.0 ** 90, 0.0, 1.0],
             "f32": [2.0 ** -100, 2.0 ** 90, 0.0, 1.0]}[name]
    table = np.array([[0, 1, 2]] * 4, dtype=np.int32)
    query = rng.standard_normal((4, 4, 64)) * np.array(sizes)[:, None, None]
    query = _cuda(query, cuda_device, dtype)
    query[3, 1, 5] = float("nan")
    query[3, 2, 6] = float("inf")
    args = (_cuda(kp, cuda_device), _cuda(vp, cuda_device), _cuda(table, cuda_device),
            torch.full((4,), 40, dtype=torch.int32, device=cuda_device))
    got = mi.paged_decode_mxfp4(query, *args)
    q = query.double().cpu().numpy()
    k, v = mo.rows(kp, table[0], 40), mo.rows(vp, table[0], 40)
    for r in (0, 2, 3):
        heads = [0, 3] if r == 3 else [0, 1, 2, 3]
        want = mo.attention(q[r:r + 1, heads], k, v, 0.125)
        _close(got[r:r + 1, heads], *want, dtype, DECODE_STEP[dtype])
    if name == "f16":
        _close(got[1:2], *mo.attention(q[1:2], k, v, 0.125), dtype, DECODE_STEP[dtype])
    else:  # scores of 2^90: the largest takes everything
        best = np.argmax(q[1] @ k[:, 0].T, -1)
        assert np.array_equal(got[1].double().cpu().numpy(), _cuda(v[best, 0], cuda_device, dtype).double().cpu().numpy())
    assert bool(torch.isnan(got[3, 1:3]).all())


@gpu
def test_decode_flags_bad_pages_and_lengths(cuda_device):
    rng = np.random.default_rng(6)
    kp, vp = _pages(rng, 4, 16, 1, 64)
    query = torch.randn(2, 4, 64, device=cuda_device, dtype=torch.bfloat16)
    args = (query, _cuda(kp, cuda_device), _cuda(vp, cuda_device))
    table = torch.tensor([[0, 7], [1, -1]], dtype=torch.int32, device=cuda_device)
    mi.paged_decode_mxfp4(*args, table, torch.tensor([32, 16], dtype=torch.int32, device=cuda_device))
    assert mi.read_device_status(cuda_device) == _lib.DEV_BAD_BLOCK
    table = torch.tensor([[0, 3], [1, 2]], dtype=torch.int32, device=cuda_device)
    full = mi.paged_decode_mxfp4(*args, table, torch.tensor([32, 32], dtype=torch.int32, device=cuda_device))
    assert mi.read_device_status(cuda_device) == 0
    # a length past the table's columns is clamped to them and flagged, a negative one is none
    long = mi.paged_decode_mxfp4(*args, table, torch.tensor([1000, -5], dtype=torch.int32, device=cuda_device))
    assert mi.read_device_status(cuda_device) == _lib.DEV_BAD_BLOCK
    assert torch.equal(long[0], full[0]) and bool((long[1] == 0).all())


@gpu
@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_decode_views_and_out(cuda_device, name):
    """A query that is a view, int64 tables, an output given by the caller, a table without columns."""
    rng = np.random.default_rng(7)
    dtype = DTYPES[name]
    ctxs = [30, 9, 64]
    kp, vp = _pages(rng, 9, 16, 2, 64)
    table = _cuda(_table(rng, ctxs, 9, 16), cuda_device)
    lens = torch.tensor(ctxs, dtype=torch.int32, device=cuda_device)
    pages = _cuda(kp, cuda_device), _cuda(vp, cuda_device)
    packed = torch.randn(3, 12, 64, device=cuda_device).to(dtype)
    query = packed[:, 2:10]
    want = mi.paged_decode_mxfp4(query.contiguous(), *pages, table, lens)
    out = torch.empty(3, 8, 64, dtype=dtype, device=cuda_device)
    wide = torch.full((3, 9), -1, dtype=torch.int64, device=cuda_device)
    wide[:, :table.shape[1]] = table
    got = mi.paged_decode_mxfp4(query, *pages, wide, lens.long(), out=out)
    assert got is out
    limit = 2 * torch.finfo(dtype).eps if dtype == torch.bfloat16 else 1e-5
    assert float((got.double() - want.double()).abs().max()) <= limit * float(want.abs().max())
    assert torch.equal(mi.paged_decode_mxfp4(query.contiguous(), *pages, table, lens), want)  # the same again
    none = mi.paged_decode_mxfp4(query, *pages, table[:, :0], lens)
    assert bool((none == 0).all())
    assert mi.paged_decode_mxfp4(query[:0], *pages, table[:0], lens[:0]).shape == (0, 8, 64)


@gpu
def test_cache_past_32_bit_offsets(cuda_device):
    """Pages that lie more than 4 GiB into the pool are stored, gathered and attended to."""
    hkv, d, bs = 8, 128, 64
    page = hkv * 4 * 1088
    nb = (1 << 32) // page + 40
    kt = torch.zeros(nb, hkv, 4, 1088, dtype=torch.uint8, device=cuda_device)
    vt = torch.zeros_like(kt)
    rng = np.random.default_rng(8)
    ctx = 100
    table = np.array([[nb - 1, nb - 7]], dtype=np.int32)
    pos = np.arange(ctx)
    slots = table[0, pos // bs].astype(np.int64) * bs + pos % bs
    rows = _cuda(rng.standard_normal((2, ctx, hkv, d)), cuda_device, torch.bfloat16)
    mi.store_kv_mxfp4(kt, vt, _cuda(slots, cuda_device), rows[0], rows[1])
    tt = _cuda(table, cuda_device)
    k, v = mi.gather_paged_kv_mxfp4(kt, vt, tt, [ctx])
    want_k, want_v = (mo.decode(*mo.encode(r.double().cpu().numpy())) for r in rows)
    assert np.array_equal(k.double().cpu().numpy(), want_k) and np.array_equal(v.double().cpu().numpy(), want_v)
    assert int(kt[:nb - 7].max()) == 0
    query = _cuda(rng.standard_normal((1, 16, d)), cuda_device, torch.bfloat16)
    got = mi.paged_decode_mxfp4(query, kt, vt, tt, torch.tensor([ctx], dtype=torch.int32, device=cuda_device))
    want = mo.attention(query.double().cpu().numpy(), want_k, want_v, d ** -0.5)
    _close(got, *want, torch.bfloat16, DECODE_STEP[torch.bfloat16])
    mi.check_device_status(cuda_device)


# ---------------------------------------------------------------------------
# prefill, and a run of them together
# ---------------------------------------------------------------------------
PREFILL_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10, torch.float32: 0.0}


def _prefill_case(device, name, hkv, group, d, bs, q_lens, ctxs, seed=0, scale=None, edit=None, **kw):
    rng = np.random.default_rng(seed + d + group)
    dtype = DTYPES[name]
    nb = sum(-(-c // bs) for c in ctxs) + 2
    kp, vp = _pages(rng, nb, bs, hkv, d)
    table = _table(rng, ctxs, nb, bs)
    if edit is not None:
        edit(kp, vp, table)
    query = _cuda(rng.standard_normal((sum(q_lens), hkv * group, d)), device, dtype)
    cu_q, cu_k = (torch.tensor([0, *np.cumsum(x)], dtype=torch.int32, device=device) for x in (q_lens, ctxs))
    args = (query, _cuda(kp, device), _cuda(vp, device), cu_q, cu_k, _cuda(table, device))
    got = mi.paged_prefill_mxfp4(*args, max_seqlen_q=max(q_lens), total_k=sum(ctxs), scale=scale, **kw)
    free = mi.paged_prefill_mxfp4(*args, max_seqlen_q=max(q_lens), scale=scale)
    mi.check_device_status(device)
    q = query.double().cpu().numpy()
    at = np.cumsum([0, *q_lens])
    parts = [mo.attention(q[at[r]:at[r + 1]], mo.rows(kp, table[r], c), mo.rows(vp, table[r], c),
                          d ** -0.5 if scale is None else scale) for r, c in enumerate(ctxs)]
    return got, free, [np.concatenate(x) for x in zip(*parts)], dtype


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hkv,group,d,bs", [
    (8, 2, 128, 16), (2, 4, 64, 64), (1, 3, 96, 32), (2, 7, 128, 32), (1, 5, 64, 16), (1, 16, 64, 256), (4, 1, 128, 48)])
def test_prefill_matches_the_formula(cuda_device, name, hkv, group, d, bs):
    q_lens, ctxs = [1, 40, 7, 130, 1], [90, 40, 135, 201, 1]
    got, free, want, dtype = _prefill_case(cuda_device, name, hkv, group, d, bs, q_lens, ctxs)
    for x in (got, free):  # the bound on the contexts only decides the split over the keys
        _close(x, *want, dtype, PREFILL_STEP[dtype])


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("q_lens,ctxs", [([3], [5000]), ([64], [2000]), ([1, 17], [4097, 63]), ([33], [33])])
def test_prefill_small_chunks_over_long_contexts(cuda_device, name, d, q_lens, ctxs):
    got, free, want, dtype = _prefill_case(cuda_device, name, 2, 4, d, 16, q_lens, ctxs)
    for x in (got, free):
        _close(x, *want, dtype, PREFILL_STEP[dtype])


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("scale", [2.0, 0.0, -0.3])
def test_prefill_scales(cuda_device, name, scale):
    got, _, want, dtype = _prefill_case(cuda_device, name, 1, 3, 64, 16, [50, 20], [70, 150], scale=scale)
    _close(got, *want, dtype, PREFILL_STEP[dtype])


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
def test_prefill_nan_blocks_reach_only_rows_that_see_them(cuda_device, name, d):
    """A NaN value block of a key in the chunk: NaN in its 32 dims for the rows from it on; a NaN key block: those
    rows alone."""
    place = {}

    def edit(kp, vp, table):
        kc, kb = mo.unpack(kp)
        vc, vb = mo.unpack(vp)
        vb[table[0, 60 // 16], 60 % 16, 0, 1] = 255  # position 60 of 90, row 10 of 40
        kb[table[0, 80 // 16], 80 % 16, 0, 0] = 255  # position 80, row 30
        kp[:], vp[:] = mo.pack(kc, kb), mo.pack(vc, vb)

    got, _, _, _ = _prefill_case(cuda_device, name, 1, 3, d, 16, [40], [90], edit=edit)
    nan = torch.isnan(got).cpu()
    assert not bool(nan[:10].any()) and bool(nan[30:].all())
    assert bool(nan[10:30, :, 32:64].all()) and int(nan[10:30].sum()) == 20 * 3 * 32


@gpu
@pytest.mark.parametrize("d", [64, 128])
def test_prefill_leaves_rows_of_no_sequence_and_flags_bad_pages(cuda_device, d):
    rng = np.random.default_rng(31)
    kp, vp = _pages(rng, 6, 16, 1, d)
    query = torch.randn(12, 2, d, device=cuda_device, dtype=torch.float16)
    cu_q = torch.tensor([0, 3, 8], dtype=torch.int32, device=cuda_device)
    cu_k = torch.tensor([0, 20, 60], dtype=torch.int32, device=cuda_device)
    table = torch.tensor([[0, 1, -1], [2, 3, 4]], dtype=torch.int32, device=cuda_device)
    out = torch.full_like(query, 7.0)
    args = (query, _cuda(kp, cuda_device), _cuda(vp, cuda_device), cu_q, cu_k)
    mi.paged_prefill_mxfp4(*args, table, max_seqlen_q=5, out=out)
    mi.check_device_status(cuda_device)
    assert bool((out[8:] == 7.0).all()) and not bool((out[:8] == 7.0).all(-1).any())
    table[1, 1] = 9
    mi.paged_prefill_mxfp4(*args, table, max_seqlen_q=5)
    assert mi.read_device_status(cuda_device) == _lib.DEV_BAD_BLOCK
    # a context past the table's columns
    cu_k[2] = 20 + 70
    table[1, 1] = 3
    mi.paged_prefill_mxfp4(*args, table, max_seqlen_q=5)
    assert mi.read_device_status(cuda_device) & _lib.DEV_BAD_BLOCK


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
def test_a_prompt_in_chunks_then_tokens(cuda_device, name):
    """CachedAttention on a 4-bit layer: two prefill chunks, then decode steps, then a fork by copy-on-write."""
    from microinfer_b200.layer.cached_attention import CachedAttention
    from microinfer_b200.layer.metadata import AttentionMetadata

    dtype = DTYPES[name]
    gen = torch.Generator().manual_seed(11)
    hq, hkv, d, bs = 8, 2, 128, 16
    pool = mi.MXFP4KVCache(1, 12, bs, hkv, d, device=cuda_device)
    attn = CachedAttention()
    attn.bind_cache(pool.layer(0))
    tables = [[3, 7, 1, 10], [0, 5, 2]]
    width = 4
    table = torch.full((2, width), -1, dtype=torch.int32)
    for r, t in enumerate(tables):
        table[r, :len(t)] = torch.tensor(t)
    lens = [0, 0]
    history = [np.zeros((2, 0, hkv, d)) for _ in range(2)]

    def step(new, prefill):
        rows = sum(new)
        q, k, v = (torch.randn(rows, h, d, generator=gen).to(dtype).to(cuda_device) for h in (hq, hkv, hkv))
        at, slots, want = 0, [], []
        for r, n in enumerate(new):
            for pos in range(lens[r], lens[r] + n):
                slots.append(tables[r][pos // bs] * bs + pos % bs)
            coded = np.stack([mo.decode(*mo.encode(t[at:at + n].double().cpu().numpy())) for t in (k, v)])
            history[r] = np.concatenate([history[r], coded], 1)
            lens[r] += n
            want.append(mo.attention(q[at:at + n].double().cpu().numpy(), *history[r], d ** -0.5))
            at += n
        fields = dict(slot_mapping=torch.tensor(slots, dtype=torch.int32, device=cuda_device),
                      block_tables=table.to(cuda_device))
        if prefill:
            cu_q, cu_k = (torch.tensor([0, *np.cumsum(x)], dtype=torch.int32, device=cuda_device)
                          for x in (new, lens))
            meta = AttentionMetadata.build(is_prefill=True, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k,
                                           max_seqlen_q=max(new), max_seqlen_k=max(lens), **fields)
        else:
            meta = AttentionMetadata.build(is_prefill=False, validate_cache_write=False,
                                           context_lens=torch.tensor(lens, dtype=torch.int32, device=cuda_device),
                                           **fields)
        got = attn(q, k, v, meta)
        _close(got, *(np.concatenate(x) for x in zip(*want)), dtype,
               (PREFILL_STEP if prefill else DECODE_STEP)[dtype])

    step([20, 9], True)
    step([23, 20], True)
    for _ in range(4):
        step([1, 1], False)
    # sequence 1 goes on in a private copy of its last page
    pool.copy_blocks([(tables[1][2], 9)])
    tables[1][2] = 9
    table[1, 2] = 9
    step([1, 1], False)
    mi.check_device_status(cuda_device)


@gpu
def test_two_graphs_and_an_eager_call_on_their_own_streams(cuda_device):
    """Captured decode steps replayed together on two streams, with an eager one beside them, share nothing."""
    rng = np.random.default_rng(12)
    ctxs = [3000, 17, 800]
    cases = []
    for seed in range(3):
        kp, vp = _pages(rng, 260, 16, 2, 128)
        table = _cuda(_table(rng, ctxs, 260, 16), cuda_device)
        query = torch.randn(3, 8, 128, device=cuda_device, dtype=torch.bfloat16)
        lens = torch.tensor(ctxs, dtype=torch.int32, device=cuda_device)
        cases.append((query, _cuda(kp, cuda_device), _cuda(vp, cuda_device), table, lens))
    want = [mi.paged_decode_mxfp4(*c) for c in cases]
    streams = [torch.cuda.Stream(cuda_device) for _ in range(3)]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for c, s in zip(cases[:2], streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(mi.paged_decode_mxfp4(*c))
        graphs.append(g)
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            third = mi.paged_decode_mxfp4(*cases[2])
        torch.cuda.synchronize()
        for got, w in zip([*outs, third], want):
            assert torch.equal(got, w)


@gpu
def test_under_torch_compile(cuda_device):
    rng = np.random.default_rng(13)
    kp, vp = _pages(rng, 6, 16, 2, 64)
    kt, vt = _cuda(kp, cuda_device), _cuda(vp, cuda_device)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=cuda_device)
    lens = torch.tensor([20, 32], dtype=torch.int32, device=cuda_device)
    slots = torch.tensor([2 * 16 + 3, 51], dtype=torch.int32, device=cuda_device)
    q, k, v = (torch.randn(2, h, 64, device=cuda_device, dtype=torch.bfloat16) for h in (4, 2, 2))

    def fn(q, k, v, kt, vt):
        mi.store_kv_mxfp4(kt, vt, slots, k, v)
        return mi.paged_decode_mxfp4(q + 0, kt, vt, table, lens) * 2

    want = fn(q, k, v, kt.clone(), vt.clone())
    got = torch.compile(fn, fullgraph=True, backend="aot_eager")(q, k, v, kt, vt)
    assert torch.equal(got, want)


@gpu
def test_transposed_query_under_torch_compile(cuda_device):
    rng = np.random.default_rng(14)
    kp, vp = _pages(rng, 6, 16, 2, 64)
    kt, vt = _cuda(kp, cuda_device), _cuda(vp, cuda_device)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=cuda_device)
    lens = torch.tensor([20, 32], dtype=torch.int32, device=cuda_device)
    cu_q = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda_device)
    cu_k = torch.tensor([0, 20, 52], dtype=torch.int32, device=cuda_device)
    heads_first = torch.randn(4, 2, 64, device=cuda_device, dtype=torch.bfloat16)

    def fn(x):
        q = x.transpose(0, 1)
        a = mi.paged_decode_mxfp4(q, kt, vt, table, lens)
        b = mi.paged_prefill_mxfp4(q, kt, vt, cu_q, cu_k, table, max_seqlen_q=1)
        return a.view(2, 256), b.view(2, 256)

    for got, want in zip(torch.compile(fn, fullgraph=True, backend="aot_eager")(heads_first), fn(heads_first)):
        assert torch.equal(got, want)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 96, 128])
def test_results_over_the_query_and_shared_pages(cuda_device, name, d):
    """`out` may be the query itself; rows of the table may name the same pages, and one page twice."""
    rng = np.random.default_rng(15)
    dtype = DTYPES[name]
    kp, vp = _pages(rng, 40, 16, 2, d)
    pages = _cuda(kp, cuda_device), _cuda(vp, cuda_device)
    one = rng.integers(0, 40, 200).astype(np.int32)
    one[7] = one[3]
    table = _cuda(np.stack([one, one, one[::-1]]), cuda_device)
    lens = torch.tensor([3200, 3185, 1700], dtype=torch.int32, device=cuda_device)
    query = _cuda(rng.standard_normal((3, 8, d)), cuda_device, dtype)
    q = query.double().cpu().numpy()
    names = [one, one, one[::-1]]
    parts = [mo.attention(q[r:r + 1], mo.rows(kp, names[r], int(c)), mo.rows(vp, names[r], int(c)), d ** -0.5)
             for r, c in enumerate(lens.tolist())]
    want = [np.concatenate(x) for x in zip(*parts)]
    over = query.clone()
    assert mi.paged_decode_mxfp4(over, *pages, table, lens, out=over) is over
    _close(over, *want, dtype, DECODE_STEP[dtype])
    over = query.clone()
    cu_q = torch.arange(4, dtype=torch.int32, device=cuda_device)
    cu_k = torch.cat([cu_q[:1], lens.cumsum(0).int()])
    if d != 96:  # computed from the pages: the rows are read before they are written
        mi.paged_prefill_mxfp4(over, *pages, cu_q, cu_k, table, max_seqlen_q=1, out=over)
        _close(over, *want, dtype, PREFILL_STEP[dtype])
    mi.check_device_status(cuda_device)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("group", [1, 6, 9])
def test_decode_every_head_dim(cuda_device, name, d, group):
    """Long and short contexts of every head_dim, scales far apart, sequences that cross CTAs."""
    ctxs = [7000, 0, 1, 31, 33, 1500]
    got, want, dtype = _decode_case(cuda_device, name, 2, group, d, 32, ctxs, spread=6.0)
    mi.check_device_status(cuda_device)
    assert bool((got[1] == 0).all())
    _close_or_past(got, *want, dtype, DECODE_STEP[dtype])


@gpu
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
def test_decode_nan_and_zero_blocks_of_every_head_dim(cuda_device, d):
    """A NaN block of V is NaN in its 32 dims of its sequence alone; a NaN of K in all; zero blocks are zeros."""
    nb = d // 32
    rng = np.random.default_rng(d)
    kp, vp = _pages(rng, 12, 16, 1, d)
    scales = vp.reshape(12, 1, 1, -1)[..., nb * 256:].reshape(12, 16, nb)  # a view
    kscales = kp.reshape(12, 1, 1, -1)[..., nb * 256:].reshape(12, 16, nb)
    scales[2, 5, nb - 1] = 255
    scales[6, 3, :] = 0
    kscales[9, 0, 0] = 255
    table = np.arange(12, dtype=np.int32).reshape(3, 4)
    kt, vt, tt = _cuda(kp, cuda_device), _cuda(vp, cuda_device), _cuda(table, cuda_device)
    query = torch.randn(3, 4, d, device=cuda_device)
    got = mi.paged_decode_mxfp4(query, kt, vt, tt, torch.full((3,), 60, dtype=torch.int32, device=cuda_device))
    nan = torch.isnan(got)
    assert bool(nan[0, :, d - 32:].all()) and not bool(nan[0, :, :d - 32].any())
    assert not bool(nan[1].any()) and bool(nan[2].all())
    want = mo.attention(query[1:2].double().cpu().numpy(), mo.rows(kp, table[1], 60), mo.rows(vp, table[1], 60), d ** -0.5)
    _close(got[1:2], *want, torch.float32, DECODE_STEP[torch.float32])


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("group", [1, 5])
def test_prefill_every_head_dim(cuda_device, name, d, group):
    """Chunks of one token and of several tiles, a context split over its keys; in shapes that are computed
    from the pages also a context shorter than its chunk, whose first rows see no key."""
    short = d != 128 and not (name == "f32" and d > 128)
    q_lens, ctxs = [140, 1, 3, 20, 9], [140, 3000, 3, 77, 5 if short else 9]
    got, free, want, dtype = _prefill_case(cuda_device, name, 2, group, d, 32, q_lens, ctxs)
    if short:
        assert bool((got[164:168] == 0).all())
    _close(got, *want, dtype, PREFILL_STEP[dtype])
    _close(free, *want, dtype, PREFILL_STEP[dtype])


@gpu
@pytest.mark.parametrize("d", [32, 96, 160, 192, 224, 256])
def test_prefill_nan_blocks_of_every_head_dim(cuda_device, d):
    nb = d // 32
    rng = np.random.default_rng(d)
    kp, vp = _pages(rng, 6, 16, 1, d)
    vp.reshape(6, 1, 1, -1)[..., nb * 256:].reshape(6, 16, nb)[4, 6, nb - 1] = 255  # key 70
    table = np.arange(6, dtype=np.int32).reshape(1, 6)
    cu = torch.tensor([0, 96], dtype=torch.int32, device=cuda_device)
    query = torch.randn(96, 3, d, device=cuda_device, dtype=torch.bfloat16)
    got = mi.paged_prefill_mxfp4(query, _cuda(kp, cuda_device), _cuda(vp, cuda_device), cu, cu,
                                 _cuda(table, cuda_device), max_seqlen_q=96)
    nan = torch.isnan(got)
    assert bool(nan[70:, :, d - 32:].all()) and int(nan.sum()) == 26 * 3 * 32


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 96, 256])
def test_prefill_values_past_fp16(cuda_device, name, d):
    """V blocks of 2^14 to 2^40 reach the rows that see them, with their weight, and no row before."""
    def edit(kp, vp, table):
        code, byte = mo.unpack(vp)
        for i, pos in enumerate([5, 6, 17, 40, 63, 64, 70, 89]):
            byte[table[0, pos // 16], pos % 16, 0, i % (d // 32)] = 127 + [14, 15, 20, 40][i % 4]
        vp[:] = mo.pack(code, byte)

    got, free, want, dtype = _prefill_case(cuda_device, name, 1, 3, d, 16, [86], [90], edit=edit)
    for x in (got, free):
        _close_or_past(x, *want, dtype, PREFILL_STEP[dtype])
    assert bool(torch.isfinite(got[0]).all())  # position 4: before the first of them

