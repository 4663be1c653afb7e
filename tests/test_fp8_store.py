"""The 8-bit cache: its layout, what its entry points refuse, the quantising store and the gather."""

import ctypes

import numpy as np
import pytest
import torch

import microinfer_b200 as mi
from microinfer_b200 import _lib
from oracle import fp8_oracle as fo
from tests.fp8_support import DTYPES, cuda, pages, table_of

gpu = pytest.mark.gpu


# ---------------------------------------------------------------------------
# host side
# ---------------------------------------------------------------------------
def test_oracle_codes_and_layout():
    for code in range(127):
        assert fo.codes_of(fo.GRID[code]) == code and fo.codes_of(-fo.GRID[code]) == code + 128
    ties = (fo.GRID[1:] + fo.GRID[:-1]) / 2
    assert all(c % 2 == 0 for c in fo.codes_of(ties))
    want = torch.tensor(np.linspace(-500, 500, 4001)).clamp(-448, 448).to(torch.float8_e4m3fn)
    assert np.array_equal(fo.codes_of(np.linspace(-500, 500, 4001)), want.view(torch.uint8).numpy())
    assert fo.byte_for([0, 448, 448.0001, 224, 2.0 ** -140, 3.4e38]).tolist() == [0, 127, 128, 126, 1, 246]
    rng = np.random.default_rng(0)
    for d in (32, 64, 96, 128, 224):
        code = rng.integers(0, 256, (3, 32, 2, d)).astype(np.uint8)
        byte = rng.integers(0, 247, (3, 2, 2)).astype(np.uint8)
        for value in (False, True):
            packed = fo.pack(code, byte, value)
            again = fo.unpack(packed, value)
            assert np.array_equal(again[0], code) and np.array_equal(again[1], byte)
    v = fo.pack(code, byte, True)
    # of a first part of 64: token 11 (half 1, pair 1, last 1), dim 21 (octet 2, the fifth)
    assert v[1, 1, 0, 512 + 2 * 64 + 16 + 5 * 2 + 1] == code[1, 11, 1, 21]
    # of the last part of 32 of 224: token 6 (half 0, pair 3), dim 192 + 9 (the third quad, the second)
    assert v[2, 0, 1, 192 * 16 + 2 * 32 + 3 * 8 + 1 * 2] == code[2, 16 + 6, 0, 201]


def test_page_bytes_and_pool():
    lib = _lib.load()
    assert lib.mi_fp8_page_bytes(16, 128) == 2064
    assert lib.mi_fp8_page_bytes(64, 96) == 4 * 1552
    for bs, d in ((8, 128), (24, 64), (16, 48), (16, 288), (0, 64)):
        assert lib.mi_fp8_page_bytes(bs, d) < 0
    pool = mi.FP8KVCache(2, 3, 32, 4, 128, device="cpu")
    assert pool.num_bytes == 2 * 2 * 3 * 4 * 2 * 2064
    layer = pool.layer(1)
    assert layer.block_size == 32 and layer.head_dim == 128
    with pytest.raises(ValueError, match="layer outside"):
        pool.layer(2)
    for bad in ((2, 3, 8, 4, 128), (2, 3, 16, 4, 40), (2, 3, 16, 4, 512), (0, 3, 16, 4, 64)):
        with pytest.raises(ValueError):
            mi.FP8KVCache(*bad, device="cpu")


def test_refusals_before_any_launch():
    page = torch.zeros(4, 2, 1, 1040, dtype=torch.uint8)
    rows = torch.zeros(3, 2, 64)
    slots = torch.zeros(3, dtype=torch.int32)
    table = torch.zeros(3, 1, dtype=torch.int32)
    lens = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensors"):
        mi.store_kv_fp8(page, page, slots, rows, rows)
    with pytest.raises(ValueError, match="uint8"):
        mi.store_kv_fp8(page.int(), page.int(), slots, rows, rows)
    for size in (1024, 1032, 16, 272):
        cut = page[..., :size].contiguous()
        with pytest.raises(ValueError, match="16 \\* head_dim"):
            mi.store_kv_fp8(cut, cut, slots, rows, rows)
    with pytest.raises(ValueError, match="contiguous"):
        mi.store_kv_fp8(page[..., :528], page[..., :528], slots, rows, rows)
    with pytest.raises(ValueError, match="heads"):
        mi.store_kv_fp8(page, page, slots, rows[:, :1].contiguous(), rows[:, :1].contiguous())
    with pytest.raises(ValueError, match="share a dtype"):
        mi.store_kv_fp8(page, page, slots, rows, rows.half())
    with pytest.raises(ValueError, match="dtype"):
        mi.store_kv_fp8(page, page, slots, rows.double(), rows.double())
    with pytest.raises(ValueError, match="one entry per token"):
        mi.store_kv_fp8(page, page, slots[:2], rows, rows)
    with pytest.raises(ValueError, match="int32 or int64"):
        mi.store_kv_fp8(page, page, slots.float(), rows, rows)
    query = torch.zeros(3, 4, 64)
    with pytest.raises(ValueError, match="CUDA tensors"):
        mi.paged_decode_fp8(query, page, page, table, lens)
    with pytest.raises(ValueError, match="head dimensions"):
        mi.paged_decode_fp8(query[..., :32], page, page, table, lens)
    with pytest.raises(ValueError, match="divisible"):
        mi.paged_decode_fp8(query[:, :3], page, page, table, lens)
    with pytest.raises(ValueError, match="one row per request"):
        mi.paged_decode_fp8(query, page, page, table[:2], lens)
    with pytest.raises(ValueError, match="one entry per request"):
        mi.paged_decode_fp8(query, page, page, table, lens[:2])
    with pytest.raises(ValueError, match="dtype"):
        mi.paged_decode_fp8(query.double(), page, page, table, lens)
    with pytest.raises(ValueError, match="out must"):
        mi.paged_decode_fp8(query, page, page, table, lens, out=query[:2])
    with pytest.raises(ValueError, match="num_requests"):
        mi.paged_prefill_fp8(query, page, page, lens, lens, table, max_seqlen_q=1)
    cu = torch.zeros(4, dtype=torch.int32)
    for bad in (dict(max_seqlen_q=0), dict(max_seqlen_q=1, total_k=-1), dict(max_seqlen_q=1, max_seqlen_k=-1)):
        with pytest.raises(ValueError, match=list(bad)[-1]):
            mi.paged_prefill_fp8(query, page, page, cu, cu, table, **bad)
    with pytest.raises(ValueError, match="CUDA tensors"):
        mi.gather_paged_kv_fp8(page, page, table, [1, 1, 1])


@pytest.mark.parametrize("shape", [(4, 0, 1, 1040), (4, 2, 0, 1040), (4, 2, 1, 0)])
def test_pages_without_heads_or_tokens_are_refused(shape):
    page = torch.zeros(shape, dtype=torch.uint8)
    table, lens = torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="pages"):
        mi.paged_decode_fp8(torch.zeros(3, 4, 64), page, page, table, lens)
    with pytest.raises(ValueError, match="pages"):
        mi.gather_paged_kv_fp8(page, page, table, [1, 1, 1])


def test_store_of_one_kv_head_takes_any_head_stride():
    page = torch.zeros(4, 1, 1, 1040, dtype=torch.uint8)
    turned = torch.zeros(1, 3, 64).transpose(0, 1)  # the stride of a single head means nothing
    with pytest.raises(ValueError, match="CUDA tensors"):  # every other check is passed
        mi.store_kv_fp8(page, page, torch.zeros(3, dtype=torch.int32), turned, turned)


def test_fake_results_are_contiguous_like_the_real_ones():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        query = torch.empty(4, 3, 64).transpose(0, 1)
        page = torch.empty(4, 2, 1, 1040, dtype=torch.uint8)
        table, lens, cu = (torch.empty(n, dtype=torch.int32) for n in ((3, 1), 3, 4))
        ops = torch.ops.microinfer_b200
        for got in (ops.paged_decode_fp8(query, page, page, table, lens),
                    ops.paged_prefill_fp8(query, page, page, cu, cu, table, 1)):
            assert got.shape == query.shape and got.is_contiguous()


def test_c_entries_refuse_bad_arguments():
    lib = _lib.load()
    buf = ctypes.create_string_buffer(64)
    p = ctypes.cast(buf, ctypes.c_void_p)
    a = ctypes.c_void_p(256)  # aligned, never touched: every call below ends on the host

    def store(dtype=2, bs=16, d=64, n=1, pages=a, index=0, ws=None, size=0, nb=4):
        return lib.mi_store_kv_fp8(pages, a, nb, bs, 2, d, p, index, p, p, dtype, 128, 128, n, ws, size, None, None)

    assert store(n=0) == 0
    assert store(dtype=7) < 0 and store(bs=8) < 0 and store(d=48) < 0 and store(n=-1) < 0
    assert store(pages=None) < 0 and store(index=3) < 0 and store(n=1 << 31) < 0
    long = 100000
    need = lib.mi_store_kv_fp8_workspace_bytes(long, 40, 16)
    assert need == 40 * 16 * 4 and lib.mi_store_kv_fp8_workspace_bytes(8, 40, 16) == 0
    assert lib.mi_store_kv_fp8_workspace_bytes(long, 0, 16) == 0 and lib.mi_store_kv_fp8_workspace_bytes(long, 4, 8) == 0
    for ws, size in ((None, need), (a, need - 1), (ctypes.c_void_p(260), need)):
        assert store(n=long, nb=40, ws=ws, size=size) < 0
        assert b"workspace" in lib.mi_last_error()

    def decode(hq=4, stride=2, n=1, ws=None, q=a, d=64, size=0):
        return lib.mi_paged_decode_fp8(a, q, a, a, 4, 16, hq, 2, d, 2, p, stride, p, n, 0.1, ws, size, None, None)

    assert decode(n=0) == 0
    assert decode(hq=3) < 0 and decode(stride=-1) < 0 and decode(n=70000) < 0 and decode(q=None) < 0
    assert decode(d=320) < 0 and decode(q=ctypes.c_void_p(264)) < 0

    def gather(n=1, most=16, rows=16, dtype=2):
        return lib.mi_gather_paged_kv_fp8(a, a, a, a, 4, 16, 2, 64, dtype, p, 2, p, n, rows, most, None, None)

    assert gather(n=0) == 0 and gather(most=0) == 0 and gather(rows=0) == 0
    assert gather(n=-1) < 0 and gather(dtype=5) < 0 and gather(n=70000) < 0
    assert lib.mi_paged_decode_fp8_workspace_bytes(0, 8, 16, 4, 2, 64, 2, 100, 0) == 0

    def prefill(n=1, tokens=4, hq=4, stride=2, bs=16, longest=4, most=16):
        return lib.mi_paged_prefill_fp8(a, a, a, a, 4, bs, hq, 2, 64, 2, p, p, p, stride, n, tokens, longest, most, 0.1,
                                        None, 0, None, None)

    assert prefill(n=0) == 0 and prefill(tokens=0) == 0
    assert prefill(longest=0) < 0 and prefill(hq=3) < 0 and prefill(longest=(1 << 24) + 1) < 0
    assert prefill(stride=(1 << 27) + 1) < 0 and b"too long" in lib.mi_last_error()  # positions past 32 bits

    def gathered(hq=16, hkv=8, d=128, dtype=2, longest=4, rows=16, most=16, ws=a, size=1 << 30, stride=2):
        return lib.mi_paged_prefill_fp8_gathered(a, a, a, a, 4, 16, hq, hkv, d, dtype, p, p, p, stride, 1, 4, longest, most,
                                                 rows, 0.1, ws, size, None, None)

    for bad, word in ((dict(d=64), b"dense"), (dict(dtype=0), b"dense"), (dict(longest=0), b"positive"),
                      (dict(rows=0), b"positive"), (dict(size=64), b"workspace"), (dict(ws=None), b"workspace"),
                      (dict(hq=12), b"divisible"), (dict(stride=(1 << 27) + 1), b"too long")):
        assert gathered(**bad) < 0 and word in lib.mi_last_error(), bad
    need = lib.mi_paged_prefill_fp8_workspace_bytes
    assert need(1, 4096, 4096, 512, 16, 4, 2, 128, 2, 8192, 0) == 148 * (2 * 256 * 130 * 4 + 16 + 8)  # 148 SMs without a device
    assert need(1, 4096, 4096, 512, 16, 4, 2, 128, 0, 256, 0) == 0  # too few keys to split
    assert need(1, 4, 4, 4, 16, 4, 2, 128, 2, 16, 0) == 0  # little work: the other kernel, not split
    assert need(1, 4, 4, 4, 8, 4, 2, 128, 2, 16, 0) == 0


# ---------------------------------------------------------------------------
# store
# ---------------------------------------------------------------------------
def _check(got, code, byte, value):
    """Pages equal the oracle's, where a NaN may have either sign."""
    got_code, got_byte = fo.unpack(got.cpu().numpy(), value)
    assert np.array_equal(got_byte, byte)
    nan = code % 128 == 127
    assert np.array_equal(got_code % 128 == 127, nan)
    assert np.array_equal(got_code[~nan], code[~nan])


def _store_case(device, rng, dtype, nb, bs, hkv, d, slots, x, aligned=True, index=torch.int32, calls=1):
    kp, vp = pages(rng, nb, bs, hkv, d)
    kt, vt = cuda(kp, device), cuda(vp, device)
    x = cuda(x, device, dtype)
    keys, values = (t[:, :hkv * d].unflatten(1, (hkv, d)) for t in x)
    for _ in range(calls):
        mi.store_kv_fp8(kt, vt, cuda(slots, device, index), keys, values)
    mi.check_device_status(device)
    for page, got, new, value in ((kp, kt, keys, False), (vp, vt, values, True)):
        code, byte = fo.unpack(page, value)
        for _ in range(calls):
            fo.store(code, byte, slots, new.double().cpu().numpy())
        _check(got, code, byte, value)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hkv,d,bs", [(1, 32, 16), (8, 128, 16), (2, 64, 64), (3, 96, 32), (20, 256, 16), (5, 128, 16)])
@pytest.mark.parametrize("aligned", [True, False])
def test_store_in_any_order(cuda_device, name, hkv, d, bs, aligned):
    """A few tokens in no order: groups with and without their first slot, scales that rise and that stay."""
    rng = np.random.default_rng(hkv * 1000 + d + bs)
    nb, tokens = 7, 53
    pad = 0 if aligned else 3  # a row stride that rules out 16-byte loads
    x = rng.standard_normal((2, tokens, hkv * d + pad)) * np.exp(2 * rng.standard_normal((2, tokens, 1)))
    slots = rng.permutation(nb * bs)[:tokens].astype(np.int64)
    slots[[3, 17]] = -1
    _store_case(cuda_device, rng, DTYPES[name], nb, bs, hkv, d, slots, x, index=torch.int32 if aligned else torch.int64)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("d,aligned", [(128, True), (64, True), (96, True), (128, False)])
@pytest.mark.parametrize("order", ["runs", "any"])
def test_store_of_many_tokens(cuda_device, name, d, aligned, order):
    """More tokens than a scan takes: ragged runs that start and end inside groups, or slots in no order."""
    rng = np.random.default_rng(d)
    hkv, bs, nb = 3, 32, 60
    if order == "runs":
        runs = [np.arange(a, b) for a, b in ((5, 401), (416, 417), (480, 1000), (1037, 1300), (1900, 1920))]
        slots = np.concatenate([r for k in (2, 0, 4, 1, 3) for r in (runs[k], [-1] * k)])
    else:
        slots = rng.permutation(nb * bs)[:1100]
        slots[::97] = -1
    slots = slots.astype(np.int64)
    assert len(slots) > 512
    pad = 0 if aligned else 1
    x = rng.standard_normal((2, len(slots), hkv * d + pad)) * np.exp(rng.standard_normal((2, len(slots), 1)))
    _store_case(cuda_device, rng, DTYPES[name], nb, bs, hkv, d, slots, x, calls=2)


@gpu
@pytest.mark.parametrize("tokens", [511, 512, 513, 528])
def test_store_where_the_way_of_finding_groups_changes(cuda_device, tokens):
    rng = np.random.default_rng(tokens)
    slots = np.arange(7, 7 + tokens).astype(np.int64)
    x = rng.standard_normal((2, tokens, 2 * 64))
    _store_case(cuda_device, rng, torch.bfloat16, 36, 16, 2, 64, slots, x)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_a_group_filled_token_by_token(cuda_device, name):
    """Every token 8 times the last: each raises the scale and rounds the others again, once."""
    dtype = DTYPES[name]
    rng = np.random.default_rng(40)
    kt = torch.full((2, 2, 1, 16 * 64 + 16), 93, dtype=torch.uint8, device=cuda_device)  # a last owner's
    vt = kt.clone()
    state = [fo.unpack(kt.cpu().numpy(), False), fo.unpack(vt.cpu().numpy(), True)]
    for t in range(16):
        x = rng.standard_normal((2, 1, 2, 64)) * 8.0 ** (t - 8)
        x = cuda(x, cuda_device, dtype)
        mi.store_kv_fp8(kt, vt, torch.tensor([16 + t], device=cuda_device), x[0], x[1])
        for (code, byte), new in zip(state, x.double().cpu().numpy()):
            fo.store(code, byte, [16 + t], new)
        if t == 0:  # the first token's group starts anew
            assert all(byte[1, 0].max() < 127 for _, byte in state)
    for got, (code, byte), value in zip((kt, vt), state, (False, True)):
        _check(got, code, byte, value)
        assert np.array_equal(got.cpu().numpy()[0], np.full((2, 1, 1040), 93))  # the other page
    mi.check_device_status(cuda_device)


@gpu
def test_store_borders_and_values_that_are_not_finite(cuda_device):
    """Every code and every tie between two, both signs, at scales from the smallest to the largest; zero,
    denormal, infinite and NaN elements, alone and among others."""
    line = np.concatenate([fo.GRID, fo.MIDDLE, fo.MIDDLE * (1 + 2.0 ** -20), fo.MIDDLE * (1 - 2.0 ** -20)])
    line = np.concatenate([line, np.zeros(-len(line) % 64 or 64)]).reshape(-1, 64)
    groups = []
    for e in (-110, -30, 0, 5, 100, 119):
        part = np.zeros((16, 64))
        part[:len(line)] = line * (1 if e != 5 else -1)
        part[15, 63] = 448.0  # every group has the scale 2^e
        groups.append(part * 2.0 ** e)
    odd = np.zeros((4, 16, 64))
    odd[0, 3, 5] = 1e-40
    odd[1, 7, 9], odd[1, 7, 10], odd[1, 8, 0] = np.inf, 3.0, -np.nan
    odd[1, 9, 1] = -np.inf
    odd[2, 4, :] = np.nan  # nothing finite
    odd[3, 0, 0], odd[3, 1, 1] = 3.4028234e38, -2.0 ** 127
    small = np.zeros((2, 16, 64))
    small[0, 2, :] = 2.0 ** -126 * np.arange(64) / 64
    small[1, 5, 5] = 449.0
    rows = np.concatenate([*groups, *odd, *small]).astype(np.float32).reshape(-1, 1, 64)
    nb = len(rows) // 16
    kt = torch.zeros(nb, 1, 1, 1040, dtype=torch.uint8, device=cuda_device)
    vt = torch.zeros_like(kt)
    r = cuda(rows, cuda_device)
    slots = np.arange(len(rows))
    mi.store_kv_fp8(kt, vt, cuda(slots, cuda_device), r, -r)
    for got, x, value in ((kt, rows, False), (vt, -rows, True)):
        code, byte = np.zeros((nb, 16, 1, 64), np.uint8), np.zeros((nb, 1, 1), np.uint8)
        fo.store(code, byte, slots, x)
        _check(got, code, byte, value)
        assert byte.max() == 246 and byte[8, 0, 0] == 0
        assert int((got[..., 1025:] != 0).sum()) == 0
    table = torch.arange(nb, dtype=torch.int32, device=cuda_device)[None]
    k, v = mi.gather_paged_kv_fp8(kt, vt, table, [len(rows)], dtype=torch.float32)
    for got, pages_, value in ((k, kt, False), (v, vt, True)):
        want = fo.rows(pages_.cpu().numpy(), np.arange(nb), len(rows), value)
        assert np.array_equal(got.double().cpu().numpy(), want, equal_nan=True)


@gpu
@pytest.mark.parametrize("tokens", [3, 700])
def test_store_skips_and_flags_slots_outside_the_pool(cuda_device, tokens):
    kt = torch.full((2, 1, 1, 1040), 7, dtype=torch.uint8, device=cuda_device)
    vt = kt.clone()
    rows = torch.ones(tokens, 1, 64, device=cuda_device)
    slots = torch.full((tokens,), -1, device=cuda_device)
    slots[:3] = torch.tensor([-2, 32, -1])
    mi.store_kv_fp8(kt, vt, slots, rows, rows)
    assert mi.read_device_status(cuda_device) == _lib.DEV_BAD_SLOT
    assert bool((kt == 7).all()) and bool((vt == 7).all())
    slots[:3] = torch.tensor([1 << 40, 1 << 32, -(1 << 33)])
    mi.store_kv_fp8(kt, vt, slots, rows, rows)
    assert mi.read_device_status(cuda_device) == _lib.DEV_BAD_SLOT
    assert bool((kt == 7).all()) and bool((vt == 7).all())
    layer = mi.LayerFP8Cache(kt, vt)
    for bad in ([0, 32, 1], [-2, 0, 1], [5, 5, 1]):
        with pytest.raises(ValueError):
            layer.write_checked(torch.tensor(bad, device=cuda_device), rows[:3], rows[:3])
    assert bool((kt == 7).all())


@gpu
@pytest.mark.parametrize("tokens", [40, 600])
def test_the_same_slot_twice_is_one_of_the_two(cuda_device, tokens):
    """Not allowed, but padded batches do it: the slot holds one of its rows, the others theirs."""
    kt = torch.zeros(64, 1, 1, 528, dtype=torch.uint8, device=cuda_device)
    vt = torch.zeros_like(kt)
    rows = torch.arange(tokens, device=cuda_device).remainder(8).add(8.0).view(-1, 1, 1).expand(-1, 1, 32).contiguous()
    slots = torch.arange(tokens, device=cuda_device)
    slots[5] = slots[21]
    mi.store_kv_fp8(kt, vt, slots, rows, rows)
    table = torch.arange(64, dtype=torch.int32, device=cuda_device)[None]
    for got in mi.gather_paged_kv_fp8(kt, vt, table, [tokens], dtype=torch.float32):
        some = got[21].unique().tolist()
        assert some in ([rows[5, 0, 0].item()], [rows[21, 0, 0].item()])
        keep = [i for i in range(tokens) if i not in (5, 21)]
        assert torch.equal(got[keep], rows[keep])


@gpu
@pytest.mark.parametrize("heads", [1, 2])
def test_store_through_a_layer_of_rows_that_are_a_transpose(cuda_device, heads):
    layer = mi.FP8KVCache(1, 2, 16, heads, 64, device=cuda_device).layer(0)
    k, v = (torch.randn(heads, 5, 64, device=cuda_device).transpose(0, 1) for _ in range(2))
    slots = [3, 4, 20, 0, 31]
    layer.write_checked(torch.tensor(slots, device=cuda_device), k, v)
    for got, x, value in ((layer.keys, k, False), (layer.values, v, True)):
        code, byte = np.zeros((2, 16, heads, 64), np.uint8), np.zeros((2, 1, heads), np.uint8)
        fo.store(code, byte, slots, x.double().cpu().numpy())
        _check(got, code, byte, value)


# ---------------------------------------------------------------------------
# gather
# ---------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hkv,d,bs,ctxs", [
    (8, 128, 16, [1, 15, 16, 17, 0, 100]), (2, 64, 64, [130, 64, 63]), (1, 96, 256, [300]), (5, 256, 32, [33, 0, 1]),
    (3, 32, 48, [50])])
def test_gather_is_exact(cuda_device, name, hkv, d, bs, ctxs):
    rng = np.random.default_rng(d + bs)
    dtype = DTYPES[name]
    nb = sum(-(-c // bs) for c in ctxs) + 2
    kp, vp = pages(rng, nb, bs, hkv, d, spread=2.0)
    table = table_of(rng, ctxs, nb, bs, width=max(-(-c // bs) for c in ctxs) + 1)
    args = (cuda(kp, cuda_device), cuda(vp, cuda_device), cuda(table, cuda_device), ctxs)
    k, v = mi.gather_paged_kv_fp8(*args, dtype=dtype)
    out = torch.full_like(k, 3.0), torch.full_like(v, 3.0)
    cu = torch.tensor([0, *np.cumsum(ctxs)], dtype=torch.int32, device=cuda_device)
    mi.gather_paged_kv_fp8(*args, cu_seqlens_k=cu, out=out)
    mi.check_device_status(cuda_device)
    for got, again, page, value in ((k, out[0], kp, False), (v, out[1], vp, True)):
        want = np.concatenate([fo.rows(page, table[r], c, value) for r, c in enumerate(ctxs)])
        want = torch.from_numpy(want).to(dtype)
        assert torch.equal(got.cpu(), want) and torch.equal(again.cpu(), want)


@gpu
def test_gather_flags_bad_pages_and_stays_within_its_rows(cuda_device):
    rng = np.random.default_rng(1)
    kp, vp = pages(rng, 4, 16, 1, 64)
    kt, vt = cuda(kp, cuda_device), cuda(vp, cuda_device)
    table = torch.tensor([[0, 9], [-1, 2]], dtype=torch.int32, device=cuda_device)
    out = torch.full((64, 1, 64), 5.0, device=cuda_device), torch.full((64, 1, 64), 5.0, device=cuda_device)
    mi.gather_paged_kv_fp8(kt, vt, table, [32, 32], out=out)
    assert mi.read_device_status(cuda_device) == _lib.DEV_BAD_BLOCK
    assert np.array_equal(out[0][:16].double().cpu().numpy(), fo.rows(kp, [0], 16, False))
    assert bool((out[0][16:48] == 5.0).all())
    # offsets that run past the output's rows
    cu = torch.tensor([0, 40, 100], dtype=torch.int32, device=cuda_device)
    table = torch.tensor([[0, 1, 2, 3]] * 2, dtype=torch.int32, device=cuda_device)
    big = torch.full((96, 1, 64), 5.0, device=cuda_device), torch.full((96, 1, 64), 5.0, device=cuda_device)
    mi.gather_paged_kv_fp8(kt, vt, table, [10, 40], cu_seqlens_k=cu, out=(big[0][:50], big[1][:50]))
    assert mi.read_device_status(cuda_device) == _lib.DEV_BAD_SLOT
    assert bool((big[0][50:] == 5.0).all())
    with pytest.raises(ValueError, match="longer than"):
        mi.gather_paged_kv_fp8(kt, vt, table, [65, 1])
