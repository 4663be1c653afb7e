"""The C entries of the 4-bit cache, called as a C program would call them."""

import numpy as np
import pytest
import torch

import microinfer_b200 as mi
from microinfer_b200 import _lib
from tests.test_mxfp4 import _cuda, _pages

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("d,hq", [(64, 8), (128, 4), (128, 16), (256, 4)])
def test_a_workspace_that_is_not_needed_is_left_alone(cuda_device, d, hq):
    """Short tables need no workspace, so one that the caller has all the same may be of any size."""
    lib = _lib.load()
    rng = np.random.default_rng(d)
    kp, vp = _pages(rng, 4, 16, 2, d)
    kt, vt = _cuda(kp, cuda_device), _cuda(vp, cuda_device)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=cuda_device)
    lens = torch.tensor([20, 0], dtype=torch.int32, device=cuda_device)
    query = torch.randn(2, hq, d, device=cuda_device, dtype=torch.bfloat16)
    assert lib.mi_paged_decode_mxfp4_workspace_bytes(2, 4, 16, hq, 2, d, 2, 2, 0) == 0
    around = torch.full((8 << 20,), 0x5A, dtype=torch.uint8, device=cuda_device)
    small = around[64:80]
    out = torch.empty_like(query)
    code = _lib.dtype_code(query.dtype)
    _lib.call("mi_paged_decode_mxfp4", out.data_ptr(), query.data_ptr(), kt.data_ptr(), vt.data_ptr(), 4, 16, hq, 2, d,
              code, table.data_ptr(), 2, lens.data_ptr(), 2, d ** -0.5, small.data_ptr(), small.numel(),
              _lib.status_buffer(cuda_device).data_ptr(), _lib.stream_of(cuda_device))
    assert torch.equal(out, mi.paged_decode_mxfp4(query, kt, vt, table, lens))
    cu_q = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda_device)
    cu_k = torch.tensor([0, 20, 21], dtype=torch.int32, device=cuda_device)
    assert lib.mi_paged_prefill_mxfp4_workspace_bytes(2, 2, 1, hq, 2, d, 32, 0) == 0
    _lib.call("mi_paged_prefill_mxfp4", out.data_ptr(), query.data_ptr(), kt.data_ptr(), vt.data_ptr(), 4, 16, hq, 2, d,
              code, cu_q.data_ptr(), cu_k.data_ptr(), table.data_ptr(), 2, 2, 2, 1, 32, d ** -0.5, small.data_ptr(),
              small.numel(), _lib.status_buffer(cuda_device).data_ptr(), _lib.stream_of(cuda_device))
    mi.check_device_status(cuda_device)
    assert bool((around == 0x5A).all())


def test_prefill_refuses_tables_whose_positions_pass_32_bits():
    """Up to three tiles of 64 keys past the last one are looked up, so a table may hold 256 positions less than 2^31."""
    lib = _lib.load()
    p = np.zeros(64, dtype=np.uint8).ctypes.data

    def prefill(block_size, width):
        # the misaligned query is refused after the sizes and before any launch
        return lib.mi_paged_prefill_mxfp4(p, p | 1, p, p, 4, block_size, 4, 2, 64, 2, p, p, p, width, 1, 1, 1, 16, 0.1, None,
                                          0, None, None)

    unsupported, alignment = -2, prefill(16, 2)
    assert alignment < 0 and alignment != unsupported
    assert prefill(16, (2 ** 31 - 16) // 16) == unsupported  # 2^31 - 16 positions
    assert prefill(1 << 20, 2047) == alignment
    assert prefill(16, 2 ** 60) == unsupported


def test_gathered_prefill_refuses_bad_arguments():
    lib = _lib.load()
    p = np.zeros(64, dtype=np.uint8).ctypes.data

    def prefill(dtype=2, bs=16, d=128, hq=4, n=1, tokens=1, q=1, most=16, rows=16, query=p, ws=p, nbytes=0):
        return lib.mi_paged_prefill_mxfp4_gathered(p, query, p, p, 4, bs, hq, 2, d, dtype, p, p, p, 2, n, tokens, q, most, rows,
                                                   0.1, ws, nbytes, None, None)

    assert prefill(n=0) == 0 and prefill(tokens=0) == 0
    for bad in (dict(dtype=9), dict(bs=8), dict(d=48), dict(hq=3), dict(n=-1), dict(n=70000), dict(q=0), dict(most=0), dict(rows=0),
                dict(rows=-1), dict(query=None), dict(query=p | 1), dict(ws=None), dict(nbytes=100), dict(most=2 ** 40)):
        assert prefill(**bad) < 0
    size = lib.mi_paged_prefill_mxfp4_gathered_workspace_bytes
    assert size(3, 17, 10, 2, 128, 2) == 2 * 10 * 2 * 128 * 2 + 3 * 2 * 2
    assert size(0, 17, 10, 2, 128, 2) == 0 and size(3, 17, 10, 2, 128, 9) == 0
