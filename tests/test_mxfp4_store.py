"""What the quantising store takes."""

import numpy as np
import pytest
import torch

import microinfer_b200 as mi
from oracle import mxfp4_oracle as mo

gpu = pytest.mark.gpu


@pytest.mark.parametrize("shape", ["keys", "values", "both"])
def test_store_of_one_kv_head_takes_any_head_stride(shape):
    """With one kv head the stride of that dimension has no meaning (a transpose of [1, T, D] is contiguous)."""
    pages = torch.zeros(4, 1, 1, 544, dtype=torch.uint8)
    slots = torch.zeros(3, dtype=torch.int32)
    plain, turned = torch.zeros(3, 1, 64), torch.zeros(1, 3, 64).transpose(0, 1)
    assert turned.stride() == (64, 192, 1) and turned.is_contiguous()
    k, v = (turned if shape in (n, "both") else plain for n in ("keys", "values"))
    with pytest.raises(ValueError, match="CUDA tensors"):  # every other check is passed
        mi.store_kv_mxfp4(pages, pages, slots, k, v)


@gpu
@pytest.mark.parametrize("heads", [1, 2])
def test_store_through_a_layer_of_rows_that_are_a_transpose(cuda_device, heads):
    layer = mi.MXFP4KVCache(1, 2, 16, heads, 64, device=cuda_device).layer(0)
    k, v = (torch.randn(heads, 5, 64, device=cuda_device).transpose(0, 1) for _ in range(2))
    layer.write_checked(torch.tensor([3, 4, 20, 0, 31], device=cuda_device), k, v)
    table = torch.tensor([[0, 1]], dtype=torch.int32, device=cuda_device)
    for got, rows in zip(mi.gather_paged_kv_mxfp4(layer.keys, layer.values, table, [32], dtype=torch.float32), (k, v)):
        want = mo.decode(*mo.encode(rows.double().cpu().numpy()))
        assert np.array_equal(got[[3, 4, 20, 0, 31]].double().cpu().numpy(), want)
    mi.check_device_status(cuda_device)
