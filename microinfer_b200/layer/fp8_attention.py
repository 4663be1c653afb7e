"""Attention over the 8-bit paged cache (``worker.fp8_cache``).

* ``paged_decode_fp8``        one query token per request, as ``paged_decode``
* ``paged_prefill_fp8``       causal chunked prefill on a cached prefix, as ``paged_prefill``
* ``gather_paged_kv_fp8``     rows in logical order, as ``gather_paged_kv``
* ``paged_attention_fp8_meta``  dispatch on the step's metadata, as ``paged_attention_meta``

Decode reads the codes and decodes them in registers.  Prefill has three ways.  Where many rows share the keys of a
shape that the dense tensor-core kernel takes, each context is decoded once into a workspace of the query's
type (twice its pages) and that kernel attends to the rows.  Elsewhere the pages are read: by a tcgen05 kernel (16-bit
queries, head_dim 64 and 128), or by one on the warp-level tensor cores for little work and everything
else.  All give the same result up to rounding: what the tensor-core kernels cannot do (a NaN of V,
scales too far apart, K or V at the ends of the range of 16 bits, scores past 2^20) is done over by the third.  The choice goes by
the shapes and the bounds
``max_seqlen_q``, ``max_seqlen_k`` and ``total_k``, never by what the tensors hold.
Workspaces come from torch's allocator for the length of the call, so that calls on several
streams, and captured graphs, each have their own.
"""

from __future__ import annotations

import math
from functools import lru_cache

import torch

from microinfer_b200 import _lib
from microinfer_b200.layer.mxfp4_attention import _aligned, _check_query, _overlap, coded_attention_meta
from microinfer_b200.layer.paged_attention import _idx
from microinfer_b200.worker.fp8_cache import page_dims


@lru_cache(maxsize=4096)
def _decode_workspace_bytes(*shape):
    return _lib.load().mi_paged_decode_fp8_workspace_bytes(*shape)


def paged_decode_fp8(query, key_pages, value_pages, block_tables, context_lens, *,
                     scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """One query token per request over its 8-bit pages; a request without keys gives zeros.

    ``query`` [requests, Hq, D] in fp32, fp16 or bf16, any group Hq / Hkv.
    """
    if torch.compiler.is_compiling():  # an opaque node for torch.compile
        res = torch.ops.microinfer_b200.paged_decode_fp8(query, key_pages, value_pages,
                                                         block_tables, context_lens, scale)
        return res if out is None else out.copy_(res)
    nb, bs, hkv, d = page_dims(key_pages, value_pages)
    n, hq = _check_query(query, hkv, d, out)
    dtype = _lib.dtype_code(query.dtype)
    table_shape = block_tables.shape
    if len(table_shape) != 2 or table_shape[0] != n:
        raise ValueError("block_tables must have one row per request")
    if context_lens.shape != (n,):
        raise ValueError("context_lens must have one entry per request")
    if n == 0:
        return query.new_empty(query.shape) if out is None else out
    device = _lib.require_cuda(query, key_pages, value_pages, block_tables, context_lens)
    width = table_shape[1]
    if width == 0:  # no request can have a key
        return query.new_zeros(query.shape) if out is None else out.zero_()
    query, block_tables, context_lens = _aligned(query), _idx(block_tables), _idx(context_lens)
    if out is None:
        out = torch.empty_like(query)
    need = _decode_workspace_bytes(n, nb, bs, hq, hkv, d, dtype, width, device.index or 0)
    workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    _lib.call(
        "mi_paged_decode_fp8", out.data_ptr(), query.data_ptr(), key_pages.data_ptr(),
        value_pages.data_ptr(), nb, bs, hq, hkv, d, dtype, block_tables.data_ptr(), width,
        context_lens.data_ptr(), n, 1.0 / math.sqrt(d) if scale is None else float(scale),
        _lib.ptr(workspace), need, _lib.status_buffer(device).data_ptr(), _lib.stream_of(device),
    )
    return out


def _gather(keys, values, key_pages, value_pages, dims, block_tables, cu_seqlens_k, rows, most, device):
    requests, width = block_tables.shape
    _lib.call(
        "mi_gather_paged_kv_fp8", keys.data_ptr(), values.data_ptr(), key_pages.data_ptr(),
        value_pages.data_ptr(), *dims, _lib.dtype_code(keys.dtype), block_tables.data_ptr(), width,
        cu_seqlens_k.data_ptr(), requests, rows, most, _lib.status_buffer(device).data_ptr(),
        _lib.stream_of(device),
    )


def gather_paged_kv_fp8(key_pages, value_pages, block_tables, contexts, *,
                        dtype: torch.dtype = torch.bfloat16,
                        cu_seqlens_k: torch.Tensor | None = None, out=None):
    """Rows of each request in logical order, request-major, as ``dtype``.

    ``contexts`` is a host sequence of context lengths; ``cu_seqlens_k`` (device,
    cumulative) skips the host prefix sum and its copy; ``out=(keys, values)``
    (contiguous ``[sum(contexts), Hkv, D]``) writes into existing tensors of any of the types.
    """
    dims = page_dims(key_pages, value_pages)
    _, bs, hkv, d = dims
    device = _lib.require_cuda(key_pages, value_pages, block_tables, cu_seqlens_k)
    contexts = [int(c) for c in contexts]
    table_shape = block_tables.shape
    if len(table_shape) != 2 or len(contexts) != table_shape[0]:
        raise ValueError("one context per block-table row")
    if contexts and min(contexts) < 0:
        raise ValueError("contexts must be non-negative")
    total = sum(contexts)
    if out is None:
        _lib.dtype_code(dtype)
        keys = torch.empty((total, hkv, d), dtype=dtype, device=device)
        values = torch.empty_like(keys)
    else:
        keys, values = out
        want = (total, hkv, d)
        if (keys.shape != want or values.shape != want or keys.dtype != values.dtype
                or not (keys.is_contiguous() and values.is_contiguous())):
            raise ValueError("out must be two contiguous [sum(contexts), Hkv, D] tensors of one dtype")
        _lib.dtype_code(keys.dtype)
        _lib.require_cuda(key_pages, keys, values)
    if total == 0:
        return keys, values
    most = max(contexts)
    if most > table_shape[1] * bs:
        raise ValueError("a context is longer than its block-table row")
    if cu_seqlens_k is None:
        cu = [0]
        for c in contexts:
            cu.append(cu[-1] + c)
        cu_seqlens_k = torch.tensor(cu, dtype=torch.int32).to(device, non_blocking=True)
    elif cu_seqlens_k.shape != (len(contexts) + 1,):
        raise ValueError("cu_seqlens_k must have num_requests + 1 entries")
    _gather(keys, values, key_pages, value_pages, dims, _idx(block_tables), _idx(cu_seqlens_k),
            total, most, device)
    return keys, values


@lru_cache(maxsize=4096)
def _prefill_workspace_bytes(*shape):
    return _lib.load().mi_paged_prefill_fp8_workspace_bytes(*shape)


@lru_cache(maxsize=4096)
def _reads_pages(dtype, hq, hkv, d, requests, max_seqlen_q, most, device):
    """Whether prefill reads the pages itself instead of gathering for the dense kernel.

    Where the dense kernel does not take the shape; for little work, up to 5 tiles of 128 rows x 128 keys for every two SMs
    (16 to 42 us where two kernels more take 28 to 44); from 3000 keys where its tiles of 128
    rows do not fill the SMs (reading the pages splits the keys: 1 x 256 rows on 16000, 32 heads on 8, 142 us where the dense way
    takes 314), or a sequence has at most 256 rows of a kv head to gather its keys for (16 x 64 on 8000: 251, 296).
    Else the rows are worth decoding once: 1 x 4096 takes 236 us there and 312 from the pages, 4 x 1024 on 4000 314 and 431.
    """
    lib = _lib.load()
    if lib.mi_prefill_kernel_for(dtype, d, hq, hkv, 0) != 2:
        return True
    sms, rows = lib.mi_device_sm_count(device), max_seqlen_q * (hq // hkv)
    tiles = requests * hkv * -(-rows // 128)
    if 2 * tiles * -(-most // 128) <= 5 * sms:
        return True
    return most >= 3000 and (tiles <= sms or rows <= 256)


def paged_prefill_fp8(query, key_pages, value_pages, cu_seqlens_q, cu_seqlens_k, block_tables, *,
                      max_seqlen_q: int, total_k: int | None = None, scale: float | None = None,
                      out: torch.Tensor | None = None,
                      max_seqlen_k: int | None = None) -> torch.Tensor:
    """Causal chunked prefill from the 8-bit cache; also mixed batches.

    As ``paged_prefill``: request r's rows sit at the end of its context
    (``cu_seqlens_k`` is cumulative over contexts, the chunk included, which is
    already stored).  ``total_k`` is the sum of the contexts (or a bound on
    it) and sizes the workspace; without it the block table's capacity does.
    ``max_seqlen_k`` (likewise a bound) is the longest of them.
    """
    if torch.compiler.is_compiling():  # an opaque node for torch.compile
        res = torch.ops.microinfer_b200.paged_prefill_fp8(
            query, key_pages, value_pages, cu_seqlens_q, cu_seqlens_k, block_tables,
            int(max_seqlen_q), total_k, scale, max_seqlen_k)
        return res if out is None else out.copy_(res)
    dims = page_dims(key_pages, value_pages)
    _, bs, hkv, d = dims
    _check_query(query, hkv, d, out)
    _lib.dtype_code(query.dtype)
    if block_tables.ndim != 2:
        raise ValueError("block_tables must have one row per request")
    requests, width = block_tables.shape
    if cu_seqlens_q.shape != (requests + 1,) or cu_seqlens_k.shape != (requests + 1,):
        raise ValueError("cu_seqlens_q and cu_seqlens_k must have num_requests + 1 entries")
    if query.shape[0] == 0 or requests == 0:
        return query.new_empty(query.shape) if out is None else out
    if max_seqlen_q <= 0:
        raise ValueError("max_seqlen_q must be positive")
    if total_k is not None and total_k < 0:
        raise ValueError("total_k must be non-negative")
    if max_seqlen_k is not None and max_seqlen_k < 0:
        raise ValueError("max_seqlen_k must be non-negative")
    device = _lib.require_cuda(query, key_pages, value_pages, cu_seqlens_q, cu_seqlens_k, block_tables)
    most = width * bs  # keys of one request
    if max_seqlen_k is not None:
        most = min(most, int(max_seqlen_k))
    rows = requests * most
    if total_k is not None:
        rows = min(rows, int(total_k))
        most = min(most, rows)
    if rows == 0:  # no request can have a key
        return query.new_zeros(query.shape) if out is None else out.zero_()
    query, block_tables = _aligned(query), _idx(block_tables)
    cu_seqlens_q, cu_seqlens_k = _idx(cu_seqlens_q), _idx(cu_seqlens_k)
    tokens, hq, _ = query.shape
    dtype = _lib.dtype_code(query.dtype)
    if out is None:
        out = torch.empty_like(query)
    elif _overlap(out, query):  # some rows may be done twice
        query = query.clone()
    if _reads_pages(dtype, hq, hkv, d, requests, int(max_seqlen_q), most, device.index or 0):
        need = _prefill_workspace_bytes(requests, tokens, int(max_seqlen_q), dims[0], bs, hq, hkv, d, dtype, most,
                                        device.index or 0)
        workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        _lib.call(
            "mi_paged_prefill_fp8", out.data_ptr(), query.data_ptr(), key_pages.data_ptr(),
            value_pages.data_ptr(), dims[0], bs, hq, hkv, d, dtype,
            cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(), block_tables.data_ptr(), width,
            requests, tokens, int(max_seqlen_q), most,
            1.0 / math.sqrt(d) if scale is None else float(scale), _lib.ptr(workspace), need,
            _lib.status_buffer(device).data_ptr(), _lib.stream_of(device),
        )
        return out
    need = _lib.load().mi_paged_prefill_fp8_gathered_workspace_bytes(requests, most, rows, hkv, d, dtype)
    workspace = torch.empty(need, dtype=torch.uint8, device=device)
    _lib.call(
        "mi_paged_prefill_fp8_gathered", out.data_ptr(), query.data_ptr(), key_pages.data_ptr(),
        value_pages.data_ptr(), dims[0], bs, hq, hkv, d, dtype, cu_seqlens_q.data_ptr(),
        cu_seqlens_k.data_ptr(), block_tables.data_ptr(), width, requests, tokens, int(max_seqlen_q),
        most, rows, 1.0 / math.sqrt(d) if scale is None else float(scale), workspace.data_ptr(), need,
        _lib.status_buffer(device).data_ptr(), _lib.stream_of(device),
    )
    return out


def paged_attention_fp8_meta(query, key_pages, value_pages, metadata, *,
                             scale: float | None = None) -> torch.Tensor:
    """Backend dispatch on validated metadata, as ``paged_attention_meta`` over the 8-bit cache."""
    return coded_attention_meta(query, key_pages, value_pages, metadata, scale, paged_decode_fp8,
                                paged_prefill_fp8, page_dims)
