"""Attention over the 4-bit paged cache (``worker.mxfp4_cache``).

* ``paged_decode_mxfp4``        one query token per request, as ``paged_decode``
* ``paged_prefill_mxfp4``       causal chunked prefill on a cached prefix, as ``paged_prefill``
* ``gather_paged_kv_mxfp4``     rows in logical order, as ``gather_paged_kv``
* ``paged_attention_mxfp4_meta``  dispatch on the step's metadata, as ``paged_attention_meta``

Decode reads the codes and decodes them in registers.  Prefill has two ways.  Where there are tiles enough for
the dense tensor-core kernel, each context is decoded once into a workspace of the query's type (3.76 times its
pages in 16 bits) and that kernel attends to the rows: a chunk of n tokens does 4 * n * Hq flops for each of the
Hkv elements decoded, so the extra pass is a few percent of a large chunk, and most of the call
where every request has a few tokens.  Few tiles, and shapes that kernel does not take, are computed from the
pages.  Both give the same result up to rounding: sequences with what the dense kernel cannot do
(a NaN or, in fp16, a block past its range; a page that is none) are done over from the pages.
Workspaces come from torch's allocator for the length of the call, so that calls on several
streams, and captured graphs, each have their own.
"""

from __future__ import annotations

import math
from functools import lru_cache

import torch

from microinfer_b200 import _lib
from microinfer_b200.layer.paged_attention import _idx
from microinfer_b200.worker.mxfp4_cache import page_dims


def _check_query(query, hkv, d, out):
    """(tokens, Hq) of a query over a cache of these heads."""
    shape = query.shape
    if len(shape) != 3:
        raise ValueError("query must have shape [tokens, Hq, D]")
    tokens, hq, query_dim = shape
    if query_dim != d:
        raise ValueError("query and cache head dimensions differ")
    if hq == 0 or hq % hkv:
        raise ValueError("Hq must be divisible by Hkv")
    if out is not None:
        if out.shape != shape or out.dtype != query.dtype or not out.is_contiguous():
            raise ValueError("out must be contiguous, of the query's shape and dtype")
        if out.device != query.device:
            raise ValueError("out must be on the query's device")
    return tokens, hq


def _aligned(t: torch.Tensor) -> torch.Tensor:
    if not t.is_contiguous():
        return t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two contiguous tensors of as many bytes share any."""
    return abs(a.data_ptr() - b.data_ptr()) < a.numel() * a.element_size()


@lru_cache(maxsize=4096)
def _decode_workspace_bytes(*shape):
    return _lib.load().mi_paged_decode_mxfp4_workspace_bytes(*shape)


def paged_decode_mxfp4(query, key_pages, value_pages, block_tables, context_lens, *,
                       scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """One query token per request over its 4-bit pages; a request without keys gives zeros.

    ``query`` [requests, Hq, D] in fp32, fp16 or bf16, any group Hq / Hkv.
    """
    if torch.compiler.is_compiling():  # an opaque node for torch.compile
        res = torch.ops.microinfer_b200.paged_decode_mxfp4(query, key_pages, value_pages,
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
        "mi_paged_decode_mxfp4", out.data_ptr(), query.data_ptr(), key_pages.data_ptr(),
        value_pages.data_ptr(), nb, bs, hq, hkv, d, dtype, block_tables.data_ptr(), width,
        context_lens.data_ptr(), n, 1.0 / math.sqrt(d) if scale is None else float(scale),
        _lib.ptr(workspace), need, _lib.status_buffer(device).data_ptr(), _lib.stream_of(device),
    )
    return out


def _gather(keys, values, key_pages, value_pages, dims, block_tables, cu_seqlens_k, rows, most, device):
    requests, width = block_tables.shape
    _lib.call(
        "mi_gather_paged_kv_mxfp4", keys.data_ptr(), values.data_ptr(), key_pages.data_ptr(),
        value_pages.data_ptr(), *dims, _lib.dtype_code(keys.dtype), block_tables.data_ptr(), width,
        cu_seqlens_k.data_ptr(), requests, rows, most, _lib.status_buffer(device).data_ptr(),
        _lib.stream_of(device),
    )


def gather_paged_kv_mxfp4(key_pages, value_pages, block_tables, contexts, *,
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
    return _lib.load().mi_paged_prefill_mxfp4_workspace_bytes(*shape)


@lru_cache(maxsize=4096)
def _reads_pages(dtype, hq, hkv, d, requests, max_seqlen_q, device):
    """Whether prefill reads the pages itself instead of gathering for the dense kernel.

    It does where the tcgen05 kernel does not take the shape (8 x 250 tokens on 2000, 16/8 heads of
    256: 361 us, gathered 19103; 8 x 8 on nothing: 14 and 29), and where that would leave three
    quarters of the SMs without a tile of 128 rows: reading the pages splits the keys
    (128 tokens on 16000, 32/8 heads of 128: 151 us, gathered 294; 256 tokens: 317 and 297).
    Many requests of few tokens are many tiles, nearly empty in both kernels, and the dense one is faster on them
    (64 x 4 on 8192, 32/8 heads of 128: 967 us, from the pages 1484).  The rule knows neither contexts nor
    the real chunks: short contexts (4 x 64 on 64: 14 us from the pages, gathered 17) and one chunk among
    decode rows (512 tokens and 63 rows on 8192: 1864, gathered 2452) go the slower way.
    """
    if dtype == _lib.dtype_code(torch.float32) and d > 128:  # q's three parts outgrow shared memory
        return False
    lib = _lib.load()
    if lib.mi_prefill_kernel_for(dtype, d, hq, hkv, 0) != 2:
        return True
    tiles = requests * hkv * -(-max_seqlen_q * (hq // hkv) // 128)
    return 4 * tiles <= lib.mi_device_sm_count(device)


def paged_prefill_mxfp4(query, key_pages, value_pages, cu_seqlens_q, cu_seqlens_k, block_tables, *,
                        max_seqlen_q: int, total_k: int | None = None, scale: float | None = None,
                        out: torch.Tensor | None = None,
                        max_seqlen_k: int | None = None) -> torch.Tensor:
    """Causal chunked prefill from the 4-bit cache; also mixed batches.

    As ``paged_prefill``: request r's rows sit at the end of its context
    (``cu_seqlens_k`` is cumulative over contexts, the chunk included, which is
    already stored).  ``total_k`` is the sum of the contexts (or a bound on
    it) and sizes the workspace; without it the block table's capacity does.
    ``max_seqlen_k`` (likewise a bound) is the longest of them.
    """
    if torch.compiler.is_compiling():  # an opaque node for torch.compile
        res = torch.ops.microinfer_b200.paged_prefill_mxfp4(
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
    if _reads_pages(dtype, hq, hkv, d, requests, int(max_seqlen_q), device.index or 0):
        if out is None:
            out = torch.empty_like(query)
        shape = (requests, tokens, int(max_seqlen_q), hq, hkv, d, most, device.index or 0)
        need = _prefill_workspace_bytes(*shape)
        workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        _lib.call(
            "mi_paged_prefill_mxfp4", out.data_ptr(), query.data_ptr(), key_pages.data_ptr(),
            value_pages.data_ptr(), dims[0], bs, hq, hkv, d, dtype,
            cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(), block_tables.data_ptr(), width,
            requests, tokens, int(max_seqlen_q), most,
            1.0 / math.sqrt(d) if scale is None else float(scale), _lib.ptr(workspace), need,
            _lib.status_buffer(device).data_ptr(), _lib.stream_of(device),
        )
        return out
    if out is None:
        out = torch.empty_like(query)
    elif _overlap(out, query):  # some rows may be done twice
        query = query.clone()
    need = _lib.load().mi_paged_prefill_mxfp4_gathered_workspace_bytes(requests, most, rows, hkv, d, dtype)
    workspace = torch.empty(need, dtype=torch.uint8, device=device)
    _lib.call(
        "mi_paged_prefill_mxfp4_gathered", out.data_ptr(), query.data_ptr(), key_pages.data_ptr(),
        value_pages.data_ptr(), dims[0], bs, hq, hkv, d, dtype, cu_seqlens_q.data_ptr(),
        cu_seqlens_k.data_ptr(), block_tables.data_ptr(), width, requests, tokens, int(max_seqlen_q),
        most, rows, 1.0 / math.sqrt(d) if scale is None else float(scale), workspace.data_ptr(), need,
        _lib.status_buffer(device).data_ptr(), _lib.stream_of(device),
    )
    return out


def paged_attention_mxfp4_meta(query, key_pages, value_pages, metadata, *,
                               scale: float | None = None) -> torch.Tensor:
    """Backend dispatch on validated metadata, as ``paged_attention_meta`` over the 4-bit cache."""
    if query.shape[0] == 0:
        return torch.empty_like(query)
    block_tables = metadata.block_tables
    if block_tables is None:
        raise ValueError("paged attention needs metadata.block_tables")
    if metadata.is_decode and metadata.context_lens is not None:
        return paged_decode_mxfp4(query, key_pages, value_pages, block_tables,
                                  metadata.context_lens, scale=scale)
    cu_q, cu_k = metadata.cu_seqlens_q, metadata.cu_seqlens_k
    if cu_q is None:
        cu_q = torch.tensor(metadata.cu_q_cpu, dtype=torch.int32, device=query.device)
    if cu_k is None:
        if metadata.context_lens is None:
            raise ValueError("metadata needs cu_seqlens_k or context_lens")
        cu_k = torch.zeros(metadata.context_lens.numel() + 1, dtype=torch.int32,
                           device=query.device)
        torch.cumsum(metadata.context_lens, 0, out=cu_k[1:])
    max_q = metadata.max_seqlen_q or max(metadata.q_lens_cpu, default=0)
    return paged_prefill_mxfp4(query, key_pages, value_pages, cu_q, cu_k, block_tables,
                               max_seqlen_q=max_q, total_k=_total_k(query, key_pages, metadata),
                               scale=scale, max_seqlen_k=metadata.max_seqlen_k or None)


# K and V rows of a gathered prefill that may be allocated for a bound on the contexts rather than their sum.
_BOUND_BYTES = 256 << 20


def _total_k(query, key_pages, metadata) -> int | None:
    """The sum of the step's contexts, which sizes a gathered prefill, or a bound on it.

    Metadata that does not say costs one copy of the lengths to the host per step, which is
    not made where a bound will do (the longest context, or else the block table's width, for every
    request) or the host does not know yet (in a capture, whose replays may have other lengths).
    """
    total = getattr(metadata, "total_seqlen_k", 0)
    if total:
        return total
    requests, width = metadata.block_tables.shape
    _, bs, hkv, d = page_dims(key_pages, key_pages)
    bound = requests * (metadata.max_seqlen_k or width * bs)
    if (2 * bound * hkv * d * query.element_size() <= _BOUND_BYTES or torch.compiler.is_compiling()
            or (query.is_cuda and torch.cuda.is_current_stream_capturing())):
        return bound
    return sum(metadata.context_lens_cpu)
