"""The 4-bit layer behind the step's metadata."""

import numpy as np
import pytest
import torch

import microinfer_b200 as mi
from microinfer_b200.layer.mxfp4_attention import paged_attention_mxfp4_meta
from oracle import mxfp4_oracle as mo
from tests.test_mxfp4 import DECODE_STEP, PREFILL_STEP, _close, _cuda, _pages, _table
from tests.test_runner_metadata import FakeSeq

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("given", ["sum", "longest", "lens", "offsets"])
def test_prefill_workspace_follows_the_contexts(cuda_device, given):
    """One long context among short ones: K and V of the contexts, not of their number times the longest."""
    rng = np.random.default_rng(60)
    q_lens, ctxs, hkv, d, bs = [130] * 31 + [140], [130] * 31 + [20000], 8, 128, 16
    need = [-(-c // bs) for c in ctxs]
    kt = torch.zeros(sum(need), hkv, 1, 1088, dtype=torch.uint8, device=cuda_device)
    table = torch.full((32, 2000), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = torch.arange(at, at + n, dtype=torch.int32)
        at += n
    cu_q, cu_k = (torch.tensor([0, *np.cumsum(x)], dtype=torch.int32, device=cuda_device) for x in (q_lens, ctxs))
    fields = {"sum": dict(cu_seqlens_k=cu_k, max_seqlen_k=max(ctxs), total_seqlen_k=sum(ctxs)),
              "longest": dict(cu_seqlens_k=cu_k, max_seqlen_k=max(ctxs)), "offsets": dict(cu_seqlens_k=cu_k),
              "lens": dict(context_lens=torch.tensor(ctxs, dtype=torch.int32, device=cuda_device))}[given]
    meta = mi.AttentionMetadata.build(is_prefill=True, cu_seqlens_q=cu_q, max_seqlen_q=max(q_lens),
                                      block_tables=table.to(cuda_device), **fields)
    query = torch.randn(sum(q_lens), 16, d, device=cuda_device, dtype=torch.bfloat16)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = paged_attention_mxfp4_meta(query, kt, kt, meta)
    mi.check_device_status(cuda_device)
    rows = 2 * sum(ctxs) * hkv * d * 2
    assert bool((got == 0).all())
    assert torch.cuda.max_memory_allocated() - before <= rows + query.numel() * 2 + (8 << 20)


def test_runner_plans_the_sum_of_the_contexts():
    meta = mi.DeviceRunnerMetadata(16, 8, max_rows=3, device="cpu")
    batch = []
    for i, (cached, new) in enumerate([(0, 5), (16, 1), (7, 30)]):
        seq = FakeSeq(i)
        seq.token_ids = list(range(cached + new))
        seq.block_table = [2 * i, 2 * i + 1, 6][:-(-(cached + new) // 16)]
        seq.num_cached_tokens, seq.num_scheduled_tokens = cached, new
        batch.append(seq)
    plan = meta.plan_prefill(batch)
    assert plan["total_k"] == 5 + 17 + 37 and plan["max_k"] == 37


@gpu
@pytest.mark.parametrize("d,bs", [(64, 32), (128, 16), (256, 16)])
@pytest.mark.parametrize("prefill", [True, False])
@pytest.mark.parametrize("given", ["lens", "offsets"])
def test_metadata_with_and_without_offsets(cuda_device, d, bs, prefill, given):
    """Offsets are made of the lengths where the metadata has only those, and the longest chunk of the offsets."""
    if not prefill and given == "offsets":
        pytest.skip("decode has lengths")
    rng = np.random.default_rng(d)
    ctxs = [70, 5, 33]
    q_lens = [20, 5, 1] if prefill else [1, 1, 1]
    nb = sum(-(-c // bs) for c in ctxs)
    kp, vp = _pages(rng, nb, bs, 2, d)
    table = _table(rng, ctxs, nb, bs)
    lens = torch.tensor(ctxs, dtype=torch.int32, device=cuda_device)
    cu_q, cu_k = (torch.tensor([0, *np.cumsum(x)], dtype=torch.int32, device=cuda_device) for x in (q_lens, ctxs))
    fields = dict(context_lens=lens) if given == "lens" else dict(cu_seqlens_k=cu_k)
    if prefill:
        fields["cu_seqlens_q"] = cu_q
    meta = mi.AttentionMetadata.build(is_prefill=prefill, block_tables=_cuda(table, cuda_device), **fields)
    query = _cuda(rng.standard_normal((sum(q_lens), 8, d)), cuda_device, torch.bfloat16)
    got = paged_attention_mxfp4_meta(query, _cuda(kp, cuda_device), _cuda(vp, cuda_device), meta)
    mi.check_device_status(cuda_device)
    q, at = query.double().cpu().numpy(), np.cumsum([0, *q_lens])
    parts = [mo.attention(q[at[r]:at[r + 1]], mo.rows(kp, table[r], c), mo.rows(vp, table[r], c), d ** -0.5)
             for r, c in enumerate(ctxs)]
    _close(got, *[np.concatenate(x) for x in zip(*parts)], torch.bfloat16,
           (PREFILL_STEP if prefill else DECODE_STEP)[torch.bfloat16])


def test_bounds_on_the_contexts_are_checked():
    pages = torch.zeros(4, 2, 1, 544, dtype=torch.uint8)
    query, cu, table = torch.zeros(3, 4, 64), torch.zeros(2, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    for bad in (dict(total_k=-1), dict(max_seqlen_k=-1)):
        with pytest.raises(ValueError, match="must be non-negative"):
            mi.paged_prefill_mxfp4(query, pages, pages, cu, cu, table, max_seqlen_q=3, **bad)


@gpu
def test_a_captured_prefill_is_replayed_with_longer_contexts(cuda_device):
    """Without the sum of the contexts a capture is sized for the longest ones that its metadata allows."""
    rng = np.random.default_rng(70)
    hkv, d, bs, first, later = 8, 128, 16, [140, 150, 137, 200], [160, 400, 139, 200]
    q_lens = [130, 140, 137, 129]
    kp, vp = _pages(rng, 100, bs, hkv, d)
    table = _table(rng, [400] * 4, 100, bs)
    kt, vt, tt = _cuda(kp, cuda_device), _cuda(vp, cuda_device), _cuda(table, cuda_device)
    cu_q, cu_k = (torch.tensor([0, *np.cumsum(x)], dtype=torch.int32, device=cuda_device) for x in (q_lens, first))
    meta = mi.AttentionMetadata.build(is_prefill=True, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k, max_seqlen_q=max(q_lens),
                                      max_seqlen_k=400, block_tables=tt)
    query = _cuda(rng.standard_normal((sum(q_lens), 16, d)), cuda_device, torch.bfloat16)
    eager = paged_attention_mxfp4_meta(query, kt, vt, meta)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = paged_attention_mxfp4_meta(query, kt, vt, meta)
    graph.replay()
    assert torch.equal(got, eager)
    cu_k.copy_(torch.tensor([0, *np.cumsum(later)], dtype=torch.int32))
    graph.replay()
    mi.check_device_status(cuda_device)
    q, at = query.double().cpu().numpy(), np.cumsum([0, *q_lens])
    parts = [mo.attention(q[at[r]:at[r + 1]], mo.rows(kp, table[r], c), mo.rows(vp, table[r], c), d ** -0.5)
             for r, c in enumerate(later)]
    _close(got, *[np.concatenate(x) for x in zip(*parts)], torch.bfloat16, PREFILL_STEP[torch.bfloat16])


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hkv,d,bs", [(1, 64, 64), (2, 96, 16), (2, 256, 32)])
def test_cached_attention_of_other_heads(cuda_device, dtype, hkv, d, bs):
    """A chunk, one on its prefix and a token, through a bound layer; rows come as a transpose of heads first."""
    from microinfer_b200.layer.cached_attention import CachedAttention

    rng = np.random.default_rng(d)
    pool = mi.MXFP4KVCache(2, 6, bs, hkv, d, device=cuda_device)
    attn = CachedAttention()
    attn.bind_cache(pool.layer(1))
    table = [4, 1, 5, 0][:-(-34 // bs)]
    tt = torch.tensor([table], dtype=torch.int32, device=cuda_device)
    history, done = [np.zeros((0, hkv, d)) for _ in range(2)], 0
    for n in (12, 21, 1):
        q, k, v = (_cuda(rng.standard_normal((h, n, d)), cuda_device, dtype).transpose(0, 1) for h in (4 * hkv, hkv, hkv))
        slots = [table[pos // bs] * bs + pos % bs for pos in range(done, done + n)]
        done += n
        history = [np.concatenate([old, mo.decode(*mo.encode(new.double().cpu().numpy()))]) for old, new in zip(history, (k, v))]
        lens = torch.tensor([done], dtype=torch.int32, device=cuda_device)
        fields = dict(slot_mapping=torch.tensor(slots, dtype=torch.int32, device=cuda_device), block_tables=tt)
        if n > 1:
            fields.update(cu_seqlens_q=torch.tensor([0, n], dtype=torch.int32, device=cuda_device),
                          cu_seqlens_k=torch.tensor([0, done], dtype=torch.int32, device=cuda_device), max_seqlen_q=n,
                          max_seqlen_k=done, total_seqlen_k=done)
        else:
            fields.update(context_lens=lens)
        got = attn(q, k, v, mi.AttentionMetadata.build(is_prefill=n > 1, **fields))
        want = mo.attention(q.double().cpu().numpy(), *history, d ** -0.5)
        _close(got, *want, dtype, (PREFILL_STEP if n > 1 else DECODE_STEP)[dtype])
    mi.check_device_status(cuda_device)
    assert int(pool.keys[0].max()) == 0
