"""Every way in which prefill from the 8-bit cache is computed, on the cases of the one that its sizes choose.

The choice goes by sizes, most cases here are small, and each way must give the formula's result for all that it takes: so the
choice is made for it, by a bound on the chunk's length that is far above it (the tcgen05 kernel on the pages) and in place of
the rule between pages and gathered rows.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import microinfer_b200 as mi
from microinfer_b200.layer import fp8_attention
from tests import test_fp8_attention as cases
from tests.fp8_support import DTYPES, PREFILL_STEP, close, prefill_case

gpu = pytest.mark.gpu
DENSE_LOST = cases.DENSE_LOST
FAR = 1 << 20  # rows of a chunk that nothing has: tiles enough for the tcgen05 kernel


@pytest.fixture(params=["tiles", "warps", "dense"])
def way(request, monkeypatch):
    asked = mi.paged_prefill_fp8
    pages = request.param != "dense"
    lib_says = fp8_attention._reads_pages

    def rule(dtype, hq, hkv, d, requests, *sizes):
        return pages or lib_says(dtype, hq, hkv, d, 1024, 1024, 1024, sizes[-1])  # rows wherever the dense kernel takes them

    def prefill(*args, max_seqlen_q, **kw):
        return asked(*args, max_seqlen_q=FAR if request.param == "tiles" else max_seqlen_q, **kw)

    monkeypatch.setattr(fp8_attention, "_reads_pages", rule)
    monkeypatch.setattr(mi, "paged_prefill_fp8", prefill)
    return request.param


def _of(test, name):
    """The values of a parametrised test's argument(s)."""
    return next(m.args[1] for m in test.pytestmark if m.name == "parametrize" and m.args[0] == name)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("hkv,group,d,bs", _of(cases.test_prefill_matches_the_formula, "hkv,group,d,bs"))
def test_prefill_matches_the_formula(cuda_device, way, name, hkv, group, d, bs):
    cases.test_prefill_matches_the_formula(cuda_device, name, hkv, group, d, bs)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("group", [1, 5])
def test_prefill_every_head_dim(cuda_device, way, name, d, group):
    cases.test_prefill_every_head_dim(cuda_device, name, d, group)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("q_lens,ctxs", _of(cases.test_prefill_small_chunks_over_long_contexts, "q_lens,ctxs"))
def test_prefill_small_chunks_over_long_contexts(cuda_device, way, name, d, q_lens, ctxs):
    got, free, want = prefill_case(cuda_device, name, 2, 4, d, 16, q_lens, ctxs)
    for x in (got, free):
        close(x, *want, PREFILL_STEP[DTYPES[name]], lost=DENSE_LOST)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("spread,scale", _of(cases.test_prefill_scales, "spread,scale"))
def test_prefill_scales(cuda_device, way, name, spread, scale):
    cases.test_prefill_scales(cuda_device, name, spread, scale)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("large", [False, True])
def test_prefill_nan_codes_reach_only_rows_that_see_them(cuda_device, way, name, d, large):
    cases.test_prefill_nan_codes_reach_only_rows_that_see_them(cuda_device, name, d, large)


@gpu
@pytest.mark.parametrize("operand", ["keys", "values"])
@pytest.mark.parametrize("hkv,d", [(16, 128), (1, 128), (1, 64)])
def test_prefill_in_fp16_of_what_fp16_does_not_hold(cuda_device, way, operand, hkv, d):
    cases.test_prefill_in_fp16_of_what_fp16_does_not_hold(cuda_device, operand, hkv, d)


@gpu
@pytest.mark.parametrize("hkv,d", [(1, 64), (1, 128), (16, 128)])
def test_prefill_leaves_rows_of_no_sequence_and_leaves_out_bad_pages(cuda_device, way, hkv, d):
    cases.test_prefill_leaves_rows_of_no_sequence_and_leaves_out_bad_pages(cuda_device, hkv, d)


@gpu
@pytest.mark.parametrize("hkv,d", [(2, 64), (2, 128), (16, 128)])
def test_results_over_the_query_and_shared_pages(cuda_device, way, hkv, d):
    cases.test_results_over_the_query_and_shared_pages(cuda_device, "bf16", hkv, d)


@gpu
@pytest.mark.parametrize("k_byte,q_power,v_byte", [(246, -100, 246), (1, 90, 1), (246, 0, 127), (127, -120, 200), (20, 20, 10)])
@pytest.mark.parametrize("name", ["bf16", "f16"])
def test_the_whole_range_of_scales(cuda_device, way, name, k_byte, q_power, v_byte):
    cases.test_decode_and_prefill_over_the_whole_range_of_scales(cuda_device, name, k_byte, q_power, v_byte)


@gpu
def test_large_values_with_no_weight(cuda_device, way):
    cases.test_large_values_with_no_weight(cuda_device, "bf16", True)


@gpu
@pytest.mark.parametrize("d", [64, 128])
def test_what_lies_past_the_context_is_ignored(cuda_device, way, d):
    cases.test_what_lies_past_the_context_is_ignored(cuda_device, "bf16", d, True)


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("count", [1100, 2049])
def test_more_sequences_than_a_launch_takes(cuda_device, way, count, d):
    """Short chunks, some without rows, some without keys."""
    rng = np.random.default_rng(count)
    q_lens = rng.integers(0, 4, count)
    ctxs = q_lens + rng.integers(0, 30, count)
    got, free, want = prefill_case(cuda_device, "bf16", 1, 2, d, 16, q_lens.tolist(), ctxs.tolist())
    for x in (got, free):
        close(x, *want, PREFILL_STEP[torch.bfloat16], lost=DENSE_LOST)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("group,d", [(4, 64), (4, 128), (6, 128)])
def test_sizes_that_choose_for_themselves(cuda_device, name, group, d):
    """Chunks around the sizes between which the choice changes, with no hand in it."""
    for q_lens, ctxs in (([200, 30], [200, 900]), ([600], [2900]), ([70], [9000]), ([1000, 3], [1400, 5000])):
        got, free, want = prefill_case(cuda_device, name, 4, group, d, 16, q_lens, ctxs)
        for x in (got, free):
            close(x, *want, PREFILL_STEP[DTYPES[name]], lost=DENSE_LOST)
