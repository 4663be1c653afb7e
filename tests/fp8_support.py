"""What the tests of the 8-bit cache share: random pages, tables, and how far attention may be off.

Store and gather are exact (the scale is a power of two).  Attention is held to
    |got - want| <= u |want| + c * sum_k p_k |v_k| + floor
with u half a step of the output type and c from the kernels' roundings:
  scores: fp32 sums of D products, off by at most D 2^-23 S with S = scale * sum |q||k| (fp32's q goes in as two f16
          parts, off by 2^-22 of each element: within it); that and the exponential's 2^-21 move p by
          as much, in the numerator and the sum;
  p:      rounded once to f16 before the product (2^-11), in the dense kernel of bf16 prefill to bf16 (2^-8);
          fp32 carries the error in a second f16 (2^-22, within the exponential's term).
floor: f16 ends.  p times 2^12 times 2^(byte - R) with R at most 2 above the largest byte of V's scales
  loses at most half of 2^-24 a key, which is 2^-37 of the sum of p (at least 2^12) times the largest magnitude of
  a code, 448 * 2^(R - 127) <= 8 * 224 * 2^(largest byte - 127): 2^-34 of the oracle's floor.  The dense kernel of fp16
  prefill lifts p by 2^7 only and has no R: half of 2^-24 of 2^7, times 448 * 2^(byte - 127): 2^-31 of it; the tcgen05
  kernel by 2^11: 2^-33 (of keys 2^25 below the largest, which the cases held to 2^-34 do not have).
"""

import numpy as np
import torch

import microinfer_b200 as mi
from oracle import fp8_oracle as fo

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DECODE_STEP = {torch.bfloat16: 2.0 ** -11, torch.float16: 2.0 ** -11, torch.float32: 0.0}
PREFILL_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 0.0}


def bound(want, weight, size, floor, dtype, d, p_step, lost=2.0 ** -34):
    u = torch.finfo(dtype).eps / 2
    c = 2 * (d * 2.0 ** -23 * size + 2.0 ** -21) + p_step
    # below the smallest normal number the steps stay as they are there: half of one is u * smallest_normal
    return u * np.maximum(np.abs(want), torch.finfo(dtype).smallest_normal) + (c + u) * weight + floor * lost


def close(got, want, weight, size, floor, p_step, lost=2.0 ** -34):
    dtype = got.dtype
    got = got.double().cpu().numpy()
    limit = bound(want, weight, size, floor, dtype, got.shape[-1], p_step, lost)
    if dtype == torch.float16:  # from 65520 on (half a step past 65504) an infinity; what may round either way is left out
        past, near = np.abs(want) - limit >= 65520, np.abs(want) + limit >= 65504
        assert np.array_equal(got[past], np.sign(want[past]) * np.inf)
        got = np.where(near, want, got)
    assert np.isfinite(got).all()
    worst = float(np.max(np.abs(got - want) / limit, initial=0.0))
    assert worst <= 1, f"{worst:.3g} of the bound"


def pages(rng, nb, bs, hkv, d, spread=0.5):
    """Random K and V pages by way of the oracle: rows of uneven size, V's groups by exp(+-2 spread)."""
    def one(by, value):
        size = np.exp(0.5 * np.clip(rng.standard_normal((nb, bs, hkv, 1)), -2, 2))
        far = np.exp(by * np.clip(rng.standard_normal((nb, bs // 16, hkv, 1)), -2, 2)).repeat(16, 1)
        return fo.pack(*fo.encode(rng.standard_normal((nb, bs, hkv, d)) * size * far), value)
    return one(0.5, False), one(spread, True)


def table_of(rng, ctxs, nb, bs, width=None):
    need = [-(-c // bs) for c in ctxs]
    assert sum(need) <= nb
    table = np.full((len(ctxs), width or max(1, max(need))), -1, dtype=np.int32)
    perm = rng.permutation(nb).astype(np.int32)
    at = 0
    for r, k in enumerate(need):
        table[r, :k] = perm[at:at + k]
        at += k
    return table


def cuda(x, device, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x)).to(device)
    return t if dtype is None else t.to(dtype)


def decode_case(device, name, hkv, group, d, bs, ctxs, seed=0, scale=None, spread=0.5, edit=None):
    rng = np.random.default_rng(seed + d + bs + group)
    nb = sum(-(-max(c, 0) // bs) for c in ctxs) + 3
    kp, vp = pages(rng, nb, bs, hkv, d, spread)
    table = table_of(rng, [max(c, 0) for c in ctxs], nb, bs, width=max(1, max(-(-c // bs) for c in ctxs)) + 1)
    query = cuda(rng.standard_normal((len(ctxs), hkv * group, d)), device, DTYPES[name])
    if edit is not None:
        edit(kp, vp, table)
    scale = d ** -0.5 if scale is None else scale
    got = mi.paged_decode_fp8(query, cuda(kp, device), cuda(vp, device), cuda(table, device),
                              torch.tensor(ctxs, dtype=torch.int32, device=device), scale=scale)
    q = query.double().cpu().numpy()
    parts = [fo.attention(q[r:r + 1], kp, vp, table[r], max(c, 0), scale) for r, c in enumerate(ctxs)]
    return got, [np.concatenate(x) for x in zip(*parts)]


def prefill_case(device, name, hkv, group, d, bs, q_lens, ctxs, seed=0, scale=None, spread=0.5, edit=None, **kw):
    rng = np.random.default_rng(seed + d + group)
    nb = sum(-(-c // bs) for c in ctxs) + 2
    kp, vp = pages(rng, nb, bs, hkv, d, spread)
    table = table_of(rng, ctxs, nb, bs)
    if edit is not None:
        edit(kp, vp, table)
    query = cuda(rng.standard_normal((sum(q_lens), hkv * group, d)), device, DTYPES[name])
    cu_q, cu_k = (torch.tensor([0, *np.cumsum(x)], dtype=torch.int32, device=device) for x in (q_lens, ctxs))
    args = (query, cuda(kp, device), cuda(vp, device), cu_q, cu_k, cuda(table, device))
    got = mi.paged_prefill_fp8(*args, max_seqlen_q=max(q_lens), total_k=sum(ctxs), scale=scale, **kw)
    free = mi.paged_prefill_fp8(*args, max_seqlen_q=max(q_lens), scale=scale)
    mi.check_device_status(device)
    q = query.double().cpu().numpy()
    at = np.cumsum([0, *q_lens])
    parts = [fo.attention(q[at[r]:at[r + 1]], kp, vp, table[r], c, d ** -0.5 if scale is None else scale)
             for r, c in enumerate(ctxs)]
    return got, free, [np.concatenate(x) for x in zip(*parts)]
