"""Measured cases of the 4-bit paged KV cache: quantising store, gather, decode and chunked prefill.

The cache holds K and V in microscaled 4-bit floating point (MXFP4: e2m1 values, one power-of-two
scale for every 32 of them along the head dimension).  ``key_pages`` and ``value_pages`` are uint8
``[num_blocks, num_kv_heads, block_size / 16, head_dim / 32 * 272]``: for every 16 tokens of a page
and kv head, the codes ``[head_dim / 32][16 tokens][16 bytes]`` (two per byte, the even element in
the low nibble), then the scale bytes ``[16 tokens][head_dim / 32]``.  A code is a sign and one of
0, 0.5, 1, 1.5, 2, 3, 4, 6; a scale byte e stands for 2^(e - 127), 0 for zero and 255 for NaN.
A block's scale exponent is floor(log2(largest magnitude)) - 2, its byte at least 1 unless every
element is zero (then 0); values round to nearest, ties to even, and saturate at 6; a block
with a value that is not finite reads as NaN.

``own`` selects what ``run`` calls: the plain form in elementary torch operations (fp32), or the
entry points of ``microinfer_b200``.
"""

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
GROUP = 16  # tokens of one code group of a page
MX = 32  # elements that share a scale


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # One user's short chat turn: a single token on a few cached ones; launch latency is all there is.
        _decode("decode_1x150", seqs=1, lo=150, hi=150, hq=16, hkv=8, d=128, bs=16),
        # The benchmark's ordinary decode step at 16/8 heads of 128 and 16-token pages.
        _decode("decode_8x4096", seqs=8, lo=4096, hi=4096, hq=16, hkv=8, d=128, bs=16),
        # One very long document: the work has to be split over the cache's length.
        _decode("decode_1x131072", seqs=1, lo=131072, hi=131072, hq=32, hkv=8, d=128, bs=256),
        # A full server: contexts of very different lengths, some rows of the batch padding (length 0).
        _decode("decode_ragged_96", seqs=96, lo=1, hi=8191, hq=32, hkv=8, d=128, bs=16, zero=5),
        # The same in fp16 with heads of 64, seven query heads to a kv head, larger pages.
        _decode("decode_ragged_d64", seqs=40, lo=900, hi=16000, hq=14, hkv=2, d=64, bs=64, dtype="f16"),
        # fp32 activations, as the CPU-checked configurations use them.
        _decode("decode_f32", seqs=4, lo=100, hi=777, hq=16, hkv=8, d=128, bs=16, dtype="f32"),
        # Every sequence of a small batch appends one token, and the pages are read back.
        _store("store_8x1", seqs=8, lo=20, hi=90, new_lo=1, new_hi=1, hkv=8, d=128, bs=16, hq=16),
        # Prefill chunks of four sequences enter the cache and are gathered with their prefixes.
        _store("store_4x2000", seqs=4, lo=2500, hi=8191, new_lo=2000, new_hi=2000, hkv=8, d=128, bs=16, hq=16, pad=192),
        # Gather of a short fp32 cache and of 64 contexts of a prefix and a suffix (1024 + 128 tokens).
        _gather("gather_3x70", seqs=3, lo=30, hi=70, hkv=4, d=64, bs=16, dtype="f32"),
        _gather("gather_64x1152", seqs=64, lo=1152, hi=1152, hkv=8, d=128, bs=16),
        # A mixed set of chunks, most with a cached prefix, odd lengths.
        _prefill("prefill_12_ragged", seqs=12, lo=40, hi=1500, new_lo=1, new_hi=400, hq=16, hkv=8, d=128, bs=16),
        # One chunk of a long prompt on its cached prefix.
        _prefill("prefill_2048_on_14336", seqs=1, lo=16384, hi=16384, new_lo=2048, new_hi=2048, hq=32, hkv=8, d=128, bs=16),
    ]


def _case(op, name, **kw):
    kw = {"op": op, "dtype": "bf16", "zero": 0, "pad": 0, "new_lo": 0, "new_hi": 0, "lens": 1, **kw}
    return {"name": name, **kw} if name else kw


def _decode(name, **kw):
    return _case("decode", name, **kw)


def _store(name, **kw):
    return _case("store", name, **kw)


def _gather(name, **kw):
    return _case("gather", name, **kw)


def _prefill(name, **kw):
    return _case("prefill", name, **kw)


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "store", "gather", "prefill"])
    hkv = rng.choice([1, 2, 4, 8])
    common = dict(hkv=hkv, d=rng.choice([64, 128, 128]), bs=rng.choice([16, 16, 32, 64, 256]), lens=rng.randrange(1 << 30))
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f16", "f32"])
    if op == "decode":
        group = rng.choice([1, 2, 4, 4, 5, 7, 8, 16])
        seqs = _log_int(rng, 1, 128)
        most = max(1, min(131072, 400000 // seqs))
        if dtype == "f32":
            most = min(most, 4096)
        hi = _log_int(rng, 1, most)
        lo = rng.choice([1, hi, max(1, hi // 2), max(1, hi // 8)])
        return _case(op, None, seqs=seqs, lo=lo, hi=hi, hq=hkv * group, dtype=dtype, zero=rng.choice([0, 0, min(seqs - 1, 3)]), **common)
    if op == "store":
        seqs = _log_int(rng, 1, 64)
        new = _log_int(rng, 1, max(1, 8000 // seqs))
        hi = _log_int(rng, new, max(new, 30000 // seqs))
        return _case(op, None, seqs=seqs, lo=max(new, hi // 3), hi=hi, new_lo=max(1, new // 2), new_hi=new, hq=2 * hkv, dtype=dtype, pad=rng.choice([0, 0, 1, 37]), **common)
    if op == "gather":
        seqs = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, max(1, 73000 // seqs))
        return _case(op, None, seqs=seqs, lo=max(1, hi // 3), hi=hi, dtype=dtype, zero=rng.choice([0, 0, min(seqs - 1, 2)]), **common)
    group = rng.choice([1, 2, 4, 8])
    seqs = _log_int(rng, 1, 16)
    new = _log_int(rng, 1, max(1, 2000 // seqs))
    hi = _log_int(rng, new, max(new, 16000 // seqs))
    if dtype == "f32":
        new, hi = min(new, 64), min(hi, 600)
        hi = max(hi, new)
    return _case(op, None, seqs=seqs, lo=max(new, hi // 2), hi=hi, new_lo=max(1, new // 3), new_hi=new, hq=hkv * group, dtype=dtype, **common)


def _lengths(case):
    """(contexts, new tokens) of the batch: fixed by the case alone, so that its work is known."""
    rng = random.Random(case["lens"])
    ctx = [rng.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
    for r in rng.sample(range(case["seqs"]), case["zero"]):
        ctx[r] = 0
    new = [min(c, rng.randint(case["new_lo"], case["new_hi"])) for c in ctx]
    return ctx, new


def work(case):
    ctx, new = _lengths(case)
    total, tokens = sum(ctx), sum(new)
    size = 4 if case["dtype"] == "f32" else 2
    row = case["hkv"] * case["d"]
    coded = 2 * row // MX * 17  # bytes of one token's K and V in the cache
    table = 4 * sum(-(-c // case["bs"]) for c in ctx)
    if case["op"] == "decode":
        qo = 2 * case["seqs"] * case["hq"] * case["d"] * size
        return {"bytes": total * coded + qo + table + 4 * case["seqs"], "flops": 4 * case["hq"] * case["d"] * total}
    if case["op"] == "store":
        return {"bytes": tokens * (2 * row * size + coded + 4) + (total - tokens) * coded + total * 2 * row * size + table, "flops": 2 * row * (tokens + total)}
    if case["op"] == "gather":
        return {"bytes": total * (coded + 2 * row * size) + table, "flops": 2 * row * total}
    pairs = sum(n * (c - n) + n * (n + 1) // 2 for c, n in zip(ctx, new))
    return {"bytes": total * coded + 2 * tokens * case["hq"] * case["d"] * size + table, "flops": 4 * case["hq"] * case["d"] * pairs}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    ctx, new = _lengths(case)
    hkv, d, bs, dtype = case["hkv"], case["d"], case["bs"], DTYPES[case["dtype"]]
    need = [-(-c // bs) for c in ctx]
    blocks = sum(need) + 4  # a few free pages with what their last owner left there
    perm = np.random.RandomState(int(seed) % (1 << 32)).permutation(blocks).astype(np.int32)
    table = np.full((len(ctx), max(1, max(need))), -1, dtype=np.int32)
    at = 0
    for r, k in enumerate(need):
        table[r, :k] = perm[at:at + k]
        at += k

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    # Keys have channels of very different size, values tokens of somewhat different size.
    channel = torch.exp(0.6 * normal(hkv, d))
    shape = (blocks, hkv, bs // GROUP, GROUP, d)
    key_pages = _encode_pages(normal(*shape) * channel[:, None, None, :])
    value_pages = _encode_pages(normal(*shape) * torch.exp(0.4 * normal(blocks, hkv, bs // GROUP, GROUP, 1)))

    cu_k = torch.tensor([0, *np.cumsum(ctx)], dtype=torch.int32, device=dev)
    cu_q = torch.tensor([0, *np.cumsum(new)], dtype=torch.int32, device=dev)
    state = {
        "case": case, "key_pages": key_pages, "value_pages": value_pages, "contexts": ctx, "total": sum(ctx), "tokens": sum(new),
        "max_q": max(new) if new else 0, "max_ctx": max(ctx), "table": torch.from_numpy(table).to(dev), "cu_k": cu_k, "cu_q": cu_q,
        "context_lens": torch.tensor(ctx, dtype=torch.int32, device=dev), "scale": 1.0 / math.sqrt(d), "dtype": dtype,
    }
    if case["op"] == "decode":
        state["query"] = normal(len(ctx), case["hq"], d).to(dtype)
    if case["op"] == "prefill":
        state["query"] = normal(sum(new), case["hq"], d).to(dtype)
    if case["op"] == "store":
        rows = sum(new) + case["pad"]
        # K and V as a model has them: slices of the packed projection's output.
        qkv = normal(rows, case["hq"] + 2 * hkv, d)
        qkv[:, case["hq"]:case["hq"] + hkv] *= channel
        qkv = qkv.to(dtype)
        state["keys"] = qkv[:, case["hq"]:case["hq"] + hkv]
        state["values"] = qkv[:, case["hq"] + hkv:]
        pos = np.concatenate([np.arange(c - n, c) for c, n in zip(ctx, new)])
        seq = np.repeat(np.arange(len(ctx)), new)
        slots = np.full(rows, -1, dtype=np.int32)  # rows past the last token are padding
        slots[:len(pos)] = table[seq, pos // bs] * bs + pos % bs
        state["slots"] = torch.from_numpy(slots).to(dev)
    return state


def _encode_pages(x):
    """Pages [blocks, Hkv, groups, bytes] of x [blocks, Hkv, groups, 16, D]."""
    codes, scales = _quantise(x)  # [..., 16, D / 32, 16], [..., 16, D / 32]
    return torch.cat([codes.transpose(-3, -2).flatten(-3), scales.flatten(-2)], -1).contiguous()


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _quantise(x):
    """Codes [..., D / 32, 16] and scale bytes [..., D / 32] of x [..., D]."""
    x = x.float().unflatten(-1, (-1, MX))
    mag = x.abs()
    amax = mag.amax(-1)
    byte = (torch.frexp(amax).exponent - 3 + 127).clamp(min=1)
    byte = torch.where(amax == 0, 0, byte)
    finite = torch.isfinite(mag).all(-1)
    inverse = ((254 - byte) << 23).to(torch.int32).view(torch.float32)
    q = mag * torch.where(amax == 0, 0.0, inverse)[..., None]
    code = (q > 0.25).int() + (q >= 0.75) + (q > 1.25) + (q >= 1.75) + (q > 2.5) + (q >= 3.5) + (q > 5.0)
    code = code + 8 * (x < 0)
    code = torch.where(finite[..., None], code, 0)
    byte = torch.where(finite, byte, 255)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), byte.to(torch.uint8)


def _views(pages):
    """Codes [blocks, Hkv, groups, D / 32, 16 tokens, 16 bytes] and scales [blocks, Hkv, groups, 16 tokens, D / 32] of pages."""
    nb = pages.shape[-1] // 272
    return pages[..., :nb * 256].unflatten(-1, (nb, GROUP, 16)), pages[..., nb * 256:].unflatten(-1, (GROUP, nb))


def _dequantise(pages):
    """fp32 rows [slots, Hkv, D] of all pages."""
    codes, scales = _views(pages)
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=pages.device)
    value = table[torch.stack([codes & 15, codes >> 4], -1).int()].flatten(-2)  # [blocks, Hkv, groups, D / 32, 16, 32]
    byte = scales.int()
    scale = torch.where(byte == 255, float("nan"), (byte << 23).view(torch.float32))
    value = value * scale.transpose(-1, -2)[..., None]
    return value.permute(0, 2, 4, 1, 3, 5).reshape(-1, pages.shape[1], value.shape[3] * MX)


def _positions(s):
    """Slots [seqs, max context] of every position, and which of them exist."""
    bs = s["case"]["bs"]
    pos = torch.arange(max(1, s["max_ctx"]), device=s["table"].device)
    slots = s["table"][:, pos // bs] * bs + pos % bs
    return slots.clamp(min=0), pos < s["context_lens"][:, None]


def _plain_gather(s):
    row = torch.arange(s["total"], device=s["table"].device)
    seq = torch.searchsorted(s["cu_k"], row.int(), right=True) - 1
    pos = row - s["cu_k"][seq]
    bs = s["case"]["bs"]
    slots = s["table"][seq, pos // bs] * bs + pos % bs
    return {"keys": _dequantise(s["key_pages"])[slots].to(s["dtype"]), "values": _dequantise(s["value_pages"])[slots].to(s["dtype"])}


def _plain_store(s, pages, rows):
    bs = s["case"]["bs"]
    n = s["tokens"]
    slots = s["slots"][:n].long()
    block, group, token = slots // bs, slots % bs // GROUP, slots % GROUP
    codes, scales = _views(pages)
    new_codes, new_scales = _quantise(rows[:n])
    codes[block, :, group, :, token] = new_codes
    scales[block, :, group, token] = new_scales


def _softmax(x):
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == float("-inf"), 0.0, m))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, 1.0, total)  # a row without keys is zero


def _plain_decode(s):
    case = s["case"]
    slots, there = _positions(s)
    k, v = _dequantise(s["key_pages"])[slots], _dequantise(s["value_pages"])[slots]
    v = torch.where(there[..., None, None], v, 0.0)
    q = s["query"].float().unflatten(1, (case["hkv"], -1))
    x = torch.einsum("shgd,schd->shgc", q, k) * s["scale"]
    p = _softmax(torch.where(there[:, None, None], x, float("-inf")))
    return torch.einsum("shgc,schd->shgd", p, v).flatten(1, 2).to(s["dtype"])


def _plain_prefill(s):
    case = s["case"]
    dev = s["table"].device
    slots, there = _positions(s)
    k, v = _dequantise(s["key_pages"])[slots], _dequantise(s["value_pages"])[slots]
    v = torch.where(there[..., None, None], v, 0.0)
    i = torch.arange(s["max_q"], device=dev)
    new = s["cu_q"][1:] - s["cu_q"][:-1]
    token = (s["cu_q"][:-1, None] + i).clamp(max=s["tokens"] - 1)
    q = s["query"].float()[token].unflatten(2, (case["hkv"], -1))  # [seqs, max_q, Hkv, G, D]
    x = torch.einsum("sqhgd,schd->shgqc", q, k) * s["scale"]
    last = s["context_lens"][:, None] - new[:, None] + i  # position of query row i
    seen = there[:, None] & (torch.arange(slots.shape[1], device=dev) <= last[..., None])
    p = _softmax(torch.where(seen[:, None, None], x, float("-inf")))
    out = torch.einsum("shgqc,schd->sqhgd", p, v).flatten(2, 3)
    t = torch.arange(s["tokens"], device=dev)
    seq = torch.searchsorted(s["cu_q"], t.int(), right=True) - 1
    return out[seq, t - s["cu_q"][seq]].to(s["dtype"])


def run(state):
    s = state
    op = s["case"]["op"]
    if own:
        import microinfer_b200 as mi

        kp, vp = s["key_pages"], s["value_pages"]
        if op == "decode":
            return mi.paged_decode_mxfp4(s["query"], kp, vp, s["table"], s["context_lens"], scale=s["scale"])
        if op == "prefill":
            return mi.paged_prefill_mxfp4(s["query"], kp, vp, s["cu_q"], s["cu_k"], s["table"], max_seqlen_q=s["max_q"], total_k=s["total"], scale=s["scale"])
        if op == "store":
            mi.store_kv_mxfp4(kp, vp, s["slots"], s["keys"], s["values"])
        keys, values = mi.gather_paged_kv_mxfp4(kp, vp, s["table"], s["contexts"], dtype=s["dtype"], cu_seqlens_k=s["cu_k"])
        return {"keys": keys, "values": values}
    if op == "decode":
        return _plain_decode(s)
    if op == "prefill":
        return _plain_prefill(s)
    if op == "store":
        _plain_store(s, s["key_pages"], s["keys"])
        _plain_store(s, s["value_pages"], s["values"])
    return _plain_gather(s)


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
_GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _exact_rows(s, pages, r):
    """float64 [context, Hkv, D] of sequence r, token by token through its block table."""
    bs, d = s["case"]["bs"], s["case"]["d"]
    ctx = s["contexts"][r]
    if ctx == 0:
        return torch.zeros(0, pages.shape[1], d, dtype=torch.float64, device=pages.device)
    raw = pages[s["table"][r, :-(-ctx // bs)].long()].to(torch.float64)  # [n, Hkv, groups, bytes]
    n, hkv, groups, _ = raw.shape
    out = torch.empty(n, groups, GROUP, hkv, d, dtype=torch.float64, device=pages.device)
    grid = torch.tensor(_GRID, dtype=torch.float64, device=pages.device)
    for b in range(d // MX):
        byte = raw[..., b * GROUP * 16:(b + 1) * GROUP * 16].reshape(n, hkv, groups, GROUP, 16)
        e = raw[..., d // MX * 256 + b::d // MX]  # this block's scale of each token
        factor = torch.where(e == 0, 0.0, torch.pow(2.0, e - 127))
        factor = torch.where(e == 255, torch.nan, factor)[..., None]
        for half, nibble in enumerate((torch.remainder(byte, 16), torch.floor(byte / 16))):
            mag = grid[torch.remainder(nibble, 8).long()]
            value = torch.where(nibble >= 8, -mag, mag) * factor
            out[..., b * MX + half:(b + 1) * MX:2] = value.permute(0, 2, 3, 1, 4)
    return out.reshape(n * bs, hkv, d)[:ctx]


def _exact_encode(x):
    """The cache's values of x [tokens, Hkv, D], by distance to the eight magnitudes."""
    x = x.to(torch.float64)
    blocks = x.reshape(*x.shape[:-1], -1, MX)
    top = blocks.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(torch.where(top > 0, top, 1.0)))
    e = torch.where(torch.pow(2.0, e) > top, e - 1, e)
    e = torch.where(torch.pow(2.0, e + 1) <= top, e + 1, e) - 2
    unit = torch.pow(2.0, e.clamp(min=-126))
    grid = torch.tensor(_GRID, dtype=torch.float64, device=x.device)
    odd = torch.arange(8, device=x.device) % 2 * 1e-12  # of two as near, the even code
    best = ((blocks.abs() / unit).unsqueeze(-1) - grid).abs().add(odd).argmin(-1)
    value = torch.sign(blocks) * grid[best] * unit
    bad = ~torch.isfinite(blocks).all(-1, keepdim=True)
    return torch.where(bad, torch.nan, torch.where(top > 0, value, 0.0)).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    ctx, new = _lengths(case)
    keys, values, out = [], [], []
    at = 0
    for r, (c, n) in enumerate(zip(ctx, new)):
        k, v = _exact_rows(s, s["key_pages"], r), _exact_rows(s, s["value_pages"], r)
        if case["op"] == "store":
            k[c - n:] = _exact_encode(s["keys"][at:at + n])
            v[c - n:] = _exact_encode(s["values"][at:at + n])
        if case["op"] in ("store", "gather"):
            keys.append(k)
            values.append(v)
        else:
            rows = 1 if case["op"] == "decode" else n
            q = s["query"][r:r + 1] if case["op"] == "decode" else s["query"][at:at + n]
            q = q.to(torch.float64)
            o = torch.zeros_like(q)
            group = case["hq"] // case["hkv"]
            mask = torch.arange(c, device=q.device)[None] > torch.arange(c - rows, c, device=q.device)[:, None]
            for h in range(case["hq"] if c else 0):
                x = (q[:, h] @ k[:, h // group].T / math.sqrt(case["d"])).masked_fill(mask, -torch.inf)
                o[:, h] = torch.softmax(x, -1) @ v[:, h // group]
            out.append(o)
        at += n
    if case["op"] in ("store", "gather"):
        return {"keys": torch.cat(keys), "values": torch.cat(values)}
    return torch.cat(out)
