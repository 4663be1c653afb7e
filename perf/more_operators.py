"""Measured cases of the 8-bit paged KV cache: quantising store, gather, decode and chunked prefill.

The cache holds K and V as 8-bit floating point (e4m3: sign, 4 bits of exponent, 3 of mantissa; largest 448, smallest
2^-9, 0x7f and 0xff not a number, no infinity) with one power-of-two scale for every block of 16 tokens and kv head.
``key_pages`` and ``value_pages`` are uint8 ``[num_blocks, num_kv_heads, block_size / 16, 16 * head_dim + 16]``: for every
16 tokens of a page and kv head (a group) the codes, then 16 bytes of which the first is the scale: byte b stands for
2^(b - 127), 0 for zero; the other 15 are zero. Codes lie in parts of 64 dims (w = 64; a last part of 32 where head_dim is
an odd multiple of 32): K's as ``[16 tokens][w dims]``, V's as ``[2 halves][8][4 pairs][w / 8 dims][2 tokens]``, where
token = 8 * half + 2 * pair + the last index, and dim = w / 8 * the second index + the fourth.

The store quantises the tokens N of a call in a group together. With a the largest finite magnitude of their elements, the
byte they need is 0 where a = 0 and else e + 127, e the least exponent with a <= 448 * 2^e, held between 1 and 246. A call
that writes the group's first token sets the scale to that; any other raises it to that, and where it rises the group's
other codes are rounded to the new scale. Roundings are to nearest, ties to even, saturating at 448; elements that
are not finite become NaN.

``own`` selects what ``run`` calls: the plain form in elementary torch operations (fp32), or the
entry points of ``microinfer_b200``.
"""

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
GROUP = 16  # tokens that share a scale
TAIL = 16  # bytes after a group's codes, the scale first


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # One user's chat turn: a single token on a few hundred cached ones; launch latency is all there is.
        _decode("decode_1x300", seqs=1, lo=300, hi=300, hq=16, hkv=8, d=128, bs=16),
        # The benchmark's ordinary decode step: 8 sequences of 128 to 512 tokens, 16/8 heads of 128, 16-token pages.
        _decode("decode_8x512", seqs=8, lo=128, hi=512, hq=16, hkv=8, d=128, bs=16),
        # One very long document: the work has to be split over the cache's length.
        _decode("decode_1x100001", seqs=1, lo=100001, hi=100001, hq=32, hkv=8, d=128, bs=256),
        # A full server: contexts of very different lengths, some rows of the batch padding (length 0).
        _decode("decode_ragged_128", seqs=128, lo=1, hi=6000, hq=32, hkv=8, d=128, bs=16, zero=7),
        # The same in fp16 with heads of 64, seven query heads to a kv head, larger pages.
        _decode("decode_ragged_d64", seqs=33, lo=700, hi=12000, hq=14, hkv=2, d=64, bs=32, dtype="f16"),
        # fp32 activations, as the CPU-checked configurations use them.
        _decode("decode_f32", seqs=5, lo=90, hi=900, hq=16, hkv=8, d=128, bs=16, dtype="f32"),
        # Every sequence of a batch appends one token inside a block that has a scale already, and the pages are read back.
        _store("store_32x1", seqs=32, lo=20, hi=90, new_lo=1, new_hi=1, hkv=8, d=128, bs=16, hq=16),
        # Prefill chunks of four sequences enter the cache, most starting inside a block, and are gathered with their prefixes.
        _store("store_4x2047", seqs=4, lo=2500, hi=8191, new_lo=2001, new_hi=2047, hkv=8, d=128, bs=16, hq=16, pad=100),
        # Gather of 48 contexts for a kernel that takes rows.
        _gather("gather_48x1500", seqs=48, lo=1500, hi=1500, hkv=8, d=128, bs=16),
        # A mixed set of chunks, most with a cached prefix, odd lengths.
        _prefill("prefill_10_ragged", seqs=10, lo=40, hi=2000, new_lo=1, new_hi=500, hq=16, hkv=8, d=128, bs=16),
        # Chunks in fp16 with heads of 64.
        _prefill("prefill_6x300_d64", seqs=6, lo=2400, hi=2800, new_lo=300, new_hi=300, hq=14, hkv=2, d=64, bs=32, dtype="f16"),
        # One chunk of a long prompt on its cached prefix.
        _prefill("prefill_1536_on_12288", seqs=1, lo=13824, hi=13824, new_lo=1536, new_hi=1536, hq=32, hkv=8, d=128, bs=16),
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
    common = dict(hkv=hkv, d=rng.choice([64, 96, 128, 128, 128, 256]), bs=rng.choice([16, 16, 32, 64, 256]), lens=rng.randrange(1 << 30))
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f16", "f32"])
    wide = max(1, common["d"] // 128)
    if op == "decode":
        group = rng.choice([1, 2, 4, 4, 5, 7, 8, 16])
        seqs = _log_int(rng, 1, 128)
        most = max(1, min(100000, 350000 // seqs) // wide)
        if dtype == "f32":
            most = min(most, 4096)
        hi = _log_int(rng, 1, most)
        lo = rng.choice([1, hi, max(1, hi // 2), max(1, hi // 8)])
        return _case(op, None, seqs=seqs, lo=lo, hi=hi, hq=hkv * group, dtype=dtype, zero=rng.choice([0, 0, min(seqs - 1, 3)]), **common)
    if op == "store":
        seqs = _log_int(rng, 1, 64)
        new = _log_int(rng, 1, max(1, 8000 // seqs // wide))
        hi = _log_int(rng, new, max(new, 24000 // seqs // wide))
        return _case(op, None, seqs=seqs, lo=max(new, hi // 3), hi=hi, new_lo=max(1, new // 2), new_hi=new, hq=2 * hkv, dtype=dtype, pad=rng.choice([0, 0, 1, 37]), **common)
    if op == "gather":
        seqs = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, max(1, 70000 // seqs // wide))
        return _case(op, None, seqs=seqs, lo=max(1, hi // 3), hi=hi, dtype=dtype, zero=rng.choice([0, 0, min(seqs - 1, 2)]), **common)
    group = rng.choice([1, 2, 4, 8])
    seqs = _log_int(rng, 1, 16)
    new = _log_int(rng, 1, max(1, 1500 // seqs // wide))
    hi = _log_int(rng, new, max(new, 13000 // seqs // wide))
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
    groups = sum(-(-c // GROUP) for c in ctx)
    coded = 2 * row * total + 2 * case["hkv"] * groups  # bytes of the contexts' codes and scales
    table = 4 * sum(-(-c // case["bs"]) for c in ctx)
    if case["op"] == "decode":
        qo = 2 * case["seqs"] * case["hq"] * case["d"] * size
        return {"bytes": coded + qo + table + 4 * case["seqs"], "flops": 4 * case["hq"] * case["d"] * total}
    if case["op"] == "store":
        touched = sum(-(-c // GROUP) - (c - n) // GROUP for c, n in zip(ctx, new))
        stored = tokens * (2 * row * size + 2 * row + 4) + 2 * case["hkv"] * touched
        read = 2 * row * (total - tokens) + 2 * case["hkv"] * groups
        return {"bytes": stored + read + total * 2 * row * size + table, "flops": 2 * row * (tokens + total)}
    if case["op"] == "gather":
        return {"bytes": coded + total * 2 * row * size + table, "flops": 2 * row * total}
    pairs = sum(n * (c - n) + n * (n + 1) // 2 for c, n in zip(ctx, new))
    return {"bytes": coded + 2 * tokens * case["hq"] * case["d"] * size + table, "flops": 4 * case["hq"] * case["d"] * pairs}


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
    key_pages = _new_pages(normal(*shape) * channel[:, None, None, :], False)
    value_pages = _new_pages(normal(*shape) * torch.exp(0.4 * normal(blocks, hkv, bs // GROUP, GROUP, 1)), True)

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
        qkv[:, case["hq"] + hkv:] *= torch.exp(0.4 * normal(rows, hkv, 1))
        qkv = qkv.to(dtype)
        state["keys"] = qkv[:, case["hq"]:case["hq"] + hkv]
        state["values"] = qkv[:, case["hq"] + hkv:]
        pos = np.concatenate([np.arange(c - n, c) for c, n in zip(ctx, new)])
        seq = np.repeat(np.arange(len(ctx)), new)
        slots = np.full(rows, -1, dtype=np.int32)  # rows past the last token are padding
        slots[:len(pos)] = table[seq, pos // bs] * bs + pos % bs
        state["slots"] = torch.from_numpy(slots).to(dev)
    return state


def _new_pages(x, value):
    """Pages of x [blocks, Hkv, groups, 16, D], every group quantised at once."""
    byte = _scale_byte(x.abs().amax((-1, -2)))
    return _join(_round(x * _power(127 - byte)[..., None, None]), byte, value)


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _power(e):
    """fp32 2^e of whole numbers e, -126 to 127."""
    return ((e + 127).to(torch.int32) << 23).view(torch.float32)


def _scale_byte(a):
    mantissa, exponent = torch.frexp(a)  # a = mantissa * 2^exponent, mantissa in [0.5, 1); 448 = 0.875 * 2^9
    byte = exponent - 9 + (mantissa > 0.875).int() + 127
    return torch.where(a == 0, 0, byte.clamp(1, 246))


def _round(y):
    """y rounded to e4m3 values, ties to even, at most 448."""
    finite = torch.isfinite(y)
    y = torch.where(finite, y, 0.0)
    step = _power((torch.frexp(y).exponent - 1).clamp(min=-6) - 3)
    r = (torch.round(y / step) * step).clamp(-448.0, 448.0)
    return torch.where(finite, r, float("nan"))


def _values_of_bytes(device):
    byte = torch.arange(256, device=device)
    e, m = (byte >> 3) & 15, byte & 7
    v = torch.where(e > 0, (8 + m) * _power(e - 10), m * _power(torch.full_like(e, -9)))
    v = torch.where(byte & 128 > 0, -v, v)
    return torch.where(byte & 127 == 127, float("nan"), v)


def _bytes(v):
    """Codes of e4m3 values."""
    a = v.abs()
    mantissa, exponent = torch.frexp(a)
    normal = (exponent - 1 + 7) * 8 + (mantissa * 16 - 8).int()
    code = torch.where(a >= 2.0 ** -6, normal, (a * 512).int())
    code = torch.where(torch.isnan(v), 127, code)
    return (code + 128 * (v < 0)).to(torch.uint8)


def _parts(d):
    return [64] * (d // 64) + [32] * (d % 64 // 32)


def _split(pages, value):
    """Unscaled values [blocks, Hkv, groups, 16, D] and scale bytes [blocks, Hkv, groups] of pages."""
    d = pages.shape[-1] // GROUP - 1
    lut = _values_of_bytes(pages.device)
    out, at = [], 0
    for w in _parts(d):
        c = lut[pages[..., at:at + GROUP * w].int()]
        if value:  # [2, 8, 4, w / 8, 2] -> tokens (half, pair, last), dims
            c = c.unflatten(-1, (2, 8, 4, w // 8, 2)).permute(0, 1, 2, 3, 5, 7, 4, 6).flatten(3, 5).flatten(-2)
        else:
            c = c.unflatten(-1, (GROUP, w))
        out.append(c)
        at += GROUP * w
    return torch.cat(out, -1), pages[..., at].int()


def _join(v, byte, value):
    """Pages of unscaled values and scale bytes."""
    out, at = [], 0
    for w in _parts(v.shape[-1]):
        c = _bytes(v[..., at:at + w])
        if value:
            c = c.unflatten(-2, (2, 4, 2)).unflatten(-1, (8, w // 8)).permute(0, 1, 2, 3, 6, 4, 7, 5)
            c = c.flatten(3)
        else:
            c = c.flatten(-2)
        out.append(c)
        at += w
    tail = torch.zeros(*byte.shape, TAIL, dtype=torch.uint8, device=v.device)
    tail[..., 0] = byte.to(torch.uint8)
    return torch.cat([*out, tail], -1).contiguous()


def _scale(byte):
    return torch.where(byte == 0, 0.0, _power(byte - 127))


def _dequantise(pages, value):
    """fp32 rows [slots, Hkv, D] of all pages."""
    v, byte = _split(pages, value)
    v = v * _scale(byte)[..., None, None]
    return v.permute(0, 2, 3, 1, 4).reshape(-1, pages.shape[1], v.shape[-1])


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
    return {"keys": _dequantise(s["key_pages"], False)[slots].to(s["dtype"]), "values": _dequantise(s["value_pages"], True)[slots].to(s["dtype"])}


def _plain_store(s, pages, rows, value):
    n = s["tokens"]
    x = rows[:n].float()  # [tokens, Hkv, D]
    slots = s["slots"][:n].long()
    group = slots // GROUP  # of all groups, [blocks * groups, Hkv, 16, D]
    v, old = _split(pages, value)
    v = v.permute(0, 2, 1, 3, 4).flatten(0, 1)
    old = old.permute(0, 2, 1).flatten(0, 1)
    a = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    most = torch.zeros_like(old, dtype=torch.float32).scatter_reduce(0, group[:, None].expand_as(a), a, "amax")
    first = torch.zeros(old.shape[0], dtype=torch.int32, device=x.device).index_add(0, group, (slots % GROUP == 0).int()) > 0
    need = _scale_byte(most)  # 0 where the call has no token
    byte = torch.where(first[:, None], need, torch.maximum(old, need))
    grown = ~first[:, None] & (byte > old)
    factor = torch.where(grown, _scale((127 + old - byte).clamp(min=0) * (old > 0)), 1.0)
    v = _round(v * factor[..., None, None])
    v[group, :, slots % GROUP] = _round(x * _power(127 - byte)[group][..., None])
    shape = (pages.shape[0], pages.shape[2])
    pages.copy_(_join(v.unflatten(0, shape).transpose(1, 2), byte.unflatten(0, shape).transpose(1, 2), value))


def _softmax(x):
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == float("-inf"), 0.0, m))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, 1.0, total)  # a row without keys is zero


def _plain_decode(s):
    case = s["case"]
    slots, there = _positions(s)
    k, v = _dequantise(s["key_pages"], False)[slots], _dequantise(s["value_pages"], True)[slots]
    v = torch.where(there[..., None, None], v, 0.0)
    q = s["query"].float().unflatten(1, (case["hkv"], -1))
    x = torch.einsum("shgd,schd->shgc", q, k) * s["scale"]
    p = _softmax(torch.where(there[:, None, None], x, float("-inf")))
    return torch.einsum("shgc,schd->shgd", p, v).flatten(1, 2).to(s["dtype"])


def _plain_prefill(s):
    case = s["case"]
    dev = s["table"].device
    slots, there = _positions(s)
    k, v = _dequantise(s["key_pages"], False)[slots], _dequantise(s["value_pages"], True)[slots]
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
            return mi.paged_decode_fp8(s["query"], kp, vp, s["table"], s["context_lens"], scale=s["scale"])
        if op == "prefill":
            return mi.paged_prefill_fp8(s["query"], kp, vp, s["cu_q"], s["cu_k"], s["table"], max_seqlen_q=s["max_q"], total_k=s["total"], scale=s["scale"])
        if op == "store":
            mi.store_kv_fp8(kp, vp, s["slots"], s["keys"], s["values"])
        keys, values = mi.gather_paged_kv_fp8(kp, vp, s["table"], s["contexts"], dtype=s["dtype"], cu_seqlens_k=s["cu_k"])
        return {"keys": keys, "values": values}
    if op == "decode":
        return _plain_decode(s)
    if op == "prefill":
        return _plain_prefill(s)
    if op == "store":
        _plain_store(s, s["key_pages"], s["keys"], False)
        _plain_store(s, s["value_pages"], s["values"], True)
    return _plain_gather(s)


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
_GRID = [m * 2.0 ** -9 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:-1]  # of codes 0 to 126


def _two(e):
    """float64 2^e of whole numbers e, exactly (pow is not on every device)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_codes(s, pages, value, r):
    """float64 code values [context, Hkv, D] and scales [context, Hkv] of sequence r, dim by dim through its block table."""
    bs, d, hkv = s["case"]["bs"], s["case"]["d"], s["case"]["hkv"]
    ctx, dev = s["contexts"][r], pages.device
    if ctx == 0:
        return torch.zeros(0, hkv, d, dtype=torch.float64, device=dev), torch.zeros(0, hkv, dtype=torch.float64, device=dev)
    raw = pages[s["table"][r, :-(-ctx // bs)].long()]  # [n, Hkv, groups, bytes]
    raw = raw.transpose(1, 2).flatten(0, 1)  # groups in order, [n, Hkv, bytes]
    place = np.zeros((GROUP, d), dtype=np.int64)
    for tok in range(GROUP):
        for dim in range(d):
            part, start = dim // 64, dim // 64 * 64
            w = min(64, d - start)
            i = dim - start
            if value:
                inner = (((tok // 8 * 8 + i // (w // 8)) * 4 + tok % 8 // 2) * (w // 8) + i % (w // 8)) * 2 + tok % 2
            else:
                inner = tok * w + i
            place[tok, dim] = part * 64 * GROUP + inner
    byte = raw[..., torch.from_numpy(place).to(dev)].long()  # [n, Hkv, 16, D]
    grid = torch.tensor(_GRID + [math.nan], dtype=torch.float64, device=dev)
    v = grid[byte % 128] * torch.where(byte >= 128, -1.0, 1.0).to(torch.float64)
    b = raw[..., GROUP * d].long()
    scale = torch.where(b == 0, 0.0, _two(b - 127))
    return v.transpose(1, 2).flatten(0, 1)[:ctx], scale.repeat_interleave(GROUP, 0)[:ctx]


def _nearest(y):
    """e4m3 values nearest to y, by distance to the neighbours of each in the list of all of them."""
    grid = torch.tensor(_GRID, dtype=torch.float64, device=y.device)
    a = y.abs().contiguous()
    hi = torch.searchsorted(grid, a).clamp(max=len(_GRID) - 1)
    lo = (hi - 1).clamp(min=0)
    below, above = a - grid[lo], grid[hi] - a
    take_lo = (below < above) | ((below == above) & (lo % 2 == 0))  # of two as near, the even code
    v = torch.where(take_lo, grid[lo], grid[hi])
    return torch.where(torch.isfinite(y), torch.sign(y) * v, torch.nan)


def _need(a):
    """Least power of two 2^e with a <= 448 * 2^e, held in the range of the scale byte; 0 for 0."""
    e = torch.ceil(torch.log2(torch.where(a > 0, a, 448.0) / 448.0))
    e = torch.where(_two(e) * 448.0 < a, e + 1, e)
    e = torch.where(_two(e - 1) * 448.0 >= a, e - 1, e)
    return torch.where(a > 0, _two(e.clamp(-126, 119)), 0.0)


def _exact_store(code, scale, x):
    """The sequence's values after x [tokens, Hkv, D] is stored at its end, block after block."""
    ctx, n = code.shape[0], x.shape[0]
    x = x.to(torch.float64)
    out = code * scale[..., None]
    g = (ctx - n) // GROUP * GROUP
    while g < ctx:
        new = slice(max(g, ctx - n), min(g + GROUP, ctx))
        part = x[new.start - (ctx - n):new.stop - (ctx - n)]
        a = torch.where(torch.isfinite(part), part.abs(), 0.0).amax((0, 2))
        unit = _need(a)
        if new.start > g:  # tokens before these keep the block's scale alive
            old = scale[g]
            unit = torch.maximum(unit, old)
            kept = code[g:new.start] * torch.where(unit > 0, old / torch.where(unit > 0, unit, 1.0), 0.0)[:, None]
            kept = torch.where((unit > old)[:, None], _nearest(kept), kept)
            out[g:new.start] = kept * unit[:, None]
        safe = torch.where(unit > 0, unit, 1.0)[:, None]
        out[new] = torch.where(torch.isfinite(part), _nearest(part / safe) * unit[:, None], torch.nan)
        g += GROUP
    return out


def exact(case, seed):
    s = prepare(case, seed)
    ctx, new = _lengths(case)
    keys, values, out = [], [], []
    at = 0
    for r, (c, n) in enumerate(zip(ctx, new)):
        (kc, ks), (vc, vs) = _exact_codes(s, s["key_pages"], False, r), _exact_codes(s, s["value_pages"], True, r)
        if case["op"] == "store":
            k, v = _exact_store(kc, ks, s["keys"][at:at + n]), _exact_store(vc, vs, s["values"][at:at + n])
        else:
            k, v = kc * ks[..., None], vc * vs[..., None]
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
