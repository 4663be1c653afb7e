"""The 8-bit paged KV pool: K and V in 8-bit floating point with a scale for every block of 16 tokens and kv head.

An option beside ``KVCache`` for a pool that has to hold twice the tokens of a 16-bit one: e4m3 codes (sign, 4 bits
of exponent, 3 of mantissa; largest 448, smallest 2^-9, 0x7f and 0xff not a number), one power-of-two scale for every
16 tokens of a page and kv head (a group).  A layer's pages are uint8 ``[blocks, Hkv, block_size / 16, 16 * D + 16]``; the last
dimension is a group: its codes in parts of 64 dims (w = 64; a last part of 32 where D is an odd multiple of
32), K's as ``[16 tokens][w]``, V's as ``[2 halves][8][4 pairs][w / 8 dims][2 tokens]`` (token = 8 half + 2 pair + last,
dim = w / 8 * second + fourth), then the scale byte (b stands for 2^(b - 127), 0 for zero) and 15 that are zero.
Zero-filled pages hold zeros.  ``block_size`` is a multiple of 16, ``D`` of 32 (at most 256).

``store_kv_fp8`` quantises as it stores; ``layer.fp8_attention`` has what reads the pool.
"""

from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache

import torch

from microinfer_b200 import _lib
from microinfer_b200.worker.kv_cache import copy_blocks

GROUP = 16  # tokens that share a scale
TAIL = 16  # bytes after a group's codes, the scale first


def page_dims(key_pages: torch.Tensor, value_pages: torch.Tensor) -> tuple[int, int, int, int]:
    """(num_blocks, block_size, Hkv, D) of a layer's pages; raises if they are none."""
    shape = key_pages.shape
    if len(shape) != 4 or value_pages.shape != shape:
        raise ValueError("pages must be matching [blocks, Hkv, block_size / 16, bytes] tensors")
    if key_pages.dtype != torch.uint8 or value_pages.dtype != torch.uint8:
        raise ValueError("pages must be uint8")
    if not (key_pages.is_contiguous() and value_pages.is_contiguous()):
        raise ValueError("pages must be contiguous")
    blocks, hkv, groups, size = shape
    if hkv == 0 or groups == 0:
        raise ValueError("pages must have kv heads and tokens")
    head_dim = size // GROUP - 1
    if size % GROUP or head_dim <= 0 or head_dim % 32:
        raise ValueError("the last dimension of pages must be 16 * head_dim + 16 bytes")
    return blocks, groups * GROUP, hkv, head_dim


@lru_cache(maxsize=4096)
def _workspace_bytes(*shape):
    return _lib.load().mi_store_kv_fp8_workspace_bytes(*shape)


def store_kv_fp8(key_pages, value_pages, slots, keys, values):
    """Quantise keys[t] and values[t] ([T, Hkv, D]) into slot ``slots[t]`` (-1 writes nothing).

    Slots may come in any order and must be unique within a call, as for ``store_kv_slots``.  The tokens of a call
    that fall into one block of 16 are quantised together.  A call that writes the block's first slot sets
    the block's scale; any other raises it where its tokens are too large for it, and then the block's other codes are
    rounded to the new scale.  So a block is to be filled from its first slot on, as sequences do: what it held
    before that is given up, whether it is written over or not.
    """
    if torch.compiler.is_compiling():  # an opaque node for torch.compile
        torch.ops.microinfer_b200.store_kv_fp8(key_pages, value_pages, slots, keys, values)
        return
    nb, bs, hkv, d = page_dims(key_pages, value_pages)
    shape = keys.shape
    if len(shape) != 3 or values.shape != shape:
        raise ValueError("K/V shapes differ")
    tokens, heads, dim = shape
    if heads != hkv or dim != d:
        raise ValueError("K/V heads do not match the cache")
    key_stride, value_stride = keys.stride(), values.stride()
    # the stride of a single head means nothing (a transpose of [1, T, D] is contiguous)
    if (key_stride[2] != 1 or value_stride[2] != 1
            or (hkv > 1 and (key_stride[1] != d or value_stride[1] != d))):
        raise ValueError("K/V inner dimensions must be contiguous")
    if keys.dtype != values.dtype:
        raise ValueError("K/V must share a dtype")
    dtype = _lib.dtype_code(keys.dtype)
    if slots.shape != (tokens,):
        raise ValueError("slots must have one entry per token")
    index = _lib.index_code(slots.dtype)
    if tokens == 0:
        return
    device = _lib.require_cuda(key_pages, value_pages, slots, keys, values)
    slots = slots.contiguous()
    need = _workspace_bytes(tokens, nb, bs)
    workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    _lib.call(
        "mi_store_kv_fp8", key_pages.data_ptr(), value_pages.data_ptr(), nb, bs, hkv, d,
        slots.data_ptr(), index, keys.data_ptr(), values.data_ptr(), dtype, key_stride[0],
        value_stride[0], tokens, _lib.ptr(workspace), need, _lib.status_buffer(device).data_ptr(), _lib.stream_of(device),
    )


@dataclass(frozen=True)
class LayerFP8Cache:
    """One layer's pages, uint8 [blocks, Hkv, block_size / 16, bytes]; the 8-bit ``LayerKVCache``."""

    keys: torch.Tensor
    values: torch.Tensor

    def __post_init__(self):
        page_dims(self.keys, self.values)
        if self.keys.device != self.values.device:
            raise ValueError("K/V must have matching devices")

    @property
    def block_size(self) -> int:
        return self.keys.shape[2] * GROUP

    @property
    def head_dim(self) -> int:
        return self.keys.shape[3] // GROUP - 1

    def write_checked(self, slots, keys, values):
        """Validate every slot first (-1 skips), then write; invalid input writes nothing."""
        if slots.ndim != 1 or slots.dtype not in (torch.int32, torch.int64):
            raise ValueError("slots must be a 1-D integer tensor")
        expected = (slots.numel(), self.keys.shape[1], self.head_dim)
        if tuple(keys.shape) != expected or tuple(values.shape) != expected:
            raise ValueError("K/V shape must match slots and cache heads")
        if any(t.device != self.keys.device for t in (slots, keys, values)):
            raise ValueError("slots and K/V must be on the cache device")
        if torch.any(slots < -1) or torch.any(slots >= self.keys.shape[0] * self.block_size):
            raise ValueError("slot outside cache")
        valid = slots[slots >= 0]
        if valid.unique().numel() != valid.numel():
            raise ValueError("duplicate slot")
        self.write_slots(slots, keys, values)

    def write_slots(self, slots, keys, values):
        """Hot path from flat slot ids (-1 = padding): valid and unique slots assumed."""
        d = keys.shape[-1]
        if keys.stride(-1) != 1 or keys.stride(-2) != d:
            keys = keys.contiguous()
        if values.stride(-1) != 1 or values.stride(-2) != d:
            values = values.contiguous()
        store_kv_fp8(self.keys, self.values, slots, keys, values)


class FP8KVCache:
    """``KVCache`` in 8 bits: pools of zero-filled pages for all layers."""

    def __init__(self, num_layers, num_blocks, block_size, num_kv_heads, head_dim, *, device="cuda"):
        if any(n <= 0 for n in (num_layers, num_blocks, block_size, num_kv_heads, head_dim)):
            raise ValueError("cache dimensions must be positive")
        if block_size % GROUP:
            raise ValueError("block_size must be a multiple of 16")
        if head_dim % 32 or head_dim > 256:
            raise ValueError("head_dim must be a multiple of 32, at most 256")
        self.num_layers = num_layers
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.device = torch.device(device)
        shape = (num_layers, num_blocks, num_kv_heads, block_size // GROUP, GROUP * head_dim + TAIL)
        self.keys = torch.zeros(shape, dtype=torch.uint8, device=device)
        self.values = torch.zeros_like(self.keys)

    @property
    def num_bytes(self) -> int:
        return self.keys.numel() * 2

    def layer(self, index: int) -> LayerFP8Cache:
        if not 0 <= index < self.num_layers:
            raise ValueError("layer outside cache")
        return LayerFP8Cache(self.keys[index], self.values[index])

    def copy_blocks(self, pairs, *, check: bool = True):
        """Copy-on-write: page src -> dst in every layer, for K and V (as ``KVCache.copy_blocks``)."""
        copy_blocks(self.keys, self.values, pairs, check=check)
