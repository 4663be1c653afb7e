"""The 4-bit paged KV pool: K and V in microscaled 4-bit floating point (MXFP4).

An option beside ``KVCache`` for a pool that has to hold 3.76 times the tokens
of a 16-bit one: e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), one
power-of-two scale for every 32 elements along the head dimension.  A layer's
pages are uint8 ``[blocks, Hkv, block_size / 16, D / 32 * 272]``; the last
dimension is a group of 16 tokens of one kv head: the codes
``[D / 32][16 tokens][16 bytes]`` (the even element in the low nibble), then the
scale bytes ``[16 tokens][D / 32]`` (e stands for 2^(e - 127), 0 for zero, 255 for NaN).
Zero-filled pages hold zeros.  ``block_size`` is a multiple of 16, ``D`` of 32 (at most 256).

``store_kv_mxfp4`` quantises as it stores; ``layer.mxfp4_attention`` has what
reads the pool.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from microinfer_b200 import _lib
from microinfer_b200.worker.kv_cache import copy_blocks

GROUP = 16  # tokens of a group
MX = 32  # elements that share a scale
MX_BYTES = 272  # bytes of one block of 32 elements of a group's 16 tokens


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
    if size == 0 or size % MX_BYTES:
        raise ValueError(f"the last dimension of pages must be head_dim / {MX} * {MX_BYTES} bytes")
    return blocks, groups * GROUP, hkv, size // MX_BYTES * MX


def store_kv_mxfp4(key_pages, value_pages, slots, keys, values):
    """Quantise keys[t] and values[t] ([T, Hkv, D]) into slot ``slots[t]`` (-1 writes nothing).

    Slots must be unique within a call, as for ``store_kv_slots``.
    """
    if torch.compiler.is_compiling():  # an opaque node for torch.compile
        torch.ops.microinfer_b200.store_kv_mxfp4(key_pages, value_pages, slots, keys, values)
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
    _lib.call(
        "mi_store_kv_mxfp4", key_pages.data_ptr(), value_pages.data_ptr(), nb, bs, hkv, d,
        slots.data_ptr(), index, keys.data_ptr(), values.data_ptr(), dtype, key_stride[0],
        value_stride[0], tokens, _lib.status_buffer(device).data_ptr(), _lib.stream_of(device),
    )


@dataclass(frozen=True)
class LayerMXFP4Cache:
    """One layer's pages, uint8 [blocks, Hkv, block_size / 16, bytes]; the 4-bit ``LayerKVCache``."""

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
        return self.keys.shape[3] // MX_BYTES * MX

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
        store_kv_mxfp4(self.keys, self.values, slots, keys, values)


class MXFP4KVCache:
    """``KVCache`` in 4 bits: pools of zero-filled pages for all layers."""

    def __init__(self, num_layers, num_blocks, block_size, num_kv_heads, head_dim, *, device="cuda"):
        if any(n <= 0 for n in (num_layers, num_blocks, block_size, num_kv_heads, head_dim)):
            raise ValueError("cache dimensions must be positive")
        if block_size % GROUP:
            raise ValueError("block_size must be a multiple of 16")
        if head_dim % MX or head_dim > 256:
            raise ValueError("head_dim must be a multiple of 32, at most 256")
        self.num_layers = num_layers
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.device = torch.device(device)
        shape = (num_layers, num_blocks, num_kv_heads, block_size // GROUP, head_dim // MX * MX_BYTES)
        self.keys = torch.zeros(shape, dtype=torch.uint8, device=device)
        self.values = torch.zeros_like(self.keys)

    @property
    def num_bytes(self) -> int:
        return self.keys.numel() * 2

    def layer(self, index: int) -> LayerMXFP4Cache:
        if not 0 <= index < self.num_layers:
            raise ValueError("layer outside cache")
        return LayerMXFP4Cache(self.keys[index], self.values[index])

    def copy_blocks(self, pairs, *, check: bool = True):
        """Copy-on-write: page src -> dst in every layer, for K and V (as ``KVCache.copy_blocks``)."""
        copy_blocks(self.keys, self.values, pairs, check=check)
