"""Paged KV store (nv/npu/paged_kv_cache.py:1-72).

Two bf16 tensors [num_layers, num_blocks, block_size, num_kv_heads, head_dim],
allocated once; ``write`` scatters token rows into slots with the HIP store
kernel (the reference used two index_copy_ calls) and ``get_physical_cache``
hands out per-layer [num_blocks, block_size, num_kv_heads, head_dim] views.
At 128-token pages one block of K for one layer is 128 * 8 * 128 * 2 B =
256 KiB of contiguous HBM, so a page is read with long linear bursts.

``Fp4PagedKVCache`` holds the same rows in 4 bits (FP4 codes with a power-of-two
scale per 32 dims): 68 bytes per head vector instead of 256.  ``Fp8PagedKVCache``
holds them in 8 bits (e4m3 codes with a power-of-two scale per tile of 16 tokens
of a head): 128 bytes and a 16th.

Each has ``copy_blocks``: blocks of every layer copied to others in one launch.
"""
from __future__ import annotations

import torch

from . import _C


class PagedKVCache:
    def __init__(self, num_layers: int, num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int,
                 dtype: torch.dtype, device):
        self.num_layers = num_layers
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.dtype = dtype
        self.device = device
        shape = (num_layers, num_blocks, block_size, num_kv_heads, head_dim)
        self.key_cache = torch.empty(shape, dtype=dtype, device=device)
        self.value_cache = torch.empty(shape, dtype=dtype, device=device)

    @staticmethod
    def bytes_per_block(num_layers: int, block_size: int, num_kv_heads: int, head_dim: int, elem: int = 2) -> int:
        return 2 * num_layers * block_size * num_kv_heads * head_dim * elem

    def write(self, layer_idx: int, key_states: torch.Tensor, value_states: torch.Tensor,
              slot_mapping: torch.Tensor) -> None:
        total, hkv, d = key_states.shape
        if hkv != self.num_kv_heads or d != self.head_dim:
            raise ValueError(f"kv shape mismatch: got {tuple(key_states.shape)}")
        if slot_mapping.numel() != total:
            raise ValueError(f"slot_mapping numel {slot_mapping.numel()} != total_tokens {total}")
        slots = slot_mapping.to(device=self.key_cache.device, dtype=torch.int64)
        _C.kv_cache_write(key_states, value_states, self.key_cache[layer_idx], self.value_cache[layer_idx], slots)

    def get_physical_cache(self, layer_idx: int) -> tuple[torch.Tensor, torch.Tensor]:
        return self.key_cache[layer_idx], self.value_cache[layer_idx]

    def copy_blocks(self, sources, targets) -> None:
        """Blocks sources[i] to targets[i], in every layer (``_copy_blocks``)."""
        _copy_blocks((self.key_cache, self.value_cache), self.num_blocks, sources, targets)


def _copy_blocks(pools, num_blocks: int, sources, targets) -> None:
    """sources and targets: int32 tensors on the device, or block ids on the host, which are checked: blocks of the pool,
    no target twice, none that another pair reads."""
    if not isinstance(sources, torch.Tensor) or not isinstance(targets, torch.Tensor):
        pairs = [torch.as_tensor(list(x), dtype=torch.int32) for x in (sources, targets)]
        if pairs[0].shape != pairs[1].shape:
            raise ValueError(f"{pairs[0].numel()} sources for {pairs[1].numel()} targets")
        _C.check_block_pairs(*pairs, num_blocks)
        sources, targets = torch.stack(pairs).to(pools[0].device)
    _C.copy_blocks(pools, sources, targets)


class _QuantisedKVCache:
    """What the caches of a few bits share: codes and scales of a layer's keys and values in ``_pages``."""

    dtype = torch.uint8

    def __init__(self, num_layers: int, num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int, device):
        if head_dim != 128:
            raise ValueError(f"head_dim must be 128, got {head_dim}")
        if block_size < 16 or block_size & (block_size - 1):
            raise ValueError(f"block_size must be a power of two >= 16, got {block_size}")
        self.num_layers = num_layers
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.device = device

    def _slots(self, slot_mapping: torch.Tensor) -> torch.Tensor:
        return slot_mapping.to(device=self.key_codes.device, dtype=torch.int64).reshape(-1).contiguous()

    def _check_rows(self, key_states: torch.Tensor, slot_mapping: torch.Tensor) -> None:
        total, hkv, d = key_states.shape
        if hkv != self.num_kv_heads or d != self.head_dim:
            raise ValueError(f"kv shape mismatch: got {tuple(key_states.shape)}")
        if slot_mapping.numel() != total:
            raise ValueError(f"slot_mapping numel {slot_mapping.numel()} != total_tokens {total}")

    def get_physical_cache(self, layer_idx: int):
        return self._pages[layer_idx]

    @property
    def _pools(self) -> tuple[torch.Tensor, ...]:
        return self.key_codes, self.key_scales, self.value_codes, self.value_scales

    def copy_blocks(self, sources, targets) -> None:
        """Blocks sources[i] to targets[i], in every layer (``_copy_blocks``)."""
        _copy_blocks(self._pools, self.num_blocks, sources, targets)


class Fp4PagedKVCache(_QuantisedKVCache):
    """PagedKVCache whose pages are held in 4 bits; rows go in and come out in bf16.

    ``get_physical_cache`` gives a layer's ``Fp4Pages`` of keys and of values, which the
    attention layers take in the place of a bf16 cache's tensors."""

    def __init__(self, num_layers: int, num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int, device):
        super().__init__(num_layers, num_blocks, block_size, num_kv_heads, head_dim, device)
        rows = (num_layers, num_blocks, num_kv_heads, block_size)
        # zeroed, so that a page whose rows are not all written yet holds numbers
        self.key_codes, self.value_codes = (torch.zeros((*rows, _C.FP4_ROW_BYTES), dtype=torch.uint8, device=device)
                                            for _ in range(2))
        self.key_scales, self.value_scales = (
            torch.zeros((*rows, _C.FP4_ROW_SCALES), dtype=torch.uint8, device=device) for _ in range(2))
        self._pages = [(_C.Fp4Pages(kc, ks), _C.Fp4Pages(vc, vs)) for kc, ks, vc, vs in
                       zip(self.key_codes, self.key_scales, self.value_codes, self.value_scales)]

    @staticmethod
    def bytes_per_block(num_layers: int, block_size: int, num_kv_heads: int, head_dim: int) -> int:
        return 2 * num_layers * block_size * num_kv_heads * (head_dim // 2 + head_dim // 32)

    def write(self, layer_idx: int, key_states: torch.Tensor, value_states: torch.Tensor,
              slot_mapping: torch.Tensor) -> None:
        self._check_rows(key_states, slot_mapping)
        _C.kv_cache_write_fp4(key_states, value_states, *self.get_physical_cache(layer_idx), self._slots(slot_mapping))

    def read(self, layer_idx: int, slot_mapping: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """The bf16 keys and values [T, kv heads, head_dim] that the layer holds at the slots (zeros for -1)."""
        return _C.kv_cache_read_fp4(*self.get_physical_cache(layer_idx), self._slots(slot_mapping))


class Fp8PagedKVCache(_QuantisedKVCache):
    """PagedKVCache whose pages are held in 8 bits, a scale for each tile of 16 tokens of a head; rows go in and come out
    in bf16.

    A tile is filled from its first token on, by rows that follow one another in a call (``_C.kv_cache_write_fp8``), as
    the tokens of a sequence are.  ``get_physical_cache`` gives a layer's ``Fp8Pages`` of keys and of values."""

    def __init__(self, num_layers: int, num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int, device):
        super().__init__(num_layers, num_blocks, block_size, num_kv_heads, head_dim, device)
        rows = (num_layers, num_blocks, num_kv_heads, block_size)
        tiles = (num_layers, num_blocks, num_kv_heads, block_size // _C.FP8_TILE)
        self.key_codes, self.value_codes = (torch.zeros((*rows, _C.FP8_ROW_BYTES), dtype=torch.uint8, device=device)
                                            for _ in range(2))
        self.key_scales, self.value_scales = (torch.zeros(tiles, dtype=torch.uint8, device=device) for _ in range(2))
        self._pages = [(_C.Fp8Pages(kc, ks), _C.Fp8Pages(vc, vs)) for kc, ks, vc, vs in
                       zip(self.key_codes, self.key_scales, self.value_codes, self.value_scales)]

    @staticmethod
    def bytes_per_block(num_layers: int, block_size: int, num_kv_heads: int, head_dim: int) -> int:
        return 2 * num_layers * num_kv_heads * (block_size * head_dim + block_size // _C.FP8_TILE)

    def write(self, layer_idx: int, key_states: torch.Tensor, value_states: torch.Tensor,
              slot_mapping: torch.Tensor) -> None:
        """Unlike the other caches' this asks for an order: the rows of a tile follow one another in that of their slots.
        Slots on the host are checked for it; of slots on the device see ``_C.kv_cache_write_fp8``."""
        self._check_rows(key_states, slot_mapping)
        if not slot_mapping.is_cuda:
            _C.check_tile_order(slot_mapping)
        _C.kv_cache_write_fp8(key_states, value_states, *self.get_physical_cache(layer_idx), self._slots(slot_mapping))

    def read(self, layer_idx: int, slot_mapping: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """The bf16 keys and values [T, kv heads, head_dim] that the layer holds at the slots (zeros for -1)."""
        return _C.kv_cache_read_fp8(*self.get_physical_cache(layer_idx), self._slots(slot_mapping))

    def keep_tiles(self, slot_mapping: torch.Tensor) -> torch.Tensor:
        """The tiles that rows at the slots would go behind, in every layer: such rows may raise a tile's scale, which
        rounds its other tokens again.  ``restore_tiles`` takes them back."""
        return _C.kv_cache_keep_fp8(self._pools, self._slots(slot_mapping))

    def restore_tiles(self, kept: torch.Tensor) -> None:
        _C.kv_cache_restore_fp8(self._pools, kept)
