"""Copies of blocks in pools whose strides say less than their sizes."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from nano_vllm_ascend_amd import _C


def one_block_pool(layers, *block, dtype=torch.uint8, device="cpu"):
    """Contiguous [layers, 1, *block] whose stride of the one block is a whole pool's, and the memory behind it."""
    memory = torch.zeros((2, layers, *block), dtype=dtype, device=device)
    pool = memory[:1].transpose(0, 1)
    assert pool.is_contiguous() and pool.shape[:2] == (layers, 1) and pool.stride(1) == layers * pool.stride(0)
    return pool, memory


def test_a_blocks_size_is_that_of_its_values(monkeypatch):
    """The stride of a dim of size one may be anything in a contiguous tensor: a block's bytes do not come from it."""
    called = []

    def copy(at, sizes, n_pools, layers, blocks, src, dst, n, stream):
        called.append((list(sizes), n_pools, layers, blocks, n))
        return 0

    _C.load()  # binds _calls
    monkeypatch.setattr(_C, "_lib", SimpleNamespace(nvamd_copy_blocks=copy))
    monkeypatch.setattr(_C, "_calls", None)
    monkeypatch.setattr(_C, "_stream_of", lambda *a: None)
    ids = torch.zeros(1, dtype=torch.int32)
    pools = [one_block_pool(5, 4, 3)[0], one_block_pool(5, 8, dtype=torch.int16)[0], torch.zeros(5, 1, 2, 7)]
    _C.copy_blocks(pools, ids, ids)
    assert called == [([12, 16, 56], 3, 5, 1, 1)]
    _C.copy_blocks([torch.zeros(1, 6, 4, 3)], ids, ids)
    assert called[1] == ([48], 1, 1, 6, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("at_once", [False, True])
def test_a_pool_of_one_block_is_left_alone(device, monkeypatch, at_once):
    """Its only pair is the block itself, which is no copy; with another size of a block, a pair in a pool of two."""
    _C.load()  # binds _calls
    if not at_once:
        monkeypatch.setattr(_C, "_calls", None)
    pool, memory = one_block_pool(5, 16, 3, device=device)
    memory.copy_(torch.arange(memory.numel(), device=device).view_as(memory) % 251)
    want = memory.clone()
    ids = torch.zeros(1, dtype=torch.int32, device=device)
    _C.copy_blocks([pool], ids, ids)
    # one layer of two blocks: here it is the layers' stride that says nothing
    two = torch.arange(2 * 48, dtype=torch.uint8, device=device).view(2, 48)
    layer = two.as_strided((1, 2, 48), (7, 48, 1))
    assert layer.is_contiguous()
    _C.copy_blocks([layer], ids, ids + 1)
    assert torch.equal(memory, want) and torch.equal(two[0], two[1]) and two[0].tolist() == list(range(48))
