"""Rows of an 8-bit tile that do not follow one another in a call: two waves would write the tile at once, so the later ones
are not stored, and the error word says so."""
from __future__ import annotations

import re
from pathlib import Path

import pytest
import torch

from nano_vllm_ascend_amd import _C
from nano_vllm_ascend_amd.paged_kv_cache import Fp8PagedKVCache
from oracle import fp8_ref

HEADER = Path(__file__).resolve().parents[1] / "include" / "nvamd.h"
NEAR = 32  # NVAMD_FP8_ORDER_ROWS
EPS = 1e-6


def stored(slots):
    """The slots whose rows are stored: those of a run (rows that follow one another inside a tile) unless an earlier row
    lies in its tile."""
    out, seen = list(slots), set()
    for i, slot, n in fp8_ref.runs(torch.tensor(slots)):
        if slot // 16 in seen:
            out[i:i + n] = [-1] * n
        seen.add(slot // 16)
    return out


def test_the_rule():
    assert stored([1, 0]) == [1, -1] and stored([0, 2, 16]) == [0, -1, 16] and stored([5, 5]) == [5, -1]
    assert stored([0, -1, 1, 2]) == [0, -1, -1, -1] and stored([4, 40, 5, 6]) == [4, 40, -1, -1]
    assert stored([14, 15, 16, 17, 3, -1]) == [14, 15, 16, 17, -1, -1]
    header = HEADER.read_text()
    assert int(re.search(r"#define NVAMD_ERR_ORDER (\d+)u", header).group(1)) == _C.ERR_ORDER
    assert int(re.search(r"#define NVAMD_FP8_ORDER_ROWS (\d+)", header).group(1)) == NEAR
    assert "follow one another" in _C.describe_index_errors(_C.ERR_ORDER)


def test_host_slots_are_refused_however_far_apart():
    cache = Fp8PagedKVCache(1, 64, 32, 1, 128, "cpu")
    far_apart = torch.cat([torch.tensor([64]), 16 * torch.arange(10, 110), torch.tensor([65])])
    for slots in (torch.tensor([1, 0]), far_apart, far_apart.int(), far_apart[:, None]):
        k = torch.zeros(slots.numel(), 1, 128, dtype=torch.bfloat16)
        with pytest.raises(IndexError, match="do not follow one another"):
            cache.write(0, k, k, slots)
    k = torch.zeros(3, 1, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="on the GPU"):  # checked, and then refused for where the rows are
        cache.write(0, k, k, torch.tensor([15, 16, 17]))


def rows(t, heads, seed):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(t, heads, 128, generator=gen) * torch.exp(torch.randn(t, heads, 1, generator=gen))).bfloat16()


def far(n):  # n slots, each of a tile of its own, past those of the cases
    return [16 * (40 + i) + 5 for i in range(n)]


CASES = {
    "reversed": list(range(15, -1, -1)),
    "a gap": [0, 1, 3, 4, 16],
    "the same slot": [7, 7, 20, 20, 21],
    "padding between": [0, -1, 1, 32, 33],
    "another tile between": [4, 20, 5, 6, 21],
    "runs of two": [0, 1, 16, 17, 2, 3, 18, 19],
    "a slot outside between": [2, 1 << 40, 3, 48],
    "as far as is looked": [64, *far(NEAR - 1), 65, 80],
    "in order": [3, 4, 5, 16, 17, 100, -1, -1, 48],
}


def laid_out(name, many):
    """A case's slots alone, or between the rows of a long prompt."""
    slots = CASES[name]
    if not many:
        return slots
    before, after = list(range(16 * 400, 16 * 400 + 301)), list(range(16 * 500 + 9, 16 * 500 + 9 + 611))
    return before + slots + after


@pytest.mark.gpu
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("name", sorted(CASES))
def test_rows_out_of_order_are_not_stored(device, name, many):
    _C.clear_index_errors()
    hkv, bs, nb = 3, 32, 300
    slots = laid_out(name, many)
    outside = any(s >= nb * bs for s in slots)
    keep = stored([s if s < nb * bs else -1 for s in slots])
    k, v = rows(len(slots), hkv, 1), rows(len(slots), hkv, 2)
    cache = Fp8PagedKVCache(1, nb, bs, hkv, 128, device)
    pages = fp8_ref.empty_pages(nb, hkv, bs)
    for page in pages[1::2]:
        page.fill_(110)
    for pool, page in zip(cache._pools, pages):
        pool[0].copy_(page)
    fp8_ref.write(pages, k, v, torch.tensor(keep))
    cache.write(0, k.to(device), v.to(device), torch.tensor(slots, device=device))
    out_of_order = keep != [s if s < nb * bs else -1 for s in slots]
    assert out_of_order == (name != "in order")
    assert _C.index_errors() == out_of_order * _C.ERR_ORDER + outside * _C.ERR_SLOT
    for pool, page in zip(cache._pools, pages):
        assert torch.equal(pool[0].cpu(), page)
    _C.clear_index_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("name", ["reversed", "another tile between", "a slot outside between"])
def test_rows_out_of_order_are_rotated_all_the_same(device, name, many):
    """The rotation returns every row, as it does without a cache's order; of the cache it stores what a write does."""
    _C.clear_index_errors()
    hq, hkv, bs, nb = 4, 2, 32, 300
    slots = torch.tensor(laid_out(name, many), device=device)
    t = len(slots)
    q, k, v = (rows(t, h, 3 + h).to(device) for h in (hq, hkv, hkv))
    w = rows(1, 1, 9).view(128).to(device)
    angle = torch.arange(t)[:, None] * 1e6 ** (-torch.arange(64) / 64)
    table = torch.cat([angle.cos(), angle.sin()], 1).float().to(device)
    pos = torch.arange(t, device=device)
    got, want = (Fp8PagedKVCache(1, nb, bs, hkv, 128, device) for _ in range(2))
    k_out = torch.full_like(k, 7.0)
    q_out = _C.qk_norm_rope_fp8(q, k, v, w, w, pos, table, EPS, *got.get_physical_cache(0), slots, k_out=k_out)
    assert _C.index_errors() & _C.ERR_ORDER
    k_want = torch.full_like(k, 7.0)
    none = torch.full_like(slots, -1)
    q_want = _C.qk_norm_rope_fp8(q, k, v, w, w, pos, table, EPS, *want.get_physical_cache(0), none, k_out=k_want)
    assert torch.equal(q_out, q_want) and torch.equal(k_out, k_want)
    keep = stored([s if s < nb * bs else -1 for s in slots.tolist()])
    want.write(0, k_want, v, torch.tensor(keep, device=device))
    for a, b in zip(got._pools, want._pools):
        assert torch.equal(a, b)
    _C.clear_index_errors()
