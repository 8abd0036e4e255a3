"""Oracle of the KV cache held in 8 bits: the format by its definition, pages byte by byte.

No counterpart in the reference, whose cache is bf16 (nv/npu/paged_kv_cache.py:1-72).  Everything runs on the CPU in
float64, a tile at a time; pages are uint8 tensors laid out as include/nvamd.h says.  Attention over the values that the
pages hold, and its bound, are those of ``oracle.fp4_ref``: queries, weights and sums are treated alike.
"""
from __future__ import annotations

import math

import torch

TILE = 16
EMIN, EMAX = -117, 119
# magnitudes of codes 0 .. 126: 3 bits of fraction, 4 of exponent, subnormal below 2^-6
GRID = torch.tensor([m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127],
                    dtype=torch.float64)


def exponent(top: float) -> int:
    """The least e with top <= 448 * 2^e, within [EMIN, EMAX]."""
    e = EMIN
    while e < EMAX and top > 448.0 * 2.0 ** e:
        e += 1
    return e


def codes_of(x: torch.Tensor, e: int) -> torch.Tensor:
    """Codes of float64 values under the scale 2^e."""
    u = (x.abs() / 2.0 ** e).nan_to_num(0.0, 448.0).clamp(max=448.0)
    above = torch.searchsorted(GRID, u.contiguous()).clamp(1, 126)
    far, near = GRID[above] - u, u - GRID[above - 1]
    code = torch.where((far < near) | ((far == near) & (above % 2 == 0)), above, above - 1)
    code = torch.where(x.isfinite(), code, 127)
    return (code + 128 * torch.signbit(x)).to(torch.uint8)


def values_of(codes: torch.Tensor, e: int) -> torch.Tensor:
    low = (codes & 127).long()
    value = torch.where(low == 127, math.nan, GRID[low.clamp(max=126)]) * 2.0 ** e
    return torch.where(codes >= 128, -value, value)


def empty_pages(num_blocks: int, hkv: int, bs: int) -> tuple[torch.Tensor, ...]:
    """k_codes, k_scales, v_codes, v_scales."""
    codes, scales = (num_blocks, hkv, bs, 128), (num_blocks, hkv, bs // TILE)
    return tuple(torch.zeros(shape, dtype=torch.uint8) for shape in (codes, scales, codes, scales))


def _byte_index(which: int, tile: int) -> torch.Tensor:
    """Flat indices [16, 128] of a tile's codes: keys (0) or values (1)."""
    t, d = torch.arange(TILE)[:, None], torch.arange(128)
    return 2048 * tile + (1024 * (d // 64) + 64 * t + d % 64 if which == 0 else 16 * d + t)


def runs(slots: torch.Tensor):
    """(first row, slot, rows) of the rows that follow one another inside a tile."""
    slots, i = slots.tolist(), 0
    while i < len(slots):
        n = 1
        if slots[i] >= 0:
            while i + n < len(slots) and slots[i + n] == slots[i] + n and slots[i + n] % TILE:
                n += 1
            yield i, slots[i], n
        i += n


def write(pages, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Rows [T, hkv, 128] into the pages at their slots (those of slot -1 skipped)."""
    _, hkv, bs, _ = pages[0].shape
    for i, slot, n in runs(slots):
        o = slot % TILE
        for head in range(hkv):
            tile = ((slot // bs * hkv + head) * bs + slot % bs) // TILE
            for which, rows in enumerate((k, v)):
                codes, scales = pages[2 * which].view(-1), pages[2 * which + 1].view(-1)
                at = _byte_index(which, tile)
                x = rows[i:i + n, head].double()
                fine = x[x.isfinite()]
                e = exponent(fine.abs().max().item() if fine.numel() else 0.0)
                if o > 0:
                    held = int(scales[tile]) - 127
                    if e > held:
                        codes[at] = codes_of(values_of(codes[at], held), e)
                    e = max(e, held)
                elif which == 1:
                    codes[at] = 0  # (keys behind the rows are left as they are: nothing reads them)
                codes[at[o:o + n]] = codes_of(x, e)
                scales[tile] = e + 127


def read(pages, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """float64 keys and values [T, hkv, 128] at the slots (zeros for -1)."""
    _, hkv, bs, _ = pages[0].shape
    out = torch.zeros((2, len(slots), hkv, 128), dtype=torch.float64)
    for i, slot in enumerate(slots.tolist()):
        for head in range(hkv) if slot >= 0 else ():
            tile = ((slot // bs * hkv + head) * bs + slot % bs) // TILE
            for which in range(2):
                byte = pages[2 * which].view(-1)[_byte_index(which, tile)[slot % TILE]]
                out[which, i, head] = values_of(byte, int(pages[2 * which + 1].view(-1)[tile]) - 127)
    return out[0], out[1]


def read_sequence(pages, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``read`` of many slots at once."""
    _, hkv, bs, _ = pages[0].shape
    tile = ((slots // bs)[:, None] * hkv + torch.arange(hkv)) * (bs // TILE) + (slots % bs // TILE)[:, None]
    t, d = (slots % TILE)[:, None, None], torch.arange(128)
    out = []
    for which, at in enumerate((1024 * (d // 64) + 64 * t + d % 64, 16 * d + t)):
        byte = pages[2 * which].view(-1)[2048 * tile[..., None] + at]
        step = torch.pow(2.0, pages[2 * which + 1].view(-1)[tile].double() - 127)[..., None]
        out.append(values_of(byte, 0) * step)
    return out[0], out[1]


def write_sequences(pages, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """``write`` of many rows at once, every tile from its first token on."""
    _, hkv, bs, _ = pages[0].shape
    begins = slots % TILE == 0
    assert len(slots) == 0 or (begins[0] and ((slots[1:] == slots[:-1] + 1) | begins[1:]).all())
    run = begins.long().cumsum(0) - 1
    tile = ((slots // bs)[:, None] * hkv + torch.arange(hkv)) * (bs // TILE) + (slots % bs // TILE)[:, None]  # [T, hkv]
    t, d = (slots % TILE)[:, None, None], torch.arange(128)
    steps = torch.pow(2.0, torch.arange(EMIN, EMAX + 1).double())
    for which, (rows, at) in enumerate(((k, 1024 * (d // 64) + 64 * t + d % 64), (v, 16 * d + t))):
        x = rows.double()
        top = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
        tops = torch.zeros(int(begins.sum()), hkv, dtype=torch.float64)
        tops.scatter_reduce_(0, run[:, None].expand(-1, hkv), top, "amax")
        e = torch.searchsorted(448.0 * steps, tops).clamp(max=len(steps) - 1) + EMIN  # the least that reaches it
        codes, scales = pages[2 * which].view(-1), pages[2 * which + 1].view(-1)
        if which == 1:
            codes.view(-1, 2048)[tile[begins]] = 0
        e = e[run]
        codes[2048 * tile[..., None] + at] = codes_of(x / torch.pow(2.0, e.double())[..., None], 0)
        scales[tile] = (e + 127).to(torch.uint8)
