"""Oracle of the KV cache held in 4 bits: the format by its definition, pages byte by byte, attention in 64 bits.

No counterpart in the reference, whose cache is bf16 (nv/npu/paged_kv_cache.py:1-72).  Everything runs on the CPU in
float64; pages are uint8 tensors laid out as include/nvamd.h says.
"""
from __future__ import annotations

import math

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
EMIN, EMAX = -125, 125


def quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes [.., 128] and scale bytes [.., 4] of bf16 rows [.., 128]."""
    x = x.to(torch.float64).unflatten(-1, (4, 32))
    top = x.abs().amax(-1)
    exps = torch.arange(EMIN, EMAX + 1)
    fits = top[..., None] <= 7.0 * torch.pow(2.0, exps.double())  # the least exponent that fits, or the largest
    first = torch.where(fits.any(-1), fits.int().argmax(-1), len(exps) - 1)
    e = exps[first]
    finite = x.isfinite().all(-1)
    u = torch.where(finite[..., None], x.abs() / torch.pow(2.0, e.double())[..., None], 0.0)
    dist = (u[..., None] - GRID).abs()
    dist[..., 1::2] += 1e-9 * (dist[..., 1::2] == dist.min(-1, keepdim=True).values)  # a tie goes to the even code
    code = dist.argmin(-1) + 8 * torch.signbit(torch.where(finite[..., None], x, 0.0))
    return code.flatten(-2).to(torch.uint8), torch.where(finite, e + 127, 255).to(torch.uint8)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """float64 rows of codes [.., 128] and scale bytes [.., 4]."""
    x = GRID[(codes & 7).long()] * torch.where(codes >= 8, -1.0, 1.0)
    step = torch.where(scales == 255, math.nan, torch.pow(2.0, scales.double() - 127))
    return (x.unflatten(-1, (4, 32)) * step[..., None]).flatten(-2)


def empty_pages(num_blocks: int, hkv: int, bs: int) -> tuple[torch.Tensor, ...]:
    """k_codes, k_scales, v_codes, v_scales."""
    return tuple(torch.zeros((num_blocks, hkv, bs, w), dtype=torch.uint8) for w in (64, 4, 64, 4))


def _places(num_blocks: int, hkv: int, bs: int, slots: torch.Tensor):
    """Flat byte indices of rows: [T, hkv, 64] of key and value codes and [T, hkv, 4] of their scales."""
    tile = ((slots // bs)[:, None] * hkv + torch.arange(hkv)) * (bs // 16) + (slots % bs // 16)[:, None]  # [T, hkv]
    t = (slots % 16)[:, None, None]
    byte, q = torch.arange(64), torch.arange(4)
    codes, scales = 1024 * tile[..., None], 64 * tile[..., None]
    return codes + 64 * t + byte, scales + 16 * (t % 4) + 4 * q + t // 4, codes + 16 * byte + t, scales + 16 * q + t


def write(pages, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Rows [T, hkv, 128] into the pages at their slots (those of slot -1 skipped)."""
    nb, hkv, bs, _ = pages[0].shape
    keep = slots >= 0
    at = _places(nb, hkv, bs, slots[keep])
    code, scale = quantise(k[keep])
    pages[0].view(-1)[at[0]] = code[..., 0::2] | (code[..., 1::2] << 4)
    pages[1].view(-1)[at[1]] = scale
    code, scale = quantise(v[keep])
    code = code.unflatten(-1, (4, 2, 16))
    pages[2].view(-1)[at[2]] = (code[..., 0, :] | (code[..., 1, :] << 4)).flatten(-2)
    pages[3].view(-1)[at[3]] = scale


def read(pages, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """float64 keys and values [T, hkv, 128] at the slots (zeros for -1)."""
    nb, hkv, bs, _ = pages[0].shape
    at = _places(nb, hkv, bs, slots.clamp(min=0))
    byte = pages[0].view(-1)[at[0]]
    k = values(torch.stack((byte & 15, byte >> 4), -1).flatten(-2), pages[1].view(-1)[at[1]])
    byte = pages[2].view(-1)[at[2]].unflatten(-1, (4, 16))
    v = values(torch.stack((byte & 15, byte >> 4), -2).flatten(-3), pages[3].view(-1)[at[3]])
    gone = (slots < 0)[:, None, None]
    return k.masked_fill(gone, 0.0), v.masked_fill(gone, 0.0)


def norm_rope(x: torch.Tensor, weight: torch.Tensor, positions: torch.Tensor, table: torch.Tensor,
              eps: float) -> torch.Tensor:
    """RoPE(RMSNorm_head(x) * w) of [T, heads, 128] in float64; table fp32 [positions, 64 cos + 64 sin]."""
    x = x.double()
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + float(torch.tensor(eps, dtype=torch.float32)))
    y = y * weight.double()
    cos, sin = table.double()[positions][:, None].split(64, -1)
    lo, hi = y.split(64, -1)
    return torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), -1)


def to_bf16(x: torch.Tensor) -> torch.Tensor:
    """bf16 of float64 values with one rounding (``.bfloat16()`` rounds to 32 bits on the way): the 32-bit value nearest
    towards zero, with its last bit set where anything was cut off, rounds to bf16 as the value itself does."""
    f = x.float()
    f = torch.where(f.double().abs() > x.abs(), torch.nextafter(f, torch.zeros_like(f)), f)
    bits = f.view(torch.int32) | (f.double() != x).int()
    return bits.view(torch.float32).bfloat16()


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows [n, hq, 128] that are the last n positions of keys / values [m, hkv, 128], causal; and a bound of the error of an
    evaluation with 32-bit scores and sums, weights rounded to bf16 (the sum taking the same rounded weights) and a
    bf16 result.  Every rounding to bf16 is off by at most 2^-8 of the value.  With A = sum p |v|:
      weights: numerator and sum are each off by 2^-8 of A and of 1:              2 * 2^-8 * A
      scores: 128 products and sums of 2^-24 of sum |q k| each, the product with the scale and the exponential's argument
        some 2^-22 of the largest score: an exponent off by d scales every weight by at most e^d, numerator and sum
        alike:                                                                    2 * (e^d - 1) * A
      queries: of a block of 32 dims the values below 2^-9 of its largest are off by at most 2^-17 of that, which adds
        2^-17 max |q| sum |k| over them to the error of a score
      result:                                                                     2^-8 * (|out| + the above)
    Rows that see no key are zero."""
    n, hq, _ = q.shape
    m, hkv, _ = k.shape
    out, tol = torch.zeros(n, hq, 128, dtype=torch.float64), torch.zeros(n, hq, 128, dtype=torch.float64)
    seen = torch.arange(m)[None, :] <= (m - n + torch.arange(n))[:, None]
    for h in range(hq):
        kk, vv, qq = k[:, h // (hq // hkv)], v[:, h // (hq // hkv)], q[:, h].double()
        s = torch.where(seen, qq @ kk.T * scale, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
        total = p.sum(-1, keepdim=True)
        p = torch.where(total > 0, p / total, torch.where(total.isnan(), math.nan, 0.0))
        # a masked weight times an infinite or NaN value is nothing
        out[:, h] = torch.where(seen.any(-1, keepdim=True), (p @ vv.nan_to_num(0.0, 0.0, 0.0)), 0.0)
        hit = seen.double() @ (~vv.isfinite()).double()
        out[:, h] = torch.where(hit > 0, math.nan, out[:, h])
        a = p.nan_to_num(0.0) @ vv.nan_to_num(0.0, 0.0, 0.0).abs()
        mass = (qq.abs() @ kk.nan_to_num(0.0).abs().T * abs(scale)).amax(-1, keepdim=True)
        top = qq.abs().unflatten(-1, (4, 32)).amax(-1, keepdim=True).expand(-1, -1, 32).flatten(1)
        lost = torch.where(qq.abs() < 2.0 ** -9 * top, 2.0 ** -17 * top, 0.0) @ kk.nan_to_num(0.0).abs().T * abs(scale)
        d = 2.0 * (130 * 2.0 ** -24 * mass + 2.0 ** -22 * mass + lost.amax(-1, keepdim=True))
        part = (2 * 2.0 ** -8 + 2 * torch.expm1(d)) * a
        tol[:, h] = part + 2.0 ** -8 * (out[:, h].abs() + part) + 1e-30
    return out, tol
