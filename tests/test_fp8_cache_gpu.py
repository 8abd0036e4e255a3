"""The KV cache held in 8 bits on the GPU: rows written and read byte for byte, and the norm + rotation that writes them,
against the 64-bit oracle; copies of blocks.

Stored bytes have to be the oracle's exactly: quantisation works on bf16 values and powers of two, and the norm and
rotation run in 64 bits, where the odds that two orders of summation fall on two sides of a rounding border are some
2^-40 a value."""
from __future__ import annotations

import math

import pytest
import torch

from nano_vllm_ascend_amd import _C
from nano_vllm_ascend_amd.layers import RMSNorm, RotaryEmbedding, qk_norm_rope
from nano_vllm_ascend_amd.paged_kv_cache import Fp4PagedKVCache, Fp8PagedKVCache, PagedKVCache
from oracle import fp4_ref, fp8_ref

pytestmark = pytest.mark.gpu
EPS = 1e-6


@pytest.fixture(autouse=True)
def clean_word(device):
    _C.clear_index_errors()
    yield
    _C.clear_index_errors()
    torch.cuda.synchronize()


def rows(t, h, seed, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(t, h, 128, generator=gen)
    return (x * torch.exp(spread * torch.randn(t, h, 1, generator=gen))).bfloat16()


def filled(nb, hkv, bs, seed):
    """Pages of random bytes under scales of about one: what is not written has to stay as it was."""
    gen = torch.Generator().manual_seed(seed)
    pages = fp8_ref.empty_pages(nb, hkv, bs)
    return tuple(torch.randint(*((0, 256) if i % 2 == 0 else (115, 125)), p.shape, generator=gen, dtype=torch.uint8)
                 for i, p in enumerate(pages))


def on(device, pages):
    kc, ks, vc, vs = (p.to(device) for p in pages)
    return _C.Fp8Pages(kc, ks), _C.Fp8Pages(vc, vs)


def same(got, want):
    for name, a, b in zip(("key scales", "key codes", "value scales", "value codes"),
                          (got[0].scales, got[0].codes, got[1].scales, got[1].codes), (want[1], want[0], want[3], want[2])):
        a = a.cpu()
        if "codes" in name:  # 127 and 255 are NaN
            a, b = a.masked_fill(a == 255, 127), b.masked_fill(b == 255, 127)
        off = (a != b).nonzero().tolist()
        assert not off, f"{len(off)} {name} differ, the first at {off[:4]}"


def some_slots(t, nb, bs, order, seed):
    """Consecutive rows in pages of a seeded order, from a page's start or from inside a tile; or rows of sequences of a
    few tokens each, of which each begins somewhere in pages of its own."""
    gen = torch.Generator().manual_seed(seed)
    if order == "short":
        parts, at, page = [], 0, torch.randperm(nb, generator=gen)
        while at < t:
            n, start = (int(torch.randint(1, 20, (1,), generator=gen)), int(torch.randint(0, bs, (1,), generator=gen)))
            n = min(n, t - at, bs - start)
            parts.append(page[len(parts)] * bs + torch.arange(start, start + n))
            at += n
        return torch.cat(parts)
    start = {"page": 0, "odd": 5}[order]
    pages = torch.randperm(nb, generator=gen)
    at = torch.arange(start, start + t)
    return pages[at // bs] * bs + at % bs


SIZES = [(1, 8, 128), (1, 1, 16), (2, 3, 16), (11, 2, 32), (15, 8, 32), (16, 8, 128), (17, 5, 16), (33, 8, 64), (100, 1, 256),
         (257, 4, 128), (512, 1, 32), (513, 2, 64), (2049, 1, 64), (2100, 2, 16)]  # one row to a wave up to 512


@pytest.mark.parametrize("order", ["page", "odd", "short"])
@pytest.mark.parametrize("t, hkv, bs", SIZES)
def test_write_is_exact_and_touches_nothing_else(device, t, hkv, bs, order):
    nb = -(-(t + 5) // bs) + 2 if order != "short" else t + 1
    slots = some_slots(t, nb, bs, order, t)
    if t > 4:
        slots[[0, t - 1]] = -1  # padding rows (not between rows of one tile)
    k, v = rows(t, hkv, 1 + t), rows(t, hkv, 2 + t)
    pages = filled(nb, hkv, bs, t)
    got = on(device, pages)
    fp8_ref.write(pages, k, v, slots)
    _C.kv_cache_write_fp8(k.to(device), v.to(device), *got, slots.to(device))
    same(got, pages)
    back = _C.kv_cache_read_fp8(*got, slots.to(device))
    want = fp8_ref.read_sequence(pages, slots.clamp(min=0))
    for a, b in zip(back, want):
        assert torch.equal(a.cpu().double(), b.masked_fill((slots < 0)[:, None, None], 0.0))
    assert _C.index_errors() == 0


@pytest.mark.parametrize("first", [0, 3, 15, 16])
def test_a_tile_filled_row_by_row(device, first):
    """A decode loop's writes behind a prompt's: scales rise, what the tiles hold follows them."""
    hkv, bs, nb = 2, 32, 3
    pages = fp8_ref.empty_pages(nb, hkv, bs)
    got = on(device, pages)
    k, v = rows(60, hkv, first), rows(60, hkv, first + 1)
    grow = torch.pow(2.0, torch.arange(60) / 5.0 - 6)[:, None, None]
    k, v = (k * grow).bfloat16(), (v / grow).bfloat16()
    slots = torch.tensor([1, 2])[torch.arange(60) // bs] * bs + torch.arange(60) % bs
    at = 0
    for n in [first] + [1] * 20 + [5, 12]:
        rng = slice(at, at + n)
        fp8_ref.write(pages, k[rng], v[rng], slots[rng])
        _C.kv_cache_write_fp8(k[rng].to(device), v[rng].to(device), *got, slots[rng].to(device))
        at += n
        same(got, pages)
    raised = (pages[1] > 0).sum()
    assert raised == -(-at // 16) * hkv


@pytest.mark.parametrize("first", [0, 1])
def test_write_of_every_bf16_value(device, first):
    """Each of the 65,536 bit patterns, as the largest of its tile and beside a larger value that sets the scale; from a
    tile's first token on, and behind a row of its own."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).view(4096, 16)
    k = torch.zeros(4096, 16, 1, 128, dtype=torch.bfloat16)
    k[:, :, 0, 3] = bits
    v = torch.zeros(65536, 16, 1, 128, dtype=torch.bfloat16)[:4096]
    v[:, :, 0, 127] = bits
    v[:, :, 0, 2] = (bits.float().abs().nan_to_num(0.0, 0.0) * 2.7).clamp(max=3e38).bfloat16()
    slots = torch.arange(65536)
    pages = fp8_ref.empty_pages(512, 1, 128)
    got = on(device, pages)
    if first:
        head = slots.view(4096, 16)[:, 0]
        fp8_ref.write(pages, k[:, 3], v[:, 3], head)
        _C.kv_cache_write_fp8(k[:, 3].to(device), v[:, 3].to(device), *got, head.to(device))
    k, v, at = (x.reshape(4096, 16, *x.shape[2:])[:, first:].reshape(-1, *x.shape[2:])
                for x in (k, v, slots.view(4096, 16)))
    fp8_ref.write(pages, k, v, at)
    _C.kv_cache_write_fp8(k.to(device), v.to(device), *got, at.to(device))
    same(got, pages)
    for a, b in zip(_C.kv_cache_read_fp8(*got, slots.to(device)), fp8_ref.read_sequence(pages, slots)):
        assert torch.equal(a.cpu().double().nan_to_num(1e300), b.nan_to_num(1e300))


def test_an_infinity_or_a_nan_reads_as_nan_alone(device):
    k, v = rows(20, 2, 3), rows(20, 2, 4)
    k[3, 1, 70], k[5, 0, 0], v[7, 1, 127] = math.inf, math.nan, -math.inf
    cache = Fp8PagedKVCache(2, 4, 16, 2, 128, device)
    slots = torch.arange(20, device=device) + 3
    cache.write(1, k.to(device), v.to(device), slots)
    got_k, got_v = cache.read(1, slots)
    bad_k, bad_v = torch.zeros(20, 2, 128, dtype=torch.bool), torch.zeros(20, 2, 128, dtype=torch.bool)
    bad_k[3, 1, 70], bad_k[5, 0, 0], bad_v[7, 1, 127] = True, True, True
    assert torch.equal(got_k.isnan().cpu(), bad_k) and torch.equal(got_v.isnan().cpu(), bad_v)
    assert not cache.key_codes[0].any() and not cache.value_scales[0].any()  # the other layer
    cache.write(1, k[6:8].to(device) * 1000, v[8:10].to(device) * 1000, slots[-1] + torch.arange(1, 3, device=device))
    assert torch.equal(cache.read(1, slots)[0].isnan().cpu(), bad_k)  # still, under another scale


def test_views_and_strides(device):
    t, nb, bs = 40, 5, 16
    fused = rows(t, 8, 9).to(device)  # [T, 8, 128]: rows of a fused projection
    k, v = fused[:, 2:4], fused[:, 5:7]
    slots = some_slots(t, nb, bs, "odd", 1)
    pages = filled(nb, 2, bs, 7)
    got = on(device, pages)
    fp8_ref.write(pages, k.cpu(), v.cpu(), slots)
    _C.kv_cache_write_fp8(k, v, *got, slots.to(device))
    same(got, pages)
    wide = torch.full((t, 8, 128), 7.0, dtype=torch.bfloat16, device=device)
    order = torch.randperm(t, generator=torch.Generator().manual_seed(1))  # reading takes any order
    _C.kv_cache_read_fp8(*got, slots[order].to(device), k_out=wide[:, 1:3], v_out=wide[:, 4:6])
    want = fp8_ref.read(pages, slots[order])
    assert torch.equal(wide[:, 1:3].cpu().double(), want[0]) and torch.equal(wide[:, 4:6].cpu().double(), want[1])
    assert wide[:, [0, 3, 6, 7]].eq(7).all()


def test_empty_calls(device):
    got = on(device, filled(2, 2, 16, 0))
    none = torch.zeros(0, 2, 128, dtype=torch.bfloat16, device=device)
    slots = torch.zeros(0, dtype=torch.int64, device=device)
    _C.kv_cache_write_fp8(none, none, *got, slots)
    k, v = _C.kv_cache_read_fp8(*got, slots)
    assert k.shape == v.shape == (0, 2, 128)


@pytest.mark.parametrize("t", [8, 3000])
def test_slots_outside_the_cache_are_skipped_and_reported(device, t):
    k, v = rows(t, 2, 1), rows(t, 2, 2)
    slots = torch.full((t,), -1)
    slots[:8] = torch.tensor([3, 4, 64, 17, -1, -2, 1 << 40, 5])  # the cache has 64
    keep = torch.where((slots < 64) & (slots >= 0), slots, -1)
    keep[7] = slots[7] = 33
    pages = filled(4, 2, 16, 3)
    got = on(device, pages)
    fp8_ref.write(pages, k, v, keep)
    _C.kv_cache_write_fp8(k.to(device), v.to(device), *got, slots.to(device))
    assert _C.index_errors() == _C.ERR_SLOT
    same(got, pages)
    _C.clear_index_errors()
    for a, b in zip(_C.kv_cache_read_fp8(*got, slots.to(device)), fp8_ref.read(pages, keep)):
        assert torch.equal(a.cpu().double().nan_to_num(1e300), b.nan_to_num(1e300))
    assert _C.index_errors() == _C.ERR_SLOT
    _C.clear_index_errors()
    previous = _C.set_range_checks(True)
    try:
        with pytest.raises(IndexError):
            _C.kv_cache_write_fp8(k.to(device), v.to(device), *got, slots.to(device))
        with pytest.raises(IndexError, match="tile of 16"):
            _C.kv_cache_write_fp8(k[:3].to(device), v[:3].to(device), *got, torch.tensor([4, 3, 9], device=device))
    finally:
        _C.set_range_checks(previous)


def table_of(positions):
    freqs = torch.outer(torch.arange(positions, dtype=torch.float32),
                        1.0 / 1e6 ** (torch.arange(0, 128, 2, dtype=torch.float32) / 128))
    return torch.cat((freqs.cos(), freqs.sin()), 1).contiguous()


@pytest.mark.parametrize("keys", [False, True])
@pytest.mark.parametrize("t, hq, hkv, bs, order", [(1, 16, 8, 128, "page"), (1, 1, 1, 16, "odd"), (7, 16, 8, 16, "short"),
                                                   (33, 40, 8, 64, "odd"), (130, 16, 8, 128, "page"),
                                                   (300, 2, 1, 32, "odd"), (65, 24, 3, 256, "short"),
                                                   (2060, 9, 2, 128, "odd"), (2049, 3, 1, 16, "page"),
                                                   (512, 9, 5, 32, "odd"), (513, 17, 5, 32, "short")])
def test_norm_rope_stores_the_code_of_the_exact_key(device, t, hq, hkv, bs, order, keys):
    nb, table = (-(-(t + 5) // bs) + 1 if order != "short" else t), table_of(40960)
    gen = torch.Generator().manual_seed(t)
    qkv = rows(t, hq + 2 * hkv, t, spread=0.3)
    qw, kw = ((1 + 0.1 * torch.randn(128, generator=gen)).bfloat16() for _ in range(2))
    pos = torch.randint(0, 40960, (t,), generator=gen)
    slots = some_slots(t, nb, bs, order, t)
    if t > 4:
        slots[[0, t - 1]] = -1
    q, k, v = qkv.split([hq, hkv, hkv], 1)
    want_q, want_k = (fp4_ref.to_bf16(fp4_ref.norm_rope(x, w, pos, table, EPS)) for x, w in ((q, qw), (k, kw)))
    pages = filled(nb, hkv, bs, t)
    got = on(device, pages)
    fp8_ref.write(pages, want_k, v, slots)
    dq, dk, dv = qkv.to(device).split([hq, hkv, hkv], 1)
    before = dk.clone()
    k_out = torch.empty(t, hkv, 128, dtype=torch.bfloat16, device=device) if keys else None
    q_out = _C.qk_norm_rope_fp8(dq, dk, dv, qw.to(device), kw.to(device), pos.to(device), table.to(device), EPS, *got,
                                slots.to(device), k_out=k_out)
    same(got, pages)
    assert torch.equal(q_out.cpu(), want_q) and torch.equal(dq.cpu(), q) and torch.equal(dk, before)
    if keys:
        assert torch.equal(k_out.cpu(), want_k)  # padding rows too
    assert _C.index_errors() == 0


def spread_out(gen, *shape, low, high):
    """Normal numbers times powers of two of exponents low .. high, within bf16's largest."""
    e = torch.randint(low, high + 1, shape[:-1] + (1,), generator=gen).double()
    return (torch.randn(*shape, generator=gen).double() * torch.pow(2.0, e)).clamp(-3.38e38, 3.38e38).bfloat16()


@pytest.mark.parametrize("low, high, weight_low, weight_high, eps", [
    (118, 126, 8, 8, 1e-6), (-120, 126, -60, 60, 1e-6), (-133, 126, -100, 100, 2e-38)])
def test_norm_rope_over_the_whole_range_of_bf16(device, low, high, weight_low, weight_high, eps):
    t, hq, hkv, bs, table = 200, 4, 2, 32, table_of(4096)
    gen = torch.Generator().manual_seed(high - low)
    qkv = spread_out(gen, t, hq + 2 * hkv, 128, low=low, high=high)
    qw, kw = (spread_out(gen, 128, 1, low=weight_low, high=weight_high)[:, 0].contiguous() for _ in range(2))
    pos, slots = torch.randint(0, 4096, (t,), generator=gen), some_slots(t, 8, bs, "odd", 1)
    q, k, v = qkv.split([hq, hkv, hkv], 1)
    want_q, want_k = (fp4_ref.to_bf16(fp4_ref.norm_rope(x, w, pos, table, eps)) for x, w in ((q, qw), (k, kw)))
    pages = filled(8, hkv, bs, 2)
    got = on(device, pages)
    fp8_ref.write(pages, want_k, v, slots)
    dq, dk, dv = qkv.to(device).split([hq, hkv, hkv], 1)
    k_out = torch.empty(t, hkv, 128, dtype=torch.bfloat16, device=device)
    q_out = _C.qk_norm_rope_fp8(dq, dk, dv, qw.to(device), kw.to(device), pos.to(device), table.to(device), eps, *got,
                                slots.to(device), k_out=k_out)
    assert torch.equal(q_out.cpu(), want_q) and torch.equal(k_out.cpu(), want_k)
    same(got, pages)


@pytest.mark.parametrize("t", [50, 2100])
def test_norm_rope_in_place_through_the_layer_equals_the_two_steps(device, t):
    """qk_norm_rope with an 8-bit cache rewrites q and k, as with a bf16 one; what it stored is what a write of that k
    stores."""
    hq, hkv = 16, 8
    cache, twin = (Fp8PagedKVCache(2, t // 16 + 3, 16, hkv, 128, device) for _ in range(2))
    norms = [RMSNorm(128, EPS).to(device, torch.bfloat16) for _ in range(2)]
    for m, seed in zip(norms, (1, 2)):
        m.weight.data = (1 + 0.1 * torch.randn(128, generator=torch.Generator().manual_seed(seed))).bfloat16().to(device)
    rotary = RotaryEmbedding(128, 4096, 1e6).to(device)
    qkv = rows(t, hq + 2 * hkv, 5, spread=0.3).to(device)
    q, k, v = qkv.split([hq, hkv, hkv], 1)
    raw_v, pos = v.clone(), torch.arange(t, device=device) + 7
    want_q = fp4_ref.norm_rope(q.cpu(), norms[0].weight.cpu(), pos.cpu(), rotary.cos_sin.cpu(), EPS)
    slots = torch.arange(t, device=device) + 9
    qk_norm_rope(q, k, v, *norms, rotary, pos, cache, 1, slots)
    assert torch.equal(q.cpu(), fp4_ref.to_bf16(want_q)) and torch.equal(v, raw_v)
    twin.write(1, k, v, slots)
    for name in ("key_codes", "key_scales", "value_codes", "value_scales"):
        assert torch.equal(getattr(cache, name), getattr(twin, name))


@pytest.mark.parametrize("t", [4, 2052])
def test_norm_rope_reports_positions_and_slots(device, t):
    q, k, v = (rows(t, h, h).to(device) for h in (2, 1, 1))
    w = torch.ones(128, dtype=torch.bfloat16, device=device)
    table = table_of(64)
    got = on(device, filled(2, 1, 16, 1))
    pos, slots = torch.zeros(t, dtype=torch.int64), torch.full((t,), -1)
    pos[:4], slots[:4] = torch.tensor([0, 63, 64, -1]), torch.arange(4)
    out = _C.qk_norm_rope_fp8(q, k, v, w, w, pos.to(device), table.to(device), EPS, *got, slots.to(device))
    assert _C.index_errors() == _C.ERR_POSITION
    want = fp4_ref.norm_rope(q.cpu(), w.cpu(), pos.clamp(0, 63), table, EPS)  # clamped to the table
    assert torch.equal(out.cpu(), fp4_ref.to_bf16(want))
    _C.clear_index_errors()
    slots[:4] = torch.tensor([0, 1, 32, -1])
    _C.qk_norm_rope_fp8(q, k, v, w, w, pos.clamp(0, 63).to(device), table.to(device), EPS, *got, slots.to(device))
    assert _C.index_errors() == _C.ERR_SLOT


def test_calls_go_to_the_current_stream_and_replay_from_a_graph(device):
    t, hq, hkv, bs, nb = 9, 4, 2, 16, 4
    table, w = table_of(256).to(device), torch.ones(128, dtype=torch.bfloat16, device=device)
    qkv, pos = rows(t, hq + 2 * hkv, 1).to(device), torch.arange(t, device=device)
    slots = (torch.arange(t) + 3).to(device)
    q, k, v = qkv.split([hq, hkv, hkv], 1)
    got, want = on(device, filled(nb, hkv, bs, 1)), on(device, filled(nb, hkv, bs, 1))
    q_out, k_back, v_back = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)

    def step(pages, out):
        _C.qk_norm_rope_fp8(q, k, v, w, w, pos, table, EPS, *pages, slots, q_out=out)
        return _C.kv_cache_read_fp8(*pages, slots, k_out=k_back, v_out=v_back)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(got, q_out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(got, q_out)
    step(want, torch.empty_like(q))
    for seed in (2, 3, 4):
        qkv.copy_(rows(t, hq + 2 * hkv, seed))
        slots.copy_(torch.arange(t) + 5 * seed)
        graph.replay()
        replayed = q_out.clone(), k_back.clone(), v_back.clone()
        torch.cuda.synchronize()
        eager = torch.empty_like(q)
        step(want, eager)
        assert torch.equal(replayed[0], eager)
        assert torch.equal(replayed[1], k_back) and torch.equal(replayed[2], v_back)
        want_k, want_v = fp8_ref.read(tuple(p.cpu() for p in (*want[0], *want[1])), slots.cpu())
        assert torch.equal(k_back.cpu().double(), want_k) and torch.equal(v_back.cpu().double(), want_v)


# -------------------------------------------------------------------------------------------- copies of blocks
def random_bytes(t, seed):
    view = t.view(torch.uint8) if t.dtype is not torch.uint8 else t
    view.random_(0, 256, generator=torch.Generator(device=t.device).manual_seed(seed))


def cache_of(kind, device, layers=3, blocks=9, bs=32, hkv=2):
    sizes = layers, blocks, bs, hkv, 128
    if kind == "bf16":
        cache = PagedKVCache(*sizes, torch.bfloat16, device)
        return cache, [cache.key_cache, cache.value_cache]
    cache = (Fp4PagedKVCache if kind == "fp4" else Fp8PagedKVCache)(*sizes, device)
    return cache, [cache.key_codes, cache.key_scales, cache.value_codes, cache.value_scales]


@pytest.mark.parametrize("sizes", [dict(), dict(layers=1, blocks=2, bs=16, hkv=1), dict(bs=256, hkv=8), dict(hkv=3, bs=16)])
@pytest.mark.parametrize("kind", ["bf16", "fp4", "fp8"])
def test_copy_blocks_copies_every_layer_and_nothing_else(device, kind, sizes):
    cache, pools = cache_of(kind, device, **sizes)
    for i, p in enumerate(pools):
        random_bytes(p, i)
    n = cache.num_blocks
    src, dst = ([0], [n - 1]) if n < 9 else ([3, 7, 0, 5], [8, 1, 2, 5])  # one to itself
    want = [p.clone() for p in pools]
    for w in want:
        w.view(torch.uint8)[:, dst] = w.view(torch.uint8)[:, src].clone()
    cache.copy_blocks(src, dst)
    assert all(torch.equal(p.view(torch.uint8), w.view(torch.uint8)) for p, w in zip(pools, want))
    for w in want:
        w.view(torch.uint8)[:, [dst[0]]] = w.view(torch.uint8)[:, [n // 2]]
    cache.copy_blocks(torch.tensor([n // 2], dtype=torch.int32, device=device),
                      torch.tensor([dst[0]], dtype=torch.int32, device=device))
    assert all(torch.equal(p.view(torch.uint8), w.view(torch.uint8)) for p, w in zip(pools, want))
    cache.copy_blocks([], [])
    assert _C.index_errors() == 0


@pytest.mark.parametrize("width", [1, 5, 16, 24, 4096, 16384, 16400, 40_000, 50_001])
def test_copy_blocks_of_odd_sizes(device, width):
    pools = [torch.empty(2, 7, width, dtype=torch.uint8, device=device), torch.empty(2, 7, 3, 2, device=device)]
    if width % 16 == 0:  # a pool that begins beside 16 bytes
        base = torch.empty(2 * 7 * width + 8, dtype=torch.uint8, device=device)
        pools.append(base[8:].view(2, 7, width))
    for i, p in enumerate(pools):
        random_bytes(p, i)
    want = [p.clone() for p in pools]
    for w in want:
        w[:, [2, 3]] = w[:, [6, 0]]
    _C.copy_blocks(pools, *(torch.tensor(x, dtype=torch.int32, device=device) for x in ([6, 0], [2, 3])))
    assert all(torch.equal(p.view(torch.uint8), w.view(torch.uint8)) for p, w in zip(pools, want))


def test_copy_blocks_skips_and_reports_blocks_outside_the_pool(device):
    pool = torch.empty(2, 5, 64, dtype=torch.uint8, device=device)
    random_bytes(pool, 1)
    want = pool.clone()
    want[:, 4] = want[:, 1]
    src = torch.tensor([5, 1, -1, 0], dtype=torch.int32, device=device)
    dst = torch.tensor([0, 4, 2, 1 << 30], dtype=torch.int32, device=device)
    _C.copy_blocks([pool], src, dst)
    assert _C.index_errors() == _C.ERR_BLOCK and torch.equal(pool, want)
    _C.clear_index_errors()
    before = _C.set_range_checks(True)
    try:
        with pytest.raises(IndexError, match="outside"):
            _C.copy_blocks([pool], src, dst)
        with pytest.raises(IndexError, match="twice"):
            _C.copy_blocks([pool], src[1:2].expand(2).contiguous(), dst[1:2].expand(2).contiguous())
    finally:
        _C.set_range_checks(before)
    assert torch.equal(pool, want)


def test_copy_blocks_past_32_bits(device):
    """A pool of 6 GB whose blocks lie past 4 GiB, and blocks of 1 GiB."""
    pool = torch.empty(1, 6, 1 << 30, dtype=torch.uint8, device=device)
    for b in (1, 5):
        random_bytes(pool[0, b], b)
    _C.copy_blocks([pool], *(torch.tensor([b], dtype=torch.int32, device=device) for b in (5, 0)))
    _C.copy_blocks([pool], *(torch.tensor([b], dtype=torch.int32, device=device) for b in (1, 4)))
    assert torch.equal(pool[0, 0], pool[0, 5]) and torch.equal(pool[0, 4], pool[0, 1])


def test_copy_blocks_replays_from_a_graph_and_follows_the_stream(device):
    cache, pools = cache_of("fp8", device)
    for i, p in enumerate(pools):
        random_bytes(p, i)
    src, dst = (torch.zeros(2, dtype=torch.int32, device=device) for _ in range(2))
    cache.copy_blocks(src, dst)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.copy_blocks(src, dst)
    for a, b in (([0, 1], [2, 3]), ([3, 8], [4, 0]), ([5, 5], [5, 6])):
        want = [p.clone() for p in pools]
        for w in want:
            w[:, b] = w[:, a].clone()
        src.copy_(torch.tensor(a, dtype=torch.int32))
        dst.copy_(torch.tensor(b, dtype=torch.int32))
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, w) for p, w in zip(pools, want))


def test_copies_are_made_at_once_only_if_they_are_plain(device, monkeypatch):
    """csrc/calls.cpp leaves what _C.py refuses to it; without it the same copies are made from Python."""
    pools = [torch.empty(2, 6, 40, dtype=torch.uint8, device=device), torch.empty(2, 6, 3, 2, device=device)]
    ids = torch.arange(3, dtype=torch.int32, device=device)
    for bad in (([], ids, ids), (pools * 5, ids, ids), ([pools[0].cpu()], ids, ids), ([pools[0][:, :5]], ids, ids),
                ([pools[0], pools[1][:1]], ids, ids), ([pools[0][0]], ids, ids), (pools, ids.long(), ids),
                (pools, ids, ids[:2]), (pools, ids.cpu(), ids), (pools, ids, ids.repeat_interleave(2)[::2])):
        assert _C._calls.copy(*bad) is None
        with pytest.raises(ValueError):
            _C.copy_blocks(*bad)
    results = []
    for at_once in (True, False):
        if not at_once:
            monkeypatch.setattr(_C, "_calls", None)
        for i, p in enumerate(pools):
            random_bytes(p, i)
        _C.copy_blocks(iter(pools) if not at_once else tuple(pools), ids, ids + 3)
        results.append([p.clone() for p in pools])
    assert all(torch.equal(a, b) for a, b in zip(*results)) and torch.equal(results[0][0][:, :3], results[0][0][:, 3:])
