"""The KV cache held in 4 bits on the GPU: rows written and read byte for byte, and the norm + rotation that writes them,
against the 64-bit oracle.

Stored bytes have to be the oracle's exactly: quantisation works on bf16 values and powers of two, and the norm and
rotation run in 64 bits, where the odds that two orders of summation fall on two sides of a rounding border are some
2^-40 a value."""
from __future__ import annotations

import math

import pytest
import torch

from nano_vllm_ascend_amd import _C
from nano_vllm_ascend_amd.layers import RMSNorm, RotaryEmbedding, qk_norm_rope
from nano_vllm_ascend_amd.paged_kv_cache import Fp4PagedKVCache
from oracle import fp4_ref

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
    return (x * torch.exp(spread * torch.randn(t, h, 4, generator=gen)).repeat_interleave(32, -1)).bfloat16()


def filled(nb, hkv, bs, seed):
    """Pages of random bytes: what is not written has to stay as it was."""
    gen = torch.Generator().manual_seed(seed)
    return tuple(torch.randint(0, 256, (nb, hkv, bs, w), generator=gen, dtype=torch.uint8) for w in (64, 4, 64, 4))


def on(device, pages):
    kc, ks, vc, vs = (p.to(device) for p in pages)
    return _C.Fp4Pages(kc, ks), _C.Fp4Pages(vc, vs)


def same(got, want):
    for name, a, b in zip(("key codes", "key scales", "value codes", "value scales"), (*got[0], *got[1]), want):
        off = (a.cpu() != b).nonzero().tolist()
        assert not off, f"{len(off)} {name} differ, the first at {off[:4]}"


def some_slots(t, nb, bs, order, seed):
    gen = torch.Generator().manual_seed(seed)
    if order == "shuffled":
        return torch.randperm(nb * bs, generator=gen)[:t]
    start = {"page": 0, "odd": 5}[order]  # consecutive rows, from a page's start or from inside a tile
    pages = torch.randperm(nb, generator=gen)
    at = torch.arange(start, start + t)
    return pages[at // bs] * bs + at % bs


@pytest.mark.parametrize("order", ["page", "odd", "shuffled"])
@pytest.mark.parametrize("t, hkv, bs", [(1, 8, 128), (1, 1, 16), (2, 3, 16), (15, 8, 32), (16, 8, 128), (17, 5, 16),
                                        (33, 8, 64), (100, 1, 256), (257, 8, 128), (1000, 2, 16)])
def test_write_is_exact_and_touches_nothing_else(device, t, hkv, bs, order):
    nb = -(-(t + 5) // bs) + 2
    slots = some_slots(t, nb, bs, order, t)
    if t > 4:
        slots[[1, t // 2]] = -1  # padding rows
    k, v = rows(t, hkv, 1 + t), rows(t, hkv, 2 + t)
    pages = filled(nb, hkv, bs, t)
    got = on(device, pages)
    fp4_ref.write(pages, k, v, slots)
    _C.kv_cache_write_fp4(k.to(device), v.to(device), *got, slots.to(device))
    same(got, pages)
    back = _C.kv_cache_read_fp4(*got, slots.to(device))
    for a, b in zip(back, fp4_ref.read(pages, slots)):
        assert torch.equal(a.cpu().double(), b)
    assert _C.index_errors() == 0


def test_write_of_every_bf16_value(device):
    """Each of the 65,536 bit patterns, among zeros and beside a larger value that sets the scale."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    k = torch.zeros(65536, 1, 128, dtype=torch.bfloat16)
    k[:, 0, 3] = bits
    k[:, 0, 32 + 17] = bits
    k[:, 0, 32 + 2] = (bits.float().abs() * 2.7).clamp(max=3e38).bfloat16()
    k[:, 0, 64] = bits
    k[:, 0, 65] = 4.0
    v = k.flip(-1).contiguous()
    slots = torch.arange(65536)
    pages = fp4_ref.empty_pages(512, 1, 128)
    got = on(device, pages)
    fp4_ref.write(pages, k, v, slots)
    _C.kv_cache_write_fp4(k.to(device), v.to(device), *got, slots.to(device))
    same(got, pages)
    for a, b in zip(_C.kv_cache_read_fp4(*got, slots.to(device)), fp4_ref.read(pages, slots)):
        assert torch.equal(a.cpu().double().nan_to_num(1e300), b.nan_to_num(1e300))


def test_a_block_with_an_infinity_or_a_nan_reads_as_nan(device):
    k = rows(20, 2, 3)
    k[3, 1, 70], k[5, 0, 0], v = math.inf, math.nan, rows(20, 2, 4)
    v[7, 1, 127] = -math.inf
    cache = Fp4PagedKVCache(2, 4, 16, 2, 128, device)
    slots = torch.arange(20, device=device) + 3
    cache.write(1, k.to(device), v.to(device), slots)
    got_k, got_v = cache.read(1, slots)
    bad_k, bad_v = torch.zeros(20, 2, 128, dtype=torch.bool), torch.zeros(20, 2, 128, dtype=torch.bool)
    bad_k[3, 1, 64:96], bad_k[5, 0, :32], bad_v[7, 1, 96:] = True, True, True
    assert torch.equal(got_k.isnan().cpu(), bad_k) and torch.equal(got_v.isnan().cpu(), bad_v)
    assert not cache.key_codes[0].any() and not cache.value_scales[0].any()  # the other layer


def test_views_and_strides(device):
    t, nb, bs = 40, 5, 16
    fused = rows(t, 8, 9).to(device)  # [T, 8, 128]: rows of a fused projection
    k, v = fused[:, 2:4], fused[:, 5:7]
    slots = some_slots(t, nb, bs, "odd", 1)
    pages = filled(nb, 2, bs, 7)
    got = on(device, pages)
    fp4_ref.write(pages, k.cpu(), v.cpu(), slots)
    _C.kv_cache_write_fp4(k, v, *got, slots.to(device))
    same(got, pages)
    wide = torch.full((t, 8, 128), 7.0, dtype=torch.bfloat16, device=device)
    _C.kv_cache_read_fp4(*got, slots.to(device), k_out=wide[:, 1:3], v_out=wide[:, 4:6])
    want = fp4_ref.read(pages, slots)
    assert torch.equal(wide[:, 1:3].cpu().double(), want[0]) and torch.equal(wide[:, 4:6].cpu().double(), want[1])
    assert wide[:, [0, 3, 6, 7]].eq(7).all()


def test_empty_calls(device):
    got = on(device, filled(2, 2, 16, 0))
    none = torch.zeros(0, 2, 128, dtype=torch.bfloat16, device=device)
    slots = torch.zeros(0, dtype=torch.int64, device=device)
    _C.kv_cache_write_fp4(none, none, *got, slots)
    k, v = _C.kv_cache_read_fp4(*got, slots)
    assert k.shape == v.shape == (0, 2, 128)


def test_slots_outside_the_cache_are_skipped_and_reported(device):
    k, v = rows(6, 2, 1), rows(6, 2, 2)
    slots = torch.tensor([3, 64, 17, -1, -2, 1 << 40])  # the cache has 64
    keep = torch.where((slots < 64) & (slots >= 0), slots, -1)
    pages = filled(4, 2, 16, 3)
    got = on(device, pages)
    fp4_ref.write(pages, k, v, keep)
    _C.kv_cache_write_fp4(k.to(device), v.to(device), *got, slots.to(device))
    assert _C.index_errors() == _C.ERR_SLOT
    same(got, pages)
    _C.clear_index_errors()
    for a, b in zip(_C.kv_cache_read_fp4(*got, slots.to(device)), fp4_ref.read(pages, keep)):
        assert torch.equal(a.cpu().double().nan_to_num(1e300), b.nan_to_num(1e300))
    assert _C.index_errors() == _C.ERR_SLOT
    _C.clear_index_errors()
    previous = _C.set_range_checks(True)
    try:
        with pytest.raises(IndexError):
            _C.kv_cache_write_fp4(k.to(device), v.to(device), *got, slots.to(device))
    finally:
        _C.set_range_checks(previous)


def table_of(positions):
    freqs = torch.outer(torch.arange(positions, dtype=torch.float32),
                        1.0 / 1e6 ** (torch.arange(0, 128, 2, dtype=torch.float32) / 128))
    return torch.cat((freqs.cos(), freqs.sin()), 1).contiguous()


@pytest.mark.parametrize("keys", [False, True])
@pytest.mark.parametrize("t, hq, hkv, bs, order", [(1, 16, 8, 128, "page"), (1, 1, 1, 16, "odd"), (7, 16, 8, 16, "shuffled"),
                                                   (33, 40, 8, 64, "odd"), (130, 16, 8, 128, "page"),
                                                   (300, 2, 1, 32, "odd"), (65, 24, 3, 256, "shuffled")])
def test_norm_rope_stores_the_code_of_the_exact_key(device, t, hq, hkv, bs, order, keys):
    nb, table = -(-(t + 5) // bs) + 1, table_of(40960)
    gen = torch.Generator().manual_seed(t)
    qkv = rows(t, hq + 2 * hkv, t, spread=0.3)
    qw, kw = ((1 + 0.1 * torch.randn(128, generator=gen)).bfloat16() for _ in range(2))
    pos = torch.randint(0, 40960, (t,), generator=gen)
    slots = some_slots(t, nb, bs, order, t)
    if t > 4:
        slots[2] = -1
    q, k, v = qkv.split([hq, hkv, hkv], 1)
    want_q, want_k = (fp4_ref.to_bf16(fp4_ref.norm_rope(x, w, pos, table, EPS)) for x, w in ((q, qw), (k, kw)))
    pages = filled(nb, hkv, bs, t)
    got = on(device, pages)
    fp4_ref.write(pages, want_k, v, slots)
    dq, dk, dv = qkv.to(device).split([hq, hkv, hkv], 1)
    before = dk.clone()
    k_out = torch.empty(t, hkv, 128, dtype=torch.bfloat16, device=device) if keys else None
    q_out = _C.qk_norm_rope_fp4(dq, dk, dv, qw.to(device), kw.to(device), pos.to(device), table.to(device), EPS, *got,
                                slots.to(device), k_out=k_out)
    same(got, pages)
    assert torch.equal(q_out.cpu(), want_q) and torch.equal(dq.cpu(), q) and torch.equal(dk, before)
    if keys:
        assert torch.equal(k_out.cpu(), want_k)
    assert _C.index_errors() == 0


def spread_out(gen, *shape, low, high):
    """Normal numbers times powers of two of exponents low .. high, within bf16's largest."""
    e = torch.randint(low, high + 1, shape[:-1] + (1,), generator=gen).double()
    return (torch.randn(*shape, generator=gen).double() * torch.pow(2.0, e)).clamp(-3.38e38, 3.38e38).bfloat16()


@pytest.mark.parametrize("low, high, weight_low, weight_high, eps", [
    (118, 126, 8, 8, 1e-6),         # x w is past 32 bits' largest, the normed value is not
    (-120, 126, -60, 60, 1e-6),
    (-104, -90, -50, -36, 2e-38),   # x w is below their least normal one
    (-133, 126, -100, 100, 2e-38),  # results past bf16's largest, and below its least, among them
])
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
    fp4_ref.write(pages, want_k, v, slots)
    dq, dk, dv = qkv.to(device).split([hq, hkv, hkv], 1)
    k_out = torch.empty(t, hkv, 128, dtype=torch.bfloat16, device=device)
    q_out = _C.qk_norm_rope_fp4(dq, dk, dv, qw.to(device), kw.to(device), pos.to(device), table.to(device), eps, *got,
                                slots.to(device), k_out=k_out)
    assert torch.equal(q_out.cpu(), want_q) and torch.equal(k_out.cpu(), want_k)
    same(got, pages)


def test_norm_rope_in_place_through_the_layer_equals_the_two_steps(device):
    """qk_norm_rope with a 4-bit cache rewrites q and k, as with a bf16 one; what it stored is what a write of that k stores."""
    t, hq, hkv = 50, 16, 8
    cache, twin = (Fp4PagedKVCache(2, 6, 16, hkv, 128, device) for _ in range(2))
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


def test_norm_rope_reports_positions_and_slots(device):
    q, k, v = (rows(4, h, h).to(device) for h in (2, 1, 1))
    w = torch.ones(128, dtype=torch.bfloat16, device=device)
    table = table_of(64)
    got = on(device, filled(2, 1, 16, 1))
    pos = torch.tensor([0, 63, 64, -1])
    out = _C.qk_norm_rope_fp4(q, k, v, w, w, pos.to(device), table.to(device), EPS, *got,
                              torch.tensor([0, 1, 2, 3], device=device))
    assert _C.index_errors() == _C.ERR_POSITION
    want = fp4_ref.norm_rope(q.cpu(), w.cpu(), pos.clamp(0, 63), table, EPS)  # clamped to the table
    assert torch.equal(out.cpu(), fp4_ref.to_bf16(want))
    _C.clear_index_errors()
    _C.qk_norm_rope_fp4(q, k, v, w, w, pos.clamp(0, 63).to(device), table.to(device), EPS, *got,
                        torch.tensor([0, 1, 32, -1], device=device))
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
        _C.qk_norm_rope_fp4(q, k, v, w, w, pos, table, EPS, *pages, slots, q_out=out)
        return _C.kv_cache_read_fp4(*pages, slots, k_out=k_back, v_out=v_back)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(got, q_out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(got, q_out)
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
        want_k, want_v = fp4_ref.read(tuple(p.cpu() for p in (*want[0], *want[1])), slots.cpu())
        assert torch.equal(k_back.cpu().double(), want_k) and torch.equal(v_back.cpu().double(), want_v)


@pytest.mark.parametrize("checks", [False, True])
def test_no_memory_raises_as_torch_does(device, checks):
    """Results of 2 x 4 GiB under a limit on torch's allocator of about 1 GiB: the allocation fails, nothing is launched."""
    got = on(device, filled(2, 8, 16, 0))
    slots = torch.zeros(1 << 21, dtype=torch.int64, device=device)
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(device).total_memory
    before = _C.set_range_checks(checks)
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (1 << 30)) / total)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            _C.kv_cache_read_fp4(*got, slots)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
        _C.set_range_checks(before)
