"""CPU checks of the KV cache held in 4 bits: the oracle against the format's definition by hand, the argument checks
of the C ABI and the refusals of the Python entry points."""
from __future__ import annotations

import importlib
import math
import subprocess
import sys
import warnings

import pytest
import torch

from nano_vllm_ascend_amd import _C, build
from nano_vllm_ascend_amd.paged_kv_cache import Fp4PagedKVCache
from oracle import fp4_ref

EINVAL, EUNSUPPORTED, EWORKSPACE = -1, -2, -3
A = 0x10000  # aligned stand-in address: no failing call dereferences it


def row(*head, fill=0.0):
    x = torch.full((128,), fill, dtype=torch.bfloat16)
    x[:len(head)] = torch.tensor(head, dtype=torch.float64).bfloat16()
    return x


# -------------------------------------------------------------------------------------------- the format
def test_scale_is_the_least_power_that_seven_steps_of_reach_the_maximum():
    for top, byte in ((7.0, 127), (7.03125, 128), (6.0, 127), (3.5, 126), (3.515625, 127), (1.0, 125), (1.75, 125),
                      (1.7578125, 126), (2.0 ** -130, 2), (0.0, 2), (2.0 ** 127, 252), (3.3e38, 252)):
        codes, scales = fp4_ref.quantise(row(top))
        assert scales.tolist() == [byte, 2, 2, 2], top
        step = 2.0 ** (byte - 127)
        if 2 < byte < 252:
            assert top <= 7 * step and top > 7 * step / 2


def test_codes_round_to_nearest_with_ties_to_the_even_code():
    x = row(0.24, 0.25, 0.26, 0.74, 0.75, 1.25, 1.26, 1.75, 2.5, 2.53, 3.5, 5.0, 5.03, 7.0, -0.25, -0.75, -5.0, -7.0)
    codes, scales = fp4_ref.quantise(x)
    assert scales[0] == 127
    assert codes[:18].tolist() == [0, 0, 1, 1, 2, 2, 3, 4, 4, 5, 6, 6, 7, 7, 8, 10, 14, 15]
    got = fp4_ref.values(codes, scales)
    assert got[:13].tolist() == [0, 0, .5, .5, 1, 1, 1.5, 2, 2, 3, 4, 4, 6]


def test_a_block_with_an_infinity_or_a_nan_reads_as_nan_alone():
    x = row(*[1.0] * 128)
    x[40], x[100] = math.inf, math.nan
    codes, scales = fp4_ref.quantise(x)
    assert scales.tolist() == [125, 255, 125, 255]
    got = fp4_ref.values(codes, scales)
    assert got[:32].eq(1).all() and got[32:64].isnan().all() and got[64:96].eq(1).all() and got[96:].isnan().all()


def test_no_value_is_off_by_more_than_a_step():
    gen = torch.Generator().manual_seed(1)
    x = (torch.randn(500, 128, generator=gen) * torch.exp(3 * torch.randn(500, 1, generator=gen))).bfloat16()
    codes, scales = fp4_ref.quantise(x)
    step = torch.pow(2.0, scales.double() - 127).repeat_interleave(32, -1)
    off = (fp4_ref.values(codes, scales) - x.double()).abs() / step
    assert off.max() <= 1.0                                        # 4 .. 7 round to 4 or 6
    assert off[(x.double().abs() <= 4 * step)].max() <= 0.5        # 2 .. 4: half of the unit between them
    assert off[(x.double().abs() <= 2 * step)].max() <= 0.25


def test_values_round_to_bf16_once():
    x = torch.tensor([1.00390625, 1.00390625 + 1e-12, 1.01171875, 1.01171875 - 1e-12, -1.00390625 - 1e-12, 0.0, 0.5],
                     dtype=torch.float64)
    assert fp4_ref.to_bf16(x).tolist() == [1.0, 1.0078125, 1.015625, 1.0078125, -1.0078125, 0.0, 0.5]


def test_pages_hold_rows_where_the_layout_says():
    pages = fp4_ref.empty_pages(3, 2, 32)
    k, v = row(*[6.0, -1.0]), row(*[0.0] * 17, 6.0)
    both = torch.zeros(1, 2, 128, dtype=torch.bfloat16)
    ks, vs = both.clone(), both.clone()
    ks[0, 1], vs[0, 1] = k, v
    slot = 2 * 32 + 16 + 5  # page 2, tile 1, token 5 of the tile
    fp4_ref.write(pages, ks, vs, torch.tensor([slot]))
    page = (2 * 2 + 1) * 32  # rows before head 1 of page 2
    assert pages[0].view(-1)[64 * (page + 21)] == 7 | (10 << 4)
    assert pages[1].view(-1)[4 * (page + 16) + 16 * (5 % 4) + 4 * 0 + 5 // 4] == 127
    assert pages[2].view(-1)[64 * (page + 16) + 16 * 1 + 5] == 7 << 4  # dim 17 = 16 + r of block 0, r = 1
    assert pages[3].view(-1)[4 * (page + 16) + 5] == 127
    got_k, got_v = fp4_ref.read(pages, torch.tensor([slot, -1]))
    assert torch.equal(got_k[0, 1], k.double()) and torch.equal(got_v[0, 1], v.double())
    assert not got_k[1].any() and not got_v[1].any()


# -------------------------------------------------------------------------------------------- the C ABI
CACHE = dict(kc=A, ks=A, vc=A, vs=A, nb=64, bs=128)


def test_write_and_read_argument_errors():
    lib = _C.load()
    for fn in (lib.nvamd_kv_cache_write_fp4, lib.nvamd_kv_cache_read_fp4):
        def call(**over):
            args = dict(k=A, k_stride=1024, v=A, v_stride=1024, **CACHE, slots=A, t=4, hkv=8, d=128, stream=None)
            args.update(over)
            return fn(*args.values())

        assert call(t=0) == 0
        assert call(t=-1) == EINVAL and call(nb=0) == EINVAL and call(hkv=0) == EINVAL
        assert call(d=64) == EUNSUPPORTED and call(bs=8) == EUNSUPPORTED and call(bs=48) == EUNSUPPORTED
        for name in ("k", "v", "kc", "ks", "vc", "vs"):
            assert call(**{name: 0}) == EINVAL and call(**{name: A + 8}) == EINVAL, name
        assert call(slots=0) == EINVAL
        assert call(k_stride=1016) == EINVAL and call(v_stride=1028) == EINVAL
        assert call(t=1 << 27) == EUNSUPPORTED and call(t=2 ** 31 - 1) == EUNSUPPORTED


def test_norm_rope_argument_errors():
    lib = _C.load()

    def call(**over):
        args = dict(q_out=A, qo_stride=2048, k_out=None, ko_stride=0, q=A, q_stride=4096, k=A, k_stride=4096, v=A,
                    v_stride=4096, qw=A, kw=A, pos=A, table=A, max_pos=4096, **CACHE, slots=A, t=4, hq=16, hkv=8, d=128,
                    eps=1e-6, stream=None)
        args.update(over)
        return lib.nvamd_qk_norm_rope_fp4(*args.values())

    assert call(t=0) == 0
    assert call(d=64) == EUNSUPPORTED and call(bs=12) == EUNSUPPORTED
    for name in ("q_out", "q", "k", "v", "qw", "kw", "table", "kc", "ks", "vc", "vs"):
        assert call(**{name: 0}) == EINVAL and call(**{name: A + 4}) == EINVAL, name
    assert call(pos=0) == EINVAL and call(slots=0) == EINVAL and call(max_pos=0) == EINVAL and call(hq=0) == EINVAL
    assert call(k_out=A, ko_stride=1016) == EINVAL and call(k_out=A + 8, ko_stride=1024) == EINVAL
    assert call(qo_stride=2040) == EINVAL


def test_decode_argument_errors():
    lib = _C.load()

    def call(**over):
        args = dict(out=A, out_stride=2048, q=A, q_stride=2048, **CACHE, bt=A, bt_stride=8, bt_width=8, lens=A, batch=4,
                    hq=16, hkv=8, d=128, scale=128 ** -0.5, max_ctx=1024, ws=A, ws_bytes=1 << 24, stream=None)
        args.update(over)
        return lib.nvamd_paged_decode_fp4(*args.values())

    assert call(batch=0) == 0
    for name in ("out", "q", "kc", "ks", "vc", "vs"):
        assert call(**{name: 0}) == EINVAL and call(**{name: A + 8}) == EINVAL, name
    assert call(bt=0) == EINVAL and call(lens=0) == EINVAL and call(batch=-1) == EINVAL
    assert call(hq=12) == EINVAL and call(bt_stride=4) == EINVAL and call(max_ctx=0) == EINVAL
    assert call(d=64) == EUNSUPPORTED and call(bs=8) == EUNSUPPORTED
    assert call(batch=2049, ws_bytes=1 << 40) == EUNSUPPORTED      # more than 16,384 (sequence, kv head) units
    assert call(max_ctx=131073, ws_bytes=1 << 40) == EUNSUPPORTED
    assert call(bt_width=1 << 25, bt_stride=1 << 25) == EUNSUPPORTED  # 2^32 tokens
    need = _C.paged_decode_workspace_size(4, 16, 8, 1024)
    assert call(ws_bytes=need - 1) == EWORKSPACE and call(ws=0) == EWORKSPACE and call(ws=A + 8) == EINVAL


@pytest.mark.parametrize("batch, hq, hkv, bound", [(1, 1, 1, 1), (4, 16, 8, 512), (4, 16, 8, 513), (100, 40, 8, 40960),
                                                   (7, 17, 1, 131072)])
def test_the_shared_workspace_holds_the_partitions_of_4_bit_decode(batch, hq, hkv, bound):
    """A counter for each of 16,384 units; records of 132 floats a head for partitions of 512 tokens or more."""
    records = batch * hkv * -(-bound // 512) * (hq // hkv)
    assert _C.paged_decode_workspace_size(batch, hq, hkv, bound) >= 4 * 16384 + 4 * 132 * records


def test_fused_decode_argument_errors():
    lib = _C.load()

    def call(**over):
        args = dict(out=A, out_stride=2048, q=A, q_stride=4096, k=A, k_stride=4096, v=A, v_stride=4096, qw=A, kw=A, pos=A,
                    table=A, max_pos=4096, eps=1e-6, **CACHE, slots=A, bt=A, bt_stride=8, bt_width=8, lens=A, batch=4,
                    hq=16, hkv=8, d=128, scale=128 ** -0.5, max_ctx=1024, ws=A, ws_bytes=1 << 24, stream=None)
        args.update(over)
        return lib.nvamd_paged_decode_fused_fp4(*args.values())

    assert call(batch=0) == 0
    for name in ("out", "q", "k", "v", "qw", "kw", "table", "kc", "ks", "vc", "vs"):
        assert call(**{name: 0}) == EINVAL and call(**{name: A + 8}) == EINVAL, name
    assert call(pos=0) == EINVAL and call(slots=0) == EINVAL and call(max_pos=0) == EINVAL and call(bt=0) == EINVAL
    assert call(k_stride=1016) == EINVAL and call(v_stride=4092) == EINVAL
    assert call(d=64) == EUNSUPPORTED and call(max_ctx=131073, ws_bytes=1 << 40) == EUNSUPPORTED
    assert call(ws_bytes=100) == EWORKSPACE


def test_prefill_argument_errors():
    lib = _C.load()

    def call(**over):
        args = dict(out=A, out_stride=2048, q=A, q_stride=2048, **CACHE, bt=A, bt_stride=8, bt_width=8, cu=A, kv=A,
                    n=2, tokens=64, max_q=64, hq=16, hkv=8, d=128, scale=128 ** -0.5, ws=None, ws_bytes=0, stream=None)
        args.update(over)
        return lib.nvamd_paged_prefill_fp4(*args.values())

    assert call(n=0) == 0 and call(max_q=0) == 0 and call(tokens=0) == 0
    for name in ("out", "q", "kc", "ks", "vc", "vs"):
        assert call(**{name: 0}) == EINVAL and call(**{name: A + 8}) == EINVAL, name
    assert call(bt=0) == EINVAL and call(cu=0) == EINVAL and call(kv=0) == EINVAL
    assert call(scale=0.0) == EINVAL and call(scale=math.nan) == EINVAL and call(tokens=-1) == EINVAL
    assert call(hq=12) == EINVAL and call(n=65536) == EINVAL and call(bt_width=16) == EINVAL
    assert call(d=64) == EUNSUPPORTED and call(bs=8) == EUNSUPPORTED
    assert call(bt_width=1 << 25, bt_stride=1 << 25) == EUNSUPPORTED
    assert call(bt_width=(1 << 23) + 1, bt_stride=1 << 25) == EUNSUPPORTED  # past 2^30 tokens
    need = lib.nvamd_paged_prefill_fp4_workspace_size
    size = need(2, 10, 16, 8, 128, 320)
    # 2 x 8 units of 2 x 16 rows, the keys cut in 256 / 32 pieces, 528 bytes a row
    assert size == 2 * 8 * 32 * 8 * 528
    long = dict(max_q=10, bt_width=320, bt_stride=320)
    assert call(**long, ws=A, ws_bytes=size - 1) == EWORKSPACE and call(**long, ws=A + 8, ws_bytes=size) == EINVAL
    assert need(2, 10, 16, 8, 128, 31) == 0                        # short contexts
    assert need(32, 2000, 16, 8, 128, 320) == 0                    # a full card
    assert need(1, 1, 1, 1, 16, 1 << 20) == 16 * 32 * 528           # 32 pieces at most
    for bad in ((0, 10, 16, 8, 128, 320), (2, 0, 16, 8, 128, 320), (2, 10, 4, 8, 128, 320), (2, 10, 16, 0, 128, 320)):
        assert need(*bad) == 0


# -------------------------------------------------------------------------------------------- Python entry points
def pages(nb=4, hkv=8, bs=16):
    return _C.Fp4Pages(torch.zeros(nb, hkv, bs, 64, dtype=torch.uint8), torch.zeros(nb, hkv, bs, 4, dtype=torch.uint8))


def heads(t, h, d=128, dtype=torch.bfloat16):
    return torch.zeros(t, h, d, dtype=dtype)


def test_pages_have_the_shape_of_a_bf16_cache():
    assert pages(5, 2, 32).shape == (5, 32, 2, 128)
    cache = Fp4PagedKVCache(3, 5, 32, 2, 128, "cpu")
    keys, values = cache.get_physical_cache(1)
    assert keys.shape == values.shape == (5, 32, 2, 128) and keys.codes.is_contiguous()
    per_block = sum(t[0].numel() for t in (*keys, *values)) * 3
    assert Fp4PagedKVCache.bytes_per_block(3, 32, 2, 128) == per_block
    for bad in (dict(block_size=8), dict(block_size=24), dict(head_dim=64)):
        with pytest.raises(ValueError):
            Fp4PagedKVCache(**{**dict(num_layers=1, num_blocks=2, block_size=16, num_kv_heads=1, head_dim=128,
                                      device="cpu"), **bad})
    with pytest.raises(ValueError, match="kv shape"):
        cache.write(0, heads(4, 8), heads(4, 8), torch.arange(4))
    with pytest.raises(ValueError, match="slot_mapping"):
        cache.write(0, heads(4, 2), heads(4, 2), torch.arange(3))


@pytest.mark.parametrize("match, args", [
    ("Fp4Pages", (heads(4, 8), heads(4, 8), torch.zeros(4, 16, 8, 128), pages(), torch.arange(4))),
    ("codes must be", (heads(4, 8), heads(4, 8), pages(), pages(nb=3), torch.arange(4))),
    ("scales must be", (heads(4, 8), heads(4, 8), _C.Fp4Pages(pages().codes, pages(nb=3).scales), pages(),
                        torch.arange(4))),
    ("contiguous uint8", (heads(4, 8), heads(4, 8), _C.Fp4Pages(pages().codes.to(torch.int8), pages().scales), pages(),
                          torch.arange(4))),
    ("bfloat16", (heads(4, 8, dtype=torch.float16), heads(4, 8), pages(), pages(), torch.arange(4))),
    ("value_states must be", (heads(4, 8), heads(3, 8), pages(), pages(), torch.arange(4))),
    ("not dense", (heads(4, 16)[:, ::2], heads(4, 8), pages(), pages(), torch.arange(4))),
    ("slot_mapping", (heads(4, 8), heads(4, 8), pages(), pages(), torch.arange(5))),
    ("slot_mapping", (heads(4, 8), heads(4, 8), pages(), pages(), torch.arange(4, dtype=torch.int32))),
    ("on the GPU", (heads(4, 8), heads(4, 8), pages(), pages(), torch.arange(4))),
])
def test_write_refuses(match, args):
    with pytest.raises(ValueError, match=match):
        _C.kv_cache_write_fp4(*args)


def test_read_refuses():
    with pytest.raises(ValueError, match="k_out must be"):
        _C.kv_cache_read_fp4(pages(), pages(), torch.arange(4), k_out=heads(5, 8))
    with pytest.raises(ValueError, match="on the GPU"):
        _C.kv_cache_read_fp4(pages(), pages(), torch.arange(4))


def test_norm_rope_refuses():
    table, w, pos = torch.zeros(64, 128), torch.ones(128, dtype=torch.bfloat16), torch.arange(4)

    def call(q=heads(4, 16), k=heads(4, 8), v=heads(4, 8), qw=w, kw=w, pos=pos, table=table, slots=torch.arange(4), **out):
        _C.qk_norm_rope_fp4(q, k, v, qw, kw, pos, table, 1e-6, pages(), pages(), slots, **out)

    for match, over in (("q must be", dict(q=heads(4, 16)[:, 0])), ("k must be", dict(k=heads(5, 8))),
                        ("v must be", dict(v=heads(4, 4))), ("q_weight", dict(qw=w.float())),
                        ("k_weight", dict(kw=w[:64])), ("positions", dict(pos=pos.int())),
                        ("cos_sin", dict(table=table.double())), ("cos_sin", dict(table=table[:, :64])),
                        ("slot_mapping", dict(slots=torch.arange(3))), ("q_out must be", dict(q_out=heads(4, 8))),
                        ("k_out must be", dict(k_out=heads(4, 16))), ("on the GPU", {})):
        with pytest.raises(ValueError, match=match):
            call(**over)
    fused = heads(4, 32)
    with pytest.raises(ValueError, match="row stride"):  # written in place of rows that lie further apart
        call(q=fused[:, :16], q_out=fused.view(-1)[:4 * 16 * 128].view(4, 16, 128))


def test_attention_refuses():
    bt, lens, ws = torch.zeros(4, 3, dtype=torch.int32), torch.ones(4, dtype=torch.int32), torch.zeros(64)
    q = heads(4, 16)

    def decode(out=q, q=q, bt=bt, lens=lens, ws=ws):
        _C.paged_decode_fp4(out, q, pages(), pages(), bt, lens, 0.1, 48, ws)

    for match, over in (("shape mismatch", dict(out=heads(3, 16))), ("must be bfloat16", dict(q=heads(4, 16, dtype=torch.float32))), ("block_tables", dict(bt=bt.long())),
                        ("block_tables", dict(bt=bt[:3])), ("block_tables", dict(bt=torch.cat([bt, bt]))),
                        ("rows must be dense", dict(bt=torch.zeros(4, 6, dtype=torch.int32)[:, ::2])),
                        ("context_lens", dict(lens=lens.long())), ("context_lens", dict(lens=lens[:3])),
                        ("on the GPU", {})):
        with pytest.raises(ValueError, match=match):
            decode(**over)
    cu = torch.tensor([0, 1, 4], dtype=torch.int32)

    def prefill(cu=cu, kv=lens, bt=bt):
        _C.paged_prefill_fp4(q, q, pages(), pages(), bt, cu, kv, 4, 0.1)

    for match, over in (("cu_seqlens", dict(cu=cu.long())), ("kv_lens", dict(kv=lens[:1])),
                        ("block_tables", dict(bt=bt[:1])), ("on the GPU", {})):
        with pytest.raises(ValueError, match=match):
            prefill(**over)


def test_block_tables_whose_rows_overlap_are_refused():
    """One table for several sequences by a stride of 0, or windows of one list: a row at the table's width from the one
    before would lie outside its memory."""
    q, kv, w = heads(4, 16), heads(4, 8), torch.ones(128, dtype=torch.bfloat16)
    lens, pos, ws = torch.ones(4, dtype=torch.int32), torch.arange(4), torch.zeros(64)
    cu = torch.arange(5, dtype=torch.int32)
    one = torch.zeros(1, 3, dtype=torch.int32)

    def decode(bt, n=4):
        _C.paged_decode_fp4(None, q[:n], pages(), pages(), bt, lens[:n], 0.1, 48, ws)

    def fused(bt, n=4):
        _C.paged_decode_fused_fp4(None, q[:n], kv[:n], kv[:n], w, w, pos[:n], torch.zeros(64, 128), 1e-6, pages(), pages(),
                                  pos[:n], bt, lens[:n], 0.1, 48, ws)

    def prefill(bt, n=4):
        _C.paged_prefill_fp4(q[:n], q[:n], pages(), pages(), bt, cu[:n + 1], lens, 1, 0.1)

    for call in (decode, fused, prefill):
        for bt in (one.expand(4, 3), torch.zeros(6, dtype=torch.int32).as_strided((4, 3), (1, 1)),
                   torch.zeros(9, dtype=torch.int32).as_strided((4, 3), (2, 1))):
            with pytest.raises(ValueError, match="block_tables overlap"):
                call(bt)
        for bt in (one, one[0].expand(1, 3)):  # a single row's stride says nothing
            with pytest.raises(ValueError, match="on the GPU"):
                call(bt, 1)
        with pytest.raises(ValueError, match="on the GPU"):
            call(torch.zeros(12, dtype=torch.int32).as_strided((4, 3), (3, 1)))


def test_numbers_past_32_bits_are_refused():
    """The C ABI takes them as ints, and a conversion would keep their lower half."""
    q, kv, w = heads(4, 16), heads(4, 8), torch.ones(128, dtype=torch.bfloat16)
    lens, pos, ws = torch.ones(4, dtype=torch.int32), torch.arange(4), torch.zeros(64)
    cu, table = torch.arange(5, dtype=torch.int32), torch.zeros(4, 3, dtype=torch.int32)
    far = torch.empty(4, (1 << 32) + 3, dtype=torch.int32, device="meta")[:, :3]  # rows 2^32 + 3 apart

    def decode(bt=table, bound=48):
        _C.paged_decode_fp4(None, q, pages(), pages(), bt, lens, 0.1, bound, ws)

    def fused(bt=table, bound=48):
        _C.paged_decode_fused_fp4(None, q, kv, kv, w, w, pos, torch.zeros(64, 128), 1e-6, pages(), pages(), pos, bt, lens,
                                  0.1, bound, ws)

    def prefill(bt=table, bound=1):
        _C.paged_prefill_fp4(q, q, pages(), pages(), bt, cu, lens, bound, 0.1)

    for call in (decode, fused, prefill):
        with pytest.raises(ValueError, match="row stride of block_tables .* 32 bits"):
            call(bt=far)
        for bound in ((1 << 32) + 48, 1 << 31, -(1 << 32) + 48):
            with pytest.raises(ValueError, match="max_.*_len .* 32 bits"):
                call(bound=bound)


# -------------------------------------------------------------------------------------------- without csrc/calls.cpp
CALLS = "nano_vllm_ascend_amd._calls"


@pytest.fixture
def unloaded(monkeypatch):
    monkeypatch.setattr(_C, "_lib", None)
    monkeypatch.setattr(_C, "_calls", None)


def test_the_library_loads_without_the_extension(unloaded, monkeypatch):
    monkeypatch.setitem(sys.modules, CALLS, None)  # an import of it fails
    with pytest.warns(RuntimeWarning, match="_calls.so cannot be used"):
        _C.load()
    assert _C._calls is None and _C.version() > 0 and _C.paged_decode_workspace_size(4, 16, 8, 1024) > 0
    for call in (lambda: _C.kv_cache_write_fp4(heads(4, 8), heads(4, 8), pages(), pages(), torch.arange(4)),
                 lambda: _C.kv_cache_read_fp4(pages(), pages(), torch.arange(4))):
        with pytest.raises(ValueError, match="on the GPU"):
            call()


def test_an_extension_of_another_abi_is_not_used(unloaded, monkeypatch):
    other = type(sys)(CALLS)
    other.ABI_VERSION, other.bind = _C.load().nvamd_version() + 1, None
    monkeypatch.setattr(_C, "_lib", None)
    monkeypatch.setitem(sys.modules, CALLS, other)
    with pytest.warns(RuntimeWarning, match="version .* of the C ABI"):
        _C.load()
    assert _C._calls is None


def test_the_extension_is_used_where_it_is_built(unloaded):
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        _C.load()
    assert _C._calls is importlib.import_module(CALLS)


def test_the_library_is_built_without_the_extension(monkeypatch, tmp_path):
    def no_torch():
        raise ImportError("no module named torch")

    def link(cmd, **_):
        open(cmd[-1], "w").close()
        return subprocess.CompletedProcess(cmd, 0, "", "")

    stale = tmp_path / "_calls.so"
    stale.touch()
    for name, value in (("LIB_PATH", tmp_path / "libnvamd.so"), ("CALLS_PATH", stale), ("OBJ_DIR", tmp_path / "obj"),
                        ("_compile", lambda src: tmp_path / src.name), ("_build_calls", no_torch)):
        monkeypatch.setattr(build, name, value)
    monkeypatch.setattr(build.subprocess, "run", link)
    with pytest.warns(RuntimeWarning, match="no module named torch"):
        build.build(verbose=False)
    assert (tmp_path / "libnvamd.so").exists() and not stale.exists()


def test_the_attention_layer_keeps_one_workspace_for_each_device():
    """Calls that go to and fro between devices find the workspace that they left; only one that was outgrown is kept beside it."""
    from nano_vllm_ascend_amd.layers import HipPagedAttention
    layer = HipPagedAttention(4, 2, 128)
    first = {d: layer.workspace(2, 600, torch.device(d)) for d in ("cpu", "meta")}
    assert all(space.device.type == d for d, space in first.items())
    for _ in range(3):
        for d, space in first.items():
            assert layer.workspace(1, 512, torch.device(d)) is space
    assert layer._outgrown == []
    grown = layer.workspace(3, 512, torch.device("cpu"))
    assert grown is not first["cpu"] and len(layer._outgrown) == 1 and layer._outgrown[0] is first["cpu"]
    assert layer.workspace(4, 600, torch.device("cpu")) is grown  # to a power of two
    assert layer.workspace(2, 600, torch.device("meta")) is first["meta"]
