"""CPU checks of the KV cache held in 8 bits and of copies of blocks: the oracle against the format's definition by hand,
the argument checks of the C ABI and the refusals of the Python entry points."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from nano_vllm_ascend_amd import _C
from nano_vllm_ascend_amd.paged_kv_cache import Fp4PagedKVCache, Fp8PagedKVCache, PagedKVCache
from oracle import fp8_ref

EINVAL, EUNSUPPORTED, EWORKSPACE = -1, -2, -3
A = 0x10000  # aligned stand-in address: no failing call dereferences it


def row(*head, fill=0.0):
    x = torch.full((1, 1, 128), fill, dtype=torch.bfloat16)
    x[0, 0, :len(head)] = torch.tensor(head, dtype=torch.float64).bfloat16()
    return x


# -------------------------------------------------------------------------------------------- the format
def test_scale_is_the_least_power_that_448_steps_of_reach_the_maximum():
    for top, e in ((448.0, 0), (450.0, 1), (224.0, -1), (226.0, 0), (1.0, -8), (1.75, -8), (1.7578125, -7), (0.0, -117),
                   (2.0 ** -130, -117), (2.0 ** 127, 119), (3.38e38, 119)):
        assert fp8_ref.exponent(torch.tensor(top).bfloat16().item()) == e, top


def test_codes_are_e4m3_with_ties_to_the_even_code():
    x = torch.tensor([0.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -6, 1.0, 1.0625, 1.1875, 15.5, 448.0, 464.0, 1e9, -1.0625, -0.0],
                     dtype=torch.float64)
    codes = fp8_ref.codes_of(x, 0).tolist()
    assert codes == [0, 0, 2, 8, 56, 56, 58, 88, 126, 126, 126, 184, 128]
    every = torch.arange(256, dtype=torch.uint8)
    back = fp8_ref.codes_of(fp8_ref.values_of(every, 5), 5)
    assert torch.equal(back[every % 128 != 127], every[every % 128 != 127])
    assert fp8_ref.codes_of(torch.tensor([math.inf, -math.inf, math.nan], dtype=torch.float64), 3).tolist()[:2] == [127, 255]
    # e4m3 as torch has it
    grid = every.view(torch.float8_e4m3fn).double()
    assert torch.equal(fp8_ref.values_of(every, 0).nan_to_num(999.0), grid.nan_to_num(999.0))


def test_pages_hold_rows_where_the_layout_says():
    pages = fp8_ref.empty_pages(3, 2, 32)
    ks, vs = torch.zeros(1, 2, 128, dtype=torch.bfloat16), torch.zeros(1, 2, 128, dtype=torch.bfloat16)
    ks[0, 1, 70], vs[0, 1, 17] = 448.0, -448.0
    slot = 2 * 32 + 16 + 5  # page 2, tile 1, token 5 of the tile
    fp8_ref.write(pages, ks, vs, torch.tensor([slot]))
    tile = (2 * 2 + 1) * 2 + 1
    assert pages[0].view(-1)[2048 * tile + 1024 + 64 * 5 + 6] == 126 and pages[0].count_nonzero() == 1
    assert pages[2].view(-1)[2048 * tile + 16 * 17 + 5] == 254
    assert pages[1].view(-1)[tile] == pages[3].view(-1)[tile] == 127
    got = fp8_ref.read(pages, torch.tensor([slot, -1]))
    assert torch.equal(got[0][0], ks[0].double()) and torch.equal(got[1][0], vs[0].double()) and not got[0][1].any()


def test_rows_behind_others_raise_the_scale_and_keep_what_the_tile_holds():
    pages = fp8_ref.empty_pages(1, 1, 16)
    fp8_ref.write(pages, row(1.0, 1.125, 2.0 ** -14), row(1.0), torch.tensor([0]))
    assert pages[1][0, 0, 0] == 127 - 8
    fp8_ref.write(pages, row(0.5), row(0.25), torch.tensor([1]))   # smaller: the scale stays
    assert pages[1][0, 0, 0] == 127 - 8
    fp8_ref.write(pages, row(9.0), row(1.0), torch.tensor([2]))    # 448 * 2^-5 = 14
    assert pages[1][0, 0, 0] == 127 - 5 and pages[3][0, 0, 0] == 127 - 8
    k, v = fp8_ref.read(pages, torch.arange(3))
    assert k[0, 0, :3].tolist() == [1.0, 1.125, 2.0 ** -14] and k[1, 0, 0] == 0.5 and k[2, 0, 0] == 9.0
    assert v[:, 0, 0].tolist() == [1.0, 0.25, 1.0]
    fp8_ref.write(pages, row(2.0), row(2.0), torch.tensor([0]))    # a first token starts the tile anew
    assert pages[1][0, 0, 0] == 127 - 7
    assert list(fp8_ref.runs(torch.tensor([5, 6, 14, 15, 16, 17, -1, 18, 3, 2]))) == [
        (0, 5, 2), (2, 14, 2), (4, 16, 2), (7, 18, 1), (8, 3, 1), (9, 2, 1)]


def test_no_value_is_off_by_more_than_a_rounding():
    gen = torch.Generator().manual_seed(1)
    x = (torch.randn(64, 2, 128, generator=gen) * torch.exp(2 * torch.randn(64, 2, 1, generator=gen))).bfloat16()
    pages = fp8_ref.empty_pages(4, 2, 16)
    fp8_ref.write(pages, x, x, torch.arange(64))
    k, v = fp8_ref.read_sequence(pages, torch.arange(64))
    step = torch.pow(2.0, pages[1].double() - 127).transpose(1, 2).reshape(4, 2, 1).repeat_interleave(16, 0)
    assert ((k - x.double()).abs() <= torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * step)).all()
    assert torch.equal(k, v) and torch.equal(k, fp8_ref.read(pages, torch.arange(64))[0])


# -------------------------------------------------------------------------------------------- the C ABI
CACHE = dict(kc=A, ks=A, vc=A, vs=A, nb=64, bs=128)


def test_write_and_read_argument_errors():
    lib = _C.load()
    for fn in (lib.nvamd_kv_cache_write_fp8, lib.nvamd_kv_cache_read_fp8):
        def call(**over):
            args = dict(k=A, k_stride=1024, v=A, v_stride=1024, **CACHE, slots=A, t=4, hkv=8, d=128, stream=None)
            args.update(over)
            return fn(*args.values())

        assert call(t=0) == 0
        assert call(t=-1) == EINVAL and call(nb=0) == EINVAL and call(hkv=0) == EINVAL
        assert call(d=64) == EUNSUPPORTED and call(bs=8) == EUNSUPPORTED and call(bs=48) == EUNSUPPORTED
        for name in ("k", "v", "kc", "ks", "vc", "vs"):
            assert call(**{name: 0}) == EINVAL, name
        for name in ("k", "v", "kc", "vc"):
            assert call(**{name: A + 8}) == EINVAL, name
        assert call(slots=0) == EINVAL
        assert call(k_stride=1016) == EINVAL and call(v_stride=1028) == EINVAL
        assert call(t=1 << 27) == EUNSUPPORTED and call(t=2 ** 31 - 1) == EUNSUPPORTED
        wide = dict(hkv=40_000, k_stride=40_000 * 128, v_stride=40_000 * 128)
        assert call(**wide) == EUNSUPPORTED


def test_norm_rope_argument_errors():
    lib = _C.load()

    def call(**over):
        args = dict(q_out=A, qo_stride=2048, k_out=None, ko_stride=0, q=A, q_stride=4096, k=A, k_stride=4096, v=A,
                    v_stride=4096, qw=A, kw=A, pos=A, table=A, max_pos=4096, **CACHE, slots=A, t=4, hq=16, hkv=8, d=128,
                    eps=1e-6, stream=None)
        args.update(over)
        return lib.nvamd_qk_norm_rope_fp8(*args.values())

    assert call(t=0) == 0
    assert call(d=64) == EUNSUPPORTED and call(bs=12) == EUNSUPPORTED
    for name in ("q_out", "q", "k", "v", "qw", "kw", "table", "kc", "vc"):
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
        return lib.nvamd_paged_decode_fp8(*args.values())

    assert call(batch=0) == 0
    for name in ("out", "q", "kc", "vc"):
        assert call(**{name: 0}) == EINVAL and call(**{name: A + 8}) == EINVAL, name
    assert call(ks=0) == EINVAL and call(vs=0) == EINVAL
    assert call(bt=0) == EINVAL and call(lens=0) == EINVAL and call(batch=-1) == EINVAL
    assert call(hq=12) == EINVAL and call(bt_stride=4) == EINVAL and call(max_ctx=0) == EINVAL
    assert call(d=64) == EUNSUPPORTED and call(bs=8) == EUNSUPPORTED
    assert call(batch=2049, ws_bytes=1 << 40) == EUNSUPPORTED      # more than 16,384 (sequence, kv head) units
    assert call(max_ctx=131073, ws_bytes=1 << 40) == EUNSUPPORTED
    assert call(bt_width=1 << 25, bt_stride=1 << 25) == EUNSUPPORTED  # 2^32 tokens
    need = _C.paged_decode_workspace_size(4, 16, 8, 1024)
    assert call(ws_bytes=need - 1) == EWORKSPACE and call(ws=0) == EWORKSPACE and call(ws=A + 8) == EINVAL


def test_fused_decode_argument_errors():
    lib = _C.load()

    def call(**over):
        args = dict(out=A, out_stride=2048, q=A, q_stride=4096, k=A, k_stride=4096, v=A, v_stride=4096, qw=A, kw=A, pos=A,
                    table=A, max_pos=4096, eps=1e-6, **CACHE, slots=A, bt=A, bt_stride=8, bt_width=8, lens=A, batch=4,
                    hq=16, hkv=8, d=128, scale=128 ** -0.5, max_ctx=1024, ws=A, ws_bytes=1 << 24, stream=None)
        args.update(over)
        return lib.nvamd_paged_decode_fused_fp8(*args.values())

    assert call(batch=0) == 0
    for name in ("out", "q", "k", "v", "qw", "kw", "table", "kc", "vc"):
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
        return lib.nvamd_paged_prefill_fp8(*args.values())

    assert call(n=0) == 0 and call(max_q=0) == 0 and call(tokens=0) == 0
    for name in ("out", "q", "kc", "vc"):
        assert call(**{name: 0}) == EINVAL and call(**{name: A + 8}) == EINVAL, name
    assert call(ks=0) == EINVAL and call(vs=0) == EINVAL
    assert call(bt=0) == EINVAL and call(cu=0) == EINVAL and call(kv=0) == EINVAL
    assert call(scale=0.0) == EINVAL and call(scale=math.nan) == EINVAL and call(tokens=-1) == EINVAL
    assert call(hq=12) == EINVAL and call(n=65536) == EINVAL and call(bt_width=16) == EINVAL
    assert call(d=64) == EUNSUPPORTED and call(bs=8) == EUNSUPPORTED
    assert call(bt_width=(1 << 23) + 1, bt_stride=1 << 25) == EUNSUPPORTED  # past 2^30 tokens
    need = lib.nvamd_paged_prefill_fp8_workspace_size
    size = need(2, 10, 16, 8, 128, 320)
    # 2 x 8 units of 2 x 16 rows, the keys cut in 256 / 32 pieces, 528 bytes a row
    assert size == 2 * 8 * 32 * 8 * 528
    long = dict(max_q=10, bt_width=320, bt_stride=320)
    assert call(**long, ws=A, ws_bytes=size - 1) == EWORKSPACE and call(**long, ws=A + 8, ws_bytes=size) == EINVAL
    assert need(2, 10, 16, 8, 128, 31) == 0                        # short contexts
    for bad in ((0, 10, 16, 8, 128, 320), (2, 0, 16, 8, 128, 320), (2, 10, 4, 8, 128, 320), (2, 10, 16, 0, 128, 320)):
        assert need(*bad) == 0


def test_copy_blocks_argument_errors():
    lib = _C.load()

    def call(pools=(A, A), sizes=(4096, 32), n_pools=2, layers=3, blocks=10, src=A, dst=A, n=4):
        at = (ctypes.c_void_p * len(pools))(*pools) if pools is not None else None
        size = (ctypes.c_int64 * len(sizes))(*sizes) if sizes is not None else None
        return lib.nvamd_copy_blocks(at, size, n_pools, layers, blocks, src, dst, n, None)

    assert call(n=0) == 0 and call(layers=0) == 0
    assert call(pools=None) == EINVAL and call(sizes=None) == EINVAL and call(pools=(A, 0)) == EINVAL
    assert call(sizes=(4096, 0)) == EINVAL and call(n_pools=0) == EINVAL and call(blocks=0) == EINVAL
    assert call(src=0) == EINVAL and call(dst=0) == EINVAL and call(n=-1) == EINVAL and call(layers=-1) == EINVAL
    assert call(pools=(A,) * 9, sizes=(16,) * 9, n_pools=9) == EUNSUPPORTED
    assert call(n=65536) == EUNSUPPORTED and call(layers=65536) == EUNSUPPORTED
    assert call(sizes=(4096, (1 << 32) + 1)) == EUNSUPPORTED


# -------------------------------------------------------------------------------------------- Python entry points
def pages(nb=4, hkv=8, bs=16):
    return _C.Fp8Pages(torch.zeros(nb, hkv, bs, 128, dtype=torch.uint8), torch.zeros(nb, hkv, bs // 16, dtype=torch.uint8))


def heads(t, h, d=128, dtype=torch.bfloat16):
    return torch.zeros(t, h, d, dtype=dtype)


def test_pages_have_the_shape_of_a_bf16_cache():
    assert pages(5, 2, 32).shape == (5, 32, 2, 128)
    cache = Fp8PagedKVCache(3, 5, 32, 2, 128, "cpu")
    keys, values = cache.get_physical_cache(1)
    assert keys.shape == values.shape == (5, 32, 2, 128) and keys.codes.is_contiguous()
    per_block = sum(t[0].numel() for t in (*keys, *values)) * 3
    assert Fp8PagedKVCache.bytes_per_block(3, 32, 2, 128) == per_block
    for bad in (dict(block_size=8), dict(block_size=24), dict(head_dim=64)):
        with pytest.raises(ValueError):
            Fp8PagedKVCache(**{**dict(num_layers=1, num_blocks=2, block_size=16, num_kv_heads=1, head_dim=128,
                                      device="cpu"), **bad})
    with pytest.raises(ValueError, match="kv shape"):
        cache.write(0, heads(4, 8), heads(4, 8), torch.arange(4))
    with pytest.raises(ValueError, match="slot_mapping"):
        cache.write(0, heads(4, 2), heads(4, 2), torch.arange(3))


FP4_PAGES = _C.Fp4Pages(torch.zeros(4, 8, 16, 64, dtype=torch.uint8), torch.zeros(4, 8, 16, 4, dtype=torch.uint8))


@pytest.mark.parametrize("match, args", [
    ("Fp8Pages", (heads(4, 8), heads(4, 8), torch.zeros(4, 16, 8, 128), pages(), torch.arange(4))),
    ("Fp8Pages", (heads(4, 8), heads(4, 8), FP4_PAGES, FP4_PAGES, torch.arange(4))),
    ("Fp8Pages", (heads(4, 8), heads(4, 8), pages(), FP4_PAGES, torch.arange(4))),
    ("codes must be", (heads(4, 8), heads(4, 8), pages(), pages(nb=3), torch.arange(4))),
    ("scales must be", (heads(4, 8), heads(4, 8), _C.Fp8Pages(pages().codes, pages(nb=3).scales), pages(),
                        torch.arange(4))),
    ("contiguous uint8", (heads(4, 8), heads(4, 8), _C.Fp8Pages(pages().codes.to(torch.int8), pages().scales), pages(),
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
        _C.kv_cache_write_fp8(*args)


def test_pages_of_one_kind_are_refused_by_the_other_kinds_calls():
    with pytest.raises(ValueError, match="Fp4Pages"):
        _C.kv_cache_write_fp4(heads(4, 8), heads(4, 8), pages(), pages(), torch.arange(4))
    with pytest.raises(ValueError, match="Fp4Pages"):
        _C.kv_cache_read_fp4(pages(), pages(), torch.arange(4))
    with pytest.raises(ValueError, match="Fp8Pages"):
        _C.kv_cache_read_fp8(FP4_PAGES, FP4_PAGES, torch.arange(4))


def test_range_checks_want_the_rows_of_a_tile_in_order():
    for good in ([0, 1, 2], [5, 6, 16, 17, 3 * 16], [40, 8, 200], [-1, 4, -1, -1, 80], [], [3]):
        _C.check_tile_order(torch.tensor(good, dtype=torch.int64))
    for bad in ([1, 0], [0, 2], [5, 16, 6], [7, 7], [0, 1, 3], [4, 20, 5], [0, -1, 1]):
        with pytest.raises(IndexError, match="tile of 16 slots"):
            _C.check_tile_order(torch.tensor(bad))


def test_read_and_norm_rope_refuse():
    with pytest.raises(ValueError, match="k_out must be"):
        _C.kv_cache_read_fp8(pages(), pages(), torch.arange(4), k_out=heads(5, 8))
    with pytest.raises(ValueError, match="on the GPU"):
        _C.kv_cache_read_fp8(pages(), pages(), torch.arange(4))
    table, w, pos = torch.zeros(64, 128), torch.ones(128, dtype=torch.bfloat16), torch.arange(4)

    def call(q=heads(4, 16), k=heads(4, 8), v=heads(4, 8), qw=w, kw=w, pos=pos, table=table, slots=torch.arange(4), **out):
        _C.qk_norm_rope_fp8(q, k, v, qw, kw, pos, table, 1e-6, pages(), pages(), slots, **out)

    for match, over in (("q must be", dict(q=heads(4, 16)[:, 0])), ("k must be", dict(k=heads(5, 8))),
                        ("v must be", dict(v=heads(4, 4))), ("q_weight", dict(qw=w.float())),
                        ("positions", dict(pos=pos.int())), ("cos_sin", dict(table=table[:, :64])),
                        ("slot_mapping", dict(slots=torch.arange(3))), ("q_out must be", dict(q_out=heads(4, 8))),
                        ("k_out must be", dict(k_out=heads(4, 16))), ("on the GPU", {})):
        with pytest.raises(ValueError, match=match):
            call(**over)


def test_attention_refuses():
    bt, lens, ws = torch.zeros(4, 3, dtype=torch.int32), torch.ones(4, dtype=torch.int32), torch.zeros(64)
    q = heads(4, 16)

    def decode(out=q, q=q, bt=bt, lens=lens, ws=ws, bound=48):
        _C.paged_decode_fp8(out, q, pages(), pages(), bt, lens, 0.1, bound, ws)

    for match, over in (("shape mismatch", dict(out=heads(3, 16))),
                        ("must be bfloat16", dict(q=heads(4, 16, dtype=torch.float32))),
                        ("block_tables", dict(bt=bt.long())), ("block_tables", dict(bt=bt[:3])),
                        ("rows must be dense", dict(bt=torch.zeros(4, 6, dtype=torch.int32)[:, ::2])),
                        ("block_tables overlap", dict(bt=bt[:1].expand(4, 3))), ("32 bits", dict(bound=(1 << 32) + 48)),
                        ("context_lens", dict(lens=lens.long())), ("context_lens", dict(lens=lens[:3])),
                        ("on the GPU", {})):
        with pytest.raises(ValueError, match=match):
            decode(**over)
    cu = torch.tensor([0, 1, 4], dtype=torch.int32)

    def prefill(cu=cu, kv=lens, bt=bt, bound=4):
        _C.paged_prefill_fp8(q, q, pages(), pages(), bt, cu, kv, bound, 0.1)

    for match, over in (("cu_seqlens", dict(cu=cu.long())), ("kv_lens", dict(kv=lens[:1])),
                        ("block_tables", dict(bt=bt[:1])), ("32 bits", dict(bound=1 << 32)), ("on the GPU", {})):
        with pytest.raises(ValueError, match=match):
            prefill(**over)


def test_copy_blocks_refuses():
    pool, ids = torch.zeros(2, 6, 16), torch.arange(3, dtype=torch.int32)
    for match, pools, src, dst in (
            ("1 to 8 pools", [], ids, ids), ("1 to 8 pools", [pool] * 9, ids, ids),
            ("pools must be", [pool, torch.zeros(2, 5, 16)], ids, ids), ("pools must be", [torch.zeros(6, 16)], ids, ids),
            ("pools must be", [pool.transpose(0, 1)], ids, ids), ("pools must be", [torch.zeros(2, 0, 16)], ids, ids),
            ("sources", [pool], ids.long(), ids), ("targets", [pool], ids, ids[:2]), ("targets", [pool], ids, ids.long()),
            ("sources", [pool], torch.arange(6, dtype=torch.int32)[::2], ids), ("on the GPU", [pool], ids, ids)):
        with pytest.raises(ValueError, match=match):
            _C.copy_blocks(pools, src, dst)


@pytest.mark.parametrize("cache", [PagedKVCache(2, 6, 16, 1, 128, torch.bfloat16, "cpu"),
                                   Fp4PagedKVCache(2, 6, 16, 1, 128, "cpu"), Fp8PagedKVCache(2, 6, 16, 1, 128, "cpu")])
def test_copies_of_host_block_ids_are_checked(cache):
    for src, dst in (([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0], [6]), ([-1], [2])):
        with pytest.raises(IndexError):
            cache.copy_blocks(src, dst)
    with pytest.raises(ValueError, match="sources for"):
        cache.copy_blocks([0, 1], [2])
    with pytest.raises(ValueError, match="on the GPU"):
        cache.copy_blocks([0, 3], [2, 3])  # a block to itself is no copy


def test_the_oracle_writes_many_rows_as_it_writes_a_few():
    gen = torch.Generator().manual_seed(2)
    x = (torch.randn(50, 2, 128, generator=gen) * torch.exp(3 * torch.randn(50, 2, 1, generator=gen))).bfloat16()
    x[7, 1, 3], x[30, 0, 0] = math.nan, math.inf
    slots = torch.cat([torch.arange(64, 97), torch.arange(16, 33)])
    one, many = fp8_ref.empty_pages(4, 2, 32), fp8_ref.empty_pages(4, 2, 32)
    fp8_ref.write(one, x, x.flip(0), slots)
    fp8_ref.write_sequences(many, x, x.flip(0), slots)
    assert all(torch.equal(a, b) for a, b in zip(one, many))
