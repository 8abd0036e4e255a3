"""A decode step that is launched ahead and dropped leaves no trace in an 8-bit cache.

Its rows may raise the scale that they share with up to 15 tokens before them, whose codes are then rounded again; the step
that is made in its place belongs to another batch, and its rows may differ in their last bits and not raise it.
"""
from __future__ import annotations

import pytest
import torch
from test_overlap_trace import FakeKVModel, _fold, make_llm, make_schedule, run_product

from nano_vllm_ascend_amd import LLM, _C
from nano_vllm_ascend_amd.paged_kv_cache import Fp8PagedKVCache
from nano_vllm_ascend_amd.qwen3 import CausalLMOutput

EINVAL, EUNSUPPORTED, EWORKSPACE, A = -1, -2, -3, 0x10000
TILE = 16


# -------------------------------------------------------------------------------------------- the engine, on the CPU
class TileModel(FakeKVModel):
    """Whose rows raise the scale of their tile by as much as their token and their batch's size ask for, and whose tokens
    depend on the scales of the whole context."""

    def __init__(self, block_size):
        super().__init__(block_size)
        self.scales: dict[int, int] = {}

    def __call__(self, input_ids_flat, position_ids_flat, kv_cache, attn_metadata, is_prefill, logits_indices=None):
        md = attn_metadata
        ctx = md.context_lens.tolist()
        for token, slot in zip(input_ids_flat.tolist(), md.slot_mapping.tolist()):
            self.cache[slot] = token
            held = self.scales.get(slot // TILE, 0) if slot % TILE else 0
            self.scales[slot // TILE] = max(held, (7 * token + 31 * len(ctx)) % 101)
        bt = md.block_tables.tolist()
        rows = []
        for i, n in enumerate(ctx):
            slots = [bt[i][p // self.bs] * self.bs + p % self.bs for p in range(n)]
            rows.append(_fold(self.cache[s] + 1000 * self.scales[s // TILE] for s in slots))
        logits = torch.zeros(len(rows), 509)
        logits[torch.arange(len(rows)), torch.tensor(rows, dtype=torch.long)] = 1.0
        return CausalLMOutput(logits=logits)


class Tiles:
    """The scales of a cache that can put its tiles back, as an Fp8PagedKVCache does."""

    def __init__(self, model):
        self.scales, self.restored = model.scales, 0

    def keep_tiles(self, slots):
        return {s // TILE: self.scales[s // TILE] for s in slots.tolist() if s % TILE}

    def restore_tiles(self, kept):
        self.scales.update(kept)
        self.restored += 1


def tile_llm(monkeypatch, overlap, **cfg):
    llm = make_llm(monkeypatch, overlap=overlap, **cfg)
    llm.runner.model = llm.runner.decode_graph_runner.model = TileModel(cfg["block_size"])
    llm.runner.kv_cache = Tiles(llm.runner.model)
    return llm


@pytest.mark.parametrize("seed, block_size", [(1, 16), (2, 32), (3, 128)])
def test_overlapped_tokens_are_the_synchronous_loops(monkeypatch, seed, block_size):
    """Steps are dropped where a request samples EOS."""
    cfg = dict(block_size=block_size, num_blocks=2000 // block_size, max_num_seqs=4, prefix=False)
    schedule = make_schedule(seed, 9, block_size, 5, 90, 10, 60, 0)
    _, plain, _ = run_product(tile_llm(monkeypatch, False, **cfg), schedule, -1)
    eos = plain[1][len(plain[1]) // 2]
    _, want, reasons = run_product(tile_llm(monkeypatch, False, **cfg), schedule, eos)
    assert "eos" in reasons.values()
    llm = tile_llm(monkeypatch, True, **cfg)
    _, got, _ = run_product(llm, schedule, eos)
    stats = llm.runner.overlap_stats
    assert got == want and stats["used"] > 0
    assert llm.runner.kv_cache.restored == stats["discarded"] > 0


# -------------------------------------------------------------------------------------------- the entry points
def test_argument_errors():
    lib = _C.load()
    size = lib.nvamd_kv_cache_kept_size_fp8
    assert size(1, 1, 1) == 2 * 2048 + 16 and size(28, 32, 8) == 28 * 32 * 8 * 4112
    assert size(0, 1, 1) == size(1, 0, 1) == size(1, 1, 0) == 0

    def keep(kept=A, space=3 * 5 * 2 * 4112, kc=A, ks=A, vc=A, vs=A, layers=3, blocks=4, bs=16, slots=A, n=5, hkv=2, d=128):
        return lib.nvamd_kv_cache_keep_fp8(kept, space, kc, ks, vc, vs, layers, blocks, bs, slots, n, hkv, d, None)

    def restore(kept=A, space=3 * 5 * 2 * 4112, kc=A, ks=A, vc=A, vs=A, layers=3, blocks=4, bs=16, n=5, hkv=2, d=128):
        return lib.nvamd_kv_cache_restore_fp8(kept, space, kc, ks, vc, vs, layers, blocks, bs, n, hkv, d, None)

    for call in (keep, restore):
        assert call(n=0) == 0
        for bad in (dict(kept=0), dict(kept=A + 8), dict(kc=0), dict(ks=0), dict(vc=A + 4), dict(vs=0), dict(layers=0),
                    dict(blocks=0), dict(n=-1), dict(hkv=0)):
            assert call(**bad) == EINVAL, bad
        for bad in (dict(bs=8), dict(bs=48), dict(d=64), dict(layers=1 << 16, n=1 << 14)):
            assert call(**bad) == EUNSUPPORTED, bad
        assert call(space=3 * 5 * 2 * 4112 - 1) == EWORKSPACE
    assert keep(slots=0) == EINVAL


def test_what_python_refuses():
    cache = Fp8PagedKVCache(2, 4, 16, 2, 128, "cpu")
    pools = cache._pools
    slots = torch.arange(3)
    for match, p, s in (("as many layers", (pools[0], pools[1][:1], *pools[2:]), slots),
                        ("contiguous", (pools[0].transpose(0, 1), *pools[1:]), slots),
                        ("codes must be", (pools[0][..., :64].contiguous(), *pools[1:]), slots),
                        ("slot_mapping", pools, slots.int()), ("slot_mapping", pools, slots[None]),
                        ("on the GPU", pools, slots)):
        with pytest.raises(ValueError, match=match):
            _C.kv_cache_keep_fp8(p, s)
    kept = torch.zeros(3, 2 * 2 * 4112, dtype=torch.uint8)
    for match, k in (("kept must be", kept[:, :-1]), ("kept must be", kept[0]), ("kept must be", kept.view(torch.int8)),
                     ("kept must be", kept.T), ("on the GPU", kept)):
        with pytest.raises(ValueError, match=match):
            _C.kv_cache_restore_fp8(pools, k)


def rows(n, hkv, seed, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(n, hkv, 128, generator=gen)).bfloat16()


@pytest.mark.gpu
@pytest.mark.parametrize("hkv, bs", [(1, 16), (3, 32), (8, 128)])
def test_tiles_are_put_back(device, hkv, bs):
    """Every number of tokens before the row; what the tile holds of them is again what it was, in each layer, and all
    other tiles stay as they are."""
    layers, nb = 3, -(-16 * 20 // bs)
    cache = Fp8PagedKVCache(layers, nb, bs, hkv, 128, device)
    tiles = torch.randperm(nb * bs // TILE, generator=torch.Generator().manual_seed(hkv))[:18]
    before = [int(x) for x in tiles[:16]]  # the x-th holds x tokens
    slots = torch.cat([16 * t + torch.arange(x) for x, t in enumerate(before)])
    for layer in range(layers):
        k = rows(len(slots), hkv, layer)
        cache.write(layer, k.to(device), k.flip(0).to(device), slots.to(device))
    at = torch.tensor([16 * t + x for x, t in enumerate(before)] + [-1, nb * bs, -7, 16 * int(tiles[17])])
    held = [p.clone() for p in cache._pools]
    kept = cache.keep_tiles(at.to(device))
    assert kept.shape == (20, layers * hkv * 4112) and all(torch.equal(a, b) for a, b in zip(held, cache._pools))
    loud = rows(16, hkv, 9, 1e4).to(device)
    for layer in range(layers):
        cache.write(layer, loud, loud, at[:16].to(device))
    assert not torch.equal(cache.read(1, slots.to(device))[0], cache_of(held, nb, bs).read(1, slots.to(device))[0])
    cache.restore_tiles(kept)
    for layer in range(layers):
        for got, want in zip(cache.read(layer, slots.to(device)), cache_of(held, nb, bs).read(layer, slots.to(device))):
            assert torch.equal(got, want)
    scale_at = {(t // (bs // TILE), t % (bs // TILE)) for t in before[:1]}  # begun by its row: its scale is that row's
    for p, h in zip(cache._pools[1::2], held[1::2]):
        same = (p == h).all(dim=(0, 2)).cpu()
        assert all(bool(same[b, t]) for b in range(nb) for t in range(bs // TILE) if (b, t) not in scale_at)
    others = [t for t in range(nb * bs // TILE) if t not in before]
    for p, h in zip(cache._pools[::2], held[::2]):
        p, h = (x.view(layers, nb, hkv, -1, 2048).transpose(2, 3).flatten(1, 2)[:, others] for x in (p, h))
        assert torch.equal(p, h)
    cache.restore_tiles(kept[:0])
    cache.keep_tiles(at[:0].to(device))


def cache_of(pools, nb, bs):
    """A cache that holds these bytes."""
    layers, _, hkv = pools[0].shape[:3]
    cache = Fp8PagedKVCache(layers, nb, bs, hkv, 128, pools[0].device)
    for p, h in zip(cache._pools, pools):
        p.copy_(h)
    return cache


@pytest.mark.gpu
def test_a_kept_place_outside_the_pool_is_not_restored(device):
    """Of a larger cache, say: nothing is written."""
    big, small = Fp8PagedKVCache(1, 8, 16, 1, 128, device), Fp8PagedKVCache(1, 2, 16, 1, 128, device)
    big._pools[0].fill_(1)
    kept = big.keep_tiles(torch.tensor([16 * 7 + 3, 16 * 2 + 1], device=device))
    small.restore_tiles(kept)
    assert not any(p.any() for p in small._pools)


def small_llm(overlap, **kw):
    from dataclasses import replace

    from nano_vllm_ascend_amd.config import QWEN3_0_6B

    llm = LLM(replace(QWEN3_0_6B, num_hidden_layers=2), max_model_len=512, num_blocks=32, max_num_seqs=4, seed=1,
              kv_cache_dtype="fp8", enable_overlap=overlap, **kw)
    llm.runner.tokenizer.eos_token_id = -1
    return llm


def held_rows(llm, i, n):
    bs, table = llm.runner.block_size, torch.tensor(llm.runner.block_manager.block_tables[i])
    pos = torch.arange(n)
    return [x for layer in range(2) for x in llm.runner.kv_cache.read(layer, table[pos // bs] * bs + pos % bs)]


@pytest.mark.gpu
@pytest.mark.parametrize("drop", ["fork", "submit"])
@pytest.mark.parametrize("block_size", [16, 128])
def test_a_dropped_step_whose_row_raised_its_tile(device, drop, block_size):
    """The dropped step's rows are replaced by larger ones, which raise their tiles: the cache and the tokens are those of
    the synchronous loop all the same."""
    results = []
    for overlap in (False, True):
        llm = small_llm(overlap, block_size=block_size)
        ids = [llm.submit(list(range(s, s + n)), max_new_tokens=30) for s, n in ((3, 37), (50, 122))]
        for _ in range(6):
            llm.step()
        if overlap:
            ahead = llm.runner._in_flight
            slots = ahead.entry.buffers["slot_mapping"]
            assert (slots % TILE != 0).all()
            for layer in range(2):
                loud = rows(2, 8, layer, 300.0).to(device)
                llm.runner.kv_cache.write(layer, loud, loud, slots)
        ids.append(llm.fork(ids[0]) if drop == "fork" else llm.submit([9, 8, 7], max_new_tokens=20))
        for _ in range(3):
            llm.step()
        if overlap:
            assert llm.runner.overlap_stats["discarded"] > 0
        llm.runner._drop_in_flight()
        n = [llm.runner.block_manager.seq_lens[i] for i in ids]
        state = [x.cpu() for i, m in zip(ids, n) for x in held_rows(llm, i, m)]
        out = {}
        while llm.has_unfinished():
            out.update((o["request_id"], o["token_ids"]) for o in llm.step())
        results.append((n, state, out))
    (n0, state0, out0), (n1, state1, out1) = results
    assert n0 == n1 and out0 == out1
    assert all(torch.equal(a, b) for a, b in zip(state0, state1))
