"""A queued request whose cached prefix is overwritten while it waits.

A block of the prefix cache that nobody uses is the pool's to hand out.  A request is planned on the cached blocks that it
finds when it is submitted; what they hold when it is admitted may be another request's.  The model here samples from the
whole context that it reads back through the block table, so a token differs wherever a row of the context does.
"""
from __future__ import annotations

from types import SimpleNamespace

import pytest
from host_pack import HostPackedBlockManager
from test_overlap_trace import make_llm

BS = 4
SHARED = [7, 3, 9, 1]  # a block of tokens


def llm_of(monkeypatch, num_blocks, overlap, max_num_seqs=2):
    llm = make_llm(monkeypatch, block_size=BS, num_blocks=num_blocks, max_num_seqs=max_num_seqs, prefix=True,
                   overlap=overlap)

    def copy_blocks(sources, targets):
        for s, t in zip(sources, targets):
            for i in range(BS):
                if s * BS + i in llm.runner.model.cache:
                    llm.runner.model.cache[t * BS + i] = llm.runner.model.cache[s * BS + i]

    llm.runner.kv_cache = SimpleNamespace(copy_blocks=copy_blocks)
    return llm


def alone(monkeypatch, prompt, n):
    return llm_of(monkeypatch, 64, False).generate([prompt], max_new_tokens=n)[0]["token_ids"]


def run(llm):
    out = {}
    while llm.has_unfinished():
        out.update((o["request_id"], o["token_ids"]) for o in llm.step())
    return out


def seed_prefix(llm):
    """Leaves SHARED cached in block 0, the last of the free ones."""
    llm.generate([SHARED + [2]], max_new_tokens=1)
    assert llm.runner.block_manager.free_block_ids[-1] == 0


@pytest.mark.parametrize("overlap", [False, True])
def test_a_running_requests_growth_takes_the_cached_block(monkeypatch, overlap):
    llm = llm_of(monkeypatch, 6, overlap, max_num_seqs=1)
    seed_prefix(llm)
    first, second = [11, 12, 13, 14], SHARED + [5]
    a = llm.submit(first, max_new_tokens=20)  # grows over all six blocks
    b = llm.submit(second, max_new_tokens=6)
    waiting = llm.scheduler.waiting[1]
    assert waiting.cached_block_ids == [0] and waiting.reserved_blocks == 2
    out = run(llm)
    assert out[a] == alone(monkeypatch, first, 20)
    assert out[b] == alone(monkeypatch, second, 6)
    assert waiting.cached_block_ids == [] and waiting.reserved_blocks == 3
    assert llm.scheduler.reserved_blocks_total == 0 and len(llm.runner.block_manager.free_block_ids) == 6


@pytest.mark.parametrize("overlap", [False, True])
def test_a_forks_growth_takes_the_cached_block(monkeypatch, overlap):
    """Forked at a block's end: the fork itself copies nothing, the branches take their blocks in the next step."""
    llm = llm_of(monkeypatch, 8, overlap)
    seed_prefix(llm)
    first, second = [11, 12, 13, 14, 15, 16], SHARED + [5]
    a = llm.submit(first, max_new_tokens=9)
    for _ in range(3):
        llm.step()
    m = llm.runner.block_manager
    assert m.seq_lens[a] == 2 * BS
    m.prepare_prefill_metadata(["other"], [4 * BS], [0], [[]])
    assert m.free_block_ids == [1, 0]
    b = llm.submit(second, max_new_tokens=3)
    (waiting,) = llm.scheduler.waiting
    child = llm.fork(a)
    assert waiting.cached_block_ids == [0]
    llm.step()
    assert m.block_tables[a][2] == 1 and m.block_tables[child][2] == 0
    m.free_slot("other")
    out = run(llm)
    assert out[a] == out[child] == alone(monkeypatch, first, 9)
    assert out[b] == alone(monkeypatch, second, 3) and waiting.cached_block_ids == []


@pytest.mark.parametrize("prefix_last", [False, True])
def test_requests_admitted_together_do_not_take_each_others_prefix(monkeypatch, prefix_last):
    """The block that one of them finds cached is the first that the other would get."""
    llm = llm_of(monkeypatch, 6, False)
    seed_prefix(llm)
    m = llm.runner.block_manager
    m.prepare_prefill_metadata(["other"], [5 * BS], [0], [[]])
    prompts = [SHARED + [5], [21, 22, 23]]
    ids = [llm.submit(p, max_new_tokens=2) for p in prompts[:: -1 if prefix_last else 1]]
    m.free_slot("other")
    assert m.free_block_ids[0] == 0
    out = run(llm)
    for i, p in zip(ids, prompts[:: -1 if prefix_last else 1]):
        assert out[i] == alone(monkeypatch, p, 2)
    assert llm.runner.prefill_stats["cached_tokens"] == BS  # the prefix was used, too


def test_holds_prefix():
    m = HostPackedBlockManager(num_blocks=4, block_size=BS, device="cpu")
    tokens = list(range(3 * BS))
    m.prepare_prefill_metadata([0], [3 * BS], [0], [[]])
    m.cache_full_blocks(0, tokens)
    assert m.holds_prefix(tokens, []) and m.holds_prefix(tokens, [0, 1]) and m.holds_prefix(tokens + [9], [0, 1, 2])
    assert not m.holds_prefix(tokens, [1, 0]) and not m.holds_prefix(tokens, [0, 2]) and not m.holds_prefix(tokens, [3])
    assert not m.holds_prefix([5] + tokens[1:], [0])
    m.free_slot(0)
    assert m.holds_prefix(tokens, [0, 1, 2])  # free blocks keep what they hold
    m.prepare_prefill_metadata([1], [2 * BS], [0], [[]])  # takes 3 and 2
    assert m.holds_prefix(tokens, [0, 1]) and not m.holds_prefix(tokens, [0, 1, 2])
    m.free_slot(1)
    m.clear_prefix_cache()
    assert not m.holds_prefix(tokens, [0])
