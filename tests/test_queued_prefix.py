"""Requests whose cached prefix lies in blocks that the pool may hand out.

A block of the prefix cache that nobody uses is the pool's to hand out.  The model here samples from the
whole context that it reads back through the block table, so a token differs wherever a row of the context does.
"""
from __future__ import annotations

from types import SimpleNamespace

import pytest
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
