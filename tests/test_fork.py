"""Requests that branch: block tables, budgets and states on the CPU, tokens on the GPU."""
from __future__ import annotations

import sys
from dataclasses import replace
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent / "golden"))
from host_pack import HostPackedBlockManager  # noqa: E402
from test_continuous_batching import ScriptedRunner, engine  # noqa: E402

from nano_vllm_ascend_amd import LLM, SamplingParams  # noqa: E402
from nano_vllm_ascend_amd.config import QWEN3_0_6B  # noqa: E402
from nano_vllm_ascend_amd.model_runner import ModelRunner  # noqa: E402


def manager(num_blocks=8, block_size=4):
    return HostPackedBlockManager(num_blocks=num_blocks, block_size=block_size, device="cpu")


def prefill(m, slot, n):
    m.prepare_prefill_metadata([slot], [n], [0], [[]])


def test_a_fork_shares_full_blocks_and_copies_the_rest():
    m = manager()
    prefill(m, 0, 10)
    assert m.fork_slot(0, 1) == [(2, 3)]
    assert m.block_tables == {0: [0, 1, 2], 1: [0, 1, 3]} and m.seq_lens == {0: 10, 1: 10}
    assert [m.blocks[b].ref_count for b in range(4)] == [2, 2, 1, 1]
    md = m.prepare_decode_metadata([0, 1], [10, 10], 1)
    assert md.slot_mapping.tolist() == [2 * 4 + 2, 3 * 4 + 2] and md.context_lens.tolist() == [11, 11]
    m.free_slot(0)
    assert m.free_block_ids[-1] == 2 and m.blocks[0].ref_count == 1  # what the fork still uses stays
    m.free_slot(1)
    assert sorted(m.free_block_ids) == list(range(8)) and m.block_tables == {}


def test_a_fork_at_a_blocks_end_copies_nothing():
    m = manager()
    prefill(m, 0, 8)
    assert m.fork_slot(0, 1) == [] and m.block_tables[1] == [0, 1]
    md = m.prepare_decode_metadata([0, 1], [8, 8], 1)
    assert md.slot_mapping.tolist() == [2 * 4, 3 * 4]  # each its own next block
    prefill(m, 2, 1)
    assert m.fork_slot(2, 3) == [(4, 5)] and m.block_tables[3] == [5]


def test_a_fork_without_a_block_changes_nothing():
    m = manager(num_blocks=3)
    prefill(m, 0, 10)
    with pytest.raises(RuntimeError, match="out of free blocks"):
        m.fork_slot(0, 1)
    assert m.block_tables == {0: [0, 1, 2]} and [b.ref_count for b in m.blocks] == [1, 1, 1]
    with pytest.raises(ValueError, match="in use"):
        m.fork_slot(0, 0)
    with pytest.raises(KeyError):
        m.fork_slot(5, 1)


def forking_engine(**kw):
    llm = engine(**kw)
    llm.runner.forks = []
    llm.runner.fork = lambda seq, child: llm.runner.forks.append((seq.seq_id, child.seq_id))
    return llm


def run(llm):
    out = {}
    while llm.has_unfinished():
        out.update((o["request_id"], o["token_ids"]) for o in llm.step())
    return out


def test_a_fork_goes_on_from_the_present_state():
    llm = forking_engine(max_num_seqs=3, total_blocks=16)
    a = llm.submit("abc", max_new_tokens=5)
    b = llm.submit("abcd", max_new_tokens=3)
    llm.step()  # prefill
    llm.step()
    llm.step()
    child = llm.fork(a)
    assert llm.runner.forks == [(a, child)] and child not in (a, b)
    seq, new = llm.scheduler.running[a], llm.scheduler.running[child]
    assert new.generated_token_ids == seq.generated_token_ids and new.generated_token_ids is not seq.generated_token_ids
    assert new.cache_position == seq.cache_position and new.next_token_id == seq.next_token_id
    assert llm.scheduler.reserved_blocks_total == seq.reserved_blocks + llm.scheduler.running[b].reserved_blocks + 2
    out = run(llm)
    assert out[a] == out[child] == [0, 1, 2, 3, 4] and out[b] == [10, 11, 12]
    assert llm.scheduler.reserved_blocks_total == 0
    assert sorted(llm.runner.ids("free")) == [a, b, child]


def test_a_forks_own_budget_and_sampling():
    llm = forking_engine()
    a = llm.submit("abc", max_new_tokens=6, temperature=0.5)
    for _ in range(3):
        llm.step()
    child = llm.fork(a, max_new_tokens=3, top_k=4)
    assert llm.scheduler.running[child].sampling_params == SamplingParams(temperature=0.5, top_k=4)
    assert llm.scheduler.running[a].sampling_params == SamplingParams(temperature=0.5)
    out = run(llm)
    assert out[child] == [0, 1, 2] and out[a] == [0, 1, 2, 3, 4, 5]


def test_forks_that_are_refused():
    llm = forking_engine(max_num_seqs=2, total_blocks=4)
    a = llm.submit("abc", max_new_tokens=5)  # two blocks
    with pytest.raises(ValueError, match="not running"):
        llm.fork(a)                           # waits for its prefill
    with pytest.raises(ValueError, match="not running"):
        llm.fork(99)
    llm.step()
    llm.step()
    llm.step()
    with pytest.raises(ValueError, match="is spent"):
        llm.fork(a, max_new_tokens=2)
    with pytest.raises(RuntimeError, match="no room"):
        llm.fork(a, max_new_tokens=10)        # three or more blocks
    llm.fork(a)
    with pytest.raises(RuntimeError, match="no room"):
        llm.fork(a)                           # two sequences at most
    assert len(llm.runner.forks) == 1 and len(llm.scheduler.running) == 2
    run(llm)
    with pytest.raises(ValueError, match="not running"):
        llm.fork(a)


class PoolRunner(ScriptedRunner):
    """Whose prompts and forks take blocks of a real pool of 8, in which requests find their prefixes."""

    def __init__(self):
        super().__init__()
        self.block_size, self.enable_prefix_cache = 4, True
        self.block_manager = manager(num_blocks=8)
        self.copied = []
        self.kv_cache = SimpleNamespace(copy_blocks=lambda sources, targets: self.copied.append((sources, targets)))

    prepare_sequences = ModelRunner.prepare_sequences
    fork = ModelRunner.fork

    def _drop_in_flight(self):
        pass

    def prefill(self, seqs):
        super().prefill(seqs)
        for seq in seqs:
            prefill(self.block_manager, seq.seq_id, seq.estimated_prompt_len)


def test_a_fork_that_takes_a_cached_block_leaves_no_request_waiting_for_it():
    llm = engine(max_num_seqs=2)
    llm.runner = PoolRunner()
    llm.engine_core.runner = llm.runner
    m = llm.runner.block_manager
    prefill(m, "before", 4)  # its block, 0, stays cached behind the other free ones
    m.cache_full_blocks("before", torch.arange(1, 5))
    a = llm.submit("a" * 10, max_new_tokens=3)
    llm.scheduler.waiting[0].cached_block_ids, llm.scheduler.waiting[0].cached_prefix_len = [], 0
    llm.step()
    m.free_slot("before")
    prefill(m, "other", 16)
    assert m.free_block_ids == [0]
    b = llm.submit("b" * 11, max_new_tokens=3)
    (waiting,) = llm.scheduler.waiting
    assert waiting.seq_id == b and waiting.cached_block_ids == [0] and waiting.runtime_prompt_len == 7
    reserved = waiting.reserved_blocks
    llm.fork(a)
    assert llm.runner.copied == [((3,), (0,))]
    assert waiting.cached_block_ids == [] and waiting.cached_prefix_len == 0 and waiting.runtime_prompt_len == 11
    assert waiting.runtime_prompt_token_ids.tolist() == list(range(1, 12)) and waiting.reserved_blocks == reserved + 1


# -------------------------------------------------------------------------------------------- on the GPU
SMALL = replace(QWEN3_0_6B, num_hidden_layers=2)


def make_llm(kind, **kw):
    llm = LLM(SMALL, **{**dict(max_model_len=512, num_blocks=64, max_num_seqs=8, seed=1, kv_cache_dtype=kind), **kw})
    llm.runner.tokenizer.eos_token_id = -1
    return llm


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("kind", ["bf16", "fp4", "fp8"])
@pytest.mark.parametrize("n", [5, 126, 127, 128, 300])
def test_a_greedy_fork_gives_the_tokens_of_its_parent(device, kind, n, graph):
    """Forks of a request between any two steps, around the ends of its blocks, and of a fork: each gives the tokens of the
    request run alone, whichever of them ends first."""
    prompt = torch.randint(0, 10000, (n,), generator=torch.Generator().manual_seed(n)).tolist()
    want = make_llm(kind, enable_decode_graph=False).generate([prompt], max_new_tokens=24)[0]["token_ids"]
    llm = make_llm(kind, enable_decode_graph=graph)
    first = llm.submit(prompt, max_new_tokens=20)
    ids = {first: 20}
    for _ in range(2):
        llm.step()
    for budget in (24, 9):
        ids[llm.fork(first, max_new_tokens=budget)] = budget
        llm.step()
    ids[llm.fork(max(ids), max_new_tokens=12)] = 12
    out = {}
    while llm.has_unfinished():
        out.update((o["request_id"], o["token_ids"]) for o in llm.step())
    assert {i: len(t) for i, t in out.items()} == ids
    for i, budget in ids.items():
        assert out[i] == want[:budget], i
    m = llm.runner.block_manager
    assert len(m.free_block_ids) == 64 and not m.block_tables and all(b.ref_count == 0 for b in m.blocks)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "fp4", "fp8"])
def test_forks_that_sample_write_to_blocks_of_their_own(device, kind):
    """Branches with tokens of their own: what the parent's blocks hold, and the parent's tokens, do not change."""
    prompt = list(range(140))
    want = make_llm(kind).generate([prompt], max_new_tokens=16)[0]["token_ids"]
    llm = make_llm(kind)
    parent = llm.submit(prompt, max_new_tokens=16)
    llm.step()
    children = [llm.fork(parent, temperature=5.0) for _ in range(5)]
    m = llm.runner.block_manager
    tables = [m.block_tables[i] for i in (parent, *children)]
    assert len({t[0] for t in tables}) == 1 and len({t[1] for t in tables}) == 6
    cache = llm.runner.kv_cache
    pools = ([cache.key_cache, cache.value_cache] if kind == "bf16"
             else [cache.key_codes, cache.key_scales, cache.value_codes, cache.value_scales])
    for pool in pools:  # each has the parent's bytes
        for t in tables[1:]:
            assert torch.equal(pool[:, t[1]].view(torch.uint8), pool[:, tables[0][1]].view(torch.uint8))
    out = {}
    while llm.has_unfinished():
        out.update((o["request_id"], o["token_ids"]) for o in llm.step())
    assert out[parent] == want
    assert len({tuple(out[i]) for i in children}) == 5 and all(out[i][0] == want[0] for i in children)
