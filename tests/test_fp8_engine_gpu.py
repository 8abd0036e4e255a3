"""The engine with its KV cache held in 8 bits: LLM(kv_cache_dtype="fp8")."""
from __future__ import annotations

from dataclasses import replace

import pytest
import torch
from test_fp4_engine_gpu import LOGIT_TOL, SMALL, WIDE, logits_after, prompts_for

from nano_vllm_ascend_amd import LLM
from nano_vllm_ascend_amd.paged_kv_cache import Fp8PagedKVCache, PagedKVCache
from oracle.qwen3_ref import Qwen3Ref


def make_llm(config=SMALL, graph=True, **kw):
    llm = LLM(config, **{**dict(max_model_len=512, num_blocks=64, max_num_seqs=4, enable_decode_graph=graph, seed=1,
                                retain_logits=True, kv_cache_dtype="fp8"), **kw})
    llm.runner.tokenizer.eos_token_id = -1
    return llm


def held(cache, table, n, bs, layers, device):
    pos = torch.arange(n)
    where = (table.long()[pos // bs] * bs + pos % bs).to(device)
    return [tuple(x.cpu() for x in cache.read(layer, where)) for layer in range(layers)]


@pytest.mark.gpu
@pytest.mark.parametrize("config", [SMALL, WIDE], ids=["gqa2", "gqa5"])
@pytest.mark.parametrize("block_size", [16, 128])
def test_decode_attends_to_what_the_cache_holds(device, config, block_size):
    """A decode step's logits are the oracle's on the keys and values that the engine's cache holds by then."""
    llm = make_llm(config, enable_overlap=False, block_size=block_size)
    assert isinstance(llm.runner.kv_cache, Fp8PagedKVCache)
    prompts = prompts_for([37, 150, 5], seed=3)
    for p in prompts:
        llm.submit(p, max_new_tokens=6)
    llm.step()  # the prompts
    ref = Qwen3Ref(dict(llm.runner.model.state_dict()), config, round_bf16=True, max_positions=512)
    seen = []
    llm.runner.metadata_hook = lambda kind, slots, md: seen.append((md.block_tables, md.context_lens))
    for _ in range(4):
        llm.step()
        tables, ctx = seen[-1]
        running = list(llm.scheduler.running.values())
        assert len(running) == len(prompts)
        for row, seq in enumerate(running):
            n = int(ctx[row])
            history = held(llm.runner.kv_cache, tables[row], n, block_size, config.num_hidden_layers, device)
            token = (prompts[row] + list(seq.generated_token_ids))[n - 1]
            want = logits_after(ref, history, token, n - 1)
            assert (llm.runner.last_logits[row].float().cpu() - want).abs().max().item() <= LOGIT_TOL


@pytest.mark.gpu
def test_what_the_cache_holds_is_near_the_bf16_cache(device):
    """After a prompt and a few steps each value is off by a rounding to e4m3 of its tile (2^-4 of it or 2^-10 of the
    tile's scale, which is below 2^-7 of its largest), of rows that differ by what the cache's precision does to them: the
    first layer's not at all."""
    prompt = prompts_for([60], seed=8)[0]
    caches = []
    for kind in ("bf16", "fp8"):
        llm = make_llm(kv_cache_dtype=kind, enable_overlap=False)
        llm.submit(prompt, max_new_tokens=9)
        for _ in range(9):
            llm.step()
        caches.append(llm.runner.kv_cache)
    table = torch.arange(1)
    k8, v8 = held(caches[1], table, 60, 128, 1, device)[0]
    for a, b in ((caches[0].key_cache[0, 0, :60], k8), (caches[0].value_cache[0, 0, :60], v8)):
        a, b = a.cpu().double(), b.double()
        top = torch.cat([a, a.new_zeros(4, *a.shape[1:])]).unflatten(0, (4, 16)).abs().amax((1, 3))  # [tile, head]
        step = 2.0 ** -17 * top.repeat_interleave(16, 0)[:60, :, None] * 2  # 2^-10 of a scale of 2^-8 of twice the largest
        # (the bf16 path rounds the normed key before its rotation: 2^-7 more of the row's largest, 2^-8 twice)
        slack = 2.0 ** -7 * a.abs().amax(-1, keepdim=True)
        assert ((a - b).abs() <= 2.0 ** -4 * a.abs() + step + slack).all()


@pytest.mark.gpu
def test_graph_and_overlap_give_the_eager_tokens(device):
    """The captured decode step, launched ahead or not, equals the eager one; and the sequences do not see each other."""
    prompts = prompts_for([37, 200, 5, 128], seed=4)
    want = [r["token_ids"] for r in make_llm(graph=False).generate(prompts, max_new_tokens=20)]
    graph = make_llm()
    assert [r["token_ids"] for r in graph.generate(prompts, max_new_tokens=20)] == want
    assert graph.runner.decode_graph_stats()["replays"] > 10 and graph.runner.overlap_stats["used"] > 5
    again = graph.generate(prompts[::-1], max_new_tokens=20)
    assert [r["token_ids"] for r in again[::-1]] == want


@pytest.mark.gpu
@pytest.mark.parametrize("beside", [[], [90, 5]], ids=["alone", "beside_prompts_without_a_hit"])
def test_a_prompt_takes_the_route_of_its_own_prefix(device, beside):
    """The logits of a prompt with cached blocks are the oracle's on the keys and values that the cache holds; those of
    prompts without any, in the same step, the oracle's on its own keys and values, as if they ran alone."""
    llm = make_llm(enable_prefix_cache=True)
    ref = Qwen3Ref(dict(llm.runner.model.state_dict()), SMALL, round_bf16=True, max_positions=512)
    shared = prompts_for([300], seed=5)[0]
    llm.generate([shared + [1, 2, 3]], max_new_tokens=2)
    prompts = prompts_for(beside, seed=6)
    prompts.insert(1, shared + [7, 8])  # between the others
    seen = {}
    llm.runner.metadata_hook = lambda kind, slots, md: seen.update(
        (slot, (md.block_tables[row], int(md.context_lens[row]))) for row, slot in enumerate(slots))
    ids = [llm.submit(p, max_new_tokens=6) for p in prompts]
    llm.step()
    llm.runner.metadata_hook = None
    for row, (seq_id, prompt) in enumerate(zip(ids, prompts)):
        seq = llm.scheduler.running[seq_id]
        table, n = seen[seq_id]
        assert n == len(prompt) and (seq.cached_prefix_len == 256) == (len(prompt) == 302)
        if seq.cached_prefix_len:
            history = held(llm.runner.kv_cache, table, n, llm.runner.block_size, SMALL.num_hidden_layers, device)
            want = logits_after(ref, history, prompt[-1], n - 1)
        else:
            ref.reset()
            want = ref.forward(prompt).reshape(-1)
        got = llm.runner.last_logits[row].float().cpu()
        assert (got - want).abs().max().item() <= LOGIT_TOL, (row, (got - want).abs().max().item())
        assert seq.next_token_id == int(got.argmax())


@pytest.mark.gpu
def test_the_pool_holds_twice_the_tokens(device):
    llm = make_llm(num_blocks=None, npu_memory_utilization=0.2)
    args = (SMALL.num_hidden_layers, llm.runner.block_size, SMALL.num_key_value_heads, SMALL.head_dim)
    assert PagedKVCache.bytes_per_block(*args) / Fp8PagedKVCache.bytes_per_block(*args) == 256 / (128 + 1 / 16)
    pool = sum(getattr(llm.runner.kv_cache, n).nbytes for n in ("key_codes", "key_scales", "value_codes", "value_scales"))
    assert pool == llm.runner.num_blocks * Fp8PagedKVCache.bytes_per_block(*args)


def test_unknown_kinds_are_refused():
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        LLM(replace(SMALL), num_blocks=4, kv_cache_dtype="int8")
