"""The engine with its KV cache held in 4 bits: LLM(kv_cache_dtype="fp4")."""
from __future__ import annotations

import random
from dataclasses import replace

import pytest
import torch

from nano_vllm_ascend_amd import LLM
from nano_vllm_ascend_amd.config import QWEN3_0_6B
from nano_vllm_ascend_amd.paged_kv_cache import Fp4PagedKVCache, PagedKVCache
from oracle.qwen3_ref import Qwen3Ref

SMALL = replace(QWEN3_0_6B, num_hidden_layers=2)
WIDE = replace(QWEN3_0_6B, num_hidden_layers=2, num_attention_heads=40, num_key_value_heads=8)

# Logits of the 2-layer model in bf16 from one history: two orders of summation move one by a few hundredths at most
# (the bound of the bf16 engine's tests).
LOGIT_TOL = 0.08


def prompts_for(lens, seed=0):
    rng = random.Random(seed)
    return [[rng.randint(0, 10000) for _ in range(n)] for n in lens]


def make_llm(config=SMALL, graph=True, **kw):
    llm = LLM(config, **{**dict(max_model_len=512, num_blocks=64, max_num_seqs=4, enable_decode_graph=graph, seed=1,
                                retain_logits=True, kv_cache_dtype="fp4"), **kw})
    llm.runner.tokenizer.eos_token_id = -1
    return llm


def logits_after(ref: Qwen3Ref, history, token: int, pos: int) -> torch.Tensor:
    """The oracle's logits of a token at a position whose keys and values of every layer up to and with its own are
    ``history[layer]`` ([pos + 1, kv heads, 128] each)."""
    cfg, w = ref.cfg, ref.w
    hq, hkv, d = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim
    at = torch.tensor([pos])
    h = w["model.embed_tokens"][torch.tensor([[token]])]
    for i, (keys, values) in enumerate(history):
        p = f"model.layers.{i}."
        x = ref._norm(h, w[p + "input_layernorm.weight"])
        q = ref._r(x @ w[p + "self_attn.qkv_weight"].T)[..., : hq * d].reshape(1, 1, hq, d)
        q = ref._rope(ref._norm(q, w[p + "self_attn.q_norm.weight"]), at)[0, 0]
        k, v = (t.float().repeat_interleave(hq // hkv, 1) for t in (keys, values))
        s = torch.einsum("hd,khd->hk", q, k) * d ** -0.5
        a = ref._r(torch.einsum("hk,khd->hd", torch.softmax(s, -1), v)).reshape(1, 1, hq * d)
        h = ref._r(h + ref._r(a @ w[p + "self_attn.o_weight"].T))
        x = ref._norm(h, w[p + "post_attention_layernorm.weight"])
        gu = ref._r(x @ w[p + "mlp.gate_up_weight"].T)
        inter = cfg.intermediate_size
        act = ref._r(ref._r(torch.nn.functional.silu(gu[..., :inter])) * gu[..., inter:])
        h = ref._r(h + ref._r(act @ w[p + "mlp.down_weight"].T))
    return ref._r(ref._norm(h, w["model.norm.weight"])[0, 0] @ w["model.embed_tokens"].T).float()


@pytest.mark.gpu
@pytest.mark.parametrize("config", [SMALL, WIDE], ids=["gqa2", "gqa5"])
def test_decode_attends_to_what_the_cache_holds(device, config):
    """A decode step's logits are the oracle's on the keys and values that the engine's cache holds by then."""
    llm = make_llm(config, enable_overlap=False)
    assert isinstance(llm.runner.kv_cache, Fp4PagedKVCache)
    prompts = prompts_for([37, 150, 5], seed=3)
    for p in prompts:
        llm.submit(p, max_new_tokens=6)
    llm.step()  # the prompts
    ref = Qwen3Ref(dict(llm.runner.model.state_dict()), config, round_bf16=True, max_positions=512)
    bs, cache = llm.runner.block_size, llm.runner.kv_cache
    seen = []
    llm.runner.metadata_hook = lambda kind, slots, md: seen.append((md.block_tables, md.context_lens))
    for _ in range(4):
        llm.step()
        tables, ctx = seen[-1]
        running = list(llm.scheduler.running.values())
        assert len(running) == len(prompts)
        for row, seq in enumerate(running):
            n = int(ctx[row])
            pos = torch.arange(n)
            where = (tables[row].long()[pos // bs] * bs + pos % bs).to(device)
            history = [tuple(x.cpu() for x in cache.read(layer, where)) for layer in range(config.num_hidden_layers)]
            token = (prompts[row] + list(seq.generated_token_ids))[n - 1]
            want = logits_after(ref, history, token, n - 1)
            assert (llm.runner.last_logits[row].float().cpu() - want).abs().max().item() <= LOGIT_TOL


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
def test_prefix_hits_read_the_4_bit_pages(device):
    """A prompt whose first blocks are cached runs on the paged route, and gives the same tokens each time that it hits."""
    llm = make_llm(enable_prefix_cache=True)
    shared = prompts_for([300], seed=5)[0]
    llm.generate([shared + [1, 2, 3]], max_new_tokens=2)
    runs = [llm.generate([shared + [7, 8]], max_new_tokens=8)[0]["token_ids"] for _ in range(2)]
    assert llm.runner.prefill_stats["paged_batches"] == 2 and llm.runner.prefill_stats["cached_tokens"] == 2 * 256
    assert runs[0] == runs[1]


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

    def hook(kind, slots, md):
        assert kind == "prefill"
        seen.update((slot, (md.block_tables[row], int(md.context_lens[row]))) for row, slot in enumerate(slots))

    llm.runner.metadata_hook = hook
    ids = [llm.submit(p, max_new_tokens=6) for p in prompts]
    llm.step()
    llm.runner.metadata_hook = None
    assert list(llm.scheduler.running) == ids and llm.runner.last_logits.shape[0] == len(prompts)
    bs, cache = llm.runner.block_size, llm.runner.kv_cache
    for row, (seq_id, prompt) in enumerate(zip(ids, prompts)):
        seq = llm.scheduler.running[seq_id]
        table, n = seen[seq_id]
        assert n == len(prompt) and (seq.cached_prefix_len == 256) == (len(prompt) == 302)
        if seq.cached_prefix_len:
            pos = torch.arange(n)
            where = (table.long()[pos // bs] * bs + pos % bs).to(device)
            history = [tuple(x.cpu() for x in cache.read(layer, where)) for layer in range(SMALL.num_hidden_layers)]
            want = logits_after(ref, history, prompt[-1], n - 1)
        else:
            ref.reset()
            want = ref.forward(prompt).reshape(-1)
        got = llm.runner.last_logits[row].float().cpu()
        assert (got - want).abs().max().item() <= LOGIT_TOL, (row, (got - want).abs().max().item())
        assert seq.next_token_id == int(got.argmax())


@pytest.mark.gpu
def test_the_pool_holds_as_many_more_tokens(device):
    llm = make_llm(num_blocks=None, npu_memory_utilization=0.2)
    args = (SMALL.num_hidden_layers, llm.runner.block_size, SMALL.num_key_value_heads, SMALL.head_dim)
    assert PagedKVCache.bytes_per_block(*args) / Fp4PagedKVCache.bytes_per_block(*args) == 256 / 68
    pool = sum(getattr(llm.runner.kv_cache, n).nbytes for n in ("key_codes", "key_scales", "value_codes", "value_scales"))
    assert pool == llm.runner.num_blocks * Fp4PagedKVCache.bytes_per_block(*args)


def test_unknown_kinds_are_refused():
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        LLM(SMALL, num_blocks=4, kv_cache_dtype="int4")
