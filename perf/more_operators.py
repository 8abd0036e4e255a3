"""Operators of a KV cache held in 8 bits and of a cache's blocks: one pass of each, with plain forms beside them.

Kinds of case (the value of ``"kind"``):
  store    rows of keys and values are quantised into the cache at their slots, behind what their blocks of tokens hold.
  rope     queries and keys are normalised per head and rotated to their positions; the rotated keys and the raw values
           go into the cache at their slots, the queries come out in bf16, and with ``keys`` the rotated keys too.
  decode   one query token per sequence attends to its cached context.
  prefill  the last tokens of each sequence attend, causally, to the cached prefix and themselves, all in the cache.
  copy     blocks of a cache (``cache``: 8-bit, 4-bit or bf16) are copied to others, in every layer.
Store and rope return what the cache then holds, in bf16, of every token of the tiles that they wrote to.

The cache.  A page (of ``block_size`` tokens) of a head is tiles of 16 tokens.  A tile's keys (values) share a scale 2^e,
a byte e + 127, and a value's code is x / 2^e in e4m3 (nearest, ties to the even code, saturated at 448; an infinity or a
NaN is the code 127, NaN).  Rows that begin a tile set e to the least integer with max|x| <= 448 * 2^e over them, within
[-117, 119] (infinities and NaNs do not count); rows that go behind others raise it to theirs if that is larger, and the
tile's other codes are then rounded to the new scale.  A layer's keys (values) are codes [blocks, kv heads, block_size,
128] and scales [blocks, kv heads, block_size / 16], bytes.  Of a tile, with t the token and d the dim:
  key codes    byte 1024 (d / 64) + 64 t + d % 64
  value codes  byte 16 d + t

Sequence lengths are fixed by a case's own values, so a case's work does not depend on the seed; tensors and block
tables come from the seed.  Queries, keys and values are N(0, 1), as normed heads are, and a few channels of the keys
are four times as large, as trained models have them.
"""
from __future__ import annotations

import math
import random

import torch

own = False

D = 128               # head_dim of every configuration
TILE = 16             # tokens that share a scale
EPS = 1e-6
THETA = 1.0e6
MAX_POSITIONS = 40960
SCALE = D ** -0.5


def listed() -> list[dict]:
    return [
        # The smallest call: one token's rows into a conversation, in the middle of a tile; launch latency counts.
        store("store_1", 1, start=1000),
        # The rows of a long prompt behind a cached turn that ends inside a tile, an odd number of them.
        store("store_12345", 12345, start=1029),
        # The norms and rotation of a decode step of 32 requests, three of them padding of a captured batch.
        rope("rope_decode_b32", 32, 256, 2304, pad=3),
        # The same of a batch of ragged prompts, whose attention then runs on the rotated keys themselves.
        rope("rope_prompts_b32", 32, 64, 2048, keys=True),
        # A few short chats: latency counts.
        decode("decode_b4_ctx512", 4, 1, 512, bound=512),
        # The headline workload: 32 requests in the middle of generation.
        decode("decode_b32_ctx2304", 32, 256, 2304, bound=4096),
        # The load workload: 100 requests of 2048 prompt tokens, somewhere in their 2048 output tokens.
        decode("decode_b100_ctx4096", 100, 2048, 4096, bound=4096),
        # Long documents at eight query heads per kv head: a few requests up to the models' 40,960 positions, which also
        # bound the launch.
        decode("decode_gqa8_b4_ctx40960", 4, 8192, 40960, hq=64, hkv=8, bound=40960),
        # Short follow-ups (a chat's next turn) on a cached conversation, in pages of 16 tokens.
        prefill("prefill_turns_b8", 8, 1, 64, cached=1040, block_size=16),
        # Prompts admitted at once behind a shared system prompt.
        prefill("prefill_prefix_b32_2048", 32, 512, 2048, cached=1152),
        # A request that branches: its last, partly filled block, in every layer.
        copy("copy_fork_1", 1, blocks=16),
        # A batch's blocks moved at once, as when requests are gathered at one end of the pool.
        copy("copy_blocks_48", 48, blocks=112, cache="bf16"),
    ]


def store(name, tokens, start=0, hkv=8, block_size=128, pad=0):
    """``start``: tokens that the sequence has in the cache already."""
    return _named(name, kind="store", tokens=tokens, start=start, hkv=hkv, block_size=block_size, pad=pad)


def rope(name, batch, lo, hi, hq=16, hkv=8, block_size=128, keys=False, pad=0):
    """Without ``keys`` one token per sequence (a decode step), with it every token of each (prompts)."""
    return _named(name, kind="rope", batch=batch, lo=lo, hi=hi, hq=hq, hkv=hkv, block_size=block_size, keys=keys,
                  pad=pad)


def decode(name, batch, lo, hi, hq=16, hkv=8, block_size=128, bound=0):
    return _named(name, kind="decode", batch=batch, lo=lo, hi=hi, hq=hq, hkv=hkv, block_size=block_size, bound=bound)


def prefill(name, batch, lo, hi, hq=16, hkv=8, block_size=128, cached=0):
    return _named(name, kind="prefill", batch=batch, lo=lo, hi=hi, hq=hq, hkv=hkv, block_size=block_size,
                  cached=cached)


def copy(name, n, blocks, cache="fp8", layers=28, hkv=8, block_size=128):
    """``n`` of a pool's ``blocks`` are copied to as many others."""
    return _named(name, kind="copy", n=n, blocks=blocks, cache=cache, layers=layers, hkv=hkv, block_size=block_size)


def _named(name, **case):
    return {"name": name, **case} if name else case


HEADS = [(16, 8), (16, 8), (16, 8), (32, 8), (40, 8), (64, 8), (8, 8), (16, 4), (24, 8), (2, 1), (16, 1)]


def _log(rng, lo, hi) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(["store", "rope", "decode", "decode", "decode", "prefill", "prefill", "copy"])
    hq, hkv = rng.choice(HEADS)
    bs = rng.choice([128, 128, 128, 64, 32, 16, 256])
    if kind == "store":
        tokens = _log(rng, 1, 40_000)
        return store(None, tokens, rng.choice([0, 16, rng.randint(1, 4000)]), hkv, bs, rng.choice([0, min(3, tokens - 1)]))
    if kind == "rope":
        keys = rng.random() < 0.5
        hi = _log(rng, 8, 4096)
        batch = _log(rng, 1, max(1, min(100, 40_000 // hi if keys else 100)))
        return rope(None, batch, max(1, hi // rng.choice([1, 4, 32])), hi, hq, hkv, bs, keys,
                    rng.choice([0, batch // 4]))
    if kind == "decode":
        hi = _log(rng, 64, 40960)
        batch = _log(rng, 1, max(1, min(128, 300_000 // hi)))
        lo = rng.choice([0, 1, hi // 2, max(1, hi - 100)])
        return decode(None, batch, lo, hi, hq, hkv, bs, rng.choice([0, 4096 * -(-hi // 4096), 40960]))
    if kind == "prefill":
        hi = _log(rng, 4, 4000)
        cached = rng.choice([0, 16, 256, 1040, 4096])
        batch = _log(rng, 1, max(1, min(32, 24_000 // hi, 300_000_000 // (hi * (hi + cached) * hq // 8))))
        return prefill(None, batch, rng.choice([0, 1, hi // 2]), hi, hq, hkv, bs, cached)
    n = _log(rng, 1, 48)
    return copy(None, n, 2 * n + rng.randint(0, 16), rng.choice(["fp8", "fp8", "fp4", "bf16"]), rng.randint(1, 28), hkv,
                rng.choice([128, 64, 16]))


# ------------------------------------------------------------------------------------------------ sizes
def _lens(case) -> list[int]:
    """Context lengths (decode; rope of single tokens) or new tokens (prefill, rope of prompts) of each sequence; one
    of them is the longest that the case allows."""
    rng = random.Random(1_000_003 * case["batch"] + 1_009 * case["lo"] + case["hi"])
    lens = [rng.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
    lens[rng.randrange(len(lens))] = case["hi"]
    return lens


def _spans(case) -> list[tuple[int, int]]:
    """First new position and end of each sequence of a store or rope case."""
    if case["kind"] == "store":
        return [(case["start"], case["start"] + case["tokens"] - case["pad"])]
    return [(0 if case["keys"] else n - 1, n) for n in _lens(case)]


def _widths(case) -> list[int]:
    """Bytes of a block of one layer in each of the cache's arrays."""
    rows = case["hkv"] * case["block_size"]
    return {"fp8": [rows * D, rows // TILE] * 2, "fp4": [rows * D // 2, rows * D // 32] * 2,
            "bf16": [rows * D * 2] * 2}[case["cache"]]


def work(case) -> dict:
    hkv = case["hkv"]
    if case["kind"] == "copy":
        return {"bytes": 2 * case["n"] * case["layers"] * sum(_widths(case)), "flops": 0}
    if case["kind"] in ("store", "rope"):
        spans = _spans(case)
        t = sum(end - first for first, end in spans)
        behind = sum(end - first // TILE * TILE for first, end in spans)  # with the tokens before them in their tiles
        scales = 2 * hkv * sum(-(-end // TILE) - first // TILE for first, end in spans)
        # k, v read; cache written; its codes read and returned in bf16
        rows = hkv * (t * (4 * D + 2 * D) + behind * (2 * D + 4 * D)) + 2 * scales + 8 * (t + behind)
        if case["kind"] == "store":
            return {"bytes": rows, "flops": 4 * D * hkv * t}
        heads = t * (case["hq"] + (hkv if case["keys"] else 0))
        q_rows = 4 * D * t * case["hq"] + (2 * D * t * hkv if case["keys"] else 0) + 4 * D * t + 8 * t
        return {"bytes": rows + q_rows, "flops": 10 * D * (heads + 2 * t * hkv)}
    hq, lens = case["hq"], _lens(case)
    if case["kind"] == "decode":
        total = sum(lens)
        pages = -(-total // case["block_size"]) + len(lens)
        cache = 2 * hkv * (D * total + total // TILE + len(lens))
        return {"bytes": cache + 4 * D * hq * len(lens) + 4 * pages, "flops": 4 * D * hq * total}
    cached = case["cached"]
    pairs = sum(n * cached + n * (n + 1) // 2 for n in lens)
    total = sum(lens)
    keys = total + cached * len(lens)
    return {"bytes": 2 * hkv * (D * keys + keys // TILE) + 4 * D * hq * total, "flops": 4 * D * hq * pairs}


# ------------------------------------------------------------------------------------------------ states
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, *shape, mean=0.0, std=1.0):
    return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(mean, std, generator=gen)


def _pages(lens, bs, seed):
    """A pool that holds every sequence with a block to spare, and its table: distinct blocks in a seeded order, the
    spare one (used by nothing) last in the pool."""
    need = [-(-n // bs) for n in lens]
    perm = torch.randperm(max(sum(need), 1), generator=torch.Generator().manual_seed(int(seed)))
    tables = torch.zeros((len(lens), max(max(need), 1)), dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = perm[at:at + n].to(torch.int32)
        at += n
    return len(perm) + 1, tables


def _empty_cache(blocks, case):
    """Codes and scales of keys and values that no row has been written to, and the codes' values."""
    def byte(*shape):
        return torch.zeros((blocks, case["hkv"], *shape), dtype=torch.uint8, device="cuda")

    bs = case["block_size"]
    positive = [m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)]
    positive[127] = math.nan
    return {"k_codes": byte(bs, D), "k_scales": byte(bs // TILE), "v_codes": byte(bs, D), "v_scales": byte(bs // TILE),
            "grid": torch.tensor(positive + [-x for x in positive], device="cuda")}


def _channels(gen):
    """Every 16th channel of the keys, from a seeded one on, is four times as large."""
    at = torch.randint(0, 16, (1,), generator=gen, device="cuda")
    return torch.where(torch.arange(D, device="cuda") % 16 == at, 4.0, 1.0).bfloat16()


@torch.no_grad()
def prepare(case, seed) -> dict:
    return {"store": _prepare_rows, "rope": _prepare_rows, "decode": _prepare_attention,
            "prefill": _prepare_attention, "copy": _prepare_copy}[case["kind"]](case, seed)


def _slots(tables, seq, pos, bs):
    return tables[seq, pos // bs].to(torch.int64) * bs + pos % bs


def _fill(state, gen, slots):
    """Random keys and values at slots that are whole tiles, some at a time."""
    channels = _channels(gen)
    for part in slots.split(1 << 17):
        k, v = (_normal(gen, len(part), state["case"]["hkv"], D) for _ in range(2))
        _store(state, k * channels, v, *_plan(part))


def _prepare_rows(case, seed):
    gen, bs, hkv = _generator(seed), case["block_size"], case["hkv"]
    spans = _spans(case)
    blocks, tables = _pages([end for _, end in spans], bs, seed)

    def positions(begin_of):
        parts = [torch.arange(begin_of(first), end) for first, end in spans]
        seq = torch.repeat_interleave(torch.arange(len(parts)), torch.tensor([len(p) for p in parts]))
        return seq, torch.cat(parts)

    seq, pos = positions(lambda first: first)
    slots = torch.cat([_slots(tables, seq, pos, bs), torch.full((case["pad"],), -1)])  # a padded batch's have none
    state = {"case": case, **_empty_cache(blocks, case), "slots": slots.cuda()}
    behind_seq, behind = positions(lambda first: first // TILE * TILE)
    state["written"] = _slots(tables, behind_seq, behind, bs).cuda()  # every token of the tiles that are written to
    firsts = torch.tensor([first for first, _ in spans])
    held = behind[behind < firsts[behind_seq]]
    if len(held):  # tiles that hold tokens already: whole ones, whose further tokens the rows then replace
        tiles, at = torch.unique_consecutive(
            torch.stack((behind_seq, behind // TILE))[:, behind < firsts[behind_seq]], dim=1), torch.arange(TILE)
        _fill(state, gen, _slots(tables, tiles[0].repeat_interleave(TILE),
                                 (tiles[1][:, None] * TILE + at).flatten(), bs).cuda())
    plan = _plan(state["slots"][: len(pos)])
    pos = torch.cat([pos, torch.zeros(case["pad"], dtype=torch.int64)])
    hq, t = case.get("hq", 0), len(slots)
    qkv = _normal(gen, t, hq + 2 * hkv, D)
    qkv[:, hq:hq + hkv] *= _channels(gen)
    state.update(plan=plan, q=qkv[:, :hq], k=qkv[:, hq:hq + hkv],
                 v=qkv[:, hq + hkv:])  # views into a fused projection's rows
    if case["kind"] == "rope":
        freqs = torch.outer(torch.arange(MAX_POSITIONS, dtype=torch.float32),
                            1.0 / THETA ** (torch.arange(0, D, 2, dtype=torch.float32) / D))
        state.update(positions=pos.cuda(), table=torch.cat((freqs.cos(), freqs.sin()), 1).contiguous().cuda(),
                     q_weight=_normal(gen, D, mean=1.0, std=0.02), k_weight=_normal(gen, D, mean=1.0, std=0.02),
                     q_out=torch.empty((t, hq, D), dtype=torch.bfloat16, device="cuda"),
                     k_out=torch.empty((t, hkv, D), dtype=torch.bfloat16, device="cuda") if case["keys"] else None)
    return state


def _prepare_attention(case, seed):
    gen, lens, bs, cached = _generator(seed), _lens(case), case["block_size"], case.get("cached", 0)
    kv_lens = [n + cached for n in lens]
    blocks, tables = _pages(kv_lens, bs, seed)
    state = {"case": case, **_empty_cache(blocks, case)}
    _fill(state, gen, torch.arange(blocks * bs, device="cuda"))
    tokens = len(lens) if case["kind"] == "decode" else sum(lens)
    qkv = _normal(gen, max(tokens, 1), (case["hq"] + 2 * case["hkv"]), D)
    state.update(q=qkv[:tokens, : case["hq"]], tables=tables.cuda(),
                 kv_lens=torch.tensor(kv_lens, dtype=torch.int32).cuda())
    if case["kind"] == "prefill":
        state["cu"] = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    return state


def _prepare_copy(case, seed):
    gen, nb = _generator(seed), case["blocks"]
    pools = [torch.empty((case["layers"], nb, w), dtype=torch.uint8, device="cuda").random_(0, 256, generator=gen)
             for w in _widths(case)]
    perm = torch.randperm(nb, generator=torch.Generator().manual_seed(int(seed))).to(torch.int32).cuda()
    return {"case": case, "pools": pools, "sources": perm[: case["n"]].contiguous(),
            "targets": perm[nb - case["n"]:].contiguous()}


# ------------------------------------------------------------------------------------------------ one pass
_layers = {}  # a program's attention layers, which keep their workspaces


def run(state):
    case = state["case"]
    if not own:
        return {"store": _plain_store, "rope": _plain_rope, "decode": _plain_decode, "prefill": _plain_prefill,
                "copy": _plain_copy}[case["kind"]](state)
    from nano_vllm_ascend_amd import _C
    from nano_vllm_ascend_amd.layers import HipPagedAttention

    if case["kind"] == "copy":
        _C.copy_blocks(state["pools"], state["sources"], state["targets"])
        return state["pools"]
    keys = _C.Fp8Pages(state["k_codes"], state["k_scales"])
    values = _C.Fp8Pages(state["v_codes"], state["v_scales"])
    if case["kind"] == "store":
        _C.kv_cache_write_fp8(state["k"], state["v"], keys, values, state["slots"])
        return _C.kv_cache_read_fp8(keys, values, state["written"])
    if case["kind"] == "rope":
        _C.qk_norm_rope_fp8(state["q"], state["k"], state["v"], state["q_weight"], state["k_weight"],
                            state["positions"], state["table"], EPS, keys, values, state["slots"],
                            q_out=state["q_out"], k_out=state["k_out"])
        k_out = [] if state["k_out"] is None else [state["k_out"]]
        return [state["q_out"], *k_out, *_C.kv_cache_read_fp8(keys, values, state["written"])]
    if case["kind"] == "prefill":
        out = torch.empty(state["q"].shape, dtype=torch.bfloat16, device="cuda")
        return _C.paged_prefill_fp8(out, state["q"], keys, values, state["tables"], state["cu"], state["kv_lens"],
                                    case["hi"], SCALE)
    heads = case["hq"], case["hkv"]
    if heads not in _layers:
        _layers[heads] = HipPagedAttention(*heads, D)
    return _layers[heads](state["q"], keys, values, state["tables"], state["kv_lens"],
                          max_context_len=max(case["bound"], case["hi"]))


def _plan(slots):
    """The tiles of the pool that slots lie in, each slot's index among them and token, whether a tile's first is one."""
    tiles, index = torch.unique(slots // TILE, return_inverse=True)
    token = slots % TILE
    begins = torch.zeros(len(tiles), dtype=torch.bool, device=slots.device)
    begins[index[token == 0]] = True
    return tiles, index, token, begins


def _places(state, tiles):
    """Page and tile of the page of tiles of the pool."""
    per_page = state["case"]["block_size"] // TILE
    return tiles // per_page, tiles % per_page


def _codes(state, name):
    """The codes of keys ("k") or values with their tiles spelled out: [page, head, tile, 2, 16, 64] or [.., 128, 16]."""
    c = state[name + "_codes"]
    nb, hkv, bs, _ = c.shape
    return c.view(nb, hkv, bs // TILE, *((2, TILE, 64) if name == "k" else (D, TILE)))


def _by_token(codes, name):
    """Tiles of codes as [.., 16, 128]."""
    return codes.transpose(-3, -2).flatten(-2) if name == "k" else codes.transpose(-1, -2)


def _step(scale):
    return (scale.int() << 23).view(torch.float32)  # 2^(byte - 127) itself (a power computed on the GPU may be a bit off)


def _exponent(top):
    """The scale bytes of maxima: the least e with top <= 448 * 2^e."""
    mantissa, exponent = torch.frexp(top)  # top = mantissa * 2^exponent, 0.5 <= mantissa < 1
    return (exponent - 9 + (mantissa > 0.875).int()).clamp(-117, 119) + 127


def _quantise(x, scale):
    """Codes of values [.., 16, 128] at the scale bytes [..] of their tiles."""
    u = x / _step(scale)[..., None, None]
    code = u.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    return torch.where(x.isfinite(), code, 127 + 128 * torch.signbit(x).to(torch.uint8))


def _store(state, k, v, tiles, index, token, begins):
    page, tile = _places(state, tiles)
    for name, rows in (("k", k), ("v", v)):
        codes, scales = _codes(state, name), state[name + "_scales"]
        held = scales[page, :, tile].int()  # [tiles, heads]
        values = state["grid"][_by_token(codes[page, :, tile], name).int()] * _step(held)[..., None, None]
        rows = rows.float()
        largest = torch.where(rows.isfinite(), rows.abs(), 0.0).amax(-1)
        top = torch.zeros(held.shape, device=held.device)
        top.scatter_reduce_(0, index[:, None].expand_as(largest), largest, "amax")
        scale = torch.where(begins[:, None], _exponent(top), torch.maximum(_exponent(top), held))
        values[index, :, token] = rows
        code = _quantise(values, scale)
        code = code.unflatten(-1, (2, 64)).transpose(-3, -2) if name == "k" else code.transpose(-1, -2)
        codes[page, :, tile] = code
        scales[page, :, tile] = scale.to(torch.uint8)


def _load(state, name, slots):
    """The values [rows, heads, 128] at slots."""
    page, tile = _places(state, slots // TILE)
    code = (_codes(state, name)[page, :, tile, :, slots % TILE].flatten(-2) if name == "k"
            else _codes(state, name)[page, :, tile, :, slots % TILE])
    return (state["grid"][code.int()] * _step(state[name + "_scales"][page, :, tile])[..., None]).bfloat16()


def _plain_store(state):
    rows = len(state["plan"][1])
    _store(state, state["k"][:rows], state["v"][:rows], *state["plan"])
    return tuple(_load(state, name, state["written"]) for name in "kv")


def _rounded(x):
    """bf16 of 64-bit values, rounded once (a cast by way of 32 bits rounds twice)."""
    mantissa, exponent = torch.frexp(x)
    return ((mantissa * 256).round() * (exponent.long() + 1015 << 52).view(torch.float64)).bfloat16()


def _plain_rope(state):
    """In 64 bits: a key next to a border of the codes goes by its exact value."""
    angle = state["table"][state["positions"]].double()[:, None]
    cos, sin = angle[..., : D // 2], angle[..., D // 2:]

    def rotated(x, weight):
        x = x.double()
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.double()
        lo, hi = y[..., : D // 2], y[..., D // 2:]
        return _rounded(torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), -1))

    q, k = rotated(state["q"], state["q_weight"]), rotated(state["k"], state["k_weight"])
    rows = len(state["plan"][1])
    _store(state, k[:rows], state["v"][:rows], *state["plan"])
    return [q, *([k] if state["case"]["keys"] else []), *(_load(state, name, state["written"]) for name in "kv")]


def _context(state):
    """Keys and values in fp32 [sequences, kv heads, width of the table in tokens, 128]."""
    tables = state["tables"].long()
    n, hkv = tables.shape[0], state["case"]["hkv"]
    for name in "kv":
        code = _by_token(_codes(state, name)[tables], name)  # [n, pages, heads, tiles, 16, 128]
        x = state["grid"][code.int()]
        x *= _step(state[name + "_scales"][tables])[..., None, None]
        yield x.permute(0, 2, 1, 3, 4, 5).reshape(n, hkv, -1, D).contiguous()


def _softmax_v(scores, seen, v):
    """softmax over the keys that are seen, times v; a row that sees none is zero."""
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return (p @ v) / torch.where(total == 0, 1.0, total)


def _plain_decode(state):
    case, q = state["case"], state["q"].float()
    k, v = _context(state)
    b, hkv, width, _ = k.shape
    scores = q.reshape(b, hkv, -1, D) @ k.transpose(-1, -2).contiguous() * SCALE
    seen = torch.arange(width, device="cuda") < state["kv_lens"][:, None, None, None]
    return _softmax_v(scores, seen, v).reshape(b, case["hq"], D).bfloat16()


def _plain_prefill(state):
    case, q, cu = state["case"], state["q"].float(), state["cu"].long()
    k, v = _context(state)
    n, hkv, width, _ = k.shape
    rows, group = case["hi"], case["hq"] // hkv
    at = torch.arange(rows, device="cuda")
    q_len = (cu[1:] - cu[:-1])[:, None]
    padded = q[(cu[:-1, None] + at).clamp(max=max(q.shape[0] - 1, 0))]  # [n, rows, hq, D]
    padded = padded.view(n, rows, hkv, group, D).permute(0, 2, 3, 1, 4).reshape(n, hkv, group * rows, D)
    scores = padded @ k.transpose(-1, -2).contiguous() * SCALE
    last = (state["kv_lens"].long()[:, None] - q_len + at).repeat(1, group)  # the last key that each row sees
    seen = torch.arange(width, device="cuda") <= last[:, None, :, None]
    out = _softmax_v(scores, seen, v).view(n, hkv, group, rows, D).permute(0, 3, 1, 2, 4).reshape(n, rows, -1, D)
    token = torch.arange(q.shape[0], device="cuda")
    seq = torch.searchsorted(cu[1:].contiguous(), token, right=True)
    return out[seq, token - cu[seq]].bfloat16()


def _plain_copy(state):
    for pool in state["pools"]:
        pool[:, state["targets"].long()] = pool[:, state["sources"].long()]
    return state["pools"]


# ------------------------------------------------------------------------------------------------ exact results
def _two_to(e):
    """2^e in 64 bits, from its exponent field."""
    return (e.long() + 1023 << 52).view(torch.float64)


def _grid64():
    """The magnitudes of codes 0 .. 126 in 64 bits."""
    code = torch.arange(127, device="cuda")
    e, m = code // 8, (code % 8).double()
    return torch.where(e == 0, m / 8, 1 + m / 8) * _two_to(torch.where(e == 0, 1, e) - 7)


def _nearest(x, step):
    """Values in 64 bits as codes of a step hold them."""
    grid, u = _grid64(), x.abs() / step
    above = torch.searchsorted(grid, u.contiguous()).clamp(1, 126)
    far, near = grid[above] - u, u - grid[above - 1]
    pick = torch.where((far < near) | ((far == near) & (above % 2 == 0)), above, above - 1)
    return torch.where(x.isfinite(), grid[pick] * step * torch.where(x < 0, -1.0, 1.0), math.nan)


def _bf16(x):
    """The bf16 number nearest to each 64-bit value, of two as near the one of even bits: of the cast's and its neighbours."""
    bits = x.bfloat16().view(torch.int16)
    near = torch.stack((bits, bits - 1, bits + 1), -1)
    off = (near.view(torch.bfloat16).double() - x[..., None]).abs()
    nearest = off == off.min(-1, keepdim=True).values
    pick = (2 * nearest.int() + (near % 2 == 0).int()).argmax(-1, keepdim=True)
    return near.gather(-1, pick)[..., 0].contiguous().view(torch.bfloat16).double()


def _cached(state, head, slots):
    """Keys and values [tokens, 128] of one kv head at the slots, in 64 bits, and their steps [tokens], byte by byte."""
    bs, hkv = state["case"]["block_size"], state["case"]["hkv"]
    grid = _grid64()
    tile = (((slots // bs * hkv + head) * bs + slots % bs) // TILE)[:, None]
    t, d = (slots % TILE)[:, None], torch.arange(D, device="cuda")[None]
    out = []
    for name, at in (("k", d // 64 * 1024 + t * 64 + d % 64), ("v", d * TILE + t)):
        byte = state[name + "_codes"].flatten()[tile * (TILE * D) + at].long()
        step = _two_to(state[name + "_scales"].flatten()[tile[:, 0]].long() - 127)
        low = byte % 128
        value = torch.where(low == 127, math.nan, grid[low.clamp(max=126)]) * torch.where(byte >= 128, -1.0, 1.0)
        out.append((value * step[:, None], step))
    return out


def _exact_rows(state, k, v):
    """What the tiles that are written to hold afterwards, in 64 bits, at ``state["written"]``."""
    written, slots = state["written"], state["slots"][state["slots"] >= 0]
    where = torch.full((int(written.max()) + 1,), -1, device="cuda")  # the row that goes to a slot
    where[slots] = torch.arange(len(slots), device="cuda")
    row = where[written]
    tiles, tile = torch.unique(written // TILE, return_inverse=True)
    begun = torch.zeros(len(tiles), dtype=torch.bool, device="cuda")
    begun[tile[(row >= 0) & (written % TILE == 0)]] = True
    out = [torch.empty((len(written), state["case"]["hkv"], D), dtype=torch.float64, device="cuda") for _ in "kv"]
    for head in range(state["case"]["hkv"]):
        for rows, (held, step), result in zip((k, v), _cached(state, head, written), out):
            x = rows[:, head][row.clamp(min=0)]
            top = torch.where(x.isfinite() & (row >= 0)[:, None], x.abs(), 0.0).max(-1).values
            top = torch.zeros(len(tiles), dtype=torch.float64, device="cuda").scatter_reduce_(0, tile, top, "amax")
            fits = torch.full_like(top, 2.0 ** -117)  # the least power of two that 448 steps of reach the maximum
            for _ in range(-117, 119):
                fits = torch.where(top > 448 * fits, fits * 2, fits)
            before = torch.zeros_like(top).scatter_reduce_(0, tile, step, "amax")
            new = torch.where(begun, fits, torch.maximum(fits, before))[tile][:, None]
            result[:, head] = _nearest(torch.where((row >= 0)[:, None], x, held), new)
    return out


@torch.no_grad()
def exact(case, seed):
    if case["kind"] == "copy":
        return None
    state = prepare(case, seed)
    if case["kind"] in ("store", "rope"):
        q, k, v = (state[x].double() for x in "qkv")
        if case["kind"] == "rope":
            turn = state["table"].double()[state["positions"]].unsqueeze(1)
            turn = torch.complex(turn[..., :64], turn[..., 64:])  # lo + i hi, turned by the angle

            def turned(x, w):
                x = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / D + EPS) * w.double()
                z = torch.complex(x[..., :64].contiguous(), x[..., 64:].contiguous()) * turn
                return torch.cat((z.real, z.imag), -1)

            q, k = turned(q, state["q_weight"]), turned(k, state["k_weight"])
        rows = _exact_rows(state, _bf16(k) if case["kind"] == "rope" else k, v)  # what is stored is the bf16 key
        return tuple(rows) if case["kind"] == "store" else [q, *([k] if case["keys"] else []), *rows]
    lens = state["kv_lens"].tolist()
    starts = state["cu"].tolist() if case["kind"] == "prefill" else list(range(len(lens) + 1))
    q, bs, group = state["q"].double(), case["block_size"], case["hq"] // case["hkv"]
    out = torch.zeros_like(q)
    for i, n in enumerate(lens):
        a, b = starts[i], starts[i + 1]
        if not n or a == b:
            continue
        pos = torch.arange(n, device="cuda")
        slots = state["tables"][i].long()[pos // bs] * bs + pos % bs
        hidden = pos[None, :] > torch.arange(n - (b - a), n, device="cuda")[:, None]
        for g in range(case["hkv"]):
            (k, _), (v, _) = _cached(state, g, slots)
            for h in range(g * group, g * group + group):
                weight = torch.softmax((q[a:b, h] @ k.T / math.sqrt(D)).masked_fill(hidden, -math.inf), -1)
                out[a:b, h] = weight @ v
    return out
