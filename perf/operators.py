"""Operators of a KV cache held in 4 bits: one pass of each, with plain forms beside them.

Kinds of case (the value of ``"kind"``):
  store    rows of keys and values are quantised into the cache at their slots and read back from it.
  rope     queries and keys are normalised per head and rotated to their positions; the rotated keys and the raw values
           go into the cache at their slots (read back from it), the queries come out in bf16, and with ``keys`` the
           rotated keys too.
  decode   one query token per sequence attends to its cached context.
  prefill  the last tokens of each sequence attend, causally, to the cached prefix and themselves, all in the cache.

The cache.  A head vector is 4 blocks of 32 consecutive dims.  A block's scale is 2^e, e the least integer with
max|x| <= 7 * 2^e, within [-125, 125]; its byte is e + 127, or 255 (every value of the block reads as NaN) if the block
holds an infinity or a NaN.  A value's code is the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 to |x| / 2^e, ties to the even
code, with the sign in bit 3.  A layer's keys (values) are codes [blocks, kv heads, block_size, 64] and scales
[blocks, kv heads, block_size, 4], bytes, whose pages hold tiles of 16 tokens (t = token % 16, q = block of 32 dims):
  key codes    byte 64 t + i: dims 2i (low nibble) and 2i + 1
  key scales   byte 16 (t % 4) + 4 q + t / 4
  value codes  byte 16 (16 q + r) + t: dims 32 q + r (low nibble) and 32 q + 16 + r, r < 16
  value scales byte 16 q + t

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
EPS = 1e-6
THETA = 1.0e6
MAX_POSITIONS = 40960
SCALE = D ** -0.5
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed() -> list[dict]:
    return [
        # The smallest call: one token's rows; launch latency counts.
        store("store_1", 1),
        # The rows of a batch of prompts, an odd number of them.
        store("store_12345", 12345),
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
        # Eight query heads per kv head at a middling batch.
        decode("decode_gqa8_b16_ctx4096", 16, 512, 4096, hq=64, hkv=8, bound=4096),
        # Long documents: a few requests up to the models' 40,960 positions, which also bound the launch.
        decode("decode_b4_ctx40960", 4, 8192, 40960, bound=40960),
        # Short follow-ups (a chat's next turn) on a cached conversation, in pages of 16 tokens.
        prefill("prefill_turns_b8", 8, 1, 64, cached=1040, block_size=16),
        # Prompts admitted at once behind a shared system prompt.
        prefill("prefill_prefix_b32_2048", 32, 512, 2048, cached=1152),
        # The rest of two long documents at five query heads per kv head.
        prefill("prefill_gqa5_b2_4000", 2, 3000, 4000, hq=40, hkv=8, cached=4096),
    ]


def store(name, tokens, hkv=8, block_size=128, pad=0):
    return _named(name, kind="store", tokens=tokens, hkv=hkv, block_size=block_size, pad=pad)


def rope(name, batch, lo, hi, hq=16, hkv=8, block_size=128, keys=False, pad=0):
    """Without ``keys`` one token per sequence (a decode step), with it every token of each (prompts)."""
    return _named(name, kind="rope", batch=batch, lo=lo, hi=hi, hq=hq, hkv=hkv, block_size=block_size, keys=keys,
                  pad=pad)


def decode(name, batch, lo, hi, hq=16, hkv=8, block_size=128, bound=0):
    return _named(name, kind="decode", batch=batch, lo=lo, hi=hi, hq=hq, hkv=hkv, block_size=block_size, bound=bound)


def prefill(name, batch, lo, hi, hq=16, hkv=8, block_size=128, cached=0):
    return _named(name, kind="prefill", batch=batch, lo=lo, hi=hi, hq=hq, hkv=hkv, block_size=block_size,
                  cached=cached)


def _named(name, **case):
    return {"name": name, **case} if name else case


HEADS = [(16, 8), (16, 8), (16, 8), (32, 8), (40, 8), (64, 8), (8, 8), (16, 4), (24, 8), (2, 1), (16, 1)]


def _log(rng, lo, hi) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(["store", "rope", "decode", "decode", "decode", "prefill", "prefill"])
    hq, hkv = rng.choice(HEADS)
    bs = rng.choice([128, 128, 128, 64, 32, 16, 256])
    if kind == "store":
        tokens = _log(rng, 1, 40_000)
        return store(None, tokens, hkv, bs, rng.choice([0, min(3, tokens - 1)]))
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
    hi = _log(rng, 4, 4000)
    cached = rng.choice([0, 16, 256, 1040, 4096])
    batch = _log(rng, 1, max(1, min(32, 24_000 // hi, 300_000_000 // (hi * (hi + cached) * hq // 8))))
    return prefill(None, batch, rng.choice([0, 1, hi // 2]), hi, hq, hkv, bs, cached)


# ------------------------------------------------------------------------------------------------ sizes
def _lens(case) -> list[int]:
    """Context lengths (decode; rope of single tokens) or new tokens (prefill, rope of prompts) of each sequence; one
    of them is the longest that the case allows."""
    rng = random.Random(1_000_003 * case["batch"] + 1_009 * case["lo"] + case["hi"])
    lens = [rng.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
    lens[rng.randrange(len(lens))] = case["hi"]
    return lens


def _tokens(case) -> int:
    """Rows of a store or rope case that have a slot."""
    if case["kind"] == "store":
        return case["tokens"] - case["pad"]
    return sum(_lens(case)) if case["keys"] else case["batch"]


def work(case) -> dict:
    hkv, row = case["hkv"], D // 2 + D // 32  # a row's bytes in the cache, of one head
    if case["kind"] in ("store", "rope"):
        t = _tokens(case)
        rows = t * hkv * (4 * D + 2 * row + 4 * D) + 8 * t  # k, v read; cache written; k, v of the cache returned
        if case["kind"] == "store":
            return {"bytes": rows, "flops": 4 * D * hkv * t}
        heads = t * (case["hq"] + (hkv if case["keys"] else 0))
        q_rows = 4 * D * t * case["hq"] + (2 * D * t * hkv if case["keys"] else 0) + 4 * D * t + 8 * t
        return {"bytes": rows + q_rows, "flops": 10 * D * (heads + 2 * t * hkv)}
    hq, lens = case["hq"], _lens(case)
    if case["kind"] == "decode":
        total = sum(lens)
        pages = -(-total // case["block_size"]) + len(lens)
        return {"bytes": 2 * row * hkv * total + 4 * D * hq * len(lens) + 4 * pages, "flops": 4 * D * hq * total}
    cached = case["cached"]
    pairs = sum(n * cached + n * (n + 1) // 2 for n in lens)
    total = sum(lens)
    return {"bytes": 2 * row * hkv * (total + cached * len(lens)) + 4 * D * hq * total, "flops": 4 * D * hq * pairs}


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
    """Codes and scales of keys and values, as bytes that no row has been written to, and the codes' values."""
    def byte(width):
        return torch.zeros((blocks, case["hkv"], case["block_size"], width), dtype=torch.uint8, device="cuda")

    return {"k_codes": byte(D // 2), "k_scales": byte(D // 32), "v_codes": byte(D // 2), "v_scales": byte(D // 32),
            "grid": torch.tensor(GRID + tuple(-x for x in GRID), device="cuda")}


def _channels(gen):
    """Every 16th channel of the keys, from a seeded one on, is four times as large."""
    at = torch.randint(0, 16, (1,), generator=gen, device="cuda")
    return torch.where(torch.arange(D, device="cuda") % 16 == at, 4.0, 1.0).bfloat16()


@torch.no_grad()
def prepare(case, seed) -> dict:
    return {"store": _prepare_rows, "rope": _prepare_rows, "decode": _prepare_attention,
            "prefill": _prepare_attention}[case["kind"]](case, seed)


def _prepare_rows(case, seed):
    gen, bs, hkv = _generator(seed), case["block_size"], case["hkv"]
    if case["kind"] == "store":
        lens = [case["tokens"] - case["pad"]]
        pos = torch.arange(lens[0])
        seq = torch.zeros_like(pos)
    else:
        lens = _lens(case)
        ends = torch.tensor([0] + lens).cumsum(0)
        if case["keys"]:
            seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
            pos = torch.arange(int(ends[-1])) - ends[seq]
        else:
            seq, pos = torch.arange(len(lens)), torch.tensor(lens) - 1
    blocks, tables = _pages(lens, bs, seed)
    slots = tables[seq, pos // bs].to(torch.int64) * bs + pos % bs
    slots = torch.cat([slots, torch.full((case["pad"],), -1)])  # rows of a padded batch have no slot
    pos = torch.cat([pos, torch.zeros(case["pad"], dtype=torch.int64)])
    hq, t = case.get("hq", 0), len(slots)
    qkv = _normal(gen, t, hq + 2 * hkv, D)
    qkv[:, hq:hq + hkv] *= _channels(gen)
    state = {"case": case, **_empty_cache(blocks, case), "slots": slots.cuda(), "q": qkv[:, :hq],
             "k": qkv[:, hq:hq + hkv], "v": qkv[:, hq + hkv:]}  # views into a fused projection's rows
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
    channels = _channels(gen)
    rows = max(1, (1 << 17) // bs) * bs  # fill the pool some tokens at a time
    for at in range(0, blocks * bs, rows):
        slots = torch.arange(at, min(at + rows, blocks * bs), device="cuda")
        k, v = (_normal(gen, len(slots), case["hkv"], D) for _ in range(2))
        _store(state, k * channels, v, slots)
    tokens = len(lens) if case["kind"] == "decode" else sum(lens)
    qkv = _normal(gen, max(tokens, 1), (case["hq"] + 2 * case["hkv"]), D)
    state.update(q=qkv[:tokens, : case["hq"]], tables=tables.cuda(),
                 kv_lens=torch.tensor(kv_lens, dtype=torch.int32).cuda())
    if case["kind"] == "prefill":
        state["cu"] = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    return state


# ------------------------------------------------------------------------------------------------ one pass
_layers = {}  # a program's attention layers, which keep their workspaces


def run(state):
    case = state["case"]
    if not own:
        return {"store": _plain_store, "rope": _plain_rope, "decode": _plain_decode, "prefill": _plain_prefill}[
            case["kind"]](state)
    from nano_vllm_ascend_amd import _C
    from nano_vllm_ascend_amd.layers import HipPagedAttention

    keys = _C.Fp4Pages(state["k_codes"], state["k_scales"])
    values = _C.Fp4Pages(state["v_codes"], state["v_scales"])
    if case["kind"] == "store":
        _C.kv_cache_write_fp4(state["k"], state["v"], keys, values, state["slots"])
        return _C.kv_cache_read_fp4(keys, values, state["slots"])
    if case["kind"] == "rope":
        _C.qk_norm_rope_fp4(state["q"], state["k"], state["v"], state["q_weight"], state["k_weight"],
                            state["positions"], state["table"], EPS, keys, values, state["slots"],
                            q_out=state["q_out"], k_out=state["k_out"])
        k_out = [] if state["k_out"] is None else [state["k_out"]]
        return [state["q_out"], *k_out, *_C.kv_cache_read_fp4(keys, values, state["slots"])]
    if case["kind"] == "prefill":
        out = torch.empty(state["q"].shape, dtype=torch.bfloat16, device="cuda")
        return _C.paged_prefill_fp4(out, state["q"], keys, values, state["tables"], state["cu"], state["kv_lens"],
                                    case["hi"], SCALE)
    heads = case["hq"], case["hkv"]
    if heads not in _layers:
        _layers[heads] = HipPagedAttention(*heads, D)
    return _layers[heads](state["q"], keys, values, state["tables"], state["kv_lens"],
                          max_context_len=max(case["bound"], case["hi"]))


def _quantise(x):
    """Codes [.., 4, 32] (0 .. 15) and scale bytes [.., 4] of bf16 rows [.., 128]."""
    x = x.float().unflatten(-1, (4, 32))
    u = x.abs()
    mantissa, exponent = torch.frexp(u.amax(-1))  # max = mantissa * 2^exponent, 0.5 <= mantissa < 1
    e = (exponent - 3 + (mantissa > 0.875).int()).clamp(-125, 125)
    fine = x.isfinite().all(-1)
    e = torch.where(fine, e, 0)
    u = torch.where(fine[..., None], torch.ldexp(u, -e[..., None]), 0.0)
    code = ((u > 0.25).to(torch.uint8) + (u >= 0.75) + (u > 1.25) + (u >= 1.75) + (u > 2.5) + (u >= 3.5) + (u > 5.0))
    return code + (x < 0).to(torch.uint8) * 8, torch.where(fine, e + 127, 255).to(torch.uint8)


def _at(state, slots):
    """Block, tile of its page and token of the tile of each slot; rows without one go to the pool's spare last slot."""
    bs = state["case"]["block_size"]
    slots = torch.where(slots < 0, state["k_codes"].shape[0] * bs - 1, slots)
    return slots // bs, slots % bs // 16, slots % 16


def _views(state):
    """The cache with its pages' tiles spelled out."""
    nb, hkv, bs, _ = state["k_codes"].shape
    return (state["k_codes"].view(nb, hkv, bs // 16, 16, 64), state["k_scales"].view(nb, hkv, bs // 16, 4, 4, 4),
            state["v_codes"].view(nb, hkv, bs // 16, 64, 16), state["v_scales"].view(nb, hkv, bs // 16, 4, 16))


def _store(state, k, v, slots):
    block, tile, t = _at(state, slots)
    kc, ks, vc, vs = _views(state)
    code, scale = _quantise(k)
    code = code.flatten(-2)
    kc[block, :, tile, t] = code[..., 0::2] | code[..., 1::2] << 4
    ks[block, :, tile, t % 4, :, t // 4] = scale
    code, scale = _quantise(v)
    vc[block, :, tile, :, t] = (code[..., :16] | code[..., 16:] << 4).flatten(-2)
    vs[block, :, tile, :, t] = scale


def _values(grid, code, scale):
    """fp32 values [.., 4, 32] of codes and scale bytes."""
    one = torch.ones_like(scale, dtype=torch.float32)
    step = torch.where(scale == 255, math.nan, torch.ldexp(one, scale.int() - 127))
    return grid[code.int()] * step[..., None]


def _load(state, slots):
    block, tile, t = _at(state, slots)
    kc, ks, vc, vs = _views(state)
    byte = kc[block, :, tile, t]
    k = _values(state["grid"], torch.stack((byte & 15, byte >> 4), -1).unflatten(-2, (4, 16)).flatten(-2),
                ks[block, :, tile, t % 4, :, t // 4])
    byte = vc[block, :, tile, :, t].unflatten(-1, (4, 16))
    v = _values(state["grid"], torch.cat((byte & 15, byte >> 4), -1), vs[block, :, tile, :, t])
    live = (slots >= 0)[:, None, None]
    return torch.where(live, k.flatten(-2), 0.0), torch.where(live, v.flatten(-2), 0.0)


def _plain_store(state):
    _store(state, state["k"], state["v"], state["slots"])
    return tuple(x.bfloat16() for x in _load(state, state["slots"]))


def _rounded(x):
    """bf16 of 64-bit values, rounded once (a cast by way of 32 bits rounds twice)."""
    mantissa, exponent = torch.frexp(x)
    return torch.ldexp((mantissa * 256).round(), exponent - 8).bfloat16()


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
    _store(state, k, state["v"], state["slots"])
    return [q, *([k] if state["case"]["keys"] else []), *(x.bfloat16() for x in _load(state, state["slots"]))]


def _context(state):
    """Keys and values in fp32 [sequences, kv heads, width of the table in tokens, 128]."""
    kc, ks, vc, vs = _views(state)
    tables = state["tables"].long()
    n, hkv = tables.shape[0], kc.shape[1]
    byte = kc[tables]  # [n, blocks, hkv, tiles, 16, 64]
    k = _values(state["grid"], torch.stack((byte & 15, byte >> 4), -1).unflatten(-2, (4, 16)).flatten(-2),
                ks[tables].permute(0, 1, 2, 3, 6, 4, 5).flatten(4, 5)).flatten(-2)
    byte = vc[tables].unflatten(-2, (4, 16))  # [n, blocks, hkv, tiles, 4, 16, 16]
    v = _values(state["grid"], torch.cat((byte & 15, byte >> 4), -2).permute(0, 1, 2, 3, 6, 4, 5),
                vs[tables].transpose(-1, -2)).flatten(-2)
    return (x.permute(0, 2, 1, 3, 4, 5).reshape(n, hkv, -1, D).contiguous() for x in (k, v))


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


# ------------------------------------------------------------------------------------------------ exact results
def _nearest(row):
    """Rows [.., 128] in 64 bits as a 4-bit cache holds them."""
    out = torch.empty_like(row)
    grid = torch.tensor(GRID, dtype=torch.float64, device=row.device)
    for q in range(4):
        x = row[..., 32 * q: 32 * q + 32]
        top = x.abs().max(dim=-1, keepdim=True).values
        step = torch.full_like(top, 2.0 ** -125)  # the least power of two that 7 steps of reach the maximum
        for e in range(-124, 126):
            step = torch.where(top > 7 * step, step * 2, step)
        u = x.abs() / step
        best = torch.zeros_like(u)
        for i in range(1, 8):  # nearer than the value below, or as near and of an even code
            above, below = (grid[i] - u).abs(), (u - grid[i - 1]).abs()
            best = torch.where((above < below) | ((above == below) & (i % 2 == 0)), grid[i], best)
        out[..., 32 * q: 32 * q + 32] = torch.where(top.isfinite(), best * step * x.sign(), math.nan)
    return out


def _bf16(x):
    """The bf16 number nearest to each 64-bit value, of two as near the one of even bits: of the cast's and its neighbours."""
    bits = x.bfloat16().view(torch.int16)
    near = torch.stack((bits, bits - 1, bits + 1), -1)
    off = (near.view(torch.bfloat16).double() - x[..., None]).abs()
    nearest = off == off.min(-1, keepdim=True).values
    pick = (2 * nearest.int() + (near % 2 == 0).int()).argmax(-1, keepdim=True)
    return near.gather(-1, pick)[..., 0].contiguous().view(torch.bfloat16).double()


def _cached(state, head, slots):
    """Keys and values [tokens, 128] of one kv head at the slots, in 64 bits, byte by byte."""
    bs, hkv = state["case"]["block_size"], state["case"]["hkv"]
    grid = torch.tensor(GRID + tuple(-x for x in GRID), dtype=torch.float64, device="cuda")
    page = ((slots // bs * hkv + head) * bs)[:, None]
    token = (slots % bs)[:, None]
    tile, t, d = page + token // 16 * 16, token % 16, torch.arange(D, device="cuda")[None]
    q, r = d // 32, d % 16

    def value(codes, at, high, scales, scale_at):
        byte = codes.flatten()[at].long()
        code = torch.where(high, byte // 16, byte % 16)
        return grid[code] * torch.pow(2.0, scales.flatten()[scale_at].double() - 127)

    return (value(state["k_codes"], 64 * (page + token) + d // 2, d % 2 == 1, state["k_scales"],
                  4 * tile + 16 * (t % 4) + 4 * q + t // 4),
            value(state["v_codes"], 64 * tile + 16 * (16 * q + r) + t, d % 32 >= 16, state["v_scales"],
                  4 * tile + 16 * q + t))


@torch.no_grad()
def exact(case, seed):
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
        none = state["slots"] < 0
        rows = [_nearest(_bf16(k) if case["kind"] == "rope" else k), _nearest(v)]  # what is stored is the bf16 key
        for x in rows:
            x[none] = 0
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
            k, v = _cached(state, g, slots)
            for h in range(g * group, g * group + group):
                weight = torch.softmax((q[a:b, h] @ k.T / math.sqrt(D)).masked_fill(hidden, -math.inf), -1)
                out[a:b, h] = weight @ v
    return out
