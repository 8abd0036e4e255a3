"""Attention over the KV cache held in 8 bits, against the 64-bit oracle on the values that the pages hold.

Tolerances are the bound that oracle.fp4_ref.attention derives for each element from the roundings that an evaluation with
bf16 weights and results makes."""
from __future__ import annotations

import math
import random

import pytest
import torch

from nano_vllm_ascend_amd import _C
from nano_vllm_ascend_amd.block_manager import PagedKVCacheMetadata
from nano_vllm_ascend_amd.layers import (HipBatchPrefillAttention, HipPagedAttention, RMSNorm, RotaryEmbedding,
                                         qk_norm_rope)
from nano_vllm_ascend_amd.paged_kv_cache import Fp8PagedKVCache
from oracle import fp4_ref, fp8_ref

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


@pytest.fixture(autouse=True)
def clean_word(device):
    _C.clear_index_errors()
    yield
    _C.clear_index_errors()
    torch.cuda.synchronize()


class Batch:
    """Sequences of the given contexts in pages of a seeded order; rows past a context and pages of nobody hold stale bytes,
    codes and scales of NaN among them."""

    def __init__(self, device, lens, hq, hkv, bs, seed=0, spread=0.5, extra_width=0):
        gen = torch.Generator().manual_seed(seed)
        need = [-(-n // bs) for n in lens]
        self.nb = sum(need) + 2
        order = torch.randperm(self.nb, generator=gen)
        self.tables = torch.zeros(len(lens), max(max(need), 1) + extra_width, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            self.tables[i, :n] = order[at:at + n]
            at += n
        self.pages = tuple(torch.randint(0, 256, p.shape, generator=gen, dtype=torch.uint8)
                           for p in fp8_ref.empty_pages(self.nb, hkv, bs))
        for p in self.pages[1::2]:
            p[p > 200] = 255
        self.slots = [self.tables[i, torch.arange(n) // bs].long() * bs + torch.arange(n) % bs
                      for i, n in enumerate(lens)]
        slots = torch.cat(self.slots)
        k, v = (torch.randn(len(slots), hkv, 128, generator=gen) for _ in range(2))
        k = k * torch.exp(spread * torch.randn(len(slots), hkv, 1, generator=gen))
        fp8_ref.write_sequences(self.pages, k.bfloat16(), v.bfloat16(), slots)
        self.lens, self.hq, self.hkv, self.bs, self.device, self.gen = lens, hq, hkv, bs, device, gen
        self.upload()

    def upload(self):
        kc, ks, vc, vs = (p.to(self.device) for p in self.pages)
        self.keys, self.values = _C.Fp8Pages(kc, ks), _C.Fp8Pages(vc, vs)

    def queries(self, t, scale=1.0):
        return (scale * torch.randn(t, self.hq, 128, generator=self.gen)).bfloat16()

    def want(self, i, q, scale=SCALE):
        """The last len(q) positions of sequence i."""
        k, v = fp8_ref.read_sequence(self.pages, self.slots[i])
        return fp4_ref.attention(q, k, v, scale)

    def decode(self, q, bound=None, scale=SCALE, out=None, workspace=None):
        bound = bound or max(max(self.lens), 1)
        if workspace is None:
            workspace = _C.alloc_paged_decode_workspace(len(self.lens), self.hq, self.hkv, bound, self.device)
        out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=self.device) if out is None else out
        return _C.paged_decode_fp8(out, q.to(self.device), self.keys, self.values, self.tables.to(self.device),
                                   torch.tensor(self.lens, dtype=torch.int32, device=self.device), scale, bound,
                                   workspace)

    def prefill(self, q, q_lens, out=None, max_q=None, scale=SCALE):
        cu = torch.tensor([0] + q_lens).cumsum(0).to(torch.int32).to(self.device)
        out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=self.device) if out is None else out
        if max_q == "strips":
            max_q = 65536 // (self.hq * len(self.lens))
        return _C.paged_prefill_fp8(out, q.to(self.device), self.keys, self.values, self.tables.to(self.device), cu,
                                    torch.tensor(self.lens, dtype=torch.int32, device=self.device),
                                    max_q or max(q_lens), scale)


def close(got, want, tol):
    got = got.cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    off = ((got - want).abs() - tol).nan_to_num(-1.0)
    assert off.max().item() <= 0, f"off by {off.max().item():.3g} over the bound at {off.argmax().item()}"


def check_decode(batch, q, got, scale=SCALE):
    for i, n in enumerate(batch.lens):
        if n == 0:
            assert not got[i].any()
            continue
        close(got[i:i + 1], *batch.want(i, q[i:i + 1], scale))


# -------------------------------------------------------------------------------------------- decode
@pytest.mark.parametrize("hq, hkv", [(1, 1), (2, 1), (16, 8), (6, 2), (4, 1), (5, 1), (16, 2), (15, 1), (16, 1), (17, 1),
                                     (40, 2)])
def test_decode_head_layouts(device, hq, hkv):
    batch = Batch(device, [1, 300, 0, 77, 64], hq, hkv, 32, seed=hq)
    q = batch.queries(5)
    check_decode(batch, q, batch.decode(q))
    assert _C.index_errors() == 0


@pytest.mark.parametrize("bs", [16, 32, 64, 128, 256])
def test_decode_contexts_around_tiles_pages_and_partitions(device, bs):
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513, 1023, 1024, 1025]
    batch = Batch(device, lens, 4, 2, bs, seed=bs)
    q = batch.queries(len(lens))
    check_decode(batch, q, batch.decode(q))
    check_decode(batch, q, batch.decode(q, bound=8192))  # a bound far past the contexts


@pytest.mark.parametrize("lens, hq, hkv", [([5000, 3], 2, 1), ([9001, 1, 0, 4097], 4, 2), ([40960], 2, 1),
                                           ([70000, 131072], 1, 1)])
def test_decode_long_contexts(device, lens, hq, hkv):
    batch = Batch(device, lens, hq, hkv, 128, seed=1)
    q = batch.queries(len(lens))
    check_decode(batch, q, batch.decode(q))


def test_decode_many_sequences(device):
    """More sequences than a wave's lanes, and enough partitions that they grow past the smallest."""
    gen = torch.Generator().manual_seed(3)
    lens = [int(x) for x in torch.randint(0, 700, (150,), generator=gen)]
    batch = Batch(device, lens, 2, 2, 16, seed=4)
    q = batch.queries(150)
    check_decode(batch, q, batch.decode(q))
    lens = [2600 + i for i in range(70)]
    batch = Batch(device, lens, 4, 4, 128, seed=5)  # 70 x 11 x 4 partitions of 256 tokens, were they that small
    q = batch.queries(70)
    check_decode(batch, q, batch.decode(q, bound=4096))


def test_decode_of_the_largest_batches(device):
    """16,384 units of a sequence and a kv head: each sequence's bits are those of a small batch."""
    gen = torch.Generator().manual_seed(39)
    lens = [int(x) for x in torch.randint(0, 40, (2048,), generator=gen)]
    batch = Batch(device, lens, 8, 8, 16, seed=40)
    q = batch.queries(2048)
    got = batch.decode(q, bound=4096)
    tables, dq, n = batch.tables.to(device), q.to(device), torch.tensor(lens, dtype=torch.int32, device=device)
    space = _C.alloc_paged_decode_workspace(100, 8, 8, 64, device)
    for at in (0, 1000, 1948):
        rows = slice(at, at + 100)
        few = _C.paged_decode_fp8(None, dq[rows], batch.keys, batch.values, tables[rows], n[rows], SCALE, 64, space)
        assert torch.equal(few, got[rows])
    for i in (0, 1, 1023, 2047):
        if lens[i]:
            close(got[i:i + 1], *batch.want(i, q[i:i + 1]))
    assert not got[n == 0].any() and _C.index_errors() == 0


def at_scale(batch, k_exp, v_exp):
    """The batch's rows with keys and values of about 2^k_exp and 2^v_exp."""
    slots = torch.cat(batch.slots)
    k, v = fp8_ref.read_sequence(batch.pages, slots)
    fp8_ref.write_sequences(batch.pages, (k * 2.0 ** k_exp).bfloat16(), (v * 2.0 ** v_exp).bfloat16(), slots)
    batch.upload()


EXPONENTS = pytest.mark.parametrize("q_exp, k_exp, v_exp", [(100, -100, 0), (-90, 90, 90), (-60, 60, -90), (0, 0, 100)])


@EXPONENTS
def test_decode_of_numbers_far_from_one(device, q_exp, k_exp, v_exp):
    batch = Batch(device, [1, 70, 600], 4, 2, 32, seed=41)
    at_scale(batch, k_exp, v_exp)
    q = batch.queries(3, scale=2.0 ** q_exp)
    check_decode(batch, q, batch.decode(q))


@pytest.mark.parametrize("hq, hkv", [(2, 1), (16, 8), (12, 2)])
def test_decode_beside_other_sequences(device, hq, hkv):
    """Contexts of up to 512 tokens give the same bits whatever runs beside them; of longer ones the cut, and with it the
    order of the sums, follows from all contexts of the call, within the bound."""
    lens = [512, 1, 3000, 200, 513, 5000] + [700] * 40
    batch = Batch(device, lens, hq, hkv, 64, seed=36)
    q = batch.queries(len(lens))
    whole = batch.decode(q)
    check_decode(batch, q, whole)
    tables, dq = batch.tables.to(device), q.to(device)
    for i in range(6):
        n = torch.tensor(lens[i:i + 1], dtype=torch.int32, device=device)
        space = _C.alloc_paged_decode_workspace(1, hq, hkv, 5000, device)
        alone = _C.paged_decode_fp8(None, dq[i:i + 1], batch.keys, batch.values, tables[i:i + 1], n, SCALE, 5000, space)
        close(alone, *batch.want(i, q[i:i + 1]))
        if lens[i] <= 512:
            assert torch.equal(alone[0], whole[i])


def test_decode_scores_far_apart(device):
    """A few keys carry all of the weight, in whichever partition they are; large and negative scales."""
    batch = Batch(device, [1500, 700], 4, 1, 64, seed=6, spread=1.5)
    q = batch.queries(2, scale=8.0)
    check_decode(batch, q, batch.decode(q))
    check_decode(batch, q, batch.decode(q, scale=-0.05), scale=-0.05)


def outliers(q):
    """A dim that is thousands of times the others, as some heads have."""
    q = q.clone()
    q[..., 5] *= 4000
    q[..., 100] *= 70
    return q


def test_decode_queries_with_outliers(device):
    """Keys without the outliers' dims: the scores come from what is left of the query."""
    batch = Batch(device, [900, 70], 4, 1, 64, seed=16)
    slots = torch.cat(batch.slots)
    k, v = fp8_ref.read_sequence(batch.pages, slots)
    k[..., 5] = k[..., 100] = 0
    fp8_ref.write_sequences(batch.pages, k.bfloat16(), v.bfloat16(), slots)
    batch.upload()
    q = outliers(batch.queries(2))
    check_decode(batch, q, batch.decode(q))


def test_decode_scores_below_any_reference(device):
    """Scores of about -1e31, all alike: every key weighs the same."""
    batch = Batch(device, [700, 40], 2, 1, 16, seed=17)
    slots = torch.cat(batch.slots)
    _, v = fp8_ref.read_sequence(batch.pages, slots)
    fp8_ref.write_sequences(batch.pages, torch.full((len(slots), 1, 128), -(2.0 ** 50)).bfloat16(), v.bfloat16(), slots)
    batch.upload()
    q = torch.full((2, 2, 128), 2.0 ** 50).bfloat16()
    got = batch.decode(q).cpu().double()
    for i, at in enumerate(batch.slots):
        _, v = fp8_ref.read_sequence(batch.pages, at)
        # equal weights are exact; 32-bit sums of up to 700 values, and one rounding
        tol = 2.0 ** -8 * v.mean(0).abs() + 1e-4 * v.abs().mean(0)
        assert ((got[i] - v.mean(0)).abs() <= tol).all()


def test_decode_replays_from_a_graph(device):
    """Contexts, tables and queries that change between the replays of a captured call."""
    batch = Batch(device, [1500, 33, 700], 4, 2, 16, seed=18)
    q = batch.queries(3).to(device)
    lens, tables = torch.tensor(batch.lens, dtype=torch.int32, device=device), batch.tables.to(device)
    out = torch.empty_like(q)
    spaces = [_C.alloc_paged_decode_workspace(3, 4, 2, 1500, device) for _ in range(2)]

    def call(out, space):
        return _C.paged_decode_fp8(out, q, batch.keys, batch.values, tables, lens, SCALE, 1500, space)

    call(out, spaces[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out, spaces[0])
    for now in ([1500, 33, 700], [3, 0, 64], [512, 1, 1], [1400, 20, 513]):
        q.copy_(batch.queries(3))
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        for _ in range(2):
            out.fill_(7.0)
            graph.replay()
            got = out.clone()
            torch.cuda.synchronize()
            assert torch.equal(got, call(torch.empty_like(q), spaces[1]))
        batch.lens, full, slots = now, batch.lens, batch.slots
        batch.slots = [s[:n] for s, n in zip(slots, now)]
        check_decode(batch, q.cpu(), got)
        batch.lens, batch.slots = full, slots


def test_decode_layer_keeps_a_captured_workspace(device):
    """A graph captured at a small batch replays right after the layer has served a larger one."""
    batch = Batch(device, [2000, 33, 700, 1100], 4, 2, 16, seed=19)
    layer = HipPagedAttention(4, 2, 128)
    lens, tables = torch.tensor(batch.lens, dtype=torch.int32, device=device), batch.tables.to(device)
    q = batch.queries(4).to(device)
    out = torch.empty_like(q)

    def call(n, out=None):
        return layer(q[:n], batch.keys, batch.values, tables[:n], lens[:n], max_context_len=2000, out=out)

    call(1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(1, out[:1])
    for _ in range(3):
        whole = call(4)
        junk = [torch.full((1 << 20,), 255, dtype=torch.uint8, device=device) for _ in range(4)]  # takes what was freed
        out.fill_(7.0)
        graph.replay()
        close(out[:1], *batch.want(0, q[:1].cpu()))
        assert out[1:].eq(7).all()
        del junk
    check_decode(batch, q.cpu(), whole)


def test_pages_past_32_bits(device):
    """Pages whose codes lie past 4 GiB, and rows of them written, read and attended to."""
    nb, bs, hkv = 2200, 256, 64
    cache = Fp8PagedKVCache(1, nb, bs, hkv, 128, device)
    assert cache.key_codes.nbytes > 1 << 32
    gen = torch.Generator().manual_seed(20)
    pages = torch.tensor([nb - 1, 0, nb // 2])
    n = 600
    slots = pages[torch.arange(n) // bs] * bs + torch.arange(n) % bs
    k, v = (torch.randn(n, hkv, 128, generator=gen).bfloat16() for _ in range(2))
    cache.write(0, k.to(device), v.to(device), slots.to(device))
    small = fp8_ref.empty_pages(3, hkv, bs)
    fp8_ref.write_sequences(small, k, v, torch.arange(n))
    kk, vv = fp8_ref.read_sequence(small, torch.arange(n))
    got = cache.read(0, slots.to(device))
    assert torch.equal(got[0].cpu().double(), kk) and torch.equal(got[1].cpu().double(), vv)
    q = torch.randn(n, hkv, 128, generator=gen).bfloat16()
    tables = pages.to(torch.int32)[None].to(device)
    lens = torch.tensor([n], dtype=torch.int32, device=device)
    keys, values = cache.get_physical_cache(0)
    for rows in (1, 20, 300):
        want, tol = fp4_ref.attention(q[:rows], kk, vv, SCALE)
        cu = torch.tensor([0, rows], dtype=torch.int32, device=device)
        out = torch.empty(rows, hkv, 128, dtype=torch.bfloat16, device=device)
        close(_C.paged_prefill_fp8(out, q[:rows].to(device), keys, values, tables, cu, lens, rows, SCALE), want, tol)
    want, tol = fp4_ref.attention(q[:1], kk, vv, SCALE)
    space = _C.alloc_paged_decode_workspace(1, hkv, hkv, n, device)
    close(_C.paged_decode_fp8(out[:1], q[:1].to(device), keys, values, tables, lens, SCALE, n, space), want, tol)


def test_decode_nan_reaches_only_its_sequence_and_dims(device):
    batch = Batch(device, [200, 300, 100], 2, 1, 32, seed=7)
    v = torch.ones(1, 1, 128, dtype=torch.bfloat16)
    bad_v, bad_k = v.clone(), v.clone()
    bad_v[0, 0, 70], bad_k[0, 0, 5] = math.inf, math.nan
    fp8_ref.write(batch.pages, v, bad_v, batch.slots[0][17:18])      # a value
    fp8_ref.write(batch.pages, bad_k, v, batch.slots[1][299:300])    # a key: every weight
    batch.upload()
    q = batch.queries(3)
    got = batch.decode(q)
    check_decode(batch, q, got)
    nan = got.isnan().cpu()
    assert nan[0, :, 70].all() and nan[0].sum() == 2
    assert nan[1].all() and not nan[2].any()


def test_a_nan_of_a_query_stays_in_its_row(device):
    batch = Batch(device, [150, 400], 4, 1, 16, seed=27)
    q = batch.queries(2)
    clean = batch.decode(q)
    q[1, 2, 77] = math.nan
    got = batch.decode(q)
    assert got[1, 2].isnan().all() and torch.equal(got[0], clean[0]) and torch.equal(got[1, :2], clean[1, :2])
    assert torch.equal(got[1, 3], clean[1, 3])
    q = batch.queries(200)
    for bound in (None, "strips", 60_000):
        clean = batch.prefill(q, [100, 100], max_q=bound)
        bad = q.clone()
        bad[130, 1, 3] = math.inf
        got = batch.prefill(bad, [100, 100], max_q=bound)
        assert got[130, 1].isnan().all()
        got[130, 1] = clean[130, 1]
        assert torch.equal(got, clean)


def test_decode_views_and_rows_behind_the_batch(device):
    batch = Batch(device, [40, 500], 6, 2, 16, seed=8, extra_width=3)
    fused = torch.zeros(2, 10, 128, dtype=torch.bfloat16)
    q = batch.queries(2)
    fused[:, 1:7] = q
    wide = torch.full((4, 9, 128), 7.0, dtype=torch.bfloat16, device=device)
    got = batch.decode(fused.to(device)[:, 1:7], out=wide[:2, 2:8])
    check_decode(batch, q, got)
    assert wide[2:].eq(7).all() and wide[:, :2].eq(7).all() and wide[:, 8:].eq(7).all()


def test_decode_bad_pages_and_contexts_stay_in_the_pool_and_are_reported(device):
    batch = Batch(device, [40, 500, 100], 2, 1, 16, seed=9)
    q = batch.queries(3)
    good = batch.decode(q)
    for entry in (batch.nb, -1, 1 << 30):
        batch.tables[1, 3] = entry
        got = batch.decode(q)
        assert _C.index_errors() == _C.ERR_BLOCK
        assert torch.equal(got[[0, 2]], good[[0, 2]])
        _C.clear_index_errors()
    batch.tables[1, 3] = 0
    for n in (-1, 513, 1 << 30):  # the table holds 512 tokens
        batch.lens[1] = n
        got = batch.decode(q, bound=1024)
        assert _C.index_errors() == _C.ERR_CONTEXT
        assert torch.equal(got[[0, 2]], good[[0, 2]])
        _C.clear_index_errors()
    batch.lens[1] = 500
    batch.decode(q, bound=400)  # the launch's bound holds less
    assert _C.index_errors() == _C.ERR_CONTEXT


def test_decode_is_the_same_whatever_runs_beside_it(device):
    """A replayed graph, a workspace that served other calls and repeated calls give the same bits."""
    batch = Batch(device, [40, 3000, 900], 8, 2, 64, seed=10)
    q = batch.queries(3).to(device)
    first = batch.decode(q)
    ws = _C.alloc_paged_decode_workspace(8, 16, 2, 8192, device)
    other = Batch(device, [700, 5000], 16, 2, 32, seed=11)
    for _ in range(3):
        other.decode(other.queries(2), workspace=ws)
        assert torch.equal(batch.decode(q, bound=4096, workspace=ws), first)
    tables, lens = batch.tables.to(device), torch.tensor(batch.lens, dtype=torch.int32, device=device)
    out = torch.empty_like(q)
    attn = HipPagedAttention(8, 2, 128)

    def call():
        return _C.paged_decode_fp8(out, q, batch.keys, batch.values, tables, lens, SCALE, 4096, ws)

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for n in (3000, 0, 17, 2999):
        lens[1] = n
        out.fill_(7.0)
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        batch.lens[1] = n
        assert torch.equal(got, attn(q, batch.keys, batch.values, tables, lens))
        check_decode(Window(batch, n), q.cpu(), got)


class Window:
    """A batch whose sequence 1 is cut to n tokens."""

    def __init__(self, batch, n):
        self.batch, self.lens = batch, [batch.lens[0], n, batch.lens[2]]

    def want(self, i, q, scale):
        k, v = fp8_ref.read_sequence(self.batch.pages, self.batch.slots[i][: self.lens[i]])
        return fp4_ref.attention(q, k, v, scale)


# -------------------------------------------------------------------------------------------- prefill
# The kernel follows the rows that a call's bounds allow: as many as there are, those of a middle size, of a large one.
BOUNDS = pytest.mark.parametrize("bound", [None, "strips", 60_000], ids=["exact", "strips", "tiles"])


def check_prefill(batch, q, q_lens, got, scale=SCALE):
    at = 0
    for i, n in enumerate(q_lens):
        if n:
            close(got[at:at + n], *batch.want(i, q[at:at + n], scale))
        at += n


@BOUNDS
@pytest.mark.parametrize("hq, hkv", [(1, 1), (2, 1), (3, 1), (4, 1), (5, 1), (16, 8), (8, 1), (14, 2), (17, 1), (40, 1)])
def test_prefill_head_layouts(device, hq, hkv, bound):
    q_lens, cached = [1, 40, 0, 130], [200, 16, 33, 0]
    batch = Batch(device, [a + b for a, b in zip(q_lens, cached)], hq, hkv, 32, seed=hq)
    q = batch.queries(sum(q_lens))
    check_prefill(batch, q, q_lens, batch.prefill(q, q_lens, max_q=bound))
    assert _C.index_errors() == 0


@BOUNDS
@pytest.mark.parametrize("bs", [16, 32, 64, 128, 256])
def test_prefill_lengths_around_tiles_and_pages(device, bs, bound):
    q_lens = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257]
    cached = [0, 1, 16, 31, 32, 5, 64, 100, 0, 128, 129, 1, 16, 300, 0, 255]
    batch = Batch(device, [a + b for a, b in zip(q_lens, cached)], 4, 2, bs, seed=bs)
    q = batch.queries(sum(q_lens))
    check_prefill(batch, q, q_lens, batch.prefill(q, q_lens, max_q=bound))


@pytest.mark.parametrize("bs", [16, 64])
def test_prefill_few_rows(device, bs):
    """Each alone, so that no call has more than a few rows."""
    for q_len, cached in ((1, 0), (1, 1), (2, 15), (3, 16), (15, 17), (16, 63), (17, 64), (31, 33), (33, 500), (64, 511),
                          (65, 512), (127, 3000), (256, 0), (300, 1)):
        batch = Batch(device, [q_len + cached], 4, 2, bs, seed=q_len)
        q = batch.queries(q_len)
        check_prefill(batch, q, [q_len], batch.prefill(q, [q_len]))


@pytest.mark.parametrize("hq, hkv, q_lens, cached, bs", [
    (16, 8, [20], [4096], 128),                    # few rows, 9 pieces
    (2, 1, [1, 3], [40_000, 5], 128),              # 32 pieces, and a context of one piece beside it
    (4, 1, [17, 0, 30], [5000, 100, 0], 16),       # a sequence without rows, one without cached keys
    (5, 1, [3], [511], 16), (5, 1, [3], [509], 16),  # two pieces, one
    (16, 8, [300], [4096], 128),                   # strips
    (6, 2, [300, 10, 100], [3000, 9000, 0], 16),
])
def test_prefill_cut_along_the_keys(device, hq, hkv, q_lens, cached, bs):
    batch = Batch(device, [a + b for a, b in zip(q_lens, cached)], hq, hkv, bs, seed=hq, extra_width=4096 // bs)
    width = batch.tables.shape[1]
    assert _C.load().nvamd_paged_prefill_fp8_workspace_size(len(q_lens), max(q_lens), hq, hkv, bs, width) > 0
    q = batch.queries(sum(q_lens))
    got = batch.prefill(q, q_lens)
    check_prefill(batch, q, q_lens, got)
    assert torch.equal(got, batch.prefill(q, q_lens)) and _C.index_errors() == 0


def test_prefill_cut_replays_from_a_graph(device):
    """Contexts that need one piece or many between the replays, and another call on another stream meanwhile."""
    batch = Batch(device, [9000, 300], 4, 2, 16, seed=9)
    q = batch.queries(40).to(device)
    cu = torch.tensor([0, 30, 40], dtype=torch.int32, device=device)
    lens, tables = torch.tensor(batch.lens, dtype=torch.int32, device=device), batch.tables.to(device)
    out = torch.empty_like(q)

    def call(out):
        return _C.paged_prefill_fp8(out, q, batch.keys, batch.values, tables, cu, lens, 32, SCALE)

    call(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    side = torch.cuda.Stream()
    for now in ([9000, 300], [40, 10], [700, 200], [8999, 12]):
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        torch.cuda.synchronize()
        out.fill_(7.0)
        graph.replay()
        with torch.cuda.stream(side):
            beside = call(torch.empty_like(q))
        torch.cuda.synchronize()
        assert torch.equal(out, beside)
        for i, (n, rows) in enumerate(zip(now, (slice(0, 30), slice(30, 40)))):
            k, v = fp8_ref.read_sequence(batch.pages, batch.slots[i][:n])
            close(out[rows], *fp4_ref.attention(q[rows].cpu(), k, v, SCALE))


@BOUNDS
@pytest.mark.parametrize("q_len, cached", [(1, 9000), (600, 4096), (1500, 0)])
def test_prefill_long(device, q_len, cached, bound):
    batch = Batch(device, [q_len + cached, 1], 2, 1, 128, seed=2)
    q = batch.queries(q_len + 1)
    check_prefill(batch, q, [q_len, 1], batch.prefill(q, [q_len, 1], max_q=bound))


@BOUNDS
def test_prefill_scores_far_apart(device, bound):
    """Maxima that rise along the keys, so that the running reference moves again and again."""
    batch = Batch(device, [400, 90], 2, 1, 16, seed=3, spread=1.5)
    q = batch.queries(300 + 90, scale=8.0)
    check_prefill(batch, q, [300, 90], batch.prefill(q, [300, 90], max_q=bound))


@BOUNDS
def test_prefill_rows_do_not_follow_their_neighbours(device, bound):
    """A row whose reference moves often, or whose scores overflow, leaves the bits of those beside it as they are."""
    batch = Batch(device, [200, 700], 4, 2, 16, seed=31, spread=1.5)
    q = batch.queries(300)
    clean = batch.prefill(q, [100, 200], max_q=bound)
    loud = q.clone()
    loud[1::4] *= 40
    loud[3::8] = 3e38
    got = batch.prefill(loud, [100, 200], max_q=bound)
    assert torch.equal(got[0::2], clean[0::2]) and not torch.equal(got[1::4], clean[1::4])


@BOUNDS
@EXPONENTS
def test_prefill_of_numbers_far_from_one(device, q_exp, k_exp, v_exp, bound):
    batch = Batch(device, [1, 70, 300], 4, 2, 32, seed=42)
    at_scale(batch, k_exp, v_exp)
    q = batch.queries(1 + 33 + 40, scale=2.0 ** q_exp)
    check_prefill(batch, q, [1, 33, 40], batch.prefill(q, [1, 33, 40], max_q=bound))


@BOUNDS
def test_prefill_queries_with_outliers(device, bound):
    batch = Batch(device, [300, 70], 4, 1, 64, seed=15)
    slots = torch.cat(batch.slots)
    k, v = fp8_ref.read_sequence(batch.pages, slots)
    k[..., 5] = k[..., 100] = 0
    fp8_ref.write_sequences(batch.pages, k.bfloat16(), v.bfloat16(), slots)
    batch.upload()
    q = outliers(batch.queries(150))
    check_prefill(batch, q, [100, 50], batch.prefill(q, [100, 50], max_q=bound))


@BOUNDS
def test_prefill_nan_reaches_the_rows_that_see_its_key_alone(device, bound):
    batch = Batch(device, [150, 150], 2, 1, 16, seed=4)
    one = torch.ones(1, 1, 128, dtype=torch.bfloat16)
    bad_v, bad_k = one.clone(), one.clone()
    bad_v[0, 0, 40], bad_k[0, 0, 100] = -math.inf, math.inf
    for at in (109, 115):  # two of a tile, the first of them in a page's last
        fp8_ref.write(batch.pages, one, bad_v, batch.slots[0][at:at + 1])
    fp8_ref.write(batch.pages, bad_k, one, batch.slots[1][120:121])
    batch.upload()
    q = batch.queries(150)  # 50 rows of the first sequence, from position 100 on, and 100 of the second, from 50 on
    got = batch.prefill(q, [50, 100], max_q=bound)
    check_prefill(batch, q, [50, 100], got)
    nan = got.isnan().cpu()
    assert not nan[:9].any() and nan[9:50, :, 40].all() and nan[9:50].sum() == 41 * 2
    assert not nan[50:120].any() and nan[120:].all()


@BOUNDS
def test_prefill_views_and_rows_behind_the_last_sequence(device, bound):
    batch = Batch(device, [40, 70], 3, 1, 16, seed=5)
    fused = torch.zeros(60, 5, 128, dtype=torch.bfloat16)
    q = batch.queries(50)
    fused[:50, 1:4] = q
    wide = torch.full((60, 5, 128), 7.0, dtype=torch.bfloat16, device=device)
    batch.prefill(fused.to(device)[:, 1:4], [20, 30], out=wide[:, 2:], max_q=bound)
    check_prefill(batch, q, [20, 30], wide[:50, 2:])
    assert wide[50:].eq(7).all() and wide[:, :2].eq(7).all()


@BOUNDS
def test_prefill_faults_are_reported_and_leave_the_others_alone(device, bound):
    batch = Batch(device, [100, 60, 200], 2, 1, 16, seed=6)
    q_lens = [20, 60, 100]
    q = batch.queries(180)
    good = batch.prefill(q, q_lens, max_q=bound)
    others = torch.cat([torch.arange(20), torch.arange(80, 180)])
    batch.tables[1, 2] = batch.nb
    got = batch.prefill(q, q_lens, max_q=bound)
    assert _C.index_errors() == _C.ERR_BLOCK and torch.equal(got[others], good[others])
    _C.clear_index_errors()
    batch.tables[1, 2] = 0
    for n in (59, 0, -1, 1 << 20):  # fewer keys than rows; more than the table holds
        batch.lens[1] = n
        got = batch.prefill(q, q_lens, max_q=bound)
        assert _C.index_errors() == _C.ERR_CONTEXT and torch.equal(got[others], good[others])
        if n <= 0:
            assert not got[20:80].any()  # rows that see no key
        _C.clear_index_errors()
    batch.lens[1] = 60
    cu = torch.tensor([0, 20, 80, 181], dtype=torch.int32, device=device)  # one row past the last
    out = torch.full((180, 2, 128), 7.0, dtype=torch.bfloat16, device=device)
    args = (batch.keys, batch.values, batch.tables.to(device), cu,
            torch.tensor(batch.lens, dtype=torch.int32, device=device))
    _C.paged_prefill_fp8(out, q.to(device), *args, 65536 // 6 if bound == "strips" else bound or 101, SCALE)
    assert _C.index_errors() == _C.ERR_CONTEXT
    assert torch.equal(out[:20], good[:20]) and out[80:].eq(7).all()


def test_prefill_bound_below_a_length_is_reported(device):
    batch = Batch(device, [100], 2, 1, 16, seed=6)
    q = batch.queries(50)
    batch.prefill(q, [50], max_q=49)
    assert _C.index_errors() == _C.ERR_CONTEXT


def test_prefill_replays_from_a_graph(device):
    batch = Batch(device, [100, 333], 4, 2, 16, seed=7)
    q = batch.queries(130).to(device)
    cu = torch.tensor([0, 30, 130], dtype=torch.int32, device=device)
    lens, tables = torch.tensor(batch.lens, dtype=torch.int32, device=device), batch.tables.to(device)
    out = torch.empty_like(q)

    def call(out):
        return _C.paged_prefill_fp8(out, q, batch.keys, batch.values, tables, cu, lens, 120, SCALE)  # 10 .. 120 rows

    call(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for seed in range(3):
        q.copy_(batch.queries(130))
        cu[1] = 10 + 20 * seed
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, call(torch.empty_like(q)))


# -------------------------------------------------------------------------------------------- bytes that nobody wrote
def with_stale_scales(batch, byte):
    """The batch's rows in pages whose other scale bytes are all `byte`, over random codes."""
    k, v = fp8_ref.read_sequence(batch.pages, torch.cat(batch.slots))
    for p in batch.pages[1::2]:
        p.fill_(byte)
    fp8_ref.write_sequences(batch.pages, k.bfloat16(), v.bfloat16(), torch.cat(batch.slots))
    batch.upload()


@BOUNDS
@pytest.mark.parametrize("byte", [0, 201, 252, 253, 254, 255])
def test_prefill_reads_no_value_past_the_keys(device, byte, bound):
    """Whatever scales unwritten tiles have; the codes behind a tile's tokens are random, NaNs among them."""
    q_lens, cached = [1, 40, 130, 20], [200, 17, 1, 0]
    batch = Batch(device, [a + b for a, b in zip(q_lens, cached)], 4, 2, 32, seed=28)
    with_stale_scales(batch, byte)
    q = batch.queries(sum(q_lens))
    check_prefill(batch, q, q_lens, batch.prefill(q, q_lens, max_q=bound))


@pytest.mark.parametrize("byte", [0, 201, 252, 253, 254, 255])
def test_decode_reads_no_value_past_the_context(device, byte):
    batch = Batch(device, [1, 40, 131, 530, 0, 65], 4, 2, 32, seed=29)
    with_stale_scales(batch, byte)
    q = batch.queries(6)
    check_decode(batch, q, batch.decode(q))


# -------------------------------------------------------------------------------------------- a whole decode step
def step_of(batch, seed, slots=None):
    """Projected rows of a new token for each sequence of the batch, whose last position is the token's."""
    gen = torch.Generator().manual_seed(seed)
    b = len(batch.lens)
    qkv = torch.randn(b, batch.hq + 2 * batch.hkv, 128, generator=gen).bfloat16().to(batch.device)
    q, k, v = qkv.split([batch.hq, batch.hkv, batch.hkv], 1)
    weights = [(1 + 0.1 * torch.randn(128, generator=gen)).bfloat16().to(batch.device) for _ in range(2)]
    angle = torch.rand(64, 64, generator=gen) * 7
    table = torch.cat((angle.cos(), angle.sin()), 1).to(batch.device)
    pos = torch.randint(0, 64, (b,), generator=gen).to(batch.device)
    if slots is None:
        slots = torch.stack([s[-1] if len(s) else torch.tensor(-1) for s in batch.slots])
    return q, k, v, *weights, pos, table, 1e-6, batch.keys, batch.values, slots.to(batch.device)


def attend(batch, q, bound, workspace, fused=None):
    tables, lens = batch.tables.to(batch.device), torch.tensor(batch.lens, dtype=torch.int32, device=batch.device)
    if fused is None:
        return _C.paged_decode_fp8(None, q, batch.keys, batch.values, tables, lens, SCALE, bound, workspace)
    return _C.paged_decode_fused_fp8(q, *fused, tables, lens, SCALE, bound, workspace)


def in_pages(batch):
    return [t.clone() for t in (*batch.keys, *batch.values)]


@pytest.mark.parametrize("hq, hkv, bs", [(16, 8, 128), (1, 1, 16), (12, 4, 32), (8, 1, 64), (40, 8, 16), (17, 1, 256),
                                         (34, 2, 128)])
def test_fused_step_has_the_bits_of_the_two_launches(device, hq, hkv, bs):
    batch = Batch(device, [1, 16, 17, 300, 0, 512, 513, 1100, 4097], hq, hkv, bs, seed=hq + bs)
    space = _C.alloc_paged_decode_workspace(9, hq, hkv, 8192, device)
    for bound in (4097, 8192):
        batch.upload()
        args = step_of(batch, seed=bound)
        raw = [t.clone() for t in args[:3]]
        want = attend(batch, _C.qk_norm_rope_fp8(*args), bound, space)
        stored = in_pages(batch)
        batch.upload()
        got = attend(batch, None, bound, space, fused=step_of(batch, seed=bound))
        assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(in_pages(batch), stored))
        assert all(torch.equal(a, b) for a, b in zip(args[:3], raw))
    assert _C.index_errors() == 0


@pytest.mark.parametrize("hq, hkv, bs", [(16, 8, 128), (34, 2, 32), (1, 1, 16)])
def test_fused_step_may_write_over_its_queries(device, hq, hkv, bs):
    """out is q itself, a view into the projection's rows: k and v beside it stay as they are."""
    batch = Batch(device, [1, 300, 0, 513, 4097], hq, hkv, bs, seed=37)
    space = _C.alloc_paged_decode_workspace(5, hq, hkv, 4097, device)
    args = step_of(batch, seed=38)
    want = attend(batch, None, 4097, space, fused=args)
    batch.upload()
    q, k, v, *rest = step_of(batch, seed=38)
    kv = k.clone(), v.clone()
    got = _C.paged_decode_fused_fp8(q, q, k, v, *rest, batch.tables.to(device),
                                    torch.tensor(batch.lens, dtype=torch.int32, device=device), SCALE, 4097, space)
    assert got is q and torch.equal(q, want) and torch.equal(k, kv[0]) and torch.equal(v, kv[1])


def test_fused_step_reports_what_it_skips_and_clamps(device):
    batch = Batch(device, [30, 40, 50], 4, 2, 16, seed=24)
    space = _C.alloc_paged_decode_workspace(3, 4, 2, 64, device)
    slots = torch.stack([s[-1] for s in batch.slots])
    before = in_pages(batch)
    for bad, word in ((torch.tensor(-1), 0), (torch.tensor(-2), _C.ERR_SLOT), (torch.tensor(batch.nb * 16), _C.ERR_SLOT)):
        attend(batch, None, 64, space, fused=step_of(batch, 25, slots=torch.stack([bad] * 3)))
        assert _C.index_errors() == word and all(torch.equal(a, b) for a, b in zip(in_pages(batch), before))
        _C.clear_index_errors()
    args = list(step_of(batch, 26, slots=slots))
    good = attend(batch, None, 64, space, fused=args)
    args[5] = args[5].clone()
    args[5][1] = 64
    got = attend(batch, None, 64, space, fused=args)
    assert _C.index_errors() == _C.ERR_POSITION and torch.equal(got[::2], good[::2])


# -------------------------------------------------------------------------------------------- the two routes of a call
def test_a_call_made_at_once_equals_one_that_python_checks(device):
    """Range checks send the calls through the checks of _C.py; without them csrc/calls.cpp makes those that are plain."""
    batch = Batch(device, [300, 5000, 20], 4, 2, 16, seed=21, extra_width=300)
    gen = torch.Generator().manual_seed(22)
    qkv = torch.randn(9, 8, 128, generator=gen).bfloat16().to(device)
    q, k, v = qkv.split([4, 2, 2], 1)
    weights = [torch.rand(128, generator=gen).bfloat16().to(device) for _ in range(2)]
    table = torch.randn(64, 128, generator=gen).to(device)
    pos = torch.arange(9, device=device)
    slots = batch.slots[0][:9].to(device)
    slots[8] = -1
    lens = torch.tensor(batch.lens, dtype=torch.int32, device=device)
    tables = batch.tables.to(device)
    cu = torch.tensor([0, 4, 8, 9], dtype=torch.int32, device=device)
    space = _C.alloc_paged_decode_workspace(3, 4, 2, 5000, device)

    def results():
        batch.upload()
        pages = batch.keys, batch.values
        got = [_C.paged_decode_fp8(None, q[:3], *pages, tables, lens, SCALE, 5000, space),
               _C.paged_decode_fp8(torch.empty(3, 4, 128, dtype=torch.bfloat16, device=device), q[:3], *pages, tables, lens,
                                   SCALE, 5000, space),
               _C.paged_prefill_fp8(torch.empty(9, 4, 128, dtype=torch.bfloat16, device=device), q, *pages, tables, cu, lens,
                                    4, SCALE)]
        _C.kv_cache_write_fp8(k, v, *pages, slots)
        got += [*pages[0], *pages[1], *_C.kv_cache_read_fp8(*pages, slots)]
        k_out = torch.zeros(9, 2, 128, dtype=torch.bfloat16, device=device)
        got.append(_C.qk_norm_rope_fp8(q, k, v, *weights, pos, table, 1e-6, *pages, slots, k_out=k_out))
        got.append(_C.qk_norm_rope_fp8(q, k, v, *weights, pos, table, 1e-6, *pages, slots, q_out=torch.empty_like(got[-1])))
        last = torch.stack([s[-1] for s in batch.slots]).to(device)
        fused = q[:3], k[:3], v[:3], *weights, pos[:3], table, 1e-6, *pages, last, tables, lens, SCALE, 5000, space
        got += [_C.paged_decode_fused_fp8(None, *fused), _C.paged_decode_fused_fp8(torch.empty_like(got[0]), *fused)]
        return [t.clone() for t in (*got, k_out, *pages[0], *pages[1])]

    at_once = results()
    before = _C.set_range_checks(True)
    try:
        checked = results()
    finally:
        _C.set_range_checks(before)
    assert len(at_once) == len(checked) and all(torch.equal(a, b) for a, b in zip(at_once, checked))


def test_what_the_library_refuses_raises(device):
    batch = Batch(device, [30], 2, 1, 16, seed=23)
    q = batch.queries(1).to(device)
    with pytest.raises(ValueError, match="workspace"):
        batch.decode(q, workspace=torch.zeros(64, dtype=torch.uint8, device=device))
    with pytest.raises(ValueError, match="invalid argument"):
        batch.prefill(q, [1], scale=-1.0)
    with pytest.raises(ValueError, match="invalid argument"):
        _C.kv_cache_write_fp8(q[:, :1].expand(4, 1, 128), q[:, :1].expand(4, 1, 128), batch.keys, batch.values,
                              torch.arange(4, device=device))
    with pytest.raises(ValueError, match="on one device|GPU"):
        _C.kv_cache_write_fp8(q[:, :1].cpu(), q[:, :1].cpu(), batch.keys, batch.values, torch.arange(1, device=device))


def irregular(name, x):
    """What an argument must not be: on the host, of another type, a row short, not dense."""
    if isinstance(x, _C.Fp8Pages):
        for i, t in enumerate(x):
            for how, bad in irregular(name, t):
                yield f"{x._fields[i]} {how}", x._replace(**{x._fields[i]: bad})
        yield "a plain tuple", tuple(x)
        return
    yield "on the host", x.cpu()
    if name != "workspace":
        yield "of another type", x.to(torch.float64)
        if name not in ("cos_sin", "cu_seqlens_q"):
            yield "a row short", x[:-1]
    if x.dim() == 1:
        yield "with gaps", x.repeat_interleave(2)[::2]
    else:
        yield "with gaps", x.repeat_interleave(2, -1)[..., ::2]


@pytest.mark.parametrize("name", ["write", "read", "rope", "decode", "decode_fused", "prefill"])
def test_what_the_checks_refuse_is_not_called_at_once(device, name):
    """csrc/calls.cpp leaves each call that _C.py refuses to it."""
    batch = Batch(device, [40, 33, 20], 4, 2, 16, seed=34)
    q, k, v, qw, kw, pos, table, eps, keys, values, slots = step_of(batch, 35)
    lens = torch.tensor(batch.lens, dtype=torch.int32, device=device)
    tables = batch.tables.to(device)
    cu = torch.arange(4, dtype=torch.int32, device=device)
    space = _C.alloc_paged_decode_workspace(3, 4, 2, 64, device)
    out = torch.empty_like(q)
    rope = dict(q=q, k=k, v=v, q_weight=qw, k_weight=kw, positions=pos, cos_sin=table, eps=eps)
    pages = dict(key_pages=keys, value_pages=values)
    where = dict(block_tables=tables, context_lens=lens, scale=SCALE, max_context_len=64, workspace=space)
    call, args = {
        "write": (_C.kv_cache_write_fp8, dict(key_states=k, value_states=v, **pages, slot_mapping=slots)),
        "read": (_C.kv_cache_read_fp8, dict(**pages, slot_mapping=slots)),
        "rope": (_C.qk_norm_rope_fp8, dict(**rope, **pages, slot_mapping=slots, q_out=out, k_out=torch.empty_like(k))),
        "decode": (_C.paged_decode_fp8, dict(out=out, q=q, **pages, **where)),
        "decode_fused": (_C.paged_decode_fused_fp8, dict(out=out, **rope, **pages, slot_mapping=slots, **where)),
        "prefill": (_C.paged_prefill_fp8, dict(out=out, q=q, **pages, block_tables=tables, cu_seqlens_q=cu, kv_lens=lens,
                                               max_q_len=1, scale=SCALE)),
    }[name]
    at_once = getattr(_C._calls, name)
    assert type(at_once(*args.values())) not in (type(None), int)
    for arg, x in args.items():
        if name == "read" and arg == "slot_mapping":
            cases = [c for c in irregular(arg, x) if c[0] != "a row short"]  # as many rows as there are slots
        else:
            cases = irregular(arg, x) if isinstance(x, (torch.Tensor, _C.Fp8Pages)) else ()
        for how, bad in cases:
            changed = {**args, arg: bad}
            assert at_once(*changed.values()) is None, (arg, how)
            with pytest.raises(ValueError):
                call(**changed)
    assert _C.index_errors() == 0


def test_calls_without_the_extension(device, monkeypatch):
    """Where csrc/calls.cpp cannot be used the same calls are made from Python."""
    batch = Batch(device, [300, 20], 4, 2, 16, seed=32)
    q = batch.queries(2)
    step = step_of(batch, 33)
    space = _C.alloc_paged_decode_workspace(2, 4, 2, 512, device)
    slots = torch.stack([s[-1] for s in batch.slots]).to(device)

    def results():
        batch.upload()
        args = (*step[:8], batch.keys, batch.values, slots)
        got = [batch.decode(q, bound=512), batch.prefill(q, [1, 1]), attend(batch, None, 512, space, fused=args)]
        batch.upload()
        args = (*step[:8], batch.keys, batch.values, slots)
        got.append(_C.qk_norm_rope_fp8(*args))
        got += _C.kv_cache_read_fp8(batch.keys, batch.values, slots)
        _C.kv_cache_write_fp8(step[1], step[2], batch.keys, batch.values, slots)
        return got + in_pages(batch)

    want = results()
    monkeypatch.setattr(_C, "_calls", None)
    assert all(torch.equal(a, b) for a, b in zip(results(), want))


def test_block_tables_whose_rows_overlap_are_refused_on_either_route(device):
    batch = Batch(device, [40, 33, 20], 4, 2, 16, seed=30)
    q, step = batch.queries(3).to(device), step_of(batch, 31)
    lens = torch.tensor(batch.lens, dtype=torch.int32, device=device)
    cu = torch.arange(4, dtype=torch.int32, device=device)
    space = _C.alloc_paged_decode_workspace(3, 4, 2, 64, device)
    pages = batch.keys, batch.values
    shared = batch.tables[:1].to(device).expand(3, -1)
    calls = {
        "decode": (_C.paged_decode_fp8, (None, q, *pages, shared, lens, SCALE, 64, space)),
        "decode_fused": (_C.paged_decode_fused_fp8, (None, *step, shared, lens, SCALE, 64, space)),
        "prefill": (_C.paged_prefill_fp8, (torch.empty_like(q), q, *pages, shared, cu, lens, 1, SCALE)),
    }
    for name, (call, args) in calls.items():
        assert getattr(_C._calls, name)(*args) is None  # left to the checks, which name what is wrong
        for checks in (False, True):
            before = _C.set_range_checks(checks)
            try:
                with pytest.raises(ValueError, match="block_tables overlap"):
                    call(*args)
            finally:
                _C.set_range_checks(before)
    whole = _C.paged_decode_fp8(None, q, *pages, shared.contiguous(), lens, SCALE, 64, space)
    one = batch.tables[0].to(device).expand(1, -1)  # a single row, whatever its stride
    assert torch.equal(_C.paged_decode_fp8(None, q[:1], *pages, one, lens[:1], SCALE, 64, space), whole[:1])


# -------------------------------------------------------------------------------------------- drawn calls
HEADS = [(1, 1), (16, 8), (14, 2), (12, 4), (40, 8), (32, 4), (7, 7), (33, 1)]


def some_length(rng, most):
    return rng.choice([0, 1, 16, rng.randint(1, 40), int(2 ** rng.uniform(0, math.log2(most)))])


@pytest.mark.parametrize("seed", range(10))
def test_decode_of_a_drawn_batch(device, seed):
    rng = random.Random(seed)
    hq, hkv = rng.choice(HEADS)
    batch = Batch(device, [some_length(rng, 6000) for _ in range(rng.randint(1, 20))], hq, hkv,
                  rng.choice([16, 32, 64, 128, 256]), seed=seed, extra_width=rng.choice([0, 5]))
    q = batch.queries(len(batch.lens))
    check_decode(batch, q, batch.decode(q, bound=rng.choice([None, 8192, 131072])))
    assert _C.index_errors() == 0


@pytest.mark.parametrize("seed", range(12))
def test_prefill_of_a_drawn_batch(device, seed):
    rng = random.Random(100 + seed)
    hq, hkv = rng.choice(HEADS)
    most = 2000 // hq + 20
    q_lens = [some_length(rng, most) for _ in range(rng.randint(1, 6))]
    lens = [n + some_length(rng, 3000) for n in q_lens]
    bs = rng.choice([16, 32, 64, 128, 256])
    batch = Batch(device, lens, hq, hkv, bs, seed=seed, extra_width=rng.choice([0, 8192 // bs]))
    q = batch.queries(sum(q_lens))
    bound = max(max(q_lens), 1)
    check_prefill(batch, q, q_lens, batch.prefill(q, q_lens, max_q=rng.choice([bound, bound, 4 * bound, bound + 1000, 20_000])))
    assert _C.index_errors() == 0


# -------------------------------------------------------------------------------------------- as they are used together
def test_prompt_then_decode_steps(device):
    """The layers as the model calls them: a prompt's rows are stored, a follow-up attends through the cache, decode steps
    store their row and attend."""
    hq, hkv, bs, nb = 8, 2, 16, 12
    cache = Fp8PagedKVCache(2, nb, bs, hkv, 128, device)
    pages = fp8_ref.empty_pages(nb, hkv, bs)
    norms = [RMSNorm(128, 1e-6).to(device, torch.bfloat16) for _ in range(2)]
    rotary = RotaryEmbedding(128, 512, 1e6).to(device)
    prefill, decode = HipBatchPrefillAttention(hq, hkv, 128, bs, 512), HipPagedAttention(hq, hkv, 128)
    gen = torch.Generator().manual_seed(1)
    order = torch.randperm(nb, generator=gen)
    tables = torch.stack([order[:6], order[6:]]).to(torch.int32)
    done = [0, 0]

    def step(new):
        """The rows of `new[i]` more tokens of each sequence, as projected; returns what the oracle makes of them."""
        pos = torch.cat([torch.arange(a, a + n) for a, n in zip(done, new)])
        seq = torch.repeat_interleave(torch.arange(2), torch.tensor(new))
        slots = tables[seq, pos // bs].long() * bs + pos % bs
        qkv = torch.randn(sum(new), hq + 2 * hkv, 128, generator=gen).bfloat16()
        q, k, v = qkv.split([hq, hkv, hkv], 1)
        q, k = (fp4_ref.to_bf16(fp4_ref.norm_rope(x, m.weight.cpu(), pos, rotary.cos_sin.cpu(), 1e-6))
                for x, m in zip((q, k), norms))
        fp8_ref.write(pages, k, v, slots)
        outs, tols, at = [], [], 0
        for i, n in enumerate(new):
            done[i] += n
            seen = torch.arange(done[i])
            kk, vv = fp8_ref.read_sequence(pages, tables[i, seen // bs].long() * bs + seen % bs)
            out, tol = fp4_ref.attention(q[at:at + n], kk, vv, SCALE)
            outs.append(out)
            tols.append(tol)
            at += n
        return qkv.to(device).split([hq, hkv, hkv], 1), pos.to(device), slots.to(device), torch.cat(outs), torch.cat(tols)

    for new in ([20, 37], [33, 5]):
        (q, k, v), pos, slots, want, tol = step(new)
        qk_norm_rope(q, k, v, *norms, rotary, pos, cache, 1, slots)
        md = PagedKVCacheMetadata(block_tables=tables.to(device), slot_mapping=slots, max_query_len=max(new),
                                  context_lens=torch.tensor(done, dtype=torch.int32, device=device),
                                  cu_seqlens_q=torch.tensor([0, new[0], sum(new)], dtype=torch.int32, device=device),
                                  use_paged_prefill=True)
        close(prefill(q, k, v, md, *cache.get_physical_cache(1)), want, tol)
    for _ in range(4):
        (q, k, v), pos, slots, want, tol = step([1, 1])
        raw = q.clone(), k.clone()
        got = decode.decode_step(q, k, v, *norms, rotary, pos, *cache.get_physical_cache(1), slots, tables.to(device),
                                 torch.tensor(done, dtype=torch.int32, device=device))
        close(got, want, tol)
        assert torch.equal(q, raw[0]) and torch.equal(k, raw[1])
    for a, b in zip((cache.key_codes, cache.key_scales, cache.value_codes, cache.value_scales), pages):
        assert torch.equal(a[1].cpu(), b)
    assert not cache.key_codes[0].any()
    assert _C.index_errors() == 0
