"""Into how many pieces a prefill over a quantised cache cuts the keys of its strips: as many as the card holds at once."""
from __future__ import annotations

import pytest
from test_fp8_attention_gpu import Batch, check_prefill

from nano_vllm_ascend_amd import _C


def pieces(kind, max_q, keys, n_seqs=1, hq=16, hkv=8, bs=128):
    """Of strips, by the workspace: a record of 528 bytes for each row of a strip of 32 and piece."""
    size = getattr(_C.load(), f"nvamd_paged_prefill_{kind}_workspace_size")(n_seqs, max_q, hq, hkv, bs, keys // bs)
    per_piece = n_seqs * hkv * -(-max_q * (hq // hkv) // 32) * 32 * 528
    assert size % per_piece == 0
    return max(size // per_piece, 1)


@pytest.mark.parametrize("max_q, n_seqs, keys, fp4, fp8", [
    (300, 1, 4096, 5, 3),   # 152 strips: 768 of the 4-bit cache fit at once, 512 of the 8-bit cache
    (300, 1, 8192, 5, 3),
    (100, 3, 4096, 4, 3),   # 168
    (500, 1, 8192, 3, 2),   # 256
    (520, 1, 8192, 2, 1),   # 264
    (600, 1, 8192, 2, 1),   # 304
    (600, 1, 16384, 2, 2),  # of long contexts two all the same
    (768, 1, 16384, 2, 2),  # 384
    (770, 1, 16384, 1, 1),  # 392
    (300, 1, 3968, 1, 1),   # short contexts: not cut
])
def test_strips_are_cut_for_one_round(max_q, n_seqs, keys, fp4, fp8):
    assert (pieces("fp4", max_q, keys, n_seqs), pieces("fp8", max_q, keys, n_seqs)) == (fp4, fp8)


@pytest.mark.gpu
@pytest.mark.parametrize("max_q, cached", [(600, 3000), (600, 470), (768, 20), (300, 5000)])
def test_strips_in_two_and_three_pieces(device, max_q, cached):
    """The launch's bound and the width of the tables decide: contexts of two pieces or three, and of one."""
    _C.clear_index_errors()
    batch = Batch(device, [40 + cached], 16, 8, 128, seed=7, extra_width=16384 // 128)
    assert pieces("fp8", max_q, batch.tables.shape[1] * 128) == (3 if max_q == 300 else 2)
    q = batch.queries(40)
    got = batch.prefill(q, [40], max_q=max_q)
    check_prefill(batch, q, [40], got)
    assert _C.index_errors() == 0
