"""Arguments of the packed attention, rotary and 4-bit product entry points on the host: sizes of workspaces, limits, and
buffers that overlap. Every call below is refused before anything is launched (the pointers are never dereferenced)."""
import pytest

import idolq_lib as L
from test_operators_host import P, attention


def workspace(seqs, total_q, total_k, max_q, max_k, heads, kv_heads, hd):
    return L.load().idolq_attention_packed_workspace(seqs, total_q, total_k, max_q, max_k, heads, kv_heads, hd)


@pytest.mark.parametrize("seqs,total_q,total_k,max_q,max_k", [
    (1000, 1000, 500000, 0, 0), (1000, 100000, 2048000, 500, 2048), (4000, 4000, 2000000, 0, 0), (20000, 20000, 1000000, 0, 0),
    (100000, 100000, 100001, 0, 0), (300, 3000, 2 ** 31 - 1, 0, 0), (60000, 120000, 2 ** 31 - 1, 64, 0)])
def test_packed_attention_workspace_does_not_grow_with_the_sequences(seqs, total_q, total_k, max_q, max_k):
    # chunks of keys: 2048 entries of 64 rows and a few, or as many as 64 MB hold
    assert workspace(seqs, total_q, total_k, max_q, max_k, 32, 8, 128) <= (2048 + 8) * 64 * 130 * 4


@pytest.mark.parametrize("seqs", [16000, 16500, 100000])
def test_packed_attention_takes_as_many_sequences_with_a_workspace_as_without(seqs):
    # out is q: what passes the limits is refused for that
    over = dict(seqs=seqs, total_q=seqs, total_k=4 * seqs, heads=32, kv_heads=8, ldq=2048, ldk=512, ldv=512, ldo=2048,
                k=0x2000, v=0x2000)
    for ws, size in ((None, 0), (P, 2 ** 40)):
        assert attention(**over, ws=ws, ws_bytes=size) == L.EINVAL
        assert b"overlap" in L.load().idolq_last_error(), L.load().idolq_last_error()
