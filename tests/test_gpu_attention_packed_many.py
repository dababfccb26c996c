"""Packed attention with thousands of sequences of which a few are long enough to be cut: the workspace's entries go by the
keys there."""
import pytest
import torch

import idolq_lib as L
from test_gpu_attention_packed import BF16, DEV, FP16, check, offsets, oracle

pytestmark = pytest.mark.gpu

# (queries, keys) of the long sequences: around one and two chunks of 128 keys next to each other, many parts, one query and 16
LONG = [(1, 5000), (16, 129), (3, 128), (2, 257), (1, 256), (5, 3), (16, 1111)]


@pytest.mark.parametrize("seqs,heads,kv,hd,dtype,bounds", [
    (16500, 8, 8, 64, BF16, {}), (1300, 16, 4, 64, FP16, {}), (1300, 16, 4, 64, BF16, dict(max_q=16, max_k=5000)),
    (1300, 16, 4, 64, BF16, dict(max_q=16, max_k=1100)), (700, 32, 4, 128, BF16, dict(max_q=16, max_k=5000))])
@pytest.mark.parametrize("rooms", [False, True])
def test_a_few_long_sequences_among_thousands(seqs, heads, kv, hd, dtype, bounds, rooms):
    # the others are one query on one key: its values come out. rooms: every sequence has 40 more rows than its keys take
    group, places = heads // kv, {0: LONG[0], seqs - 1: LONG[-1]}
    places.update({seqs // 2 + i: x for i, x in enumerate(LONG)})
    lens = [places.get(s, (1, 1)) for s in range(seqs)]
    lq, lk = [a for a, _ in lens], [b for _, b in lens]
    room = [n + 40 * rooms for n in lk]
    gen = torch.Generator().manual_seed(seqs)
    q, k, v = (torch.randn((n, w * hd), generator=gen).to(dtype).to(DEV)
               for n, w in ((sum(lq), heads), (sum(room) + 1000, kv), (sum(room) + 1000, kv)))
    cq, ck = offsets(lq).to(DEV), (offsets(room) + 1000).to(DEV)
    need = L.load().idolq_attention_packed_workspace(seqs, sum(lq), k.shape[0], bounds.get("max_q", 0), bounds.get("max_k", 0),
                                                     heads, kv, hd)
    assert 0 < need < (2048 + kv) * 64 * (hd + 2) * 4
    got = L.attention_packed(q, k, v, cq, ck, heads, kv, hd, causal=True, **bounds,
                             k_lens=torch.tensor(lk, dtype=torch.int32, device=DEV) if rooms else None)
    assert torch.equal(got, L.attention_packed(q, k, v, cq, ck, heads, kv, hd, causal=True, **bounds,
                                               k_lens=torch.tensor(lk, dtype=torch.int32, device=DEV) if rooms else None))
    one = torch.tensor([s for s in range(seqs) if s not in places])
    rows, keys = cq.cpu()[one].long(), ck.cpu()[one].long()
    want = v.cpu()[keys].double().reshape(-1, kv, 1, hd).expand(-1, kv, group, hd).reshape(-1, heads * hd)
    check(got.cpu()[rows], want, want.abs(), dtype)
    for s, (a, b) in places.items():
        r, c = int(cq[s]), int(ck[s])
        check(got[r:r + a], *oracle(q[r:r + a], k[c:c + b], v[c:c + b], [a], [b], heads, kv, hd, True), dtype)
