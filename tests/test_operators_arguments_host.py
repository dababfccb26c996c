"""Arguments of the packed attention, rotary and 4-bit product entry points on the host: sizes of workspaces, limits, and
buffers that overlap; and the switch of the packed layers' exact small calls. Every call of the library below is refused
before anything is launched (the pointers are never dereferenced)."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import idolq_lib as L
from ggml_types import GGMLQuantizationType
from idol_packed import PackedLinear, enable_fused_packed
from test_operators_host import P, attention, gemv, rotary


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


A, B, C, D = 0x100000, 0x200000, 0x300000, 0x400000    # far apart


@pytest.mark.parametrize("over", [
    dict(x=A, y=A, ldx=256, ldy=264), dict(x2=C, y2=C, ldx2=128, ldy2=256), dict(x=A, y=A + 16), dict(x=A, y=A - 512 * 3),
    dict(y=C), dict(y2=A), dict(y2=B), dict(y2=B + 512 * 2 + 510), dict(x=A, y=A + 256, ldx=512, ldy=512),
    dict(x=A, y=A + 1024 * 3, ldx=512, ldy=256), dict(x=A, y=A, ldx=512, ldy=512, x2=A + 512, y2=A + 510, ldx2=512, ldy2=512)])
def test_rotary_refuses_overlapping_outputs(over):
    # four rows of 256 elements in bf16 (x, y) and of 128 (x2, y2)
    assert rotary(**{**dict(x=A, y=B, x2=C, y2=D), **over}) == L.EINVAL
    assert b"overlap" in L.load().idolq_last_error(), L.load().idolq_last_error()


@pytest.mark.parametrize("over", [
    dict(out=A + 16), dict(out=A - 512 * 7), dict(out=C), dict(out=D), dict(out=C + 256 * 8 + 240), dict(out=C - 512 * 7 - 496),
    dict(out=A + 512, ldq=1024, ldo=264), dict(out=A + 1024 - 16, ldq=512, ldo=512)])
def test_packed_attention_refuses_outputs_over_its_inputs(over):
    # eight rows of 256 elements (q, out), nine of 128 (k, v)
    assert attention(**{**dict(q=A, k=C, v=D), **over}) == L.EINVAL
    assert b"overlap" in L.load().idolq_last_error(), L.load().idolq_last_error()


@pytest.mark.parametrize("over", [
    dict(y=A), dict(y=A + 1024 + 1022), dict(y=A - 62), dict(y=B, ldy=24), dict(y=B, y_dtype=L.F32, ldy=16),
    dict(y=B + 2), dict(y=B, y_dtype=L.F16, residual_dtype=L.BF16), dict(y=B - 32, y_dtype=L.BF16, ldy=32)])
def test_q4_gemv_refuses_outputs_over_its_inputs(over):
    # two rows of 512 (x) and of 16 elements (y, residual) in bf16
    assert gemv(**{**dict(x=A, residual=B, residual_dtype=L.BF16, w=C, bias=D), **over}) == L.EINVAL
    assert b"overlap" in L.load().idolq_last_error(), L.load().idolq_last_error()


def test_enabling_the_fused_path_again_leaves_small_exact_as_it_is():
    data = np.zeros((4, 2, 18), dtype=np.uint8)
    net = torch.nn.Sequential(*(PackedLinear(SimpleNamespace(shape=np.array([64, 4]), tensor_type=GGMLQuantizationType.Q4_0,
                                                             data=data), None) for _ in range(2)))
    assert enable_fused_packed(net) == 2 and all(m.fused and not m.small_exact for m in net)
    assert enable_fused_packed(net[1], small_exact=True) == 1
    assert enable_fused_packed(net) == 2 and not net[0].small_exact and net[1].small_exact
    enable_fused_packed(net, small_exact=False)
    assert not any(m.small_exact for m in net)
