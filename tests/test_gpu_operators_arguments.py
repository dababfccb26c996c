"""Views of one buffer that the packed attention, rotary and 4-bit product calls take as inputs and outputs, and those that
they refuse because an output overlaps an input."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import idolq_lib as L
from ggml_types import GGMLQuantizationType
from idol_packed import PackedLinear, enable_fused_packed

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16 = torch.bfloat16


def rows(n, cols, seed):
    return torch.randn((n, cols), generator=torch.Generator().manual_seed(seed)).to(BF16).to(DEV)


def test_rotary_between_columns_and_rows_of_one_buffer():
    pos = torch.arange(9, dtype=torch.int32, device=DEV)[:, None] * 7
    freqs = torch.linspace(1, 0.01, 16, device=DEV)
    turn = lambda x, k=None, **kw: L.rotary(x, 4, 64, pos, freqs, [16], k=k, kv_heads=0 if k is None else 2, **kw)  # noqa: E731
    wide = rows(9, 1024, 1)
    x, k = wide[:, :256], wide[:, 256:384]
    want_x, want_k = turn(x.contiguous(), k.contiguous())
    turn(x, k, out=wide[:, 384:640], k_out=wide[:, 640:768])
    assert torch.equal(wide[:, 384:640], want_x) and torch.equal(wide[:, 640:768], want_k)
    turn(x, k, out=x, k_out=k)
    assert torch.equal(x, want_x) and torch.equal(k, want_k)
    tall = rows(27, 256, 2)
    want = turn(tall[::3].contiguous())
    turn(tall[::3], out=tall[1::3])
    assert torch.equal(tall[1::3], want)
    with pytest.raises(ValueError, match="overlap"):
        turn(tall[:9], out=tall[1:10])
    with pytest.raises(ValueError, match="overlap"):
        turn(x, k, out=wide[:, 256:512])


def test_packed_attention_into_columns_between_its_inputs():
    wide = rows(50, 1024, 3)
    q, k, v, out = wide[:, :256], wide[:, 256:384], wide[:, 640:768], wide[:, 384:640]
    cu = torch.tensor([0, 30, 50], dtype=torch.int32, device=DEV)
    want = L.attention_packed(q, k, v, cu, cu, 4, 2, 64, causal=True)
    L.attention_packed(q, k, v, cu, cu, 4, 2, 64, causal=True, out=out)
    assert torch.equal(out, want)
    for bad in (wide[:, 200:456], wide[:, 512:768], wide[:, 8:264]):
        with pytest.raises(ValueError, match="overlap"):
            L.attention_packed(q, k, v, cu, cu, 4, 2, 64, causal=True, out=bad)


def test_q4_gemv_into_its_residual_and_columns_next_to_its_inputs():
    w = torch.randint(0, 256, (64 * 8 * 18,), generator=torch.Generator().manual_seed(4), dtype=torch.uint8).reshape(-1, 18)
    w[:, :2] = torch.tensor([0.03], dtype=torch.float16).view(torch.uint8)
    w = w.reshape(-1).to(DEV)
    wide = rows(7, 512, 5)
    x, res = wide[:, :256], wide[:, 256:320]
    call = lambda **kw: L.q4_gemv(x, w, L.KIND_Q4_0, 64, residual=res, **kw)  # noqa: E731
    want = call()
    call(out=wide[:, 320:384])
    assert torch.equal(wide[:, 320:384], want)
    call(out=res)
    assert torch.equal(res, want)
    for bad in (wide[:, 200:264], wide[:, 250:314], wide[:, 8:72]):
        with pytest.raises(ValueError, match="overlap"):
            call(out=bad)


@pytest.mark.parametrize("rows_of_x", [3, 16, 17])
def test_small_exact_calls_refuse_a_bias_of_another_type_as_longer_ones_do(rows_of_x):
    data = np.zeros((8, 4, 18), dtype=np.uint8)
    layer = PackedLinear(SimpleNamespace(shape=np.array([128, 8]), tensor_type=GGMLQuantizationType.Q4_0, data=data),
                         torch.ones(8)).to(DEV)
    enable_fused_packed(layer, small_exact=True)
    x = rows(rows_of_x, 128, 6)
    with torch.no_grad():
        with pytest.raises(ValueError, match="invalid fused linear bias"):
            layer(x)
        layer.bias.data = layer.bias.data.to(BF16)
        assert (layer(x) == 1).all()
