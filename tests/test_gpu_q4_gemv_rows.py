"""4-bit products: what a row's result depends on. Calls of 5 to 16 rows give a row the same bits as any other such call does,
and so do calls of 1 to 4; between the two, which add in different orders, each is within its bound."""
import pytest
import torch

import idolq_lib as L
from test_gpu_q4_gemv import BF16, DEV, F32, FP16, Q4_0, Q4_K, blocks, check, oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,n,k", [(Q4_0, 300, 1024), (Q4_K, 300, 1024), (Q4_0, 21, 1568), (Q4_K, 16401, 256)])
@pytest.mark.parametrize("dtype", [BF16, FP16, F32])
def test_rows_alone_and_in_company(kind, n, k, dtype):
    x = torch.randn((16, k), generator=torch.Generator().manual_seed(n)).to(dtype).to(DEV)
    b = blocks(kind, n, k, 21)
    w = b.reshape(-1).to(DEV)
    all16, four = L.q4_gemv(x, w, kind, n), L.q4_gemv(x[:4], w, kind, n)
    for m in range(5, 16):
        assert torch.equal(L.q4_gemv(x[:m], w, kind, n), all16[:m])
        assert torch.equal(L.q4_gemv(x[16 - m:], w, kind, n), all16[16 - m:])
    for r in range(4):
        assert torch.equal(L.q4_gemv(x[r:r + 1], w, kind, n)[0], four[r])
        assert torch.equal(L.q4_gemv(x[r:4], w, kind, n), four[r:])
    want, bound = oracle(x, b, kind)
    check(all16, want, bound, k, dtype)
    check(four, want[:4], bound[:4], k, dtype)


@pytest.mark.parametrize("kind", [Q4_0, Q4_K])
@pytest.mark.parametrize("m", [2, 7])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_activations_up_to_2_to_117(kind, m, dtype):
    # a group's 32 products of codes up to 15 + 16 are summed before its scale: 2^10 of the largest activation, below fp32's
    # largest; the scales bring the results back
    k = 512
    x = (torch.rand((m, k), generator=torch.Generator().manual_seed(m)) * 2 - 1).mul(2.0 ** 117).to(dtype).to(DEV)
    x[0] = 2.0 ** 117
    b = blocks(kind, 40, k, 22, std=2.0 ** -16)
    check(L.q4_gemv(x, b.reshape(-1).to(DEV), kind, 40), *oracle(x, b, kind), k, dtype)
