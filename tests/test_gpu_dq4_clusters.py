"""GPU tests of the 4-bit linear where the CTAs of a cluster add their sums and
a warp's lanes reach the cluster's barrier from loops of unequal length: an
output share of a CTA that is not a multiple of 32 lanes, on both kernels and
for every cluster size. Tolerances as in test_gpu_dq4.py."""

import pytest
import torch

from test_gpu_dq4 import check, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 2, 3, 5, 9, 11, 17, 18, 33, 130])
@pytest.mark.parametrize("N,K", [(32, 512), (128, 1152), (96, 2176), (160, 4224), (4096, 2304), (8192, 1280)])
def test_shares_that_do_not_fill_their_warps(cuda, M, N, K):
    import ltxb
    wq, s = weights(N, K, 64, torch.bfloat16, M, cuda)
    a = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(torch.bfloat16).to(cuda)
    out = ltxb.dq4_gemm(a, wq, s)
    check(out, a, wq, s)
    for _ in range(20):
        assert torch.equal(ltxb.dq4_gemm(a, wq, s), out)
    assert ltxb.device_status() == ltxb.OK
