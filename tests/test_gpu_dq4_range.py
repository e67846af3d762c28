"""GPU tests of the 4-bit linear on rows of A near bf16's ends. Tolerances as in test_gpu_dq4.py."""

import pytest
import torch

from test_gpu_dq4 import check, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group,scale_dtype", [(32, torch.float32), (64, torch.bfloat16), (128, torch.float32)])
@pytest.mark.parametrize("M", [1, 3, 8, 9, 16, 17, 40])
@pytest.mark.parametrize("size", [1e37, 2.0 ** 120, 3e38, 2.0 ** -100])
def test_rows_whose_sums_pass_the_largest_float(cuda, size, M, group, scale_dtype):
    """Finite rows whose values add up to more than f32 holds, while every output fits: one sign, and both."""
    import ltxb
    N, K = 96, 1024
    wq, s = weights(N, K, group, scale_dtype, 3, cuda)
    s = (s * 0.02).to(scale_dtype)  # |out| stays below 3e38
    a = torch.full((M, K), size)
    if M > 1:
        a[1] *= torch.randn(K, generator=torch.Generator().manual_seed(M)).clamp(-1, 1)
        a[-1, ::2] = 0
    a = a.to(torch.bfloat16).to(cuda)
    assert bool(a.isfinite().all())
    check(ltxb.dq4_gemm(a, wq, s), a, wq, s)
    assert ltxb.device_status() == ltxb.OK
