"""A cache object that lives as long as a server does: what it keeps between calls stays small."""

import pytest
import torch

from test_gpu_kv4 import filled

pytestmark = pytest.mark.gpu


def test_calls_of_ever_other_sizes_leave_little_behind(cuda):
    import ltxb
    cache, _, _ = filled([40], 1, 128, cuda)
    q = torch.randn(400, 1, 128, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(cuda)
    whole = ltxb.attention_kv4(q[:40], cache, causal=False)
    for n in range(1, 400):
        out = ltxb.attention_kv4(q[:n], cache, causal=False)
        if n <= 15:
            assert torch.equal(out, ltxb.attention_kv4(q[:n], cache, causal=False))
    assert sum(len(x) for x in vars(cache).values() if isinstance(x, dict)) <= 64
    assert torch.equal(ltxb.attention_kv4(q[:40], cache, causal=False), whole)
