"""GPU tests of the 4-bit cache's codes next to ties, where the values of a group
lie so far apart that their differences are no f32 numbers: codes are those of
the exact differences."""

from fractions import Fraction

import pytest
import torch

from oracle import kv4_ref as kr
from test_gpu_kv4 import make_cache

pytestmark = pytest.mark.gpu


def by_fractions(x, group):
    """codes by rational arithmetic, for a few rows"""
    x = x.double().reshape(-1, 128)
    out = torch.zeros(x.shape, dtype=torch.int64)
    for r in range(x.shape[0]):
        for g0 in range(0, 128, group):
            v = [Fraction(float(t)) for t in x[r, g0:g0 + group]]
            z = min(v)
            s = kr.quantise(x[r], group)[1][g0 // group]
            for i, t in enumerate(v):
                out[r, g0 + i] = round((t - z) / Fraction(float(s))) if float(s) > 0 else 0
    return out


def rows():
    """Steps of 1, of which every half is a tie, with something far smaller added or taken off."""
    g = torch.Generator().manual_seed(0)
    x = torch.zeros(10, 128)
    x[0] = torch.where(torch.arange(128) % 2 == 0, -7.5, 7.5)
    x[0, 3::8] = torch.randn(16, generator=g) * 1e-9            # next to the tie in the middle
    x[1] = x[0] * 2.0 ** 40
    x[2] = (torch.arange(128) % 31) * 0.5
    x[2] = torch.where(x[2] == 0, 1e-9, x[2])                   # the smallest is a tiny number
    x[3] = (torch.arange(128) % 31) * 0.5
    x[3, 0::32] = -1e-9
    x[4] = x[0]
    x[4, 3::8] = torch.tensor([1.0, -1.0]).repeat(8) * 2.0 ** -126
    x[5] = x[3] * 2.0 ** -100
    x[6] = -x[2]
    x[7] = x[0]
    x[7, 3::8] = torch.tensor([1.0, -1.0]).repeat(8) * 2.0 ** -14  # the differences are f32 numbers here
    x[8] = torch.where(torch.arange(128) % 2 == 0, -7.5, 7.5)
    x[8, 5::8] = 0.0
    x[9] = x[2] * 2.0 ** -133                                   # subnormal
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_codes_next_to_ties(cuda, group):
    x = rows()[:, None, :]
    n = x.shape[0]
    code, scale, zero = kr.quantise(x, group)
    assert torch.equal(code.reshape(n, 128), by_fractions(x, group))  # the oracle itself
    cache = make_cache([n], 1, group, cuda)
    cache.append(x.to(cuda), x.to(cuda))
    want = kr.values(code, scale, zero).float()
    for got in cache.read(n, dtype=torch.float32):
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("group", [32, 128])
def test_many_groups_of_ties_and_tiny_values(cuda, group):
    """2 M values: half steps of a scale, a tenth of them with a far smaller number in their place or as the smallest."""
    g = torch.Generator(device=cuda).manual_seed(group)
    n = 2048
    x = torch.randint(0, 31, (n, 8, 128), generator=g, device=cuda) * 0.5
    x[:, 0::2] -= torch.randint(0, 2, (n, 4, 1), generator=g, device=cuda) * 7.5
    tiny = torch.exp2(-16 - 40 * torch.rand(n, 8, 128, generator=g, device=cuda))
    tiny = torch.where(torch.rand(n, 8, 128, generator=g, device=cuda) < 0.5, tiny, -tiny)
    x = torch.where(torch.rand(n, 8, 128, generator=g, device=cuda) < 0.1, tiny, x)
    x = x * torch.exp2(torch.randint(-60, 60, (n, 8, 1), generator=g, device=cuda).float())
    x = x.to(torch.bfloat16)
    cache = make_cache([n], 8, group, cuda)
    cache.append(x, x)
    want = kr.held(x, group).float()
    for got in cache.read(n, dtype=torch.float32):
        assert torch.equal(got, want)
