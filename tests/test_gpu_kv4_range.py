"""GPU tests of the attention over a 4-bit cache where values or weights lie many
powers of two apart, against the float64 restatement in oracle/kv4_ref.py.

Tolerances, relative to what the result is made of and not to the largest |v|
of the cache. W = sum_t p_t max_d |v_t|, the weighted mean of the tokens'
largest values.
Many rows: K and V are f16 (2^-12 each), p too (2^-12 while it is above 2^-24 of
the row's largest; 2^-10 at 2^-26), exp2 is off by at most 2^-13. With A = max sum_d |q_d k_d| scale the scores are off by 2^-12 A, both in
a weight and in the sum it is divided by: |got - want| <= 2^-8 |want| +
(2^-9 + 2^-11 A) W."""

import math

import pytest
import torch

from oracle import kv4_ref as kr
from test_gpu_kv4 import make_cache

pytestmark = pytest.mark.gpu


def exact(q, k, v, causal, scale):
    """Attention in f64 and W, rows [n, H]."""
    n, H, _ = q.shape
    T, hk, _ = k.shape
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    kk, vv = (t.repeat_interleave(H // hk, 1) for t in (k, v))
    s = torch.einsum("nhd,thd->nht", q, kk) * scale
    if causal:
        pos = torch.arange(T - n, T)[:, None, None]
        s = s.masked_fill(torch.arange(T)[None, None] > pos, -math.inf)
    p = torch.softmax(s, -1)
    return torch.einsum("nht,thd->nhd", p, vv), torch.einsum("nht,th->nh", p, vv.abs().amax(-1))[..., None]


def agrees(got, q, k, v, causal=False, scale=1.0):
    want, w = exact(q, k, v, causal, scale)
    a = float(torch.einsum("nd,td->nt", q.double().cpu().abs().flatten(0, 1),
                           k.double().cpu().abs().flatten(0, 1)).max()) * abs(scale)
    slack = 2.0 ** -9 + 2.0 ** -11 * a
    got = got.double().cpu()
    ratio = (got - want).abs() / (2.0 ** -8 * want.abs() + slack * w)
    assert bool((ratio <= 1).all()), float(ratio.nan_to_num(math.inf).max())


def one_heavy_token(T, at, nats, device, seed=0):
    """q, k, v of one head with scores (scale 1) of about 0 and, for token `at`, `nats` more; its v is 0, the others' near 1."""
    g = torch.Generator().manual_seed(seed)
    q = 0.02 * torch.randn(256, 1, 128, generator=g)
    q[:, :, 0] = 4.0
    k = 0.1 * torch.randn(T, 1, 128, generator=g)
    k[:, :, 0] = 0.0
    k[at, :, 0] = nats / 4.0
    v = 1.0 + 0.1 * torch.randn(T, 1, 128, generator=g)
    v[at] = 0.0
    return [t.to(torch.bfloat16).to(device) for t in (q, k, v)]


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("T,at,rows,causal", [(700, 0, 256, False), (6000, 3, 256, False), (6000, 0, 200, True),
                                              (130, 129, 100, False)])
@pytest.mark.parametrize("nats", [8.0, 15.0, 17.5])
def test_many_rows_under_one_heavy_token(cuda, nats, T, at, rows, causal, group):
    """The rest of the weights add up, however far they lie below the heaviest."""
    import ltxb
    q, k, v = one_heavy_token(T, at, nats, cuda)
    q = q[:rows]
    cache = make_cache([T], 1, group, cuda)
    cache.append(k, v)
    out = ltxb.attention_kv4(q, cache, causal=causal, scale=1.0)
    agrees(out, q, kr.held(k.cpu(), group), kr.held(v.cpu(), group), causal)
    assert ltxb.device_status() == ltxb.OK
