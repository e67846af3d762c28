"""GPU tests of the attention over a 4-bit cache where values or weights lie many
powers of two apart, against the float64 restatement in oracle/kv4_ref.py.

Tolerances, relative to what the result is made of and not to the largest |v|
of the cache. W = sum_t p_t max_d |v_t|, the weighted mean of the tokens'
largest values.
Few rows: codes enter the products exactly and p * scale with 11 bits (off by at
most 2^-12), so an output is off by at most 2^-12 sum_t p_t scale_t code_t
<= 2^-12 * 2 W, f32 sums apart; half of 2^-10 W. The output's own rounding adds 2^-8 |want|.
Many rows: K and V are f16 (2^-12 each), p too (2^-12 while it is above 2^-24 of
the row's largest; 2^-10 at 2^-26), exp2 is off by at most 2^-13. With A = max sum_d |q_d k_d| scale the scores are off by 2^-12 A, both in
a weight and in the sum it is divided by: |got - want| <= 2^-8 |want| +
(2^-9 + 2^-11 A) W."""

import math

import pytest
import torch

from oracle import kv4_ref as kr
from test_gpu_kv4 import check, check_many, make_cache, rows_like

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


def agrees(got, q, k, v, causal=False, scale=1.0, many=False, where=slice(None)):
    want, w = exact(q, k, v, causal, scale)
    slack = 2.0 ** -10
    if many:
        a = float(torch.einsum("nd,td->nt", q.double().cpu().abs().flatten(0, 1),
                               k.double().cpu().abs().flatten(0, 1)).max()) * abs(scale)
        slack = 2.0 ** -9 + 2.0 ** -11 * a
    got, want, w = got.double().cpu()[where], want[where], w[where]
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
    agrees(out, q, kr.held(k.cpu(), group), kr.held(v.cpu(), group), causal, many=True)
    assert ltxb.device_status() == ltxb.OK


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T,at,rows", [(50, 7, 1), (700, 0, 8), (700, 0, 9), (6000, 5000, 16), (3000, 64, 40)])
@pytest.mark.parametrize("nats", [15.0, 30.0, 60.0])
def test_few_rows_under_one_heavy_token(cuda, nats, T, at, rows, group):
    import ltxb
    q, k, v = one_heavy_token(T, at, nats, cuda)
    q = q[:rows]
    cache = make_cache([T], 1, group, cuda)
    cache.append(k, v)
    out = ltxb.attention_kv4(q, cache, causal=False, scale=1.0)
    agrees(out, q, kr.held(k.cpu(), group), kr.held(v.cpu(), group))
    assert ltxb.device_status() == ltxb.OK


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("power", [12, 20, 28, 60])
@pytest.mark.parametrize("T,at,rows", [(40, 3, 1), (40, 39, 12), (900, 0, 3), (900, 600, 16), (5000, 130, 1)])
def test_one_huge_value_without_weight(cuda, T, at, rows, power, group):
    """A token whose V is 2^power the others', 90 nats below them: the others keep all their bits."""
    import ltxb
    g = torch.Generator().manual_seed(5)
    q = 0.5 * torch.randn(rows, 2, 128, generator=g)
    q[:, :, 0] = 4.0
    k = 0.3 * torch.randn(T, 1, 128, generator=g)
    k[at, :, 0] = -22.5
    v = torch.randn(T, 1, 128, generator=g)
    v[at] *= 2.0 ** power
    q, k, v = (t.to(torch.bfloat16).to(cuda) for t in (q, k, v))
    cache = make_cache([T], 1, group, cuda)
    cache.append(k, v)
    out = ltxb.attention_kv4(q, cache, causal=False, scale=1.0)
    agrees(out, q, kr.held(k.cpu(), group), kr.held(v.cpu(), group))
    assert ltxb.device_status() == ltxb.OK


@pytest.mark.parametrize("rows", [3, 12])
def test_values_that_change_size_along_the_cache(cuda, rows):
    """Rows that see different tokens of very different V: large and small ones by turns, seen by some rows only."""
    import ltxb
    T, group = 400, 32
    k, v = rows_like((T, 2, 128), 1, cuda).float(), rows_like((T, 2, 128), 2, cuda).float()
    t = torch.arange(T, device=cuda)
    v = v * torch.exp2(40.0 * torch.sin(t * 0.05))[:, None, None]
    q = torch.randn(rows, 4, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(cuda)
    # the scores follow -log |v|, so that small and large tokens weigh alike
    k = k - 2.4 * torch.sin(t * 0.05)[:, None, None] * q.float().mean((0, 1)) * 4
    k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
    cache = make_cache([T], 2, group, cuda)
    cache.append(k, v)
    for causal in (True, False):
        out = ltxb.attention_kv4(q, cache, causal=causal)
        agrees(out, q, kr.held(k.cpu(), group), kr.held(v.cpu(), group), causal, scale=128 ** -0.5)


UNEQUAL = [(1e-30, 1e30, 1e-30), (1e25, 1e-25, 1e30), (1.0, 1.0, 1e-37), (1e-38, 1e-5, 1.0), (1e-33, 1e33, 1.0),
           (1e-37, 2e37, 1e-20), (1e36, 1e-36, 1.0), (1e37, 1e-37, 1e28)]


@pytest.mark.parametrize("qs,ks,vs", UNEQUAL)
@pytest.mark.parametrize("rows,group", [(1, 128), (8, 64), (10, 32), (16, 64)])
def test_few_rows_of_unequal_size(cuda, rows, group, qs, ks, vs):
    """Queries, keys and values over many powers of two, up to bf16's ends."""
    import ltxb
    T, H = 200, 2
    g = torch.Generator().manual_seed(3)
    q = (torch.randn(rows, H, 128, generator=g) * qs * torch.exp2(torch.arange(rows) % 5 - 2.0)[:, None, None])
    k, v = (torch.randn(T, H, 128, generator=g) * s for s in (ks, vs))
    q, k, v = q.to(torch.bfloat16), k.to(torch.bfloat16), v.to(torch.bfloat16)
    cache = make_cache([T], H, group, cuda)
    cache.append(k.to(cuda), v.to(cuda))
    out = ltxb.attention_kv4(q.to(cuda), cache)
    kh, vh = kr.held(k, group), kr.held(v, group)
    check(out, kr.attention(q, kh, vh, True), float(vh.abs().max()))
    assert ltxb.device_status() == ltxb.OK


@pytest.mark.parametrize("qs,ks", [(1e-33, 1e33), (1e-37, 2e37), (1e36, 1e-36)])
def test_many_rows_of_unequal_size_too(cuda, qs, ks):
    """The same sizes give the same answer on both sides of the number of rows that chooses the kernel."""
    import ltxb
    T, H = 200, 2
    g = torch.Generator().manual_seed(3)
    q = (torch.randn(100, H, 128, generator=g) * qs).to(torch.bfloat16)
    k, v = (torch.randn(T, H, 128, generator=g) * ks).to(torch.bfloat16), torch.randn(T, H, 128, generator=g).to(torch.bfloat16)
    cache = make_cache([T], H, 64, cuda)
    cache.append(k.to(cuda), v.to(cuda))
    kh, vh = kr.held(k, 64), kr.held(v, 64)
    check_many(ltxb.attention_kv4(q.to(cuda), cache), kr.attention(q, kh, vh, True), q, kh, vh)
    few = q[-16:]
    check(ltxb.attention_kv4(few.to(cuda), cache), kr.attention(few, kh, vh, True), float(vh.abs().max()))
